"""Batched paged serving of the tiny Qwen3 (targets/qwen3_paged.py) against the
model's own op sequence run on each request by itself: logits of every prompt
and decode step, places that are released and taken again, a decode step
replayed as a CUDA graph, and the scoring of prompts."""
import pytest
import torch

from metal_autotune_b200 import lib
from metal_autotune_b200.targets import qwen3, qwen3_paged

pytestmark = pytest.mark.gpu

CFG = qwen3.TINY


@pytest.fixture(scope="module")
def model(cuda):
    return qwen3.build(CFG, seed=5, device="cuda")


def prompt(n, seed):
    return torch.randint(0, CFG.vocab, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


class Alone:
    """One request on the model's original ops with a dense cache."""

    def __init__(self, model):
        self.model, self.cache = model, qwen3.KVCache(CFG, device="cuda")

    def feed(self, tokens):
        self.model(torch.tensor(tokens, dtype=torch.int32, device="cuda"), self.cache)
        return self.model.last_logits[0].float()


def near(got, want):
    """bf16 activations through two layers: relative error of the logits row."""
    return float((got.float() - want).norm() / want.norm()) < 3e-2


def test_batch_follows_each_request_alone(model):
    server = qwen3_paged.PagedQwen3(model, requests=5, max_len=128, page_size=16, top_k=3)
    prompts = {0: prompt(7, 1), 2: prompt(33, 2), 3: prompt(16, 3)}  # places 1 and 4 stay idle
    alone = {r: Alone(model) for r in prompts}
    logits, picks = server.prefill(prompts)
    for i, r in enumerate(sorted(prompts)):
        assert near(logits[i], alone[r].feed(prompts[r]))
        assert int(server.tokens[r]) == int(logits[i].float().argmax()) == int(picks.top_ids[i, 0])
    for step in range(12):
        fed = server.tokens.tolist()
        logits, picks = server.decode()
        rows = server.last_places.tolist()
        assert sorted(r for r in rows if r >= 0) == sorted(alone)
        for i, r in enumerate(rows):
            if r >= 0:
                assert near(logits[i], alone[r].feed([fed[r]])), (step, r)
                lp = torch.log_softmax(logits[i].float(), -1)
                assert abs(float(picks.top_logprobs[i, 0]) - float(lp.max())) < 1e-4
                assert int(server.tokens[r]) == int(picks.top_ids[i, 0])
        if step == 5:  # one request ends, another takes its place and pages
            before = int(server.cache.free_head)
            server.release(2)
            assert int(server.cache.free_head) == before - -(-(33 + 6) // 16)
            alone[2] = Alone(model)
            new = prompt(21, 9)
            logits, _ = server.prefill({2: new})
            assert near(logits[0], alone[2].feed(new))
    assert lib.device_status() == 0


def test_decode_as_a_graph(model):
    prompts = {i: prompt(n, 20 + i) for i, n in enumerate((3, 30, 15, 64))}
    eager, graphed = (qwen3_paged.PagedQwen3(model, requests=4, max_len=128) for _ in range(2))
    for s in (eager, graphed):
        s.prefill(prompts)
        s.decode()  # warm-up
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    state = [t.clone() for t in (graphed.cache.lens, graphed.cache.free_head, graphed.cache.table, graphed.tokens)]
    with torch.cuda.graph(graph, stream=side):
        logits, picks = graphed.decode()
    for t, was in zip((graphed.cache.lens, graphed.cache.free_head, graphed.cache.table, graphed.tokens), state):
        assert torch.equal(t, was)  # capturing runs nothing
    for _ in range(20):
        want, _ = eager.decode()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(logits, want) and torch.equal(eager.tokens, graphed.tokens)
    assert torch.equal(eager.cache.lens, graphed.cache.lens) and eager.cache.lens.tolist() == [24, 51, 36, 85]


def test_score(model):
    server = qwen3_paged.PagedQwen3(model, requests=3, max_len=64)
    prompts = {0: prompt(12, 31), 1: prompt(40, 32)}
    got = server.score(prompts)
    for r, lp in enumerate(got):
        one = Alone(model)
        for i in range(len(prompts[r]) - 1):
            row = one.feed([prompts[r][i]])
            want = float(torch.log_softmax(row, -1)[prompts[r][i + 1]])
            assert abs(float(lp[i]) - want) < 0.1  # bf16 logits of both sides
    assert int(server.cache.free_head) == 0 and not bool(server.cache.lens.any())


def test_out_of_pages(model):
    server = qwen3_paged.PagedQwen3(model, requests=2, max_len=64, pages=3)
    with pytest.raises(RuntimeError, match="out of pages"):
        server.prefill({0: prompt(20, 1), 1: prompt(20, 2)})
    assert int(server.cache.free_head) == 0 and not bool(server.cache.lens.any())
    server.prefill({0: prompt(46, 1)})  # all three pages
    for want in (0, 0, 1):
        server.decode()
        assert server.refused() == want
    assert server.cache.lens.tolist() == [48, 0]
    with pytest.raises(ValueError, match="no tokens"):
        server.prefill({1: []})


def test_a_refused_place_keeps_its_token(cuda):
    """A place without a page for its pending token keeps that token, and goes on from it once pages come back."""
    model = qwen3.build(CFG, seed=5, device="cuda")
    model.norm.weight.data.neg_()  # or random tied weights pick the token that was fed, again and again
    server = qwen3_paged.PagedQwen3(model, requests=2, max_len=64, pages=4)
    prompts = {0: prompt(32, 1), 1: prompt(31, 2)}  # all four pages; place 1 has one slot left
    alone = Alone(model)
    server.prefill(prompts)
    alone.feed(prompts[0])
    first = server.tokens.tolist()
    server.decode()
    assert server.refused() == 1 and server.cache.lens.tolist() == [32, 32]
    second = server.tokens.tolist()
    assert second[0] == first[0]
    server.decode()
    assert server.refused() == 2 and server.tokens.tolist() == second
    server.release(1)
    for length in (33, 34):
        fed = server.tokens.tolist()[0]
        logits, picks = server.decode()
        assert server.refused() == 0 and int(server.cache.lens[0]) == length
        assert near(logits[0], alone.feed([fed])) and int(server.tokens[0]) == int(picks.top_ids[0, 0])

"""Batched serving of the Qwen3 target over a paged key-value cache.

The reference serves one request at a time from a dense cache
(autotuner_runtime/inference.py:131-156; targets/qwen3.py). Here a batch of
requests of any lengths shares one pool of pages per layer. A step lays its
tokens out (paged_plan), and per layer normalises, rotates and appends their
q/k/v (rope_paged_append), attends (paged_sdpa_decode for one new token per
request; sdpa over the prompt itself while it is prefilled) and runs the
region kernels of the dense path for the rest; the step's logits give each
request's next token, its log-probability, the entropy and the top
alternatives (token_logprobs).

Lengths, block tables, slots and the free list stay on the device: a decode
step reads nothing back and can be captured in a CUDA graph and replayed.

    python -m metal_autotune_b200.targets.qwen3_paged     # a small batch, printed
"""
from __future__ import annotations

import math

import torch

from .. import lib
from . import qwen3


class PagedKVCache:
    """Pages of one model's keys and values for up to `requests` requests of up
    to `max_len` tokens: per layer [pages, Hkv, page_size, D], one block table
    and one free list for all layers."""

    def __init__(self, cfg: qwen3.Qwen3Config, requests: int, max_len: int, *, pages: int | None = None, page_size: int = 16,
                 dtype=torch.bfloat16, device="cuda"):
        self.page_size = page_size
        self.width = -(-max_len // page_size)
        pages = requests * self.width if pages is None else pages
        shape = (pages, cfg.kv_heads, page_size, cfg.head_dim)
        self.layers = [(torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))
                       for _ in range(cfg.layers)]
        i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=device)  # noqa: E731
        self.table = torch.full((requests, self.width), -1, dtype=torch.int32, device=device)
        self.lens = i32(requests)
        self.free_pages = torch.arange(pages, dtype=torch.int32, device=device)
        self.free_head = i32(1)

    def plan(self, new_lens: torch.Tensor, token_cap: int, out=None) -> lib.PagedPlan:
        """Plan a step and take it over as the cache's state."""
        p = lib.paged_plan(self.lens, new_lens, self.table, self.free_pages, page_size=self.page_size, token_cap=token_cap,
                           free_head=self.free_head, out=out)
        self.lens.copy_(p.seq_lens)
        self.free_head.copy_(p.counts[4:])
        return p

    def release(self, request: int) -> None:
        """Give a finished request's pages back to the free list (reads its length: not for captured steps)."""
        held = -(-int(self.lens[request]) // self.page_size)
        head = int(self.free_head)
        self.free_pages[head - held:head] = self.table[request, :held]
        self.free_head -= held
        self.table[request, :held] = -1
        self.lens[request] = 0


class PagedQwen3:
    """Greedy batched generation with `model`'s weights (targets/qwen3.py)."""

    def __init__(self, model: qwen3.Qwen3Model, requests: int, max_len: int, *, page_size: int = 16, pages: int | None = None,
                 top_k: int = 5, rope_scaling: dict | None = None):
        cfg = model.cfg
        self.model, self.cfg, self.top_k, self.requests = model, cfg, top_k, requests
        device = model.norm.weight.device
        self.cache = PagedKVCache(cfg, requests, max_len, pages=pages, page_size=page_size, dtype=model.norm.weight.dtype,
                                  device=device)
        self.inv_freq, self.mscale = lib.rope_frequencies(cfg.head_dim, base=cfg.rope_theta, scaling=rope_scaling,
                                                          device=device)
        self.scale = 1.0 / math.sqrt(cfg.head_dim)
        # what a decode step reads and leaves for the next one
        self.tokens = torch.zeros(requests, dtype=torch.int32, device=device)
        self.active = torch.zeros(requests, dtype=torch.int32, device=device)
        self.plan_buffers = lib.PagedPlan.empty(requests, requests, device)

    def _layers(self, h: torch.Tensor, plan: lib.PagedPlan, attend):
        """The decoder layers over token rows h; attend(layer, q, k, v, k_cache, v_cache) -> [T, Hq, D] after the append."""
        cfg = self.cfg
        T, D = h.shape[0], cfg.head_dim
        kw = {"group_size": cfg.group, "bits": cfg.bits}
        qset = lambda m: (m.weight, m.scales, m.biases)  # noqa: E731
        k_rot = torch.empty(T, cfg.kv_heads, D, dtype=h.dtype, device=h.device)
        for layer, (kc, vc) in zip(self.model.layers, self.cache.layers):
            a, m = layer.self_attn, layer.mlp
            xn = lib.rms_norm(h, layer.input_layernorm.weight, cfg.eps)
            q, k, v = lib.quantized_matmul_multi(xn, [qset(a.q_proj), qset(a.k_proj), qset(a.v_proj)], **kw)
            q, k, v = q.view(T, cfg.heads, D), k.view(T, cfg.kv_heads, D), v.view(T, cfg.kv_heads, D)
            q = lib.rope_paged_append(q, k, v, plan.positions, plan.slots, kc, vc, self.inv_freq, mscale=self.mscale,
                                      q_norm_w=a.q_norm.weight, k_norm_w=a.k_norm.weight, eps=cfg.eps, out=q, k_out=k_rot)
            o = attend(q, k_rot, v, kc, vc).view(T, cfg.heads * D)
            h = lib.quantized_matmul(o, *qset(a.o_proj), residual=h, **kw)
            xn = lib.rms_norm(h, layer.post_attention_layernorm.weight, cfg.eps)
            act = lib.quantized_matmul_swiglu(xn, *qset(m.gate_proj), *qset(m.up_proj), **kw)
            h = lib.quantized_matmul(act, *qset(m.down_proj), residual=h, **kw)
        return h

    def _logits(self, h: torch.Tensor) -> torch.Tensor:
        E, cfg = self.model.embed_tokens, self.cfg
        xn = lib.rms_norm(h, self.model.norm.weight, cfg.eps)
        return lib.quantized_matmul(xn, E.weight, E.scales, E.biases, group_size=cfg.group, bits=cfg.bits)

    def _embed(self, tokens: torch.Tensor) -> torch.Tensor:
        E, cfg = self.model.embed_tokens, self.cfg
        return lib.quantized_embedding(tokens, E.weight, E.scales, E.biases, group_size=cfg.group, bits=cfg.bits)

    def prefill(self, prompts: dict[int, list[int]]) -> tuple[torch.Tensor, lib.TokenLogprobs]:
        """Take prompts into free places of the batch ({place: tokens}); returns the last positions' logits and each
        place's next token with its alternatives, in the order of the places."""
        places = sorted(prompts)
        flat, picks, logits = self._prompt_pass(prompts, places)
        for i, r in enumerate(places):
            self.tokens[r] = picks.top_ids[i, 0]
            self.active[r] = 1
        return logits, picks

    def score(self, prompts: dict[int, list[int]]) -> list[torch.Tensor]:
        """Log-probability of each prompt's tokens after its first, in places whose pages are given back."""
        places = sorted(prompts)
        flat, _, logits = self._prompt_pass(prompts, places, every=True)
        follow = torch.full_like(flat, -1)
        follow[:-1] = flat[1:]
        lp = lib.token_logprobs(logits, follow).logprob
        out, at = [], 0
        for r in places:
            n = len(prompts[r])
            out.append(lp[at:at + n - 1])
            at += n
            self.cache.release(r)
        return out

    def _prompt_pass(self, prompts, places, every=False):
        device = self.tokens.device
        lens = [len(prompts[r]) for r in places]
        if min(lens, default=0) == 0:
            raise ValueError("a prompt has no tokens")
        flat = torch.tensor([t for r in places for t in prompts[r]], dtype=torch.int32, device=device)
        new = torch.zeros(self.requests, dtype=torch.int32)
        new[places] = torch.tensor(lens, dtype=torch.int32)
        if bool((self.cache.lens.cpu()[places] != 0).any()):
            raise ValueError("a place of the batch still holds a request: release it first")
        plan = self.cache.plan(new.to(device), len(flat))
        if int(plan.counts[3]):
            for r in places:  # what the others got goes back
                self.cache.release(r)
            raise RuntimeError(f"{int(plan.counts[3])} request(s) refused: out of pages")
        starts = [sum(lens[:i]) for i in range(len(lens))]

        def attend(q, k, v, kc, vc):  # each prompt over itself
            o = torch.empty_like(q)
            for s, n in zip(starts, lens):
                at = lambda x: x[None, s:s + n].transpose(1, 2)  # noqa: E731
                lib.sdpa(at(q), at(k), at(v), scale=self.scale, causal=True, out=o[None, s:s + n], out_layout="blhd")
            return o

        h = self._layers(self._embed(flat), plan, attend)
        if every:
            return flat, None, self._logits(h)
        last = torch.tensor([s + n - 1 for s, n in zip(starts, lens)], device=device)
        logits = self._logits(h[last])
        return flat, lib.token_logprobs(logits, top_k=max(1, self.top_k)), logits

    def decode(self) -> tuple[torch.Tensor, lib.TokenLogprobs]:
        """One token for every active place: appends self.tokens, leaves the next ones there, returns the logits of all
        places (those of idle ones are of no request) and the log-probability, entropy and alternatives of each pick."""
        plan = self.cache.plan(self.active, self.requests, out=self.plan_buffers)
        # the step's tokens, one row each; rows past the last one are padding (slot -1, place 0)
        place = plan.token_seq.clamp(min=0).long()
        h = self._embed(self.tokens[place])
        table, lens = self.cache.table[place], torch.where(plan.token_seq >= 0, plan.seq_lens[place], 0)

        def attend(q, k, v, kc, vc):
            return lib.paged_sdpa_decode(q, kc, vc, table, lens, scale=self.scale)

        logits = self._logits(self._layers(h, plan, attend))
        picks = lib.token_logprobs(logits, top_k=max(1, self.top_k))
        # back to the places; rows without a slot (padding, and places that got no page: those keep the token that is
        # still to be appended) write a place past the last one
        to = torch.where(plan.slots >= 0, place, self.requests)
        self.tokens.copy_(torch.cat([self.tokens, self.tokens[:1]]).scatter(0, to, picks.top_ids[:, 0])[:self.requests])
        self.last_places = plan.token_seq
        return logits, picks

    def refused(self) -> int:
        """Places of the last decode step that got no slot for their token (no page left, or max_len reached): their row
        of that step means nothing, and their length and pending token stay, so that a later step with pages goes on
        from there. Reads the device; the step itself does not."""
        return int(self.plan_buffers.counts[3])

    def release(self, place: int) -> None:
        self.cache.release(place)
        self.active[place] = 0


def main() -> None:
    model = qwen3.build(qwen3.TINY, seed=1, device="cuda")
    g = torch.Generator().manual_seed(0)
    server = PagedQwen3(model, requests=4, max_len=256)
    prompts = {i: torch.randint(0, qwen3.TINY.vocab, (n,), generator=g).tolist() for i, n in enumerate((5, 40, 17, 1))}
    _, picks = server.prefill(prompts)
    out = {i: [int(t)] for i, t in enumerate(picks.top_ids[:, 0])}
    for _ in range(8):
        _, picks = server.decode()
        for i, t in enumerate(server.tokens.tolist()):
            out[i].append(t)
    for i, toks in out.items():
        print(f"request {i}: prompt of {len(prompts[i])} -> {toks}; last pick: log p {picks.top_logprobs[i, 0]:.3f}, "
              f"entropy {picks.entropy[i]:.3f}, alternatives {picks.top_ids[i].tolist()}")


if __name__ == "__main__":
    main()

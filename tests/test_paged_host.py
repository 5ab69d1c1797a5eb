"""Paged serving without a GPU: what the entry points refuse, before any CUDA
call, and the rotary frequency tables."""
import ctypes as C
import math

import pytest
import torch

from metal_autotune_b200 import build, lib

P = C.c_void_p(256)  # never dereferenced: the checks come first
BF, F32 = lib.MT_BF16, lib.MT_F32


@pytest.fixture(scope="module")
def mt():
    build.build_library()
    return lib.load()


def refused(mt, rc, code, text):
    assert rc == code and text in mt.mt_last_error_string(), (rc, mt.mt_last_error_string())


def test_plan_refuses(mt):
    args = dict(ctx=P, new=P, B=4, table=P, stride=8, width=8, free=P, n_free=9, head=None, page=16, cap=4)

    def plan(**kw):
        a = {**args, **kw}
        return mt.mt_paged_plan(a["ctx"], a["new"], a["B"], a["table"], a["stride"], a["width"], a["free"], a["n_free"], a["head"],
                                a["page"], a["cap"], P, P, P, P, a.get("slots", P), P, None)

    refused(mt, plan(B=-1), -1, b"B=-1")
    refused(mt, plan(page=0), -1, b"page_size 0")
    refused(mt, plan(stride=7), -1, b"row stride 7")
    refused(mt, plan(n_free=-1), -1, b"n_free=-1")
    refused(mt, plan(cap=1 << 31), -1, b"token_cap")
    refused(mt, plan(ctx=None), -1, b"null pointer")
    refused(mt, plan(slots=None), -1, b"null pointer")
    refused(mt, plan(free=None), -1, b"null pointer")


def test_plan_refuses_overlaps(mt):
    """An output over an input, the table's rows or another output, by address alone."""
    B, cap, n_free, stride, width = 6, 700, 50, 8, 5
    at = {}
    where = 1 << 20
    for name, size in dict(ctx=4 * B, new=4 * B, table=4 * stride * B, free=4 * n_free, head=4, lens=4 * B, start=4 * (B + 1), pos=4 * cap,
                           seq=4 * cap, slots=8 * cap, counts=20).items():
        at[name] = (where, size)
        where += size + 64 - size % 64

    def plan(**moved):
        a = {name: C.c_void_p(moved.get(name, p)) for name, (p, _) in at.items()}
        return mt.mt_paged_plan(a["ctx"], a["new"], B, a["table"], stride, width, a["free"], n_free, a["head"], 16, cap, a["lens"], a["start"],
                                a["pos"], a["seq"], a["slots"], a["counts"], None)

    outs, ins = ("lens", "start", "pos", "seq", "slots", "counts"), ("ctx", "new", "free", "head")
    for out in outs:
        size = at[out][1]
        for other in (*ins, *(o for o in outs if o != out)):
            first, n = at[other]
            refused(mt, plan(**{out: first}), -1, b"overlaps")
            refused(mt, plan(**{out: first + n - 4}), -1, b"overlaps")
            refused(mt, plan(**{out: first + 4 - size}), -1, b"overlaps")
    refused(mt, plan(counts=at["counts"][0], head=at["counts"][0] + 16), -1, b"counts overlaps free_head")
    refused(mt, plan(ctx=at["lens"][0]), -1, b"seq_lens overlaps ctx_lens")
    table = at["table"][0]
    for name in (*ins, "lens", "counts"):
        n = at[name][1]
        for row in (0, 3, 5):  # on a row's first entry, its last one, and from before a row into it
            refused(mt, plan(**{name: table + 4 * stride * row}), -1, b"overlaps")
            refused(mt, plan(**{name: table + 4 * (stride * row + width - 1)}), -1, b"overlaps")
            refused(mt, plan(**{name: table + 4 * stride * row + 4 - n}), -1, b"overlaps")


def test_append_refuses(mt):
    base = dict(q=P, st=4096, dims=128, page=16, T=2, Hq=32, Hkv=8, D=128, dt=BF, cache=P, inv=P)

    def append(**kw):
        a = {**base, **kw}
        return mt.mt_rope_paged_append(a["q"], P, P, a["st"], 128, 1024, 128, 1024, 128, None, None, 1e-6, P, P, a["inv"], a["dims"], 0, 1.0,
                                       P, 4096, 128, None, a["cache"], P, 10, a["page"], 16384, 2048, 128, a["T"], a["Hq"], a["Hkv"], a["D"],
                                       a["dt"], None)

    refused(mt, append(D=129), -1, b"multiple of 8")
    refused(mt, append(D=264), -1, b"up to 256")
    refused(mt, append(dims=130), -1, b"dims=130")
    refused(mt, append(dims=3), -1, b"dims=3")
    refused(mt, append(page=0), -1, b"page_size=0")
    refused(mt, append(dt=lib.MT_I32), -2, b"unsupported dtype")
    refused(mt, append(q=None), -1, b"null pointer")
    refused(mt, append(cache=None), -1, b"null pointer")
    refused(mt, append(inv=None), -1, b"null pointer")
    refused(mt, append(q=C.c_void_p(264)), -1, b"16-byte aligned")
    refused(mt, append(st=4100), -1, b"16-byte aligned")
    assert append(T=0, q=None) == 0


def test_attend_refuses(mt):
    need = mt.mt_paged_sdpa_decode_workspace_bytes(128)
    assert need > 65536
    base = dict(q=P, D=128, B=2, Hq=32, Hkv=8, page=16, stride=8, width=8, dt=BF, ws=P, nb=need, lens=P, ss=128)

    def attend(**kw):
        a = {**base, **kw}
        return mt.mt_paged_sdpa_decode(a["q"], 4096, 128, P, P, 10, a["page"], 16384, 2048, a["ss"], P, a["stride"], a["width"], a["lens"], P, 4096,
                                       128, a["B"], a["Hq"], a["Hkv"], a["D"], 0.1, a["dt"], a["ws"], a["nb"], None)

    refused(mt, attend(D=96), -1, b"head_dim 96")
    refused(mt, attend(dt=F32), -2, b"bf16 or f16")
    refused(mt, attend(Hq=30), -1, b"multiple of Hkv")
    refused(mt, attend(page=0), -1, b"page_size=0")
    refused(mt, attend(stride=4), -1, b"table stride=4")
    refused(mt, attend(lens=None), -1, b"null pointer")
    refused(mt, attend(B=1 << 16, width=1 << 16, stride=1 << 16), -2, b"2^35 rows")
    refused(mt, attend(ss=100), -1, b"16-byte aligned")
    refused(mt, attend(ws=None), -3, b"needs a workspace")
    refused(mt, attend(nb=need - 1), -3, b"needs a workspace")
    assert attend(B=0, q=None) == 0


def test_logprobs_refuses(mt):
    base = dict(x=P, stride=100, tokens=P, R=2, V=100, k=5, lp=P, ids=P, dt=BF)

    def logprobs(**kw):
        a = {**base, **kw}
        return mt.mt_token_logprobs(a["x"], a["stride"], a["tokens"], a["R"], a["V"], a["k"], a["lp"], None, None, a["ids"], P, a["dt"], None)

    refused(mt, logprobs(stride=99), -1, b"row_stride=99")
    refused(mt, logprobs(V=0), -1, b"V=0")
    refused(mt, logprobs(k=33), -1, b"top_k=33")
    refused(mt, logprobs(V=3, k=4), -1, b"top_k=4")
    refused(mt, logprobs(k=-1), -1, b"top_k=-1")
    refused(mt, logprobs(dt=lib.MT_I32), -2, b"unsupported dtype")
    refused(mt, logprobs(x=None), -1, b"null pointer")
    refused(mt, logprobs(lp=None), -1, b"null pointer")
    refused(mt, logprobs(ids=None), -1, b"null pointer")
    refused(mt, logprobs(x=C.c_void_p(257)), -1, b"aligned")
    assert logprobs(R=0, x=None) == 0


def test_wrappers_check_their_tensors(monkeypatch):
    """Shape and type errors come from the wrappers, by name, before any pointer is taken."""
    build.build_bind_library()
    cpu_workspace = lib.Workspace.__new__(lib.Workspace)
    cpu_workspace.buf = torch.zeros(16, dtype=torch.uint8)
    monkeypatch.setattr(lib.Workspace, "get", classmethod(lambda cls, n: cpu_workspace))
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)  # noqa: E731
    i = lambda *s: z(*s, dt=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="new_lens must have shape"):
        lib.paged_plan(i(3), i(2), i(3, 4), i(5), page_size=16, token_cap=3)
    with pytest.raises(ValueError, match="block_table must be int32"):
        lib.paged_plan(i(3), i(3), i(2, 4), i(5), page_size=16, token_cap=3)
    with pytest.raises(TypeError, match="ctx_lens must be torch.int32"):
        lib.paged_plan(i(3).long(), i(3), i(3, 4), i(5), page_size=16, token_cap=3)
    kc = z(4, 2, 16, 64)
    inv = torch.zeros(32)
    q, k = z(3, 4, 64), z(3, 2, 64)
    slots = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="k and v must be"):
        lib.rope_paged_append(q, k, z(3, 1, 64), i(3), slots, kc, kc, inv)
    with pytest.raises(TypeError, match="slots must be torch.int64"):
        lib.rope_paged_append(q, k, k, i(3), i(3), kc, kc, inv)
    with pytest.raises(ValueError, match="the caches must be"):
        lib.rope_paged_append(q, k, k, i(3), slots, z(4, 16, 2, 64), z(4, 16, 2, 64), inv)
    with pytest.raises(TypeError, match="the caches must be torch.bfloat16"):
        lib.rope_paged_append(q, k, k, i(3), slots, kc.half(), kc.half(), inv)
    with pytest.raises(ValueError, match="one shape and strides"):
        lib.paged_sdpa_decode(q, kc, z(4, 16, 2, 64).transpose(1, 2), i(3, 4), i(3), scale=1.0)
    with pytest.raises(ValueError, match="seq_lens must have shape"):
        lib.paged_sdpa_decode(q, kc, kc, i(3, 4), i(2), scale=1.0)
    with pytest.raises(ValueError, match="contiguous rows"):
        lib.token_logprobs(z(4, 10).t())
    with pytest.raises(ValueError, match="tokens must have shape"):
        lib.token_logprobs(z(4, 10), i(3))
    with pytest.raises(ValueError, match="CUDA tensors"):
        lib.token_logprobs(z(4, 10), i(4))


def test_binding_is_built_for_this_torch(monkeypatch, tmp_path):
    """A module that is newer than its source but was built for another torch is compiled again."""
    build.build_bind_library()
    built_for = build.BIND_STAMP.read_text()
    assert torch.__version__ in built_for
    compiled = []

    class Failed:
        returncode, stdout, stderr = 1, "", "not compiled in this test"

    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **kw: compiled.append(cmd) or Failed)
    monkeypatch.setattr(build, "BIND_STAMP", tmp_path / "stamp")
    build.BIND_STAMP.write_text(built_for)
    assert build.build_bind_library() == build.BIND_LIB and not compiled
    build.BIND_STAMP.write_text(built_for.replace(torch.__version__, "0.0"))
    with pytest.raises(RuntimeError, match="not compiled in this test"):
        build.build_bind_library()
    assert len(compiled) == 1 and not build.BIND_STAMP.exists()


# ------------------------------------------------------------------ rotary frequencies
def test_frequencies_without_scaling():
    f, m = lib.rope_frequencies(8, base=10000.0, device="cpu")
    assert m == 1.0 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001]))
    f, m = lib.rope_frequencies(8, base=10000.0, scaling={"type": "linear", "factor": 4}, device="cpu")
    assert m == 1.0 and torch.allclose(f, torch.tensor([0.25, 0.025, 0.0025, 0.00025]))


def test_frequencies_by_wavelength():
    """Short wavelengths as they are, long ones divided, a blend between that is continuous at both ends."""
    dims, base, old = 128, 5e5, 8192
    plain, _ = lib.rope_frequencies(dims, base=base, device="cpu")
    f, m = lib.rope_frequencies(dims, base=base, scaling={"type": "llama3", "factor": 8, "original_max_position": old,
                                                          "low_freq_factor": 1, "high_freq_factor": 4}, device="cpu")
    assert m == 1.0
    wave = 2 * math.pi / plain.double()
    short, long = wave <= old / 4, wave >= old
    assert bool(short.any()) and bool(long.any()) and not bool((short | long).all())
    assert torch.equal(f[short], plain[short]) and torch.allclose(f[long], plain[long] / 8, rtol=1e-6)
    mid = ~(short | long)
    k = ((old / wave - 1) / 3)[mid]
    assert torch.allclose(f[mid].double(), plain[mid].double() * (k + (1 - k) / 8), rtol=1e-6)


def test_frequencies_by_turns():
    dims, base = 128, 1e6
    plain, _ = lib.rope_frequencies(dims, base=base, device="cpu")
    f, m = lib.rope_frequencies(dims, base=base, scaling={"type": "yarn", "factor": 4, "original_max_position": 32768}, device="cpu")
    assert m == pytest.approx(0.1 * math.log(4) + 1)
    turns = 32768 * plain.double() / (2 * math.pi)
    ratio = (f.double() / plain.double())
    assert bool((ratio[turns > 40] == 1).all()) and torch.allclose(ratio[turns < 0.8], torch.tensor(0.25, dtype=torch.float64))
    assert bool((ratio.diff() <= 1e-9).all())


def test_frequencies_refuse():
    with pytest.raises(ValueError, match="must be even"):
        lib.rope_frequencies(7, device="cpu")
    with pytest.raises(ValueError, match="unknown rope scaling"):
        lib.rope_frequencies(8, scaling={"type": "x", "factor": 2}, device="cpu")
    with pytest.raises(ValueError, match="must be positive"):
        lib.rope_frequencies(8, scaling={"type": "linear", "factor": 0}, device="cpu")
    with pytest.raises(ValueError, match="must exceed"):
        lib.rope_frequencies(8, scaling={"type": "llama3", "factor": 2, "low_freq_factor": 4, "high_freq_factor": 4}, device="cpu")

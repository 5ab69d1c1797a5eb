"""Paged serving on the GPU against plain implementations in 64 bits: the step
plan (mt_paged_plan), the rotary append (mt_rope_paged_append), one-token
attention (mt_paged_sdpa_decode) and token log-probabilities
(mt_token_logprobs). Tolerances follow from the number formats: a result
rounded once to a type of unit roundoff u is within u|y|, fp32 arithmetic adds
a few 2^-24 of the magnitudes summed."""
import math

import numpy as np
import pytest
import torch

from metal_autotune_b200 import lib

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
U = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}  # unit roundoff
NAN, INF = float("nan"), float("inf")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def i32(a):
    return torch.as_tensor(a, dtype=torch.int32).cuda()


@pytest.fixture(autouse=True)
def clear_status(cuda):
    lib.device_status(clear=True)
    yield


# ------------------------------------------------------------------ plan
def plan_ref(ctx, new, table, free, head, page, cap):
    """The plan request by request; returns (table, seq_lens, query_start, positions, token_seq, slots, counts)."""
    table = table.copy()
    width = table.shape[1]
    positions, seq, slots = [0] * cap, [-1] * cap, [-1] * cap
    lens, start = [], [0]
    avail = len(free) - head
    wanted = taken = refused = 0
    for r, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(c, 0), max(n, 0)
        s = start[-1]
        start.append(s + n)
        had, need = -(-c // page), -(-(c + n) // page) - -(-c // page)
        fits = s + n <= cap and c + n <= width * page
        if not fits:
            need = 0
        ok = fits and (need == 0 or wanted + need <= avail)
        if ok:
            for j in range(need):
                table[r, had + j] = free[head + wanted + j]
            if need:
                taken = wanted + need
        wanted += need
        refused += not ok
        lens.append(c + n if ok else c)
        for i in range(n):
            if s + i < cap:
                p = c + i
                positions[s + i], seq[s + i] = p, r
                if ok and table[r, p // page] >= 0:
                    slots[s + i] = int(table[r, p // page]) * page + p % page
    return table, lens, start, positions, seq, slots, [start[-1], wanted, taken, refused, head + taken]


def run_plan(ctx, new, page, cap, width, *, n_free, head=0, pad=0, bad=False, seed=0):
    r = np.random.default_rng(seed)
    B = len(ctx)
    pages = r.permutation(100000).astype(np.int64)
    table = np.full((B, width), -7)
    k = 0
    for i, c in enumerate(ctx):
        held = min(-(-max(c, 0) // page), width)
        table[i, :held] = pages[k:k + held]
        k += held
        if bad and held and i % 3 == 0:
            table[i, held - 1] = -1  # a page that was never there
    free = pages[k:k + n_free]
    big = torch.full((B, width + pad), -9, dtype=torch.int32, device="cuda")
    dev = big[:, :width]
    dev.copy_(i32(table))
    args = (i32(ctx), i32(new), dev, i32(free))
    p = lib.paged_plan(*args, page_size=page, token_cap=cap, free_head=None if head == 0 else i32([head]))
    ref = plan_ref(list(ctx), list(new), table, free, head, page, cap)
    for name, got, want in zip(("table",) + lib.PagedPlan._fields, (dev, *p), ref):
        assert np.array_equal(got.cpu().numpy(), np.asarray(want).reshape(got.shape)), name
    if pad:
        assert bool((big[:, width:] == -9).all())
    again = lib.paged_plan(*args, page_size=page, token_cap=cap, free_head=None if head == 0 else i32([head]), out=lib.PagedPlan.empty(B, cap))
    assert all(torch.equal(x, y) for x, y in zip(p, again))


@pytest.mark.parametrize("B,page,max_new,max_ctx", [(1, 16, 1, 0), (1, 1, 40, 3), (7, 16, 1, 300), (33, 24, 90, 500), (513, 16, 3, 64),
                                                    (4097, 8, 2, 40), (9000, 128, 1, 300), (5, 7, 4000, 9)])
def test_plan(cuda, B, page, max_new, max_ctx):
    r = np.random.default_rng(B)
    ctx, new = r.integers(0, max_ctx + 1, B), r.integers(0, max_new + 1, B)
    total = int(new.sum())
    width = -(-(max_ctx + max_new) // page) + 1
    run_plan(ctx, new, page, total + 5, width, n_free=total + B, pad=3, seed=B)
    run_plan(ctx, new, page, max(total, 1), width, n_free=total + B + 11, head=11, bad=True, seed=B + 1)


def test_plan_refusals(cuda):
    ctx, new = [5, 0, 31, 16, 0, 3], [3, 40, 2, 0, 1, 1]
    run_plan(ctx, new, 16, 47, 8, n_free=50)       # everything fits
    run_plan(ctx, new, 16, 47, 8, n_free=3)        # out of pages inside the batch: later ones that need none go on
    run_plan(ctx, new, 16, 47, 8, n_free=0)
    run_plan(ctx, new, 16, 44, 8, n_free=50)       # out of token rows
    run_plan(ctx, new, 16, 0, 8, n_free=50)
    run_plan(ctx, new, 16, 47, 2, n_free=50)       # a request longer than its table row
    run_plan([5, -3], [-1, 2], 4, 8, 3, n_free=4)  # negative lengths count as 0


def test_plan_saturates(cuda):
    """Lengths whose sums pass 2^31: refused, nothing written out of place."""
    big = 2 ** 31 - 1
    table = torch.full((3, 4), -1, dtype=torch.int32, device="cuda")
    p = lib.paged_plan(i32([big, 0, 0]), i32([big, big, 1]), table, i32([1, 2]), page_size=1 << 20, token_cap=4)
    assert p.counts.tolist() == [big, 0, 0, 3, 0] and p.slots.tolist() == [-1] * 4
    assert p.seq_lens.tolist() == [big, 0, 0] and p.query_start.tolist() == [0, big, big, big]
    assert bool((table == -1).all())


def test_plan_no_requests(cuda):
    e = torch.empty(0, dtype=torch.int32, device="cuda")
    p = lib.paged_plan(e, e, torch.empty(0, 3, dtype=torch.int32, device="cuda"), e, page_size=16, token_cap=3)
    assert p.slots.tolist() == [-1, -1, -1] and p.query_start.tolist() == [0] and p.counts.tolist() == [0] * 5


def test_plan_step_after_step(cuda):
    """A step's lengths and head as the next one's inputs, with two sets of outputs in turn; head and lengths in the
    room beside the table's rows; one set for both is refused."""
    r = np.random.default_rng(4)
    B, page, width, cap, n_free = 700, 4, 40, 2600, 20000
    state = torch.full((B, width + 4), -9, dtype=torch.int32, device="cuda")
    table = state[:, :width]
    head = state[B - 1, width + 1:width + 2]
    head.zero_()
    free = i32(r.permutation(30000)[:n_free])
    lens, ref_table, ref_lens, ref_head = i32([0] * B), np.full((B, width), -9), [0] * B, 0
    sets = [lib.PagedPlan.empty(B, cap) for _ in range(2)]
    for step in range(6):
        new = r.integers(0, 6, B)
        p = lib.paged_plan(lens, i32(new), table, free, page_size=page, token_cap=cap, free_head=head, out=sets[step % 2])
        ref = plan_ref(ref_lens, list(new), ref_table, free.cpu().numpy(), ref_head, page, cap)
        for name, got, want in zip(("table",) + lib.PagedPlan._fields, (table, *p), ref):
            assert np.array_equal(got.cpu().numpy(), np.asarray(want).reshape(got.shape)), (step, name)
        lens, head = p.seq_lens, p.counts[4:]
        ref_table, ref_lens, ref_head = ref[0], ref[1], ref[6][4]
    for kw in (dict(ctx=p.seq_lens, head=None), dict(ctx=sets[0].seq_lens, head=p.counts[4:])):
        with pytest.raises(lib.MTError, match="overlaps"):
            lib.paged_plan(kw["ctx"], i32(new), table, free, page_size=page, token_cap=cap, free_head=kw["head"], out=p)


# ------------------------------------------------------------------ append
def cache_pair(pages, Hkv, page, D, dt, layout, fill=0.0):
    shape = (pages, Hkv, page, D) if layout == "hnd" else (pages, page, Hkv, D)
    mk = lambda: torch.full(shape, fill, dtype=dt, device="cuda")  # noqa: E731
    a, b = mk(), mk()
    return (a, b) if layout == "hnd" else (a.transpose(1, 2), b.transpose(1, 2))


def rotate_ref(x, pos, inv, dims, trad, mscale, w, eps):
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    a = pos.double()[:, None, None] * inv.double()
    c, s = torch.cos(a) * mscale, torch.sin(a) * mscale
    y = x.clone()
    i, j = (slice(0, dims, 2), slice(1, dims, 2)) if trad else (slice(0, dims // 2), slice(dims // 2, dims))
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    return y


APPEND = [
    # T, Hq, Hkv, D, dims, trad, norm, dtype, page, layout, max_pos
    (1, 32, 8, 128, 128, False, True, "bf16", 16, "hnd", 4096),
    (5, 32, 8, 128, 128, False, False, "f16", 16, "nhd", 131072),
    (37, 4, 2, 64, 32, True, True, "bf16", 24, "hnd", 100),
    (3, 3, 1, 80, 80, False, True, "f16", 7, "nhd", 2 ** 20),
    (6, 2, 2, 96, 24, False, True, "bf16", 8, "hnd", 50),     # half a rotation of 12: not whole lanes
    (6, 2, 1, 40, 10, False, False, "f32", 1, "hnd", 50),
    (4, 5, 3, 256, 64, True, True, "f32", 5, "nhd", 2 ** 30),
    (700, 8, 8, 64, 64, False, True, "bf16", 64, "hnd", 2 ** 31 - 1),
    (2, 4, 2, 8, 0, False, False, "bf16", 2, "hnd", 10),      # nothing rotated: a plain append
    (600, 20, 4, 128, 64, False, True, "f16", 16, "nhd", 9000),
]


@pytest.mark.parametrize("T,Hq,Hkv,D,dims,trad,norm,dtype,page,layout,max_pos", APPEND)
def test_append(cuda, T, Hq, Hkv, D, dims, trad, norm, dtype, page, layout, max_pos):
    g, dt = gen(T + D), DT[dtype]
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D + 8, generator=g, device="cuda").to(dt)  # rows wider than their parts
    q, k, v = (t.unflatten(1, (-1, D)) for t in qkv[:, :-8].split((Hq * D, Hkv * D, Hkv * D), 1))
    pos = torch.randint(0, max_pos, (T,), generator=g, device="cuda").int()
    pages = -(-T // page) + 2
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:T]
    slots[torch.rand(T, generator=g, device="cuda") < 0.1] = -1
    inv, _ = lib.rope_frequencies(dims, base=1e4) if dims else (torch.empty(0, device="cuda"), 1.0)
    weight = lambda: (1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(dt) if norm else None  # noqa: E731
    qw, kw = weight(), weight()
    ms = 1.25
    kc, vc = cache_pair(pages, Hkv, page, D, dt, layout, fill=3.0)
    k_out = torch.empty(T, Hkv, D, dtype=dt, device="cuda")
    before = qkv.clone()
    y = lib.rope_paged_append(q, k, v, pos, slots, kc, vc, inv, traditional=trad, mscale=ms, q_norm_w=qw, k_norm_w=kw, eps=1e-5, k_out=k_out)
    assert torch.equal(qkv, before)
    u = U[dtype]
    # rounding once, and fp32 arithmetic on values up to |row|max * mscale (norm: a handful of operations each)
    for got, x, w in ((y, q, qw), (k_out, k, kw)):
        ref = rotate_ref(x, pos, inv, dims, trad, ms, w, 1e-5)
        tol = 1.01 * u * ref.abs() + 32 * 2.0 ** -24 * ref.abs().amax(-1, keepdim=True)
        assert bool(((got.double() - ref).abs() <= tol).all()), (got.double() - ref).abs().max()
    real = slots >= 0
    at = (slots[real] // page, slice(None), slots[real] % page)
    assert torch.equal(kc[at], k_out[real]) and torch.equal(vc[at], v[real])
    untouched = torch.ones(pages, page, dtype=torch.bool, device="cuda")
    untouched[slots[real] // page, slots[real] % page] = False
    assert bool((kc.transpose(1, 2)[untouched] == 3.0).all()) and bool((vc.transpose(1, 2)[untouched] == 3.0).all())
    # in place, with the same bits
    kc2, vc2 = cache_pair(pages, Hkv, page, D, dt, layout)
    q2 = q.clone()
    assert lib.rope_paged_append(q2, k, v, pos, slots, kc2, vc2, inv, traditional=trad, mscale=ms, q_norm_w=qw, k_norm_w=kw, eps=1e-5, out=q2) is q2
    assert torch.equal(q2, y) and torch.equal(kc2[at], kc[at])
    assert lib.device_status() == 0


@pytest.mark.parametrize("dims,trad,norm", [(128, False, True), (64, True, False)])
def test_append_many_f32_rows(cuda, dims, trad, norm):
    test_append(cuda, 900, 8, 2, 128, dims, trad, norm, "f32", 16, "hnd", 5000)


def test_append_matches_dense_rope(cuda):
    """Without norm or scaling: the same rotation as mt_rope at each token's position, up to one rounding step."""
    g, T, H, D = gen(3), 9, 4, 128
    q = torch.randn(T, H, D, generator=g, device="cuda").bfloat16()
    k = torch.randn(T, 2, D, generator=g, device="cuda").bfloat16()
    inv, _ = lib.rope_frequencies(D, base=1e6)
    kc, vc = cache_pair(2, 2, 16, D, torch.bfloat16, "hnd")
    y = lib.rope_paged_append(q, k, k, torch.arange(40, 40 + T, device="cuda").int(), torch.arange(T, device="cuda"), kc, vc, inv)
    ref = lib.rope(q.transpose(0, 1).contiguous(), D, base=1e6, offset=40).transpose(0, 1)
    assert bool(((y.float() - ref.float()).abs() <= 2.0 ** -8 * ref.float().abs() + 1e-5).all())


def test_append_slot_past_the_cache(cuda):
    q = torch.ones(2, 2, 64, device="cuda").half()
    kc, vc = cache_pair(2, 2, 4, 64, torch.float16, "hnd")
    inv, _ = lib.rope_frequencies(64)
    lib.rope_paged_append(q, q, q, i32([0, 1]), torch.tensor([8, 2 ** 40], device="cuda"), kc, vc, inv)
    assert lib.device_status() == 0x701 and not bool(kc.any()) and not bool(vc.any())


def test_append_offsets_past_32_bits(cuda):
    """Rows more than 2^31 elements into the cache."""
    D, Hkv, page, pages = 128, 8, 64, 34000  # 2.2e9 elements, 4.5 GB a cache
    kc = torch.empty(pages, Hkv, page, D, dtype=torch.bfloat16, device="cuda")
    vc = torch.empty_like(kc)
    g = gen(1)
    q = torch.randn(3, 32, D, generator=g, device="cuda").bfloat16()
    k, v = (torch.randn(3, Hkv, D, generator=g, device="cuda").bfloat16() for _ in range(2))
    slots = torch.tensor([pages * page - 1, pages * page - 70, 5], device="cuda")
    inv, _ = lib.rope_frequencies(D)
    k_out = torch.empty_like(k)
    qr = lib.rope_paged_append(q, k, v, i32([7, 8, 9]), slots, kc, vc, inv, k_out=k_out)
    at = (slots // page, slice(None), slots % page)
    assert torch.equal(kc[at], k_out) and torch.equal(vc[at], v)
    # attention over one key is its value row
    o = lib.paged_sdpa_decode(qr[:1], kc[:, :, page - 1:], vc[:, :, page - 1:], i32([[pages - 1]]), i32([1]), scale=0.1)
    assert torch.equal(o[0].view(Hkv, 4, D), v[0][:, None].expand(Hkv, 4, D))


def test_attend_offsets_past_32_bits(cuda):
    """Pages more than 2^31 elements into the cache, by the copy engine and row by row."""
    D, Hkv, page, pages = 64, 4, 32, 270000  # 2.2e9 elements
    g = gen(2)
    kc, vc = (torch.empty(pages, Hkv, page, D, dtype=torch.float16, device="cuda") for _ in range(2))
    rows = torch.tensor([pages - 1, 3, pages - 2], device="cuda")
    for c in (kc, vc):
        c[rows] = torch.randn(3, Hkv, page, D, generator=g, device="cuda").half()
    q = torch.randn(1, 8, D, generator=g, device="cuda").half()
    table = rows[None].int()
    check_attend(q, kc, vc, table, i32([90]), 0.125, "f16")
    # the same rows as pages of 31 whose last row is never a key: no whole boxes
    check_attend(q, kc[:, :, :31], vc[:, :, :31], table, i32([93]), 0.125, "f16")


# ------------------------------------------------------------------ attention
def attend_ref(q, kc, vc, table, lens, scale):
    """64-bit result and sum p|v| per output value; keys on pages outside the cache are left out."""
    B, Hq, D = q.shape
    pages, Hkv, page, _ = kc.shape
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(out)
    for b in range(B):
        key = torch.arange(max(0, min(int(lens[b]), table.shape[1] * page)), device="cuda")
        pg = table[b].long()[key // page]
        key, pg = key[(pg >= 0) & (pg < pages)], pg[(pg >= 0) & (pg < pages)]
        if not len(key):
            continue
        k, v = kc[pg, :, key % page].double(), vc[pg, :, key % page].double()
        p = torch.softmax(torch.einsum("hgd,nhd->hgn", q[b].double().view(Hkv, -1, D), k) * scale, -1)
        out[b] = torch.einsum("hgn,nhd->hgd", p, v).reshape(Hq, D)
        mag[b] = torch.einsum("hgn,nhd->hgd", p, v.abs()).reshape(Hq, D)
    return out, mag


def attend_case(lens, Hq, Hkv, D, page, dtype, layout="hnd", seed=0, spread=2.0, extra_pages=1):
    g, dt = gen(seed), DT[dtype]
    B = len(lens)
    held = [-(-max(n, 0) // page) for n in lens]
    pages = sum(held) + extra_pages
    kc, vc = cache_pair(pages, Hkv, page, D, dt, layout, fill=NAN)  # what no request holds must not be looked at
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((B, max(max(held), 1)), 2 ** 30, dtype=torch.int32, device="cuda")
    k = 0
    for b, h in enumerate(held):
        table[b, :h] = order[k:k + h]
        k += h
        if h:
            rows = torch.zeros(h * page, dtype=torch.bool, device="cuda")
            rows[:lens[b]] = True
            for c in (kc, vc):
                c[order[k - h:k].long()] = torch.where(rows.view(h, 1, page, 1), torch.randn(h, Hkv, page, D, generator=g, device="cuda"), NAN).to(dt)
    q = (spread * torch.randn(B, Hq, D, generator=g, device="cuda")).to(dt)
    return q, kc, vc, table, i32(lens)


def check_attend(q, kc, vc, table, lens, scale, dtype, **kw):
    o = lib.paged_sdpa_decode(q, kc, vc, table, lens, scale=scale, **kw)
    ref, mag = attend_ref(q, kc, vc, table, lens, scale)
    # one rounding of the output, one of each probability, fp32 sums
    tol = 1.05 * U[dtype] * (ref.abs() + mag) + 1e-6 * (1 + mag)
    assert not bool(torch.isnan(o).any())
    assert bool(((o.double() - ref).abs() <= tol).all()), ((o.double() - ref).abs() / tol).max()
    return o


ATTEND = [
    # lens, Hq, Hkv, D, page, dtype, layout
    ([1], 32, 8, 128, 16, "bf16", "hnd"),
    ([129], 32, 8, 128, 16, "bf16", "nhd"),
    ([0], 4, 2, 64, 16, "bf16", "hnd"),
    ([0, 0, 5, 0, 64, 65, 0], 8, 2, 128, 8, "f16", "hnd"),
    ([15, 16, 17, 63, 64, 65, 127, 128, 1000], 4, 4, 64, 24, "bf16", "nhd"),
    ([300, 2, 77], 16, 2, 128, 7, "f16", "hnd"),           # 8 rows a head, pages that end inside every step
    ([100, 513], 32, 2, 64, 16, "bf16", "hnd"),            # 16 rows a head
    ([90, 33], 20, 1, 128, 1, "f16", "hnd"),               # 20 rows: two blocks; one row a page
    ([70, 1500], 9, 1, 64, 128, "bf16", "nhd"),
    ([33333], 32, 8, 128, 64, "bf16", "hnd"),              # one request over every CTA
    ([20000, 3, 0, 9000, 1], 5, 1, 128, 16, "f16", "nhd"),
    ([1] * 700, 2, 1, 64, 4, "bf16", "hnd"),               # more requests than CTAs, one key each
    (list(range(0, 1400, 7)), 8, 2, 128, 16, "bf16", "hnd"),
    ([(37 * i) % 301 for i in range(600)], 32, 8, 128, 16, "bf16", "hnd"),  # many short requests, more than are scanned at once
    ([(37 * i) % 301 for i in range(600)], 8, 8, 64, 12, "f16", "nhd"),
    ([400 + (91 * i) % 300 for i in range(300)], 6, 1, 128, 8, "bf16", "nhd"),
    ([2000, 0, 1, 900, 4097], 48, 4, 128, 32, "f16", "hnd"),  # 12 rows a head
    ([31, 32, 33, 95, 1000, 5000], 12, 2, 128, 32, "bf16", "hnd"),   # few units: steps of 32 keys, 6 rows a head
    ([7, 0, 40, 129, 3000], 4, 2, 128, 8, "f16", "nhd"),
    ([40, 777, 5], 4, 1, 128, 9, "bf16", "hnd"),
    ([20 + i for i in range(140)], 16, 4, 128, 48, "bf16", "nhd"),   # more units: steps of 16
    ([1000, 33, 64], 8, 1, 64, 32, "bf16", "hnd"),
]


@pytest.mark.parametrize("lens,Hq,Hkv,D,page,dtype,layout", ATTEND)
def test_attend(cuda, lens, Hq, Hkv, D, page, dtype, layout):
    case = attend_case(lens, Hq, Hkv, D, page, dtype, layout, seed=len(lens) + Hq)
    o = check_attend(*case, 1 / math.sqrt(D), dtype)
    for b, n in enumerate(lens):
        if n == 0:
            assert not bool(o[b].any())
    for _ in range(3):  # the same bits again, whoever arrives last
        assert torch.equal(o, lib.paged_sdpa_decode(*case, scale=1 / math.sqrt(D)))
    assert lib.device_status() == 0


def test_attend_strided(cuda):
    """q and out as views of wider rows, a table wider than it is used, a cache view with room between its rows."""
    lens, Hq, Hkv, D, page = [70, 0, 300], 8, 2, 64, 16
    q, kc, vc, table, ln = attend_case(lens, Hq, Hkv, D, page, "bf16", seed=5)
    wide = torch.zeros(3, Hq + 3, D + 8, dtype=torch.bfloat16, device="cuda")
    qv = wide[:, 1:Hq + 1, :D]
    qv.copy_(q)
    big = [torch.zeros(c.shape[0], Hkv, page + 1, D + 16, dtype=torch.bfloat16, device="cuda") for c in (kc, vc)]
    views = [b[:, :, :page, :D] for b in big]
    for w, c in zip(views, (kc, vc)):
        w.copy_(c)
    tw = torch.full((3, table.shape[1] + 5), -1, dtype=torch.int32, device="cuda")
    tw[:, :table.shape[1]] = table
    out = torch.full_like(wide, 7.0)
    o = check_attend(qv, *views, tw[:, :table.shape[1]], ln, 0.125, "bf16", out=out[:, 1:Hq + 1, :D])
    assert torch.equal(o, lib.paged_sdpa_decode(q, kc, vc, table, ln, scale=0.125))
    out[:, 1:Hq + 1, :D] = 7.0
    assert bool((out == 7.0).all())


def test_attend_large_and_equal_scores(cuda):
    """Scores in the hundreds, all scores equal, scale 0, a negative scale."""
    q, kc, vc, table, ln = attend_case([513, 40], 8, 2, 128, 16, "bf16", seed=8, spread=40.0)
    check_attend(q, kc, vc, table, ln, 0.25, "bf16")
    check_attend(q, kc, vc, table, ln, 0.0, "bf16")
    check_attend(q, kc, vc, table, ln, -0.03, "bf16")
    check_attend(torch.zeros_like(q), kc, vc, table, ln, 1.0, "bf16")


def test_attend_infinities(cuda):
    """-inf in k hides a key where q is positive; every score -inf gives zeros; NaN stays in its request and head."""
    q, kc, vc, table, ln = attend_case([100, 200, 50], 4, 2, 64, 16, "bf16", seed=9)
    q = q.abs() + 0.1
    clean = lib.paged_sdpa_decode(q, kc, vc, table, ln, scale=0.125)
    for key in range(0, 200, 3):
        kc[table[1, key // 16].long(), 1, key % 16] = -INF
    ref, mag = attend_ref(q, kc, vc, table, ln, 0.125)
    o = lib.paged_sdpa_decode(q, kc, vc, table, ln, scale=0.125)
    assert bool(((o.double() - ref).abs() <= 1.05 * U["bf16"] * (ref.abs() + mag) + 1e-6 * (1 + mag)).all())
    kc[table[1, :13].long(), 1] = -INF
    vc[table[0, 0].long(), 0, 3, 5] = NAN
    o = lib.paged_sdpa_decode(q, kc, vc, table, ln, scale=0.125)
    assert not bool(o[1, 2:].any()) and torch.equal(o[1, :2], clean[1, :2])
    bad = torch.isnan(o)
    assert bool(bad[0, :2, 5].all()) and int(bad.sum()) == 2
    assert torch.equal(o[2], clean[2])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("below", [12, 15, 17, 20])
def test_attend_strong_keys_without_a_value(cuda, D, below, dtype):
    """A few keys draw the attention and hold zeros; the output is what the thousands of keys `below` nats under them
    (within a quarter) carry, each with a probability far under the type's lowest normal number."""
    g, dt = gen(below + D), DT[dtype]
    lens, Hq, Hkv, page = [3900 + 13 * i for i in range(20)], 16, 4, 16
    q, kc, vc, table, ln = attend_case(lens, Hq, Hkv, D, page, dtype, seed=below)
    q.zero_()
    q[..., 0] = 8.0
    kc[..., 0] = torch.where(torch.isnan(kc[..., 0]), NAN, 0.02 * torch.randn(kc.shape[:-1], generator=g, device="cuda").clamp(-1.5, 1.5)).to(dt)
    vc.abs_()
    strong = torch.arange(0, 128, 16, device="cuda")  # one at least for each warp
    for b in range(len(lens)):
        at = (table[b, strong // page].long(), slice(None), strong % page)
        kc[(*at, 0)] = below / 8
        vc[at] = 0.0
    o = lib.paged_sdpa_decode(q, kc, vc, table, ln, scale=1.0)
    ref, mag = attend_ref(q, kc, vc, table, ln, 1.0)
    # the output's rounding (2^-25 where f16 is subnormal), one of each probability (f16 holds the largest as 2^15, so
    # 2^-40 of it where they are subnormal, |v| < 8), and fp32 arithmetic on scores of up to 30 in the exponent of 2
    tol = 1.05 * U[dtype] * (ref.abs() + mag) + 1e-5 * mag
    if dtype == "f16":
        tol += 2.0 ** -25 + max(lens) * 8 * 2.0 ** -40
    assert bool(((o.double() - ref).abs() <= tol).all()), ((o.double() - ref).abs() / tol).max()


@pytest.mark.parametrize("lens,Hq,Hkv,D,page", [([33333], 32, 8, 128, 16), ([9000, 40], 12, 1, 64, 24),
                                                ([1 + (2 * i) % 511 for i in range(256)], 32, 8, 128, 16)])
def test_attend_nan_in_split_requests(cuda, lens, Hq, Hkv, D, page):
    """A query row or keys of NaN give NaN however many workers (CTAs or warps) share the request, and only in their rows."""
    q, kc, vc, table, ln = attend_case(lens, Hq, Hkv, D, page, "bf16", seed=17)
    clean = lib.paged_sdpa_decode(q, kc, vc, table, ln, scale=0.1)
    bad = q.clone()
    bad[:, 3, 7] = NAN
    o = lib.paged_sdpa_decode(bad, kc, vc, table, ln, scale=0.1)
    others = torch.arange(Hq, device="cuda") != 3
    assert bool(torch.isnan(o[:, 3]).all()) and torch.equal(o[:, others], clean[:, others])
    # the first n keys of the last kv head: some n ends where the first worker's run does
    G, was = Hq // Hkv, kc.clone()
    for n in [*range(64, min(max(lens), 2600), 64), max(lens)]:
        for b in range(len(lens)):
            key = torch.arange(min(n, lens[b]), device="cuda")
            kc[table[b].long()[key // page], Hkv - 1, key % page, 1] = NAN
        o = lib.paged_sdpa_decode(q, kc, vc, table, ln, scale=0.1)
        assert bool(torch.isnan(o[:, -G:]).all()), n
        assert torch.equal(o[:, :-G], clean[:, :-G])
        kc.copy_(was)


def test_attend_missing_pages(cuda):
    """Keys on a page id outside the cache are hidden and reported; a length past the table is cut."""
    q, kc, vc, table, ln = attend_case([100, 64], 4, 2, 64, 16, "f16", seed=4)
    vc.nan_to_num_(0.0)
    kc.nan_to_num_(0.0)
    table[0, 2], table[1] = -1, kc.shape[0]
    o = check_attend(q, kc, vc, table, ln, 0.125, "f16")
    assert lib.device_status() == 0x702 and not bool(o[1].any())
    short = table[:, :2].contiguous()
    check_attend(q, kc, vc, short, i32([2 ** 31 - 1, 0]), 0.125, "f16")


def test_attend_on_a_stream_of_its_own(cuda):
    q, kc, vc, table, ln = attend_case([3000, 5, 900], 8, 2, 128, 16, "bf16", seed=6)
    want = lib.paged_sdpa_decode(q, kc, vc, table, ln, scale=0.1)
    torch.cuda.synchronize()
    side, ws = torch.cuda.Stream(), lib.Workspace(torch.cuda.current_device(), lib.paged_sdpa_decode_workspace_bytes(128))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = [lib.paged_sdpa_decode(q, kc, vc, table, ln, scale=0.1, workspace=ws) for _ in range(20)]
    here = [lib.paged_sdpa_decode(q, kc, vc, table, ln, scale=0.1) for _ in range(20)]
    torch.cuda.synchronize()
    assert all(torch.equal(want, o) for o in got + here)
    assert not bool(ws.buf[:65536].any())


# ------------------------------------------------------------------ log-probabilities
def logprob_ref(x, tokens, k):
    x = x.double().cpu().numpy()
    R, V = x.shape
    m = x.max(1, keepdims=True)
    z = x - m
    e = np.exp(z)
    s = e.sum(1, keepdims=True)
    lse = m + np.log(s)
    H = np.log(s[:, 0]) - np.where(e > 0, e * np.where(e > 0, z, 0), 0).sum(1) / s[:, 0]
    lp = np.array([x[r, t] - lse[r, 0] if 0 <= t < V else 0.0 for r, t in enumerate(tokens)])
    ids = np.lexsort((np.broadcast_to(np.arange(V), x.shape), -x), axis=1)[:, :k] if k else np.zeros((R, 0), int)
    return lp, H, lse[:, 0], ids, np.take_along_axis(x, ids, 1) - lse


def check_logprobs(x, tokens, k):
    p = lib.token_logprobs(x, i32(tokens), top_k=k)
    with np.errstate(all="ignore"):
        lp, H, lse, ids, top = logprob_ref(x, tokens, k)
    assert np.array_equal(p.top_ids.cpu().numpy(), ids)
    xs = x.float().cpu().numpy()
    # lse and log-probabilities: fp32 arithmetic on logits and sums of the row's magnitude, and the result's own rounding
    tol = 4 * 2.0 ** -24 * (np.abs(xs.max(1)) + 16)

    def near(got, want, more=0.0):
        got = got.double().cpu().numpy()
        bound = 2.0 ** -24 * np.abs(want) + (tol if want.ndim == 1 else tol[:, None]) + more
        with np.errstate(invalid="ignore"):
            assert ((got == want) | (np.abs(got - want) <= bound)).all()

    near(p.lse, lse)
    near(p.logprob, lp)
    near(p.top_logprobs, top)
    near(p.entropy, H)
    return p


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("R,V,k", [(1, 1, 1), (3, 2, 2), (2, 31, 5), (5, 1000, 32), (1, 151936, 20), (4, 50001, 7), (9, 4097, 0), (300, 8191, 3),
                                   (2, 33, 32), (700, 2048, 20)])
def test_logprobs(cuda, dtype, R, V, k):
    g = gen(R + V)
    x = (3 * torch.randn(R, V, generator=g, device="cuda")).to(DT[dtype])
    tokens = torch.randint(0, V, (R,), generator=g, device="cuda").tolist()
    p = check_logprobs(x, tokens, k)
    q = lib.token_logprobs(x, i32(tokens), top_k=k)
    assert all(torch.equal(a, b) for a, b in zip(p, q))
    assert lib.device_status() == 0


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("off", [0, 1, 3])
def test_logprobs_unaligned_rows(cuda, dtype, off):
    x = (2 * torch.randn(6, 20011, generator=gen(off), device="cuda")).to(DT[dtype])
    check_logprobs(x[:, off:20011 - 3 + off], [0, 1, 5, 19000, -1, 20007], 10)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_logprobs_ties_masks_and_extremes(cuda, dtype):
    V, dt = 40000, DT[dtype]
    low = torch.finfo(dt).min
    g = gen(11)
    x = (2 * torch.randn(12, V, generator=g, device="cuda"))
    x[0] = 1.5                                       # all equal
    x[1] = -INF
    x[1, [39999, 7, 20000]] = torch.tensor([1.0, 1.0, -2.0], device="cuda")  # three allowed tokens
    x[2] = low                                       # every logit the type's lowest
    x[3] = low
    x[3, 12345] = 4.0
    x[4] = torch.arange(V, device="cuda") * (1 / 4096)  # rising: every value passes what came before
    x[5] = -torch.arange(V, device="cuda") * (1 / 4096)
    x[6, 39998] = 60000.0 if dtype != "f16" else 600.0  # certain
    x[7] = torch.where(torch.rand(V, generator=g, device="cuda") < 0.5, 0.0, -0.0)  # -0 and 0 are equal
    x[8, 100:] = -INF
    x[9] = -60000.0
    x[9, 5:] = -INF
    x[10] = torch.where(torch.arange(V, device="cuda") >= V // 2, 50.0, -50.0)  # the later half carries everything
    x = x.to(dt)
    for k in (0, 1, 20, 32):
        check_logprobs(x, [0, 7, 3, 12345, 0, 0, 39998, 1, 50, 2, 30000, 9], k)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("R", [1, 700])
def test_logprobs_of_a_certain_token(cuda, dtype, R):
    """One value carries the row: its log-probability is 0 but for the rest's share, however large the logit, and no
    log-probability is positive."""
    V, dt = 20000, DT[dtype]
    rows = [(30.0, 0.0), (600.0, 0.0), (20000.0, 1.0), (60000.0, -100.0), (-20000.0, -INF), (-100.0, -140.0), (33.3, 0.0), (25.7, -3.0)]
    for r0 in range(0, len(rows), 1 if R == 1 else len(rows)):
        pairs = [rows[r0]] if R == 1 else [rows[i % len(rows)] for i in range(R)]
        x = torch.tensor([low for _, low in pairs], device="cuda")[:, None].repeat(1, V)
        ids = [(7919 * i + 11) % V for i in range(R)]
        x[torch.arange(R), ids] = torch.tensor([high for high, _ in pairs], device="cuda")
        x = x.to(dt)
        p = lib.token_logprobs(x, i32(ids), top_k=2)
        with np.errstate(all="ignore"):
            lp, H, _, _, top = logprob_ref(x, ids, 2)
        # the power's error, 2^-22, and a few roundings of numbers up to 1; none of the logit's size
        for got, want in ((p.logprob, lp), (p.top_logprobs[:, 0], top[:, 0])):
            assert np.all(np.abs(got.double().cpu().numpy() - want) <= 2.0 ** -21)
            assert bool((got <= 0).all())
        assert bool((p.top_logprobs <= 0).all()) and bool((p.entropy >= 0).all())
        assert np.all(np.abs(p.entropy.double().cpu().numpy() - H) <= 2.0 ** -20)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("R,V", [(1, 151936), (5, 40003), (300, 4999)])
def test_logprobs_one_range_of_ids_allowed(cuda, dtype, R, V):
    """Most parts of a row hold -inf alone, or the type's lowest value: at its start, its end and between."""
    g, dt = gen(R + V), DT[dtype]
    values = (2 * torch.randn(R, V + 1, generator=g, device="cuda")).to(dt)
    low = torch.finfo(dt).min
    for off, a, n, shut in ((0, 0, 40, -INF), (1, V // 2, 300, -INF), (1, V - 1, 1, -INF), (0, V - 700, 700, low), (1, 2, 3, low)):
        x = torch.full((R, V + 1), shut, dtype=dt, device="cuda")[:, off:off + V]
        x[:, a:a + n] = values[:, a:a + n]
        x[R // 2, 17] = low  # one finite value in an empty part
        for k in (0, 5, 32):
            check_logprobs(x, [a] * R, k)
        x[R - 1, (a + V // 2) % V] = NAN  # in a part that is else empty
        p = lib.token_logprobs(x, i32([a] * R), top_k=2)
        bad = torch.isnan(torch.stack([p.logprob, p.lse, p.entropy]))
        assert bool(bad[:, R - 1].all()) and not bool(bad[:, :R - 1].any()) and int(p.top_ids[R - 1, 0]) == (a + V // 2) % V


@pytest.mark.parametrize("R", [1, 100])
@pytest.mark.parametrize("k", [0, 20])
def test_logprobs_range_costs_what_scattered_ids_cost(cuda, R, k):
    """Empty parts of a row are not left to the slow exact form: 3 times the time of as many ids scattered is far above
    what they should take (some microseconds more) and far below what they took (9 to 12 times)."""
    V, n = 151936, 1519

    def least(ids):
        x = torch.full((R, V), -INF, device="cuda")
        x[:, ids] = torch.randn(R, n, generator=gen(1), device="cuda")
        x = x.bfloat16()
        times = []
        for _ in range(12):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(20):
                lib.token_logprobs(x, top_k=k)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    one_range = least(torch.arange(70000, 70000 + n, device="cuda"))
    scattered = least(torch.randperm(V, generator=gen(2), device="cuda")[:n])
    assert one_range < 3 * scattered, (one_range, scattered)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_logprobs_range_among_lowest_values(cuda, dtype):
    """The same where a mask writes the type's lowest value instead of -inf; parts of one very low value, and a row of it."""
    R, V, n, dt = 4, 151936, 1519, DT[dtype]
    low = torch.finfo(dt).min

    def least(x):
        times = []
        for _ in range(12):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(20):
                lib.token_logprobs(x, top_k=20)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    took = []
    for ids in (torch.arange(70000, 70000 + n, device="cuda"), torch.randperm(V, generator=gen(2), device="cuda")[:n]):
        x = torch.full((R, V), low, dtype=dt, device="cuda")
        x[:, ids] = torch.randn(R, n, generator=gen(1), device="cuda").to(dt)
        took.append(least(x))
        x[1] = low
        x[2] = -50000.0
        x[3, :100000] = -40000.0
        check_logprobs(x, [int(ids[0]), 5, 151935, 7], 20)
    assert took[0] < 3 * took[1], took


def test_logprobs_no_distribution(cuda):
    V = 5000
    x = torch.randn(5, V, generator=gen(2), device="cuda")
    x[0, 4000] = NAN
    x[1, 10] = INF
    x[2] = -INF
    x[3, [2, 4999]] = NAN
    p = lib.token_logprobs(x, i32([0, 1, 2, 3, 4]), top_k=3)
    for t in (p.logprob, p.entropy, p.lse, p.top_logprobs):
        assert bool(torch.isnan(t[:4].flatten(1) if t.dim() > 1 else t[:4]).all()) and bool(torch.isfinite(t[4]).all())
    assert int(p.top_ids[0, 0]) == 4000 and int(p.top_ids[1, 0]) == 10
    assert p.top_ids[2].tolist() == [0, 1, 2] and p.top_ids[3, :2].tolist() == [2, 4999]


def test_logprobs_tokens(cuda):
    x = torch.randn(4, 100, generator=gen(1), device="cuda").bfloat16()
    p = lib.token_logprobs(x, i32([-1, -5, 99, 0]))
    assert p.logprob[:2].tolist() == [0.0, 0.0] and p.top_ids.shape == (4, 0) and lib.device_status() == 0
    p = lib.token_logprobs(x, i32([100, 1, 1, 1]))
    assert p.logprob[0].item() == 0.0 and lib.device_status() == 0x801
    p = lib.token_logprobs(x, top_k=2)
    assert p.logprob is None and p.top_ids.shape == (4, 2)
    e = lib.token_logprobs(x[:0], i32([]), top_k=2)
    assert e.lse.numel() == 0


def test_logprobs_agree_with_the_greedy_pick(cuda):
    x = (3 * torch.randn(1, 151936, generator=gen(77), device="cuda"))
    token, logprob, lse = lib.logits_pick(x[0])
    p = lib.token_logprobs(x, token, top_k=1)
    assert int(p.top_ids[0, 0]) == int(token)
    assert abs(float(p.lse) - float(lse)) < 1e-4 and abs(float(p.logprob) - float(logprob)) < 1e-4

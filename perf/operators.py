"""The cases on which the paged-serving operators are measured.

Four operators that one step of a batched server runs over a paged key-value cache:

  plan      request lengths -> block tables, slots and positions of the step's tokens
  append    rotary positions (either layout, part of the head, scaled frequencies, optional q/k RMSNorm) of the
            step's q and k rows, k and v written to their slots of the cache
  attend    attention of one new token per request over its pages
  logprobs  log-probability of given tokens with entropy, logsumexp and the top alternatives

`run` computes an operator in its plain form (torch operations in 32 bits, rounded once) while `own` is false, and
calls the package's entry points while it is true.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # a decode step of a small server: eight requests, one new token each
        {"name": "plan decode 8", "op": "plan", "requests": 8, "tokens": 8, "max_ctx": 4096, "page": 16},
        # a mixed step of a large one: mostly decoding, some prompts entering in chunks
        {"name": "plan mixed 4096", "op": "plan", "requests": 4096, "tokens": 131072, "max_ctx": 8192, "page": 16},
        # decode rows of the 32/8-head decoder with q/k norms
        {"name": "append decode 4", "op": "append", "dtype": "bf16", "tokens": 4, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "traditional": False, "norm": True, "factor": 1.0, "max_pos": 4096, "page": 16},
        # prompt chunks of several requests entering the cache together, positions scaled for long contexts
        {"name": "append prompt 8192", "op": "append", "dtype": "bf16", "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "traditional": False, "norm": True, "factor": 8.0, "max_pos": 131072, "page": 64},
        # adjacent pairs over half of a 64-wide head, no norms, an odd number of rows, f16
        {"name": "append part 1111", "op": "append", "dtype": "f16", "tokens": 1111, "heads": 16, "kv_heads": 4, "dim": 64, "rot": 32,
         "traditional": True, "norm": False, "factor": 1.0, "max_pos": 2048, "page": 24},
        # one request just past the 128-token prompt: the latency of a single user's step
        {"name": "attend 1 x 129", "op": "attend", "dtype": "bf16", "requests": 1, "min_len": 129, "max_len": 129, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16},
        # a full server with ragged contexts
        {"name": "attend 64 x 8192", "op": "attend", "dtype": "bf16", "requests": 64, "min_len": 64, "max_len": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "page": 16},
        # one long document
        {"name": "attend 1 x 131072", "op": "attend", "dtype": "bf16", "requests": 1, "min_len": 131072, "max_len": 131072, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64},
        # heads of their own (20 of 64), pages of 24 that end inside every tile, idle slots of the batch (length 0)
        {"name": "attend 37 x 1500 f16", "op": "attend", "dtype": "f16", "requests": 37, "min_len": 0, "max_len": 1500, "heads": 20, "kv_heads": 20, "dim": 64, "page": 24},
        # the picked token of one decode step with its alternatives
        {"name": "logprobs 1", "op": "logprobs", "dtype": "bf16", "rows": 1, "vocab": 151936, "top": 20, "allowed": 1.0},
        # scoring of prompts: each token's log-probability and alternatives
        {"name": "logprobs 2048", "op": "logprobs", "dtype": "bf16", "rows": 2048, "vocab": 151936, "top": 20, "allowed": 1.0},
        # a grammar that leaves a hundredth of an odd vocabulary, f32 logits
        {"name": "logprobs 96 masked", "op": "logprobs", "dtype": "f32", "rows": 96, "vocab": 32003, "top": 5, "allowed": 0.01},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], uniform in its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "append", "attend", "attend", "logprobs"])
    page = rng.choice([8, 16, 24, 32, 64, 128])
    if op == "plan":
        requests = _spread(rng, 1, 4096)
        return {"op": op, "requests": requests, "tokens": requests if rng.random() < 0.4 else _spread(rng, requests, 131072),
                "max_ctx": _spread(rng, 16, 8192), "page": page}
    dtype = rng.choice(["bf16", "bf16", "f16"])
    heads, kv_heads = rng.choice([(32, 8), (16, 4), (8, 2), (4, 4), (20, 20), (16, 1)])
    if op == "append":
        dim, rot = rng.choice([(128, 128), (128, 128), (128, 64), (64, 64), (64, 32), (80, 80), (96, 48), (256, 64)])
        return {"op": op, "dtype": dtype, "tokens": _spread(rng, 1, min(8192, 8192 * 48 * 128 // ((heads + 2 * kv_heads) * dim))),
                "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rot, "traditional": rng.random() < 0.5,
                "norm": rng.random() < 0.5, "factor": rng.choice([1.0, 4.0, 8.0]), "max_pos": _spread(rng, 16, 131072), "page": page}
    if op == "attend":
        dim = rng.choice([128, 128, 64])
        requests = _spread(rng, 1, 128)
        longest = _spread(rng, 1, min(131072, 131072 * 8 * 128 // (kv_heads * dim * requests)))
        return {"op": op, "dtype": dtype, "requests": requests, "min_len": rng.choice([0, 1, max(1, longest // 8), longest]) if longest > 8 else longest,
                "max_len": longest, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page}
    vocab = rng.choice([151936, 128256, _spread(rng, 1000, 150000), _spread(rng, 1000, 150000) | 1])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    return {"op": op, "dtype": dtype, "rows": _spread(rng, 1, 2048 * 151936 // vocab // (2 if dtype == "f32" else 1)), "vocab": vocab,
            "top": rng.choice([0, 1, 5, 20, 32]), "allowed": rng.choice([1.0, 1.0, 1.0, 0.02])}


def _lengths(case):
    """The requests' context lengths, spread over [min_len, max_len] by their logarithm: the same set for every seed."""
    n, lo, hi = case["requests"], case["min_len"], case["max_len"]
    if n == 1 or lo == hi:
        return [hi] * n
    a, b = math.log(lo + 1), math.log(hi + 1)
    return [int(round(math.exp(a + (b - a) * i / (n - 1)))) - 1 for i in range(n)]


def _inv_freq(case):
    """Angles per position, rot / 2 of them: theta^(-2j / rot), those of long wavelength divided by `factor` (the smooth
    rule of 8192-token models stretched to longer contexts)."""
    rot, factor, theta, old = case["rot"], case["factor"], 1e6, 8192
    out = []
    for j in range(rot // 2):
        f = theta ** (-2.0 * j / rot)
        turns = old * f / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - 1.0) / (4.0 - 1.0)))
        out.append(f * keep + f / factor * (1.0 - keep))
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = torch.Generator().manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    i32 = lambda t: t.to(device="cuda", dtype=torch.int32)  # noqa: E731
    if case["op"] == "plan":
        B, cap, page = case["requests"], case["tokens"], case["page"]
        ctx = torch.randint(0, case["max_ctx"] + 1, (B,), generator=c)
        new = torch.ones(B, dtype=torch.int64)
        if cap > B:  # some of the requests bring a chunk of their prompt
            share = torch.rand(B, generator=c) * (torch.rand(B, generator=c) < 0.25)
            new += (share / max(float(share.sum()), 1e-9) * (cap - B)).long().clamp(max=8192)
        elif B > 2:
            new[torch.randint(0, B, (1,), generator=c)] = 0  # an idle place in the batch
        had = (ctx + page - 1) // page
        most = (case["max_ctx"] + min(cap - B, 8192) + 1) // page + 1
        pages = int(had.sum()) + int((new // page + 2).sum())
        order = torch.randperm(pages, generator=c)
        table = torch.full((B, most), -1, dtype=torch.int64)
        cols = torch.arange(most)[None, :]
        first = had.cumsum(0) - had
        held = cols < had[:, None]
        table[held] = order[(first[:, None] + cols)[held]]
        return {"case": case, "ctx": i32(ctx), "new": i32(new), "table": i32(table), "free": i32(order[int(had.sum()):]),
                "head": torch.zeros(1, dtype=torch.int32, device="cuda")}
    if case["op"] == "append":
        T, Hq, Hkv, D, page = case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["page"]
        dt = DTYPES[case["dtype"]]
        qkv = normal(T, (Hq + 2 * Hkv) * D).to(dt)  # one projection's rows, q, k and v side by side
        q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split((Hq * D, Hkv * D, Hkv * D), dim=1))
        # chunks of consecutive positions, one after another, each with pages of its own; a few rows are padding
        chunk = max(1, T // 8)
        start = torch.randint(0, max(1, case["max_pos"] - chunk), (T // chunk + 1,), generator=c)
        t = torch.arange(T)
        pos = start[t // chunk] + t % chunk
        per = (chunk + page - 1) // page + 1
        pages = (T // chunk + 1) * per + 1
        order = torch.randperm(pages - 1, generator=c) + 1
        slot = order[(t // chunk) * per + (pos // page - start[t // chunk] // page)] * page + pos % page
        if T > 16:
            slot[torch.randperm(T, generator=c)[: T // 64]] = -1
        cache = lambda: torch.zeros(pages, Hkv, page, D, dtype=dt, device="cuda")  # noqa: E731
        weight = lambda: (1 + 0.2 * normal(D)).to(dt) if case["norm"] else None  # noqa: E731
        return {"case": case, "q": q, "k": k, "v": v, "positions": i32(pos), "slots": slot.cuda(), "k_cache": cache(), "v_cache": cache(),
                "inv_freq": torch.tensor(_inv_freq(case), dtype=torch.float32, device="cuda"), "q_norm": weight(), "k_norm": weight(),
                "mscale": 1.0 if case["factor"] == 1.0 else 0.1 * math.log(case["factor"]) + 1.0}
    if case["op"] == "attend":
        B, Hq, Hkv, D, page = case["requests"], case["heads"], case["kv_heads"], case["dim"], case["page"]
        dt = DTYPES[case["dtype"]]
        lens = torch.tensor(_lengths(case))[torch.randperm(B, generator=c)]
        held = (lens + page - 1) // page
        pages = int(held.sum()) + 1
        order = torch.randperm(pages - 1, generator=c) + 1
        most = max(1, int(held.max()))
        table = torch.zeros(B, most, dtype=torch.int64)
        cols = torch.arange(most)[None, :]
        at = ((held.cumsum(0) - held)[:, None] + cols)
        table[cols < held[:, None]] = order[at[cols < held[:, None]]]
        return {"case": case, "q": (2 * normal(B, Hq, D)).to(dt), "k_cache": normal(pages, Hkv, page, D).to(dt),
                "v_cache": normal(pages, Hkv, page, D).to(dt), "table": i32(table), "lens": i32(lens), "scale": 1 / math.sqrt(D)}
    R, V = case["rows"], case["vocab"]
    logits = 2.5 * normal(R, V)
    tokens = torch.randint(0, V, (R,), generator=g, device="cuda")
    logits.scatter_(1, tokens[:, None], 6 + 4 * normal(R, 1))  # the tokens are mostly likely ones
    if case["allowed"] < 1:
        shut = torch.rand(R, V, generator=g, device="cuda") >= case["allowed"]
        shut.scatter_(1, tokens[:, None], False)
        logits.masked_fill_(shut, float("-inf"))
    return {"case": case, "logits": logits.to(DTYPES.get(case["dtype"], torch.float32)), "tokens": tokens.to(torch.int32)}


# ------------------------------------------------------------------ plain forms
def _plan(s):
    page, cap = s["case"]["page"], s["case"]["tokens"]
    ctx, new, table, head = s["ctx"].long().clamp(min=0), s["new"].long().clamp(min=0), s["table"].long(), s["head"].long()
    total, end = ctx + new, new.cumsum(0)
    start = end - new
    had = (ctx + page - 1) // page
    fits = (end <= cap) & (total <= table.shape[1] * page)
    need = torch.where(fits, (total + page - 1) // page - had, 0)
    last = need.cumsum(0)
    ok = fits & ((need == 0) | (last <= s["free"].numel() - head))
    j = torch.arange(table.shape[1], device="cuda")[None, :] - had[:, None]
    from_free = ok[:, None] & (j >= 0) & (j < need[:, None])
    at = ((last - need)[:, None] + j + head).clamp(0, s["free"].numel() - 1)
    table = torch.where(from_free, s["free"].long()[at], table)
    t = torch.arange(cap, device="cuda")
    real = t < end[-1]
    r = torch.searchsorted(end, t, right=True).clamp(max=end.numel() - 1)
    pos = torch.where(real, ctx[r] + t - start[r], 0)
    held = table[r, (pos // page).clamp(max=table.shape[1] - 1)]
    slots = torch.where(real & ok[r] & (held >= 0), held * page + pos % page, -1)
    taken = torch.where(ok, last, 0).amax(0, keepdim=True) * (need > 0).any()
    counts = torch.cat([end[-1:], last[-1:], taken, (~ok).sum(0, keepdim=True), head + taken])
    return {"table": table.int(), "seq_lens": torch.where(ok, total, ctx).int(), "query_start": torch.cat([torch.zeros_like(end[:1]), end]).int(),
            "positions": pos.int(), "token_seq": torch.where(real, r, -1).int(), "slots": slots, "counts": counts.int()}


def _rotate(x, weight, s):
    case, rot = s["case"], s["case"]["rot"]
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight.float()
    angle = s["positions"].float()[:, None, None] * s["inv_freq"]
    cos, sin = torch.cos(angle) * s["mscale"], torch.sin(angle) * s["mscale"]
    if case["traditional"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., : rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, x[..., rot:]], dim=-1).to(s["q"].dtype)


def _append(s):
    page = s["case"]["page"]
    q, k = _rotate(s["q"], s["q_norm"], s), _rotate(s["k"], s["k_norm"], s)
    real = (s["slots"] >= 0)[:, None, None]
    slot = s["slots"].clamp(min=0)  # padding rows write page 0, which no request holds, with what it has
    at = (slot // page, slice(None), slot % page)
    s["k_cache"][at] = torch.where(real, k, s["k_cache"][at])
    s["v_cache"][at] = torch.where(real, s["v"], s["v_cache"][at])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attend(s):
    case, table = s["case"], s["table"].long()
    B, Hq, Hkv, D = case["requests"], case["heads"], case["kv_heads"], case["dim"]
    rows = lambda c: c[table].transpose(2, 3).flatten(1, 2).float()  # noqa: E731  [B, L, Hkv, D]
    q = s["q"].float().view(B, Hkv, Hq // Hkv, D)
    w = torch.matmul(q, rows(s["k_cache"]).permute(0, 2, 3, 1)) * s["scale"]
    seen = (torch.arange(w.shape[-1], device="cuda")[None, :] < s["lens"][:, None])[:, None, None, :]
    w = w.masked_fill(~seen, float("-inf"))
    w = torch.exp(w - w.amax(-1, keepdim=True).clamp(min=-1e30))
    w = w / w.sum(-1, keepdim=True).clamp(min=1e-30)
    return torch.matmul(w, rows(s["v_cache"]).transpose(1, 2)).view(B, Hq, D).to(s["q"].dtype)


def _logprobs(s):
    x, k = s["logits"].float(), s["case"]["top"]
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    total = e.sum(-1, keepdim=True)
    lse = m + torch.log(total)
    entropy = torch.log(total) - (torch.where(e > 0, (x - m) * e, 0.0)).sum(-1, keepdim=True) / total
    picked = x.gather(-1, s["tokens"].long()[:, None]) - lse
    bits = (x + 0.0).view(torch.int32)
    order = (bits ^ ((bits >> 31) & 0x7FFFFFFF)).long()  # larger values first, then lower places
    keys = (order << 32) | (0xFFFFFFFF - torch.arange(x.shape[-1], device="cuda"))
    ids = 0xFFFFFFFF - (keys.topk(k, -1).values & 0xFFFFFFFF)
    return {"logprob": picked[:, 0], "entropy": entropy[:, 0], "lse": lse[:, 0], "top_ids": ids.int(), "top": x.gather(-1, ids) - lse}


# ------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    if not own:
        return {"plan": _plan, "append": _append, "attend": _attend, "logprobs": _logprobs}[case["op"]](s)
    from metal_autotune_b200 import lib
    if case["op"] == "plan":
        p = lib.paged_plan(s["ctx"], s["new"], s["table"], s["free"], page_size=case["page"], token_cap=case["tokens"], free_head=s["head"])
        return {"table": s["table"], "seq_lens": p.seq_lens, "query_start": p.query_start, "positions": p.positions, "token_seq": p.token_seq,
                "slots": p.slots, "counts": p.counts}
    if case["op"] == "append":
        q = lib.rope_paged_append(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["k_cache"], s["v_cache"], s["inv_freq"],
                                  traditional=case["traditional"], mscale=s["mscale"], q_norm_w=s["q_norm"], k_norm_w=s["k_norm"], eps=1e-6)
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if case["op"] == "attend":
        return lib.paged_sdpa_decode(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], scale=s["scale"])
    p = lib.token_logprobs(s["logits"], s["tokens"], top_k=case["top"])
    return {"logprob": p.logprob, "entropy": p.entropy, "lse": p.lse, "top_ids": p.top_ids, "top": p.top_logprobs}


def work(case):
    if case["op"] == "plan":  # the lengths, a page of each request and the free pages read; the token rows, lengths and new pages written
        return {"bytes": 20.0 * case["requests"] + 16.0 * case["tokens"] + 8.0 * case["tokens"] / case["page"], "flops": 0.0}
    if case["op"] == "append":
        values = case["tokens"] * (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        return {"bytes": 4.0 * values + 12.0 * case["tokens"], "flops": 8.0 * values}
    if case["op"] == "attend":
        rows, size = sum(_lengths(case)), 2.0
        return {"bytes": size * (2 * rows * case["kv_heads"] + 2 * case["requests"] * case["heads"]) * case["dim"],
                "flops": 4.0 * rows * case["heads"] * case["dim"]}
    size = 4.0 if case["dtype"] == "f32" else 2.0
    return {"bytes": case["rows"] * (size * case["vocab"] + 16 + 8 * case["top"]), "flops": 6.0 * case["rows"] * case["vocab"]}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers only
    s = prepare(case, seed)
    if case["op"] == "append":
        rot, page = case["rot"], case["page"]
        turn = torch.polar(torch.full((1, 1), s["mscale"], dtype=torch.float64, device="cuda"),
                           torch.outer(s["positions"].double(), s["inv_freq"].double()))[:, None, :]

        def rotated(x, weight):
            x = x.double()
            if weight is not None:
                x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["dim"] + 1e-6) * weight.double()
            x = x.clone()
            i, j = (slice(0, rot, 2), slice(1, rot, 2)) if case["traditional"] else (slice(0, rot // 2), slice(rot // 2, rot))
            z = torch.complex(x[..., i].contiguous(), x[..., j].contiguous()) * turn
            x[..., i], x[..., j] = z.real, z.imag
            return x

        out = {"q": rotated(s["q"], s["q_norm"])}
        to = s["slots"][s["slots"] >= 0]
        for name, rows in (("k_cache", rotated(s["k"], s["k_norm"])), ("v_cache", s["v"].double())):
            flat = s[name].double().transpose(1, 2).contiguous()  # [pages, page, Hkv, D]
            flat.view(-1, *flat.shape[2:])[to] = rows[s["slots"] >= 0]
            out[name] = flat.transpose(1, 2).contiguous()
        return out
    if case["op"] == "attend":
        out = torch.zeros(case["requests"], case["heads"], case["dim"], dtype=torch.float64, device="cuda")
        group = case["heads"] // case["kv_heads"]
        for b, n in enumerate(s["lens"].tolist()):
            if n:
                key = torch.arange(n, device="cuda")
                at = (s["table"][b].long()[key // case["page"]], slice(None), key % case["page"])
                k, v = s["k_cache"][at].double(), s["v_cache"][at].double()  # [n, Hkv, D]
                w = torch.einsum("hgd,nhd->hgn", s["q"][b].double().unflatten(0, (-1, group)), k) * s["scale"]
                out[b] = torch.einsum("hgn,nhd->hgd", torch.softmax(w, -1), v).flatten(0, 1)
        return out
    rows = {"logprob": [], "entropy": [], "lse": [], "top": []}
    for x, t in zip(s["logits"].split(256), s["tokens"].split(256)):
        x = x.double()
        lse = torch.logsumexp(x, -1, keepdim=True)
        rows["logprob"].append((x.gather(-1, t.long()[:, None]) - lse)[:, 0])
        rows["entropy"].append(-(torch.exp(x - lse) * (x - lse)).nan_to_num(0.0).sum(-1))
        rows["lse"].append(lse[:, 0])
        rows["top"].append(x.topk(case["top"], -1).values - lse)
    return {"top_ids": None, **{name: torch.cat(v) for name, v in rows.items()}}

"""Cases of the paged serving operators: paged_plan (block tables and slot maps from request lengths),
paged_append (rotary positions at each token's own position, and the new K/V rows into their pages)
and paged_attn (attention of new tokens over the paged cache, causal, or with a sliding window and
first tokens that stay visible).

``run`` computes an operator in plain torch operations, or, where ``own`` is true, calls the
library's entry points as a server loop does. Ragged batches come as in a serving step: the rows of
request b are rows q_start[b] .. q_start[b+1] of the token-wise tensors, rows behind the last
request belong to nobody and stay as they were.
"""
import math
import os
import random
import sys

import torch

own = False

BLK = 32  # elements of one Q8 block: an fp16 delta and 32 int8


def listed():
    return [
        # A decode step of TinyLlama-shaped requests (context 2048, 16-token pages): one new token each.
        dict(name="plan_decode_b64", op="plan", n_req=64, page=16, new_lo=1, new_hi=1, n_dec=64, ctx_lo=1, ctx_hi=2000,
             max_pages=128, pad=0, short=False, lens_seed=1),
        # A serving step of many requests: most decode, the rest prefill chunks of any length up to 512.
        dict(name="plan_mixed_b1000", op="plan", n_req=1000, page=16, new_lo=0, new_hi=512, n_dec=900, ctx_lo=0,
             ctx_hi=4000, max_pages=320, pad=37, short=False, lens_seed=2),
        # TinyLlama's decode batch of 16: 32 query heads, 4 kv heads, full rotary, fp16.
        dict(name="append_decode_b16", op="append", heads=32, kv_heads=4, d=64, page=16, src="f16", cache="f16",
             n_req=16, new_lo=1, new_hi=1, n_dec=16, ctx_lo=1, ctx_hi=2000, rope_pct=1.0, base=10000.0, pad=0,
             lens_seed=3),
        # StableLM-2-Zephyr's prefill chunks: 32 heads each, a quarter of each head rotated, fp16.
        dict(name="append_chunks_zephyr", op="append", heads=32, kv_heads=32, d=64, page=32, src="f16", cache="f16",
             n_req=5, new_lo=300, new_hi=1024, n_dec=1, ctx_lo=0, ctx_hi=3000, rope_pct=0.25, base=10000.0, pad=11,
             lens_seed=4),
        # MiniCPM's chunk of fp32 projections, written to a Q8 cache: 36 heads each.
        dict(name="append_chunk_minicpm_q8", op="append", heads=36, kv_heads=36, d=64, page=16, src="f32", cache="q8",
             n_req=3, new_lo=200, new_hi=777, n_dec=0, ctx_lo=0, ctx_hi=3000, rope_pct=1.0, base=10000.0, pad=0,
             lens_seed=5),
        # One TinyLlama sequence decoding near the end of its context: latency.
        dict(name="attn_decode_b1", op="attn", heads=32, kv_heads=4, d=64, page=16, cache="f16", io="f16", n_req=1,
             new_lo=1, new_hi=1, n_dec=1, ctx_lo=1990, ctx_hi=1990, window=0, sinks=0, pad=0, lens_seed=6),
        # MiniCPM's decode batch of 64 in Q8 throughout (activations and cache), ragged contexts.
        dict(name="attn_decode_b64_q8", op="attn", heads=36, kv_heads=36, d=64, page=16, cache="q8", io="q8", n_req=64,
             new_lo=1, new_hi=1, n_dec=64, ctx_lo=64, ctx_hi=1500, window=0, sinks=0, pad=0, lens_seed=7),
        # A serving step of TinyLlama: 24 decoding requests and 4 prompt chunks of odd lengths in one call.
        dict(name="attn_mixed_b28", op="attn", heads=32, kv_heads=4, d=64, page=16, cache="f16", io="f16", n_req=28,
             new_lo=100, new_hi=512, n_dec=24, ctx_lo=0, ctx_hi=1500, window=0, sinks=0, pad=5, lens_seed=8),
        # A long prompt's chunk of 2048 tokens over some 30,000 cached ones, 128-wide heads: the largest.
        dict(name="attn_chunk_30k", op="attn", heads=32, kv_heads=8, d=128, page=64, cache="f16", io="f16", n_req=1,
             new_lo=2048, new_hi=2048, n_dec=0, ctx_lo=29999, ctx_hi=29999, window=0, sinks=0, pad=0, lens_seed=9),
        # Prompts of StableLM-2-Zephyr in one call over a Q8 cache, one of them behind a cached prefix.
        dict(name="attn_prompts_q8", op="attn", heads=32, kv_heads=32, d=64, page=32, cache="q8", io="f16", n_req=4,
             new_lo=500, new_hi=1500, n_dec=0, ctx_lo=0, ctx_hi=1000, window=0, sinks=0, pad=0, lens_seed=10),
        # Streaming decode: long histories, a window of 4096 keys and 4 first tokens, 128-wide heads.
        dict(name="window_decode_b16", op="attn", heads=32, kv_heads=8, d=128, page=64, cache="f16", io="f16", n_req=16,
             new_lo=1, new_hi=1, n_dec=16, ctx_lo=2000, ctx_hi=40000, window=4096, sinks=4, pad=0, lens_seed=11),
        # Prompt chunks with a window of 1000 keys and 5 first tokens: TinyLlama's heads.
        dict(name="window_chunks", op="attn", heads=32, kv_heads=4, d=64, page=16, cache="f16", io="f16", n_req=3,
             new_lo=900, new_hi=2048, n_dec=0, ctx_lo=0, ctx_hi=6000, window=1000, sinks=5, pad=3, lens_seed=12),
    ]


#: (query heads, kv heads, head width): TinyLlama, StableLM-2, MiniCPM, OpenELM, the test models, and
#: 128-wide heads with 4 and 8 query heads per kv head.
HEADS = [(32, 4, 64), (32, 32, 64), (36, 36, 64), (12, 3, 64), (16, 4, 64), (28, 7, 64), (4, 2, 64), (3, 3, 64),
         (32, 8, 128), (8, 1, 128), (16, 16, 128)]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attn", "attn", "window"])
    page = rng.choice([16, 32, 64, 128])
    c = dict(op=op, page=page, pad=rng.choice([0, 0, 1, 17]), lens_seed=rng.randrange(1 << 30))
    if op == "plan":
        ctx_hi = _log_int(rng, 16, 30000)
        new_hi = _log_int(rng, 1, 600)
        n_req = _log_int(rng, 1, 1000)
        c.update(n_req=n_req, new_lo=rng.choice([0, 1]), new_hi=new_hi, n_dec=rng.randint(0, n_req), ctx_lo=0,
                 ctx_hi=ctx_hi, max_pages=-(-(ctx_hi + new_hi) // page) + rng.randint(0, 3), short=rng.random() < 0.25)
        return c
    heads, kv_heads, d = rng.choice(HEADS)
    c.update(heads=heads, kv_heads=kv_heads, d=d, cache=rng.choice(["f16", "q8"]))
    if op == "append":
        n_req = _log_int(rng, 1, 64)
        new_hi = _log_int(rng, 1, max(1, 4096 // n_req))
        c.update(src=rng.choice(["f16", "f32", "q8"]), n_req=n_req, new_lo=rng.choice([0, 1]), new_hi=new_hi,
                 n_dec=rng.randint(0, n_req), ctx_lo=0, ctx_hi=_log_int(rng, 16, 30000),
                 rope_pct=rng.choice([1.0, 1.0, 0.5, 0.25, 0.0]), base=rng.choice([10000.0, 500000.0]))
        return c
    decode = rng.random() < 0.5
    n_req = _log_int(rng, 1, 64 if decode else 8)
    new_hi = rng.choice([1, 1, 2, 5]) if decode else _log_int(rng, 2, 2048)
    ctx_hi = _log_int(rng, 16, 32000)
    # scores of the plain form: every request padded to the longest
    while n_req * heads * new_hi * (ctx_hi + new_hi) > 1.2e9 or n_req * kv_heads * d * (ctx_hi + new_hi) > 6e8:
        ctx_hi = max(16, ctx_hi * 2 // 3)
        n_req = max(1, n_req * 3 // 4)
    c.update(op="attn", io=rng.choice(["f16", "f16", "q8"]), n_req=n_req, new_lo=rng.choice([0, 1]), new_hi=new_hi,
             n_dec=rng.randint(0, n_req), ctx_lo=rng.choice([0, ctx_hi // 2]), ctx_hi=ctx_hi, window=0, sinks=0)
    if op == "window":
        c.update(window=_log_int(rng, 1, 8192), sinks=rng.choice([0, 1, 4, 16, 130]))
    return c


def _lens(c):
    """(cached tokens, new tokens) of each request: part of the case, the same for every seed."""
    r = random.Random(c["lens_seed"])
    got = [(r.randint(c["ctx_lo"], c["ctx_hi"]), 1 if i < c["n_dec"] else r.randint(c["new_lo"], c["new_hi"]))
           for i in range(c["n_req"])]
    if not any(n for _, n in got):
        got[-1] = (got[-1][0], 1)
    return [x for x, _ in got], [n for _, n in got]


def _cdiv(a, b):
    return -(-a // b)


# ---- inputs ------------------------------------------------------------------------------------
def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    ctx, new = _lens(c)
    if c["op"] == "plan":
        return _prepare_plan(c, ctx, new, g)
    s = _prepare_pages(c, ctx, new, g)
    return _prepare_append(c, s, g) if c["op"] == "append" else _prepare_attn(c, s, g)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _perm(n, g):
    return torch.randperm(n, generator=g, device="cuda").to(torch.int32)


def _prepare_plan(c, ctx, new, g):
    ps, n_req = c["page"], c["n_req"]
    have = [_cdiv(x, ps) for x in ctx]
    need = [_cdiv(x + n, ps) - h for x, n, h in zip(ctx, new, have)]
    spare = 7 + sum(need) // 8
    pages = _perm(sum(have) + sum(need) + spare, g)
    h = _i32(have)
    col = torch.arange(c["max_pages"], device="cuda")
    # the pages that each request has already, in the table's first columns
    start = (torch.cumsum(h, 0) - h)[:, None]
    idx = (start + col).clamp(max=pages.numel() - 1)
    table = torch.where(col < h[:, None], pages[idx], torch.full_like(pages[idx], -1))
    free = pages[sum(have):].contiguous()
    n_free = free.numel() if not c["short"] else sum(need) // 2
    rows = sum(new) + c["pad"]
    return {"case": c, "ctx": _i32(ctx), "new": _i32(new), "free": free, "n_free": _i32([n_free]), "table": table,
            "q_start": torch.zeros(n_req + 1, dtype=torch.int32, device="cuda"),
            "kv_lens": torch.zeros(n_req, dtype=torch.int32, device="cuda"),
            "pos": torch.zeros(rows, dtype=torch.int32, device="cuda"),
            "slots": torch.zeros(rows, dtype=torch.int32, device="cuda"),
            "n_used": torch.zeros(1, dtype=torch.int32, device="cuda")}


def _pool(c, n_pages, g):
    """One pool of pages: fp16 [page, kv head, token, d]; Q8 pages hold the int8 values in that order,
    then their fp16 deltas [kv head, token, d / 32]."""
    kvh, ps, d = c["kv_heads"], c["page"], c["d"]
    if c["cache"] == "f16":
        return torch.randn(n_pages, kvh, ps, d, generator=g, device="cuda", dtype=torch.float16)
    ints = torch.randint(-127, 128, (n_pages, kvh * ps * d), generator=g, device="cuda", dtype=torch.int8)
    delta = (torch.rand(n_pages, kvh * ps * d // BLK, generator=g, device="cuda") + 0.5) / 73.0
    return torch.cat([ints.view(torch.uint8), delta.to(torch.float16).view(torch.uint8)], 1)


def _rows(kind, rows, cols, g, scale=1.0):
    """Activation rows: fp16, fp32, or Q8 blocks (fp16 delta, 32 int8) as bytes."""
    if kind == "q8":
        ints = torch.randint(-127, 128, (rows, cols // BLK, BLK), generator=g, device="cuda", dtype=torch.int8)
        delta = (torch.rand(rows, cols // BLK, 1, generator=g, device="cuda") + 0.5) * (scale / 73.0)
        return torch.cat([delta.to(torch.float16).view(torch.uint8), ints.view(torch.uint8)], 2).view(rows, -1)
    x = torch.randn(rows, cols, generator=g, device="cuda") * scale
    return x.to(torch.float16) if kind == "f16" else x


def _prepare_pages(c, ctx, new, g):
    ps = c["page"]
    kv = [x + n for x, n in zip(ctx, new)]
    n_col = max(1, max(_cdiv(x, ps) for x in kv))
    used = [_cdiv(x, ps) for x in kv]
    n_pages = sum(used) + 3
    pages = _perm(n_pages, g)
    u = _i32(used)
    col = torch.arange(n_col, device="cuda")
    idx = ((torch.cumsum(u, 0) - u)[:, None] + col).clamp(max=n_pages - 1)
    table = torch.where(col < u[:, None], pages[idx], torch.full_like(pages[idx], -1))
    return {"case": c, "ctx": ctx, "new": new, "max_kv": max(kv), "max_new": max(new), "n_pages": n_pages,
            "table": table, "q_start": torch.cumsum(_i32([0] + new), 0).to(torch.int32), "kv_lens": _i32(kv),
            "rows": sum(new) + c["pad"], "k": _pool(c, n_pages, g), "v": _pool(c, n_pages, g)}


def _prepare_append(c, s, g):
    rows, hd, kd = s["rows"], c["heads"] * c["d"], c["kv_heads"] * c["d"]
    new = _i32(s["new"])
    t = torch.arange(rows, device="cuda")
    b = torch.searchsorted(s["q_start"][1:].contiguous(), t.to(torch.int32), right=True).clamp(max=c["n_req"] - 1)
    live = t < sum(s["new"])
    pos = (s["kv_lens"] - new)[b] + t - s["q_start"][b]
    page = s["table"][b, (pos // c["page"]).clamp(0, s["table"].shape[1] - 1)]
    slot = page * c["page"] + pos % c["page"]
    s["pos"] = torch.where(live, pos, -1).to(torch.int32)
    s["slots"] = torch.where(live, slot, -1).to(torch.int32)
    s["xq"], s["xk"], s["xv"] = (_rows(c["src"], rows, n, g) for n in (hd, kd, kd))
    s["q_out"] = torch.zeros(rows, hd, dtype=torch.float16, device="cuda")
    return s


def _prepare_attn(c, s, g):
    hd = c["heads"] * c["d"]
    s["q"] = _rows(c["io"], s["rows"], hd, g, 1.5)
    s["out"] = torch.zeros_like(s["q"])
    return s


# ---- one pass ----------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"plan": _own_plan, "append": _own_append, "attn": _own_attn}[op](state)
    return {"plan": _plan, "append": _append, "attn": _attn}[op](state)


def _q8_rows(x):
    """The values that Q8 rows stand for, as fp16."""
    x = x.view(x.shape[0], -1, BLK + 2)
    delta = x[..., :2].contiguous().view(torch.float16)
    return (x[..., 2:].view(torch.int8) * delta).view(x.shape[0], -1)


def _q8_pages(pool, c):
    """The values that a Q8 pool stands for, as fp16 [page, kv head, token, d]."""
    kvh, ps, d = c["kv_heads"], c["page"], c["d"]
    n = kvh * ps * d
    ints = pool[:, :n].view(torch.int8).view(-1, kvh, ps, d // BLK, BLK)
    delta = pool[:, n:].view(torch.float16).view(-1, kvh, ps, d // BLK, 1)
    return (ints * delta).view(-1, kvh, ps, d)


# ---- the framework's calls
def _lib():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "nanochatllms.cpp_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import gten_b200
    return gten_b200


def _handles(s):
    """The tensors' descriptors, which a program keeps beside its buffers."""
    c, G = s["case"], _lib()
    dt = {"f16": G.F16, "f32": G.F32, "q8": G.Q8}
    i32 = lambda t: G.GT(t, G.I32, tuple(t.shape))  # noqa: E731
    h = {k: i32(s[k]) for k in ("table", "q_start", "kv_lens")}
    if c["op"] == "plan":
        h.update({k: i32(s[k]) for k in ("ctx", "new", "free", "n_free", "pos", "slots", "n_used")})
    else:
        h["cache"] = G.PagedCache(s["k"], s["v"], dt[c["cache"]], s["n_pages"], c["page"], c["kv_heads"], c["d"])
        rows, hd, kd = s["rows"], c["heads"] * c["d"], c["kv_heads"] * c["d"]
        if c["op"] == "append":
            h.update(pos=i32(s["pos"]), slots=i32(s["slots"]), q_out=G.GT(s["q_out"], G.F16, (rows, hd)))
            h.update(xq=G.GT(s["xq"], dt[c["src"]], (rows, hd)), xk=G.GT(s["xk"], dt[c["src"]], (rows, kd)),
                     xv=G.GT(s["xv"], dt[c["src"]], (rows, kd)))
        else:
            h.update(q=G.GT(s["q"], dt[c["io"]], (rows, hd)), out=G.GT(s["out"], dt[c["io"]], (rows, hd)))
    s["handles"] = h
    return h


def _own_plan(s):
    h = s.get("handles") or _handles(s)
    _lib().paged_plan(h["ctx"], h["new"], h["free"], h["n_free"], s["case"]["page"], h["table"], h["q_start"],
                      h["kv_lens"], h["pos"], h["slots"], h["n_used"])
    return {k: s[k] for k in ("table", "q_start", "kv_lens", "pos", "slots", "n_used")}


def _own_append(s):
    h, c = s.get("handles") or _handles(s), s["case"]
    _lib().paged_append(h["xq"], h["xk"], h["xv"], h["pos"], h["slots"], h["cache"], h["q_out"], c["rope_pct"], c["base"])
    if c["cache"] == "q8":
        return {"q": s["q_out"], "k": _q8_pages(s["k"], c), "v": _q8_pages(s["v"], c)}
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _own_attn(s):
    h, c = s.get("handles") or _handles(s), s["case"]
    _lib().paged_attn(h["q"], h["cache"], h["table"], h["q_start"], h["kv_lens"], h["out"], window=c["window"],
                      n_sink=c["sinks"], max_new=s["max_new"])
    return _q8_rows(s["out"]) if c["io"] == "q8" else s["out"]


# ---- the plain forms
def _plan(s):
    c = s["case"]
    ps, rows, mp = c["page"], s["pos"].numel(), c["max_pages"]
    ctx, new = s["ctx"].long(), s["new"].long()
    n = new.clamp(min=0)
    q_end = torch.cumsum(n, 0)
    q_start = torch.cat([torch.zeros_like(q_end[:1]), q_end])
    kv = ctx + n
    have = (ctx + ps - 1) // ps
    fits = (ctx >= 0) & (new >= 0) & (kv <= mp * ps) & (q_end <= rows)
    need = torch.where(fits, (kv + ps - 1) // ps - have, 0)
    end = torch.cumsum(need, 0)
    grant = fits & ((need == 0) | (end <= s["n_free"].long()))
    col = torch.arange(mp, device="cuda")
    fresh = grant[:, None] & (col >= have[:, None]) & (col < (have + need)[:, None])
    src = ((end - need)[:, None] + col - have[:, None]).clamp(0, s["free"].numel() - 1)
    table = torch.where(fresh, s["free"][src], s["table"])
    t = torch.arange(rows, device="cuda")
    b = torch.searchsorted(q_end, t, right=True).clamp(max=c["n_req"] - 1)
    live = t < q_end[-1]
    pos = ctx[b] + t - q_start[b]
    slot = table[b, (pos // ps).clamp(0, mp - 1)].long() * ps + pos % ps
    return {"table": table, "q_start": q_start.int(), "kv_lens": torch.where(grant, kv, 0).int(),
            "pos": torch.where(live, pos, -1).int(), "slots": torch.where(live & grant[b], slot, -1).int(),
            "n_used": torch.where(grant, need, 0).sum().int().view(1)}


def _values(kind, x):
    if kind == "q8":
        x = x.view(x.shape[0], -1, BLK + 2)
        return (x[..., 2:].view(torch.int8).float() * x[..., :2].contiguous().view(torch.float16).float()).view(x.shape[0], -1)
    return x.float()


def _pages(pool, c):
    """The pool's values as fp32 [page, kv head, token, d]."""
    if c["cache"] == "f16":
        return pool.float()
    kvh, ps, d = c["kv_heads"], c["page"], c["d"]
    n = kvh * ps * d
    ints = pool[:, :n].view(torch.int8).view(-1, kvh, ps, d // BLK, BLK).float()
    return (ints * pool[:, n:].view(torch.float16).view(-1, kvh, ps, d // BLK, 1).float()).view(-1, kvh, ps, d)


def _q8_round(x):
    """fp32 values to the Q8 values that stand for them: per 32 elements delta = absmax / 127 (stored
    as fp16), q = x / delta rounded half away from zero."""
    b = x.view(*x.shape[:-1], -1, BLK)
    delta = b.abs().amax(-1, keepdim=True) / 127.0
    y = b * torch.where(delta != 0, 1.0 / delta, 0.0)
    q = torch.trunc(y + torch.copysign(torch.full_like(y, 0.5), y)).clamp(-127, 127)
    return (q * delta.to(torch.float16).float()).view(x.shape)


def _rotate(x, pos, c):
    """x [rows, heads, d]: the first rope_pct of each head rotated by its row's position, pairs half
    the rotated width apart; angles in 64 bits."""
    rd = int(c["d"] * c["rope_pct"]) // 2 * 2
    half = rd // 2
    if half == 0:
        return x
    j = torch.arange(half, device="cuda", dtype=torch.float64)
    angle = pos.double()[:, None] * torch.pow(torch.tensor(c["base"], dtype=torch.float64, device="cuda"), -2 * j / rd)
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    a, b = x[..., :half], x[..., half:rd]
    return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., rd:]], -1)


def _append(s):
    c, rows = s["case"], s["rows"]
    kvh, ps, d = c["kv_heads"], c["page"], c["d"]
    xq, xk, xv = (_values(c["src"], s[k]) for k in ("xq", "xk", "xv"))
    q = _rotate(xq.view(rows, -1, d), s["pos"], c).view(rows, -1)
    q_out = torch.where((s["pos"] >= 0)[:, None], q.to(torch.float16), s["q_out"])
    k = _rotate(xk.view(rows, kvh, d), s["pos"], c)
    v = xv.view(rows, kvh, d)
    if c["cache"] == "q8":
        k, v = _q8_round(k), v if c["src"] == "q8" else _q8_round(v)
    # the row that each slot receives (the last cell takes the rows without a slot)
    n = s["n_pages"] * ps
    t = torch.arange(rows, device="cuda")
    row = torch.full((n + 1,), -1, device="cuda", dtype=torch.long)
    row.scatter_(0, torch.where(s["slots"] >= 0, s["slots"], n).long(), t)
    row = row[:n].view(-1, 1, ps, 1)
    at = row.view(-1).clamp(min=0)
    put = lambda x, old: torch.where(row >= 0, x[at].view(-1, ps, kvh, d).transpose(1, 2), old).to(torch.float16)  # noqa: E731
    return {"q": q_out, "k": put(k, _pages(s["k"], c)), "v": put(v, _pages(s["v"], c))}


def _attn(s):
    c = s["case"]
    B, H, kvh, d, ps = c["n_req"], c["heads"], c["kv_heads"], c["d"], c["page"]
    N, P = s["max_new"], _cdiv(s["max_kv"], ps)
    G, L = H // kvh, P * ps
    q_start, kv = s["q_start"].long(), s["kv_lens"].long()
    new = q_start[1:] - q_start[:-1]
    page = s["table"][:, :P].long().clamp(min=0)
    k, v = (_pages(s[x][page].view(B * P, *s[x].shape[1:]), c).view(B, P, kvh, ps, d).transpose(1, 2).reshape(B, kvh, L, d)
            for x in ("k", "v"))
    i, j = torch.arange(N, device="cuda"), torch.arange(L, device="cuda")
    qf = _values(c["io"], s["q"])
    q = qf[(q_start[:-1, None] + i).clamp(max=s["rows"] - 1)].view(B, N, H, d).transpose(1, 2).reshape(B, kvh, G * N, d)
    pos = (kv - new)[:, None] + i
    seen = j <= pos[..., None]
    if c["window"]:
        seen = seen & ((j > pos[..., None] - c["window"]) | (j < c["sinks"]))
    x = torch.matmul(q, k.transpose(2, 3)).view(B, kvh, G, N, L)
    x.mul_(d ** -0.5).masked_fill_(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    x.sub_(torch.where(m > -math.inf, m, 0.0)).exp_()
    z = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(B, kvh, G * N, L), v).view(B, kvh, G, N, d)
    o = torch.where(z > 0, o / z, 0.0).view(B, H, N, d).transpose(1, 2)
    t = torch.arange(s["rows"], device="cuda")
    b = torch.searchsorted(q_start[1:].contiguous(), t, right=True).clamp(max=B - 1)
    got = o[b, (t - q_start[b]).clamp(0, N - 1)].reshape(s["rows"], -1)
    live = (t < q_start[-1])[:, None]
    if c["io"] == "q8":
        return torch.where(live, _q8_round(got), _values("q8", s["out"])).to(torch.float16)
    return torch.where(live, got.to(torch.float16), s["out"])


# ---- what a pass has to read, write and compute -------------------------------------------------
def _width(kind, n):
    return {"f16": 2 * n, "f32": 4 * n, "q8": n // BLK * (BLK + 2)}[kind]


def work(case):
    c = case
    ctx, new = _lens(c)
    T, ps = sum(new), c["page"]
    if c["op"] == "plan":
        pages = sum(_cdiv(x + n, ps) - _cdiv(x, ps) for x, n in zip(ctx, new))
        return {"bytes": 16 * c["n_req"] + 8 * pages + 8 * (T + c["pad"]), "flops": 0}
    hd, kd = c["heads"] * c["d"], c["kv_heads"] * c["d"]
    if c["op"] == "append":
        rot = int(c["d"] * c["rope_pct"]) // 2 * 2
        return {"bytes": T * (_width(c["src"], hd + 2 * kd) + 2 * hd + 2 * _width(c["cache"], kd) + 8),
                "flops": 3 * T * (c["heads"] + c["kv_heads"]) * rot}
    pairs = keys = 0
    for x, n in zip(ctx, new):
        if c["window"] == 0:
            pairs += n * x + n * (n + 1) // 2
            keys += x + n if n else 0
            continue
        w, k0 = c["window"], c["sinks"]
        for p in range(x, x + n):
            lo = max(0, p - w + 1)
            pairs += p + 1 - lo + min(lo, k0)
        lo = max(0, x - w + 1)
        keys += (x + n - lo + min(lo, k0)) if n else 0
    return {"bytes": 2 * T * _width(c["io"], hd) + 2 * keys * _width(c["cache"], kd) + 4 * (keys // ps + 2 * c["n_req"]),
            "flops": 4 * pairs * hd}


# ---- in 64 bits, from the definitions ------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": lambda _: None, "append": _exact_append, "attn": _exact_attn}[case["op"]](s)


def _decode64(kind, x):
    if kind != "q8":
        return x.double()
    b = x.view(x.shape[0], -1, 34)
    d = b[:, :, 0:2].contiguous().view(torch.float16).double()
    return (d * b[:, :, 2:34].contiguous().view(torch.int8).double()).flatten(1)


def _cells64(pool, c):
    """Pool as one row per slot: [slot, kv head, d] in 64 bits."""
    kvh, ps, d = c["kv_heads"], c["page"], c["d"]
    if c["cache"] == "f16":
        x = pool.double()
    else:
        nb = kvh * ps * d
        scale = pool[:, nb:].contiguous().view(torch.float16).double()
        x = pool[:, :nb].contiguous().view(torch.int8).double() * scale.repeat_interleave(BLK, 1)
        x = x.view(-1, kvh, ps, d)
    return x.permute(0, 2, 1, 3).reshape(-1, kvh, d)


def _exact_append(s):
    c = s["case"]
    d = c["d"]
    rd = int(d * c["rope_pct"]) // 2 * 2
    pos, slots = s["pos"].cpu(), s["slots"].cpu()
    live = [t for t in range(s["rows"]) if int(pos[t]) >= 0]
    at = torch.tensor(live, device="cuda")
    where = slots[live].cuda().long()
    p = s["pos"][at].double()

    def turned(x):
        z = torch.complex(x[..., : rd // 2].contiguous(), x[..., rd // 2: rd].contiguous())
        f = torch.tensor([c["base"] ** (-2.0 * j / max(rd, 1)) for j in range(rd // 2)], dtype=torch.float64, device="cuda")
        z = z * torch.polar(torch.ones_like(p)[:, None, None], (p[:, None] * f)[:, None, :])
        return torch.cat([z.real, z.imag, x[..., rd:]], -1)

    q = s["q_out"].double()
    q[at] = turned(_decode64(c["src"], s["xq"])[at].view(len(live), -1, d)).flatten(1)
    out = {"q": q}
    for name, src, turn in (("k", "xk", True), ("v", "xv", False)):
        cells = _cells64(s[name], c)
        x = _decode64(c["src"], s[src])[at].view(len(live), -1, d)
        cells[where] = turned(x) if turn else x
        out[name] = cells.view(s["n_pages"], c["page"], c["kv_heads"], d).transpose(1, 2)
    return out


def _exact_attn(s):
    c = s["case"]
    H, kvh, d, ps = c["heads"], c["kv_heads"], c["d"], c["page"]
    G = H // kvh
    out = _decode64(c["io"], s["out"])
    q64 = _decode64(c["io"], s["q"]).view(s["rows"], kvh, G, d)
    table = s["table"].long()
    row = 0
    for b, (x, n) in enumerate(zip(s["ctx"], s["new"])):
        if n == 0:
            continue
        at = torch.arange(x + n, device="cuda")
        slot = table[b, at // ps] * ps + at % ps
        pages, inv = torch.unique(slot // ps, return_inverse=True)
        local = inv * ps + slot % ps
        k, v = (_cells64(s[y][pages], c)[local].transpose(0, 1) for y in ("k", "v"))  # [kv head, key, d]
        step = max(1, int(3e8 // (H * (x + n))))
        for t in range(0, n, step):
            m = min(step, n - t)
            p = x + t + torch.arange(m, device="cuda")[:, None]
            gone = at > p
            if c["window"]:
                gone = gone | ((at <= p - c["window"]) & (at >= c["sinks"]))
            qs = q64[row + t: row + t + m].permute(1, 2, 0, 3).reshape(kvh, G * m, d)
            w = (qs @ k.transpose(1, 2)) / math.sqrt(d)
            w = torch.softmax(w.view(kvh, G, m, -1).masked_fill(gone, -math.inf), -1).view(kvh, G * m, -1)
            out[row + t: row + t + m] = (w @ v).view(kvh, G, m, d).permute(2, 0, 1, 3).reshape(m, H * d)
        row += n
    return out

"""The paged serving operators on the GPU against plain 64-bit implementations (paged_ref.py).

Bounds, derived before the first run. Planner: whole numbers, equal. Append: a rotated element is
two fp32 products and a sum of fp32 values whose cosine and sine are correct to about 2^-22, so it is off
by at most 2^-21 (|a| + |b|) before the final rounding, which adds half a step of its type (fp16: 2^-11
relative; Q8: half a delta, and the delta's own fp16 rounding). Attention: with w the softmax weights and
A = sum_j w_j |v_j|, rounding the weights to fp16 moves an output by at most 2^-11 A, fp32 sums over the
at most 2,000 keys here by 2^-12 A, and an error ds of a score by 2 ds A, where fp32 products give
ds <= 2^-17 S with S = scale sum_e |q_e k_e| (at most 128 terms of 2^-24 each); a Q8 cache or Q8 queries
enter the products rounded to fp16 (2^-11 relative: 2^-11 A for the values, ds larger by 2^-11 S each for
keys and queries). The result's own rounding comes on top."""
import numpy as np
import pytest
import torch

import gten_b200 as G
from paged_ref import (F16, F32, I32, Q8, U16, attn_bound, cache_of, gt, i32, new_pool, q8_encode, ref_attn, ref_plan,
                       ref_rope, rows_of, values_of)

pytestmark = pytest.mark.gpu


def rnd(gen, *shape):
    return torch.randn(*shape, generator=gen, device=gen.device, dtype=torch.float64)


def generator(seed, device):
    return torch.Generator(device=device).manual_seed(seed)


# ---- planner ----------------------------------------------------------------------------------------
def run_plan(ctx, new, free, n_free, ps, table, rows, gpu, stream=None):
    n, mp = len(ctx), len(table[0])
    t = {"ctx": i32(ctx, gpu), "new": i32(new, gpu), "free": i32(free, gpu), "n_free": i32([n_free], gpu),
         "table": i32(table, gpu), "q_start": i32([7] * (n + 1), gpu), "kv": i32([7] * n, gpu),
         "pos": i32([7] * rows, gpu), "slots": i32([7] * rows, gpu), "used": i32([7], gpu)}
    torch.cuda.synchronize()
    G.paged_plan(gt(t["ctx"]), gt(t["new"]), gt(t["free"]), gt(t["n_free"]), ps, gt(t["table"]), gt(t["q_start"]),
                 gt(t["kv"]), gt(t["pos"]), gt(t["slots"]), gt(t["used"]), stream=stream)
    torch.cuda.synchronize()
    return (t["table"].tolist(), t["q_start"].tolist(), t["kv"].tolist(), t["pos"].tolist(), t["slots"].tolist(),
            t["used"].item())


def plan_inputs(rng, n, ps, mp, new_hi, spare=5):
    ctx = [int(rng.integers(0, mp * ps - new_hi + 1)) for _ in range(n)]
    new = [int(rng.integers(0, new_hi + 1)) for _ in range(n)]
    have = [-(-c // ps) for c in ctx]
    need = sum(-(-(c + w) // ps) - h for c, w, h in zip(ctx, new, have))
    ids = rng.permutation(sum(have) + need + spare).tolist()
    table, at = [], 0
    for h in have:
        table.append(ids[at:at + h] + [-1] * (mp - h))
        at += h
    return ctx, new, ids[at:], need, table


@pytest.mark.parametrize("n,ps,mp,new_hi", [(1, 16, 4, 1), (1, 256, 2, 300), (7, 16, 9, 40), (512, 32, 6, 3), (513, 16, 5, 9),
                                            (1000, 64, 3, 100), (4096, 16, 3, 2)])
def test_plan_matches(gpu, n, ps, mp, new_hi):
    rng = np.random.default_rng(n + ps)
    ctx, new, free, need, table = plan_inputs(rng, n, ps, mp, new_hi)
    rows = max(1, sum(new) + 3)
    want = ref_plan(ctx, new, free, len(free), ps, table, rows)
    assert want[5] == need
    assert run_plan(ctx, new, free, len(free), ps, table, rows, gpu) == want


@pytest.mark.parametrize("case", ["few_pages", "no_pages", "few_rows", "negative", "table_full", "nothing_new"])
def test_plan_refuses_requests(gpu, case):
    rng = np.random.default_rng(3)
    ctx, new, free, need, table = plan_inputs(rng, 40, 16, 6, 30)
    rows, n_free = sum(new) + 2, len(free)
    if case == "few_pages":
        n_free = need // 2
    elif case == "no_pages":
        n_free = -1
    elif case == "few_rows":
        rows = sum(new) - 45
    elif case == "negative":
        ctx[3], new[9], new[11] = -1, -4, -2 ** 31
        ctx[20] = -2 ** 31
    elif case == "table_full":
        new[5], new[17] = 6 * 16 - ctx[5] + 1, 2000
        rows = sum(new) + 2
    else:
        new = [0] * 40
        rows = 4
    want = ref_plan(ctx, new, free, n_free, 16, table, rows)
    assert run_plan(ctx, new, free, n_free, 16, table, rows, gpu) == want


# ---- append -----------------------------------------------------------------------------------------
def append_case(gpu, seed, heads, kvh, d, ps, src, cache, qdt, rows, rope_pct, base, pos_hi, extra=0, stacked=False):
    gen = generator(seed, gpu)
    n_pages = -(-rows // ps) + 2
    slot_of = torch.randperm(n_pages * ps, generator=gen, device=gpu)[:rows].tolist()
    pos = torch.randint(0, pos_hi, (rows,), generator=gen, device=gpu).tolist()
    pos[0], pos[-1] = 0, pos_hi - 1
    if rows > 4:
        pos[2], slot_of[2] = -1, -1   # padding in the middle
        slot_of[3] = -1               # not granted: rotated, not stored
    q, k, v = rnd(gen, rows, heads * d), rnd(gen, rows, kvh * d), rnd(gen, rows, kvh * d)
    if stacked:  # column ranges of one projection output
        x = rows_of(src, torch.cat([q, k, v], 1))
        total = (heads + 2 * kvh) * d
        raw = [x[:, :x.shape[1] * heads * d // total], None, None]
        a, b = x.shape[1] * heads * d // total, x.shape[1] * (heads + kvh) * d // total
        raw = [x[:, :a], x[:, a:b], x[:, b:]]
        st = (total, 1)
        tens = [gt(r, src, (rows, n), st) for r, n in zip(raw, (heads * d, kvh * d, kvh * d))]
        raw = [r.contiguous() for r in raw]
    else:
        raw = [rows_of(src, y) for y in (q, k, v)]
        tens = [gt(r, src, (rows, y.shape[1])) for r, y in zip(raw, (q, k, v))]
    kp, vp = (new_pool(cache, n_pages, ps, kvh, d, gpu, extra, 0x55) for _ in range(2))
    out = rows_of(qdt, torch.zeros(rows, heads * d, device=gpu, dtype=torch.float64) + 3.0)
    before = [kp.raw.clone(), vp.raw.clone(), out.clone()]
    G.paged_append(*tens, gt(i32(pos, gpu)), gt(i32(slot_of, gpu)), cache_of(kp, vp), gt(out, qdt, (rows, heads * d)),
                   rope_pct, base)
    G.check()
    qv, kv, vv = (values_of(src, r, r_n) for r, r_n in zip(raw, (heads * d, kvh * d, kvh * d)))
    return dict(pos=pos, slots=slot_of, q=qv.view(rows, heads, d), k=kv.view(rows, kvh, d), v=vv.view(rows, kvh, d), kp=kp,
                vp=vp, out=out, before=before, raw=raw)


def close_rows(got, want, mag, dtype):
    """got and want [heads, d]; mag: bound on the fp32 error."""
    if dtype == F16:
        tol = mag + (want.abs() + mag) * U16 + 2.0 ** -25
    else:
        big = (want.abs() + mag).view(want.shape[0], -1, 32).amax(-1, keepdim=True).expand(-1, -1, 32).reshape(want.shape)
        tol = mag + big * (1.0 / 254 + U16) * (1 + 2.0 ** -10) + 2.0 ** -25
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), ((got - want).abs()[bad].max().item(), tol[bad].min().item())


@pytest.mark.parametrize("src", [F16, F32, Q8])
@pytest.mark.parametrize("cache,qdt", [(F16, F16), (Q8, F16), (Q8, Q8), (F16, Q8)])
@pytest.mark.parametrize("heads,kvh,d,ps,rope_pct,base,pos_hi,stacked",
                         [(4, 2, 64, 16, 1.0, 10000.0, 50, False), (3, 3, 64, 32, 0.25, 10000.0, 4000, True),
                          (8, 1, 128, 64, 1.0, 500000.0, 200000, True), (5, 5, 128, 16, 0.5, 10000.0, 2 ** 30, False),
                          (2, 1, 64, 256, 0.0, 10000.0, 9, False), (9, 3, 64, 16, 0.1, 10000.0, 77, True)])
def test_append_matches(gpu, src, cache, qdt, heads, kvh, d, ps, rope_pct, base, pos_hi, stacked):
    rows = 11
    r = append_case(gpu, heads + d + ps, heads, kvh, d, ps, src, cache, qdt, rows, rope_pct, base, pos_hi, 48, stacked)
    got_q = values_of(qdt, r["out"], heads * d).view(rows, heads, d)
    touched = torch.zeros(r["kp"].raw.shape[0] * ps, dtype=torch.bool)
    for t in range(rows):
        p, s = r["pos"][t], r["slots"][t]
        if p < 0:
            assert torch.equal(r["out"][t], r["before"][2][t])
            continue
        # an angle of up to 2^30 radians carries 2^30 * 2^-52 of its own rounding, far below the cosine's
        mag = lambda x: 2.0 ** -21 * 2 * x.abs().amax(-1, keepdim=True).expand_as(x)  # noqa: E731
        close_rows(got_q[t], ref_rope(r["q"][t], p, rope_pct, base), mag(r["q"][t]), qdt)
        if s < 0:
            continue
        touched[s] = True
        close_rows(r["kp"].get(s // ps, s % ps), ref_rope(r["k"][t], p, rope_pct, base), mag(r["k"][t]), cache)
        v = r["vp"].get(s // ps, s % ps)
        if src == Q8 and cache == Q8:
            assert torch.equal(v, r["v"][t])  # V blocks pass unchanged
        else:
            close_rows(v, r["v"][t], torch.zeros_like(r["v"][t]), cache)
    for pool, was in ((r["kp"], r["before"][0]), (r["vp"], r["before"][1])):
        now = type(pool)(pool.raw.clone(), pool.dtype, ps, kvh, d)
        old = type(pool)(was, pool.dtype, ps, kvh, d)
        for s in torch.nonzero(touched).view(-1).tolist():  # put the old rows back: nothing else may differ
            n = kvh * ps * d
            for a, b in ((now.raw, old.raw),):
                w = 2 if cache == F16 else 1
                av, bv = (z[s // ps][:w * n].view(kvh, ps, w * d) for z in (a, b))
                av[:, s % ps] = bv[:, s % ps]
                if cache == Q8:
                    av, bv = (z[s // ps][n:n + n // 16].view(kvh, ps, d // 16) for z in (a, b))
                    av[:, s % ps] = bv[:, s % ps]
        assert torch.equal(now.raw, old.raw)


def test_append_query_in_place(gpu):
    gen = generator(5, gpu)
    x = rnd(gen, 6, 4 * 64).to(torch.float16)
    k = rnd(gen, 6, 2 * 64).to(torch.float16)
    outs = []
    for inplace in (False, True):
        q = x.clone()
        o = q if inplace else torch.zeros_like(q)
        kp, vp = (new_pool(F16, 2, 16, 2, 64, gpu) for _ in range(2))
        G.paged_append(gt(q, F16), gt(k, F16), gt(k, F16), gt(i32(range(6), gpu)), gt(i32(range(6), gpu)), cache_of(kp, vp),
                       gt(o, F16))
        outs.append(o.clone())
    assert torch.equal(*outs)


def test_append_refuses_a_slot_outside_the_pool(gpu):
    gen = generator(6, gpu)
    q = rnd(gen, 2, 128).to(torch.float16)
    kp, vp = (new_pool(F16, 3, 16, 2, 64, gpu) for _ in range(2))
    out = torch.zeros_like(q)
    G.check()
    G.paged_append(gt(q, F16), gt(q, F16), gt(q, F16), gt(i32([0, 1], gpu)), gt(i32([48, 3], gpu)), cache_of(kp, vp),
                   gt(out, F16))
    with pytest.raises(G.GtenError, match="status 5"):
        G.check()
    G.check()
    assert kp.get(0, 3).abs().sum() > 0


# ---- attention --------------------------------------------------------------------------------------
class Batch:
    """Requests (kv length, new tokens) with random keys and values in scattered pages. Unused rows and
    pages hold the byte `fill` (0xff: NaN)."""

    def __init__(self, gpu, seed, lens, heads, kvh, d, ps, cache, io, pad=0, fill=0xff, extra=0, qscale=1.0, more_cols=0):
        self.gpu, self.lens, self.heads, self.kvh, self.d, self.ps = gpu, lens, heads, kvh, d, ps
        self.cache, self.io = cache, io
        gen = generator(seed, gpu)
        used = [-(-kv // ps) for kv, _ in lens]
        n_pages = sum(used) + 2
        ids = torch.randperm(n_pages, generator=gen, device=gpu).tolist()
        self.mp = max(1, max(used)) + more_cols
        self.table, at = [], 0
        for u in used:
            self.table.append(ids[at:at + u] + [-7] * (self.mp - u))
            at += u
        self.k, self.v = (new_pool(cache, n_pages, ps, kvh, d, gpu, extra, fill) for _ in range(2))
        self.keys, self.values = [], []
        for b, (kv, _) in enumerate(lens):
            for pool, vals in ((self.k, self.keys), (self.v, self.values)):
                x = rnd(gen, kv, kvh, d)
                for j in range(kv):
                    pool.put(self.table[b][j // ps], j % ps, x[j])
                vals.append(torch.stack([pool.get(self.table[b][j // ps], j % ps) for j in range(kv)]) if kv else x)
        self.new = [n for _, n in lens]
        self.rows = sum(self.new) + pad
        x = rnd(gen, max(1, self.rows), heads * d) * qscale
        self.q = rows_of(io, x)
        self.qv = values_of(io, self.q, heads * d).view(-1, heads, d)
        self.out = rows_of(io, torch.full_like(x, 3.0))
        self.q_start = [0]
        for n in self.new:
            self.q_start.append(self.q_start[-1] + n)
        self.kv_lens = [kv for kv, _ in lens]

    def tensors(self):
        shape = (max(1, self.rows), self.heads * self.d)
        return (gt(self.q, self.io, shape), cache_of(self.k, self.v), gt(i32(self.table, self.gpu)),
                gt(i32(self.q_start, self.gpu)), gt(i32(self.kv_lens, self.gpu)), gt(self.out, self.io, shape))

    def run(self, **kw):
        G.paged_attn(*self.tensors(), **kw)
        return self

    def compare(self, scale=0.0, window=0, n_sink=0, **_):
        got = values_of(self.io, self.out, self.heads * self.d).view(-1, self.heads, self.d)
        scale = scale or self.d ** -0.5
        for b, n in enumerate(self.new):
            if n == 0:
                continue
            s = self.q_start[b]
            want, A, S = ref_attn(self.qv[s:s + n], self.keys[b], self.values[b], self.kv_lens[b] - n, scale, window, n_sink)
            tol = attn_bound(want, A, S, self.cache, self.io)
            bad = ~((got[s:s + n] - want).abs() <= tol)
            assert not bool(bad.any()), (b, torch.nonzero(bad)[0].tolist(), got[s:s + n][bad][:4], want[bad][:4], tol[bad][:4])
        tail = self.out[self.q_start[-1]:]
        assert torch.equal(tail, rows_of(self.io, torch.full((max(1, self.rows), self.heads * self.d), 3.0, device=self.gpu,
                                                            dtype=torch.float64))[self.q_start[-1]:])


#: (kv length, new tokens): single tokens, page and tile ends, no history, nothing new, not granted
DECODE = [(1, 1), (16, 1), (17, 1), (127, 1), (128, 1), (129, 1), (300, 1), (5, 0), (0, 1)]
CHUNKS = [(130, 130), (1, 1), (257, 64), (200, 3), (0, 5), (64, 0), (511, 300), (90, 2)]
HEADS = [(8, 1, 64), (3, 3, 64), (4, 1, 64), (7, 7, 128), (16, 2, 128), (9, 3, 64)]


@pytest.mark.parametrize("lens", [DECODE, CHUNKS], ids=["decode", "chunks"])
@pytest.mark.parametrize("cache,io", [(F16, F16), (Q8, F16), (Q8, Q8), (F16, Q8)])
@pytest.mark.parametrize("heads,kvh,d", HEADS)
def test_attn_matches(gpu, lens, cache, io, heads, kvh, d):
    b = Batch(gpu, heads * d + kvh, lens, heads, kvh, d, 16, cache, io, pad=3, extra=64, more_cols=2)
    b.run(max_new=max(n for _, n in lens)).compare()
    G.check()


@pytest.mark.parametrize("window,n_sink", [(1, 0), (1, 1), (16, 4), (100, 0), (100, 130), (128, 128), (1000, 5), (33, 1000)])
@pytest.mark.parametrize("cache,heads,kvh,d,ps", [(F16, 4, 1, 64, 16), (Q8, 4, 4, 64, 32), (F16, 2, 1, 128, 128)])
@pytest.mark.parametrize("lens", [[(1, 1), (40, 1), (700, 1)], [(700, 4), (650, 650), (300, 40)]], ids=["decode", "chunks"])
def test_attn_window_and_sinks(gpu, window, n_sink, cache, heads, kvh, d, ps, lens):
    b = Batch(gpu, window + n_sink, lens, heads, kvh, d, ps, cache, F16, pad=1)
    kw = dict(window=window, n_sink=n_sink)
    b.run(**kw).compare(**kw)
    G.check()


@pytest.mark.parametrize("ps", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("cache,d", [(F16, 64), (Q8, 64), (F16, 128), (Q8, 128)])
def test_attn_page_sizes(gpu, ps, cache, d):
    b = Batch(gpu, ps + d, [(301, 1), (257, 200), (ps, 1), (ps + 1, 2)], 4, 2, d, ps, cache, F16, more_cols=1)
    b.run().compare()
    G.check()


@pytest.mark.parametrize("lens", [[(1500, 1)], [(1900, 1), (3, 1)], [(1600, 33)], [(1200, 129), (1100, 1)]])
@pytest.mark.parametrize("cache", [F16, Q8])
def test_attn_long_axis(gpu, lens, cache):
    """Few rows over many keys: the keys are split and joined."""
    b = Batch(gpu, len(lens), lens, 8, 1, 64, 64, cache, F16)
    b.run().compare()


@pytest.mark.parametrize("cache", [F16, Q8])
@pytest.mark.parametrize("heads,kvh,d,n", [(32, 32, 64, 3), (24, 24, 128, 2)])
def test_attn_many_items_per_worker(gpu, cache, heads, kvh, d, n):
    """Several items and many units for every worker: the rings wrap, and ranges end on units that only one
    of an item's two row tiles needs."""
    b = Batch(gpu, n, [(700 + 31 * i, 500 - 17 * i) for i in range(n)], heads, kvh, d, 32, cache, F16)
    b.run().compare()
    G.check()


@pytest.mark.parametrize("scale", [0.02, 1.0])
def test_attn_scale_and_peaked_scores(gpu, scale):
    """Scores up to about +-100: weights that underflow, and a running maximum that moves."""
    b = Batch(gpu, 3, [(400, 1), (300, 150)], 4, 1, 64, 16, F16, F16, qscale=4.0)
    b.run(scale=scale).compare(scale=scale)


def test_attn_max_new_is_only_a_hint(gpu):
    outs = []
    for max_new in (0, 1, 5, 300):
        b = Batch(gpu, 9, [(130, 65), (40, 1), (90, 5)], 4, 1, 64, 16, F16, F16)
        b.run(max_new=max_new).compare()


def poison(b, req, key, value, which):
    """Overwrites one key row of a request in the pages, not in the reference's copy."""
    pool = b.k if which == "k" else b.v
    n = pool.kvh * pool.ps * pool.d
    pg = pool.raw[b.table[req][key // pool.ps]]
    if pool.dtype == F16:
        pg[:2 * n].view(torch.float16).view(pool.kvh, pool.ps, pool.d)[:, key % pool.ps] = value
    else:
        pg[n:n + n // 16].view(torch.float16).view(pool.kvh, pool.ps, pool.d // 32)[:, key % pool.ps] = value


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf"), -65504.0])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("cache", [F16, Q8])
@pytest.mark.parametrize("lens", [[(200, 1)], [(200, 3)], [(300, 160)]], ids=["one", "few", "chunk"])
def test_attn_masked_keys_never_reach_a_row(gpu, value, which, cache, lens):
    """Non-finite keys and values where a window or the causal limit hides them: rows that do not see
    them are right, rows that see a non-finite value (or key) are not finite."""
    kv, n = lens[0]
    heads, kvh, d = 4, 2, 64
    b = Batch(gpu, 4, lens, heads, kvh, d, 16, cache, F16)
    window, n_sink = 60, 2
    hidden = kv - n - 75           # before the first row's window, behind the sinks
    poison(b, 0, hidden, value, which)
    last = kv - 1                  # seen by the last row alone
    if n > 1:
        poison(b, 0, last, value, which)
    b.run(window=window, n_sink=n_sink)
    got = b.out.view(-1, heads, d).double()
    rows = n - 1 if n > 1 else n
    want, A, S = ref_attn(b.qv[:n], b.keys[0], b.values[0], kv - n, d ** -0.5, window, n_sink)
    tol = attn_bound(want, A, S, cache, F16)
    assert bool(((got[:rows] - want[:rows]).abs() <= tol[:rows]).all())
    if n > 1 and which == "v" and value != -65504.0:
        assert not bool(torch.isfinite(got[n - 1]).any())
        if value == value and cache == F16:
            assert bool((got[n - 1] == value).all())
    if n > 1 and which == "k" and value != value:
        assert bool(torch.isnan(got[n - 1]).all())


def test_attn_strided_rows_and_table(gpu):
    b = Batch(gpu, 12, [(70, 33), (20, 1)], 4, 2, 64, 16, F16, F16, pad=1)
    wide = torch.full((b.rows, 4 * 64 + 40), 9.0, dtype=torch.float16, device=gpu)
    wide[:, 8:8 + 256] = b.q
    owide = torch.full((b.rows, 4 * 64 + 24), 5.0, dtype=torch.float16, device=gpu)
    table = torch.full((2, b.mp + 3), -9, dtype=torch.int32, device=gpu)
    table[:, :b.mp] = i32(b.table, gpu)
    t = b.tensors()
    G.paged_attn(gt(wide[:, 8:], F16, (b.rows, 256), (296, 1)), t[1], gt(table, I32, (2, b.mp), (b.mp + 3, 1)), t[3], t[4],
                 gt(owide, F16, (b.rows, 256), (280, 1)))
    assert bool((owide[:, 256:] == 5.0).all()) and bool((owide[b.q_start[-1]:, :] == 5.0).all())
    b.out[:b.q_start[-1]] = owide[:b.q_start[-1], :256]
    b.compare()


def test_attn_pages_out_of_the_window_may_be_gone(gpu):
    """Table entries of pages that no row sees may be anything; one that a row sees raises."""
    b = Batch(gpu, 13, [(400, 1), (400, 50)], 4, 1, 64, 16, F16, F16)
    kw = dict(window=64, n_sink=4)
    for r, n in ((0, 1), (1, 50)):
        for c in range(1, (400 - n - 64 + 1) // 16):
            b.table[r][c] = [-1, 10 ** 6, 2 ** 31 - 1][c % 3]
    b.run(**kw).compare(**kw)
    G.check()
    b.table[0][-1] = b.k.raw.shape[0]
    b.run(**kw)
    with pytest.raises(G.GtenError, match="status 5"):
        G.check()
    b.table[0][-1] = -1
    b.table[1][24] = 2 ** 30
    b.run(**kw)
    with pytest.raises(G.GtenError, match="status 5"):
        G.check()


@pytest.mark.parametrize("bad", ["long", "negative"])
def test_attn_lengths_outside_the_table(gpu, bad):
    b = Batch(gpu, 14, [(50, 1), (60, 2)], 4, 1, 64, 16, F16, F16)
    b.kv_lens[0] = 10 ** 9 if bad == "long" else -5
    b.run()
    with pytest.raises(G.GtenError, match="status 5"):
        G.check()
    got = b.out.view(-1, 4, 64).double()
    want, A, S = ref_attn(b.qv[1:3], b.keys[1], b.values[1], 58, 0.125, 0, 0)
    assert bool(((got[1:3] - want).abs() <= attn_bound(want, A, S, F16, F16)).all())


def test_attn_same_twice_and_on_another_stream(gpu):
    b = Batch(gpu, 15, [(700, 1), (300, 1), (400, 200)], 8, 2, 64, 16, F16, F16)
    b.run()
    first = b.out.clone()
    side = torch.cuda.Stream()
    b.out.zero_()
    side.wait_stream(torch.cuda.current_stream())
    b.run(stream=side)
    side.synchronize()
    assert torch.equal(b.out, first)


# ---- together ---------------------------------------------------------------------------------------
class Server:
    """A step loop over the three operators with device-side lengths: plan, append, attend (one layer)."""

    def __init__(self, gpu, n, rows, heads, kvh, d, ps, cache, io, n_pages, mp):
        z = lambda *s: torch.zeros(*s, dtype=torch.int32, device=gpu)  # noqa: E731
        self.gpu, self.n, self.rows, self.heads, self.kvh, self.d, self.ps = gpu, n, rows, heads, kvh, d, ps
        self.io = io
        self.ctx, self.new, self.n_free, self.used = z(n), z(n), z(1), z(1)
        self.free = torch.arange(n_pages, dtype=torch.int32, device=gpu).flip(0).contiguous()
        self.n_free.fill_(n_pages)
        self.table = torch.full((n, mp), -1, dtype=torch.int32, device=gpu)
        self.q_start, self.kv, self.pos, self.slots = z(n + 1), z(n), z(rows), z(rows)
        self.kp, self.vp = (new_pool(cache, n_pages, ps, kvh, d, gpu, 0, 0xff) for _ in range(2))
        self.cache = cache_of(self.kp, self.vp)
        cols = lambda h: h * d if io == F16 else h * d // 32 * 34  # noqa: E731
        dt = torch.float16 if io == F16 else torch.uint8
        self.q, self.qr, self.out = (torch.zeros(rows, cols(heads), dtype=dt, device=gpu) for _ in range(3))
        self.k, self.v = (torch.zeros(rows, cols(kvh), dtype=dt, device=gpu) for _ in range(2))
        self.ws = torch.empty(G.paged_attn_workspace(heads, d), dtype=torch.uint8, device=gpu)

    def step(self, max_new=0, **kw):
        r, h, kd = self.rows, self.heads * self.d, self.kvh * self.d
        G.paged_plan(gt(self.ctx), gt(self.new), gt(self.free), gt(self.n_free), self.ps, gt(self.table), gt(self.q_start),
                     gt(self.kv), gt(self.pos), gt(self.slots), gt(self.used))
        G.paged_append(gt(self.q, self.io, (r, h)), gt(self.k, self.io, (r, kd)), gt(self.v, self.io, (r, kd)), gt(self.pos),
                       gt(self.slots), self.cache, gt(self.qr, self.io, (r, h)))
        G.paged_attn(gt(self.qr, self.io, (r, h)), self.cache, gt(self.table), gt(self.q_start), gt(self.kv),
                     gt(self.out, self.io, (r, h)), max_new=max_new, workspace=self.ws, **kw)

    def advance(self):
        """What a server keeps between steps: lengths, and the free list without the pages handed out."""
        u = int(self.used.item())
        self.free = self.free[u:].contiguous()
        self.n_free -= u
        self.ctx.copy_(torch.where(self.kv > 0, self.kv, self.ctx))


@pytest.mark.parametrize("io,cache,window,n_sink", [(F16, F16, 0, 0), (Q8, Q8, 0, 0), (F16, Q8, 24, 3), (F16, F16, 24, 3)])
def test_steps_of_a_server(gpu, io, cache, window, n_sink):
    """Prompts in chunks, decode steps beside them, a request that must wait for pages: every step's rows
    against attention over the request's whole history, computed in 64 bits from what the steps were given."""
    heads, kvh, d, ps, n = 4, 2, 64, 16, 3
    srv = Server(gpu, n, 80, heads, kvh, d, ps, cache, io, 14, 12)
    gen = generator(21, gpu)
    plan = [[40, 0, 7], [30, 5, 1], [1, 64, 1], [1, 1, 1], [2, 1, 60], [1, 1, 60], [1, 1, 1]]
    hist = [([], []) for _ in range(n)]
    waited = 0
    for new in plan:
        srv.new.copy_(i32(new, gpu))
        x = [rnd(gen, srv.rows, w * d) for w in (heads, kvh, kvh)]
        for dst, y in zip((srv.q, srv.k, srv.v), x):
            dst.copy_(rows_of(io, y))
        qv, kv, vv = (values_of(io, t, w * d).view(srv.rows, w, d) for t, w in ((srv.q, heads), (srv.k, kvh), (srv.v, kvh)))
        ctx = srv.ctx.tolist()
        srv.step(window=window, n_sink=n_sink)
        G.check()
        granted = [k > 0 or w == 0 for k, w in zip(srv.kv.tolist(), new)]
        got = values_of(io, srv.out, heads * d).view(srv.rows, heads, d)
        row = 0
        for b, w in enumerate(new):
            if granted[b]:
                rot = lambda t: torch.stack([ref_rope(t[row + i], ctx[b] + i, 1.0, 10000.0) for i in range(w)])  # noqa: E731
                if w:
                    table, kvl = srv.table[b].tolist(), ctx[b] + w
                    # what the cache holds is compared by its own test; here its values are the keys
                    keys = torch.stack([srv.kp.get(table[j // ps], j % ps) for j in range(kvl)])
                    vals = torch.stack([srv.vp.get(table[j // ps], j % ps) for j in range(kvl)])
                    tol_k = 2.0 ** -7 if cache == Q8 or io == Q8 else 2.0 ** -10
                    hist[b][0].append(rot(kv))
                    hist[b][1].append(vv[row:row + w])
                    for have, should in ((keys, torch.cat(hist[b][0])), (vals, torch.cat(hist[b][1]))):
                        assert bool(((have - should).abs() <= tol_k * should.abs().amax(-1, keepdim=True)).all())
                    q = values_of(io, srv.qr, heads * d).view(srv.rows, heads, d)[row:row + w]
                    want, A, S = ref_attn(q, keys, vals, ctx[b], d ** -0.5, window, n_sink)
                    assert bool(((got[row:row + w] - want).abs() <= attn_bound(want, A, S, cache, io)).all()), (b, w)
            else:
                waited += 1
                assert bool((got[row:row + w] == 0).all())
            row += w
        srv.advance()
    assert waited > 0


def test_captured_steps_follow_the_lengths(gpu):
    """One graph of plan, append and attention, replayed for decode steps whose lengths change on the
    device, gives what the calls give."""
    heads, kvh, d, ps, n = 8, 2, 64, 16, 4
    runs = []
    for captured in (False, True):
        srv = Server(gpu, n, n, heads, kvh, d, ps, F16, F16, 40, 10)
        gen = generator(31, gpu)
        srv.new.fill_(1)
        got, graph = [], None
        for step in range(20):
            for t in (srv.q, srv.k, srv.v):
                t.copy_(rnd(gen, *t.shape).to(torch.float16))
            if step == 5:
                srv.ctx[1] = 0  # a new request takes the place of another
            if not captured:
                srv.step(max_new=1)
            else:
                if graph is None:
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph):
                        srv.step(max_new=1)
                graph.replay()
            got.append(srv.out.clone())
            # a device-side server: the pages handed out leave the front of the list by a rotation
            u = int(srv.used.item())
            srv.free.copy_(torch.roll(srv.free, -u))
            srv.ctx.copy_(srv.kv)
        G.check()
        runs.append(torch.stack(got))
    assert torch.equal(*runs)


def test_two_graphs_side_by_side(gpu):
    """Two captured calls with a workspace each, replayed at the same time on two streams."""
    bs = [Batch(gpu, 41 + i, [(900, 1), (300, 70)], 8, 2, 64, 16, F16, F16) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in bs]
    graphs = []
    for b, st in zip(bs, streams):
        b.ws = torch.empty(G.paged_attn_workspace(8, 64), dtype=torch.uint8, device=gpu)
        b.t = b.tensors()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            G.paged_attn(*b.t, workspace=b.ws)
        graphs.append(g)
    for _ in range(5):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for b in bs:
        b.compare()

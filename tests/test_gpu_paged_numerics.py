"""The paged attention where rounding would show: Q8 caches whose values cancel, long histories, and the framework's
own operators before, behind and beside it. Bounds as in test_gpu_paged.py unless they are derived here."""
import pytest
import torch

import gten_b200 as G
from paged_long import LongBatch
from paged_ref import F16, F32, Q8, U16, attn_bound, cache_of, gt, i32, new_pool, ref_attn

pytestmark = pytest.mark.gpu

#: every kernel over Q8 pages: single rows, tiles of 8 and of 16 rows, chunks of 1 and 2 query heads per kv head
KERNELS = [(2, 2, 1, 1), (4, 2, 1, 1), (16, 1, 1, 1), (2, 2, 40, 0), (4, 2, 40, 0)]


# ---- Q8 caches are exact --------------------------------------------------------------------------------
def q8_pages(pool, ints, delta):
    """Writes a Q8 pool: ints [page, kv head, row, d], deltas [page, kv head, row, d / 32]."""
    n = pool.kvh * pool.ps * pool.d
    pool.raw[:, :n] = ints.to(torch.int8).reshape(ints.shape[0], -1).view(torch.uint8)
    pool.raw[:, n:] = delta.to(torch.float16).reshape(ints.shape[0], -1).contiguous().view(torch.uint8)


def each_row(b, n):
    for r in range(len(b.lens)):
        keys, values = b.cells(b.k, r), b.cells(b.v, r)
        for i in range(n):
            yield r, i, keys, values


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kvh,n,max_new", KERNELS)
def test_q8_values_enter_exactly(gpu, d, heads, kvh, n, max_new):
    """Equal scores (queries of zeros) over values that nearly cancel: keys in turns hold + i delta and -(i - 1) delta. The
    weights are powers of two, so only the fp32 sums round (400 terms: 400 * 2^-23 of A with truncating adders) and the
    result. Values rounded to fp16 on their way would be off by up to 2^-11 of A, as the planted mistake shows."""
    b = LongBatch(gpu, 100 + d, [(400, n), (90, n)], heads, kvh, d, 16, Q8)
    gen = torch.Generator(device=gpu).manual_seed(7)
    pages = b.v.raw.shape[0]
    i = torch.randint(100, 128, (1, kvh, 1, d), generator=gen, device=gpu).expand(pages, kvh, 16, d)
    odd = (torch.arange(16, device=gpu) % 2 == 1)[:, None]
    delta = (torch.rand(1, kvh, 1, d // 32, generator=gen, device=gpu) + 0.5).expand(pages, kvh, 16, d // 32)
    q8_pages(b.v, torch.where(odd, 1 - i, i), delta)
    b.q.zero_()
    b.run(max_new=max_new)
    G.check()
    shown = False
    for r, t, keys, values in each_row(b, n):
        want, A, _ = b.want(r, t, keys, values)
        tol = A * 400 * 2.0 ** -23 + (want.abs() + A * 400 * 2.0 ** -23) * U16 + 2.0 ** -25
        assert bool(((b.row(r, t) - want[0]).abs() <= tol[0]).all()), (r, t)
        wrong = b.want(r, t, keys, values.to(torch.float16).double())[0]
        shown = shown or bool(((wrong - want).abs() > 2 * tol).any())
    assert shown


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("heads,kvh,n,max_new", KERNELS)
def test_q8_keys_enter_exactly(gpu, d, heads, kvh, n, max_new):
    """Queries of ones over keys whose elements are + i delta and -(i - 1) delta in turns, delta near 4: products of 500
    that cancel to scores of some 16. fp32 products and sums move a score by 2^-17 S; keys rounded to fp16 on their way
    would by 2^-11 S, as the planted mistake shows. Short histories: few keys to average over."""
    b = LongBatch(gpu, 200 + d, [(max(4, n), n), (max(3, n), n)], heads, kvh, d, 16, Q8)
    gen = torch.Generator(device=gpu).manual_seed(8)
    pages = b.k.raw.shape[0]
    i = torch.randint(100, 128, (pages, kvh, 16, 1), generator=gen, device=gpu).expand(pages, kvh, 16, d)
    odd = torch.arange(d, device=gpu) % 2 == 1
    delta = (3.5 + torch.rand(pages, kvh, 16, 1, generator=gen, device=gpu)).expand(pages, kvh, 16, d // 32)
    q8_pages(b.k, torch.where(odd, 1 - i, i), delta)
    b.q.fill_(1.0)
    b.run(max_new=max_new)
    G.check()
    shown = False
    for r, t, keys, values in each_row(b, n):
        want, A, S = b.want(r, t, keys, values)
        tol = attn_bound(want, A, S, F16, F16)  # no term for the cache's type
        assert bool(((b.row(r, t) - want[0]).abs() <= tol[0]).all()), (r, t)
        wrong = b.want(r, t, keys.to(torch.float16).double(), values)[0]
        shown = shown or bool(((wrong - want).abs() > 2 * tol).any())
    assert shown


# ---- long histories -------------------------------------------------------------------------------------
@pytest.mark.parametrize("cache,io", [(F16, F16), (Q8, F16), (Q8, Q8)])
@pytest.mark.parametrize("heads,kvh,d,ps", [(8, 2, 128, 64), (4, 4, 64, 16)])
@pytest.mark.parametrize("window,n_sink", [(0, 0), (4096, 4), (20000, 300)])
@pytest.mark.parametrize("kind", ["decode", "chunks"])
def test_long_histories(gpu, cache, io, heads, kvh, d, ps, window, n_sink, kind):
    """Histories of 32,000 keys. They are split over the GPU: a worker sums fewer than 3,000 keys and a join fewer than
    1,200 parts, so that attn_bound's 2^-12 of A (4,096 terms of 2^-24) holds for their fp32 sums too."""
    lens = [(32001, 1), (20000, 2), (31, 1)] if kind == "decode" else [(32001, 130), (20000, 300), (64, 64), (9000, 1)]
    b = LongBatch(gpu, 300, lens, heads, kvh, d, ps, cache, io)
    kw = dict(window=window, n_sink=n_sink)
    b.run(max_new=2 if kind == "decode" else 0, **kw)
    G.check()
    for r, (kv, n) in enumerate(lens):
        keys, values = b.cells(b.k, r), b.cells(b.v, r)
        for i in sorted({0, n // 3, n // 2, n - 1}):
            want, A, S = b.want(r, i, keys, values, **kw)
            tol = attn_bound(want, A, S, cache, io)
            assert bool(((b.row(r, i) - want[0]).abs() <= tol[0]).all()), (r, i)


# ---- beside the framework's own operators ---------------------------------------------------------------
@pytest.mark.parametrize("heads,kvh", [(4, 2), (3, 3), (8, 1)])
def test_pages_and_a_contiguous_cache(gpu, heads, kvh):
    """A layer both ways: projections by matmul_2d, then rotary_emb and qkv_attn over a contiguous cache, or the planner, the
    append and the attention over pages in steps of several lengths, then the output projection by matmul_2d. Each way's
    attention is within attn_bound of the exact one (qkv_attn also rounds its probabilities to fp16: 2^-25 per key of the
    largest value). The rotary operators' angles differ (test_gpu_paged_faults.py), so that a rotated fp16 query or key may
    be a step apart: 2^-10 relative each, 2^-9 S in a score, 2^-8 S A in an output."""
    d, ps, n, emb = 64, 16, 70, 192
    hd, kd = heads * d, kvh * d
    gen = torch.Generator(device=gpu).manual_seed(11)
    x = torch.randn(n, emb, generator=gen, device=gpu).to(torch.float16)
    w = [(torch.randn(o, i, generator=gen, device=gpu) * i ** -0.5).to(torch.float16) for o, i in
         ((hd, emb), (kd, emb), (kd, emb), (emb, hd))]
    z = lambda *s: torch.zeros(*s, dtype=torch.float16, device=gpu)  # noqa: E731
    g = lambda t: gt(t, F16)  # noqa: E731
    q, k, v = z(n, hd), z(n, kd), z(n, kd)
    for wi, o in zip(w, (q, k, v)):
        G.matmul_2d(g(x), g(wi), g(o))

    qr, kr, one = z(n, hd), z(n, kd), z(n, hd)
    G.rotary_emb(g(q), g(qr), d, 1.0)
    G.rotary_emb(g(k), g(kr), d, 1.0)
    G.qkv_attn(g(qr), g(kr), g(v), None, g(one), n)

    two = z(n, hd)
    kp, vp = (new_pool(F16, 8, ps, kvh, d, gpu) for _ in range(2))
    cache = cache_of(kp, vp)
    table, free = i32([[-1] * 6], gpu), i32([5, 0, 7, 2, 6, 1, 3, 4], gpu)
    ctx, kv, used, n_free = i32([0], gpu), i32([0], gpu), i32([0], gpu), i32([8], gpu)
    done = 0
    for step in (30, 1, 1, 17, 1, 20):
        rows = slice(done, done + step)
        starts, pos, slots = i32([0, 0], gpu), i32([0] * step, gpu), i32([0] * step, gpu)
        G.paged_plan(gt(ctx), gt(i32([step], gpu)), gt(free), gt(n_free), ps, gt(table), gt(starts), gt(kv), gt(pos), gt(slots),
                     gt(used))
        qs = z(step, hd)
        G.paged_append(g(q[rows]), g(k[rows]), g(v[rows]), gt(pos), gt(slots), cache, g(qs))
        G.paged_attn(g(qs), cache, gt(table), gt(starts), gt(kv), g(two[rows]), max_new=step if step == 1 else 0)
        u = int(used.item())
        free, done = free[u:].contiguous(), done + step
        n_free -= u
        ctx.copy_(kv)
    G.check()
    assert done == n

    outs = []
    for a in (one, two):
        o = torch.zeros(n, emb, device=gpu)
        G.matmul_2d(g(a), g(w[3]), gt(o, F32))
        outs.append(o.double())
    want, A, S = ref_attn(qr.double().view(n, heads, d), kr.double().view(n, kvh, d), v.double().view(n, kvh, d), 0, d ** -0.5, 0, 0)
    tol = 2 * attn_bound(want, A, S, F16, F16) + A * S[..., None] * 2.0 ** -8 + n * 2.0 ** -25 * float(v.double().abs().max())
    assert bool(((one.double() - two.double()).abs().view(n, heads, d) <= tol).all())
    # behind the output projection: its fp32 sums add at most 2^-16 of the magnitudes on each side
    mag = (one.double().abs() + tol.view(n, hd)) @ w[3].double().abs().T
    assert bool(((outs[0] - outs[1]).abs() <= tol.view(n, hd) @ w[3].double().abs().T + 2.0 ** -15 * mag).all())

"""Bad page ids and other input of the paged serving operators that must raise, and calls on which a kernel could
go wrong without a wrong index. Bounds as in test_gpu_paged.py."""
import pytest
import torch

import gten_b200 as G
import test_gpu_paged as tp
from paged_ref import F16, F32, Q8, attn_bound, cache_of, gt, i32, new_pool, ref_attn, ref_plan
from paged_long import LongBatch
from test_gpu_paged import Batch

pytestmark = pytest.mark.gpu


# ---- planner --------------------------------------------------------------------------------------------
def plan(gpu, ctx, new, free, table, rows, ps):
    n = len(ctx)
    t = {"ctx": i32(ctx, gpu), "new": i32(new, gpu), "free": i32(free, gpu), "n_free": i32([len(free)], gpu),
         "table": i32(table, gpu), "q_start": i32([7] * (n + 1), gpu), "kv": i32([7] * n, gpu), "pos": i32([7] * rows, gpu),
         "slots": i32([7] * rows, gpu), "used": i32([7], gpu)}
    G.paged_plan(gt(t["ctx"]), gt(t["new"]), gt(t["free"]), gt(t["n_free"]), ps, gt(t["table"]), gt(t["q_start"]),
                 gt(t["kv"]), gt(t["pos"]), gt(t["slots"]), gt(t["used"]))
    return t


@pytest.mark.parametrize("ps", [16, 64, 256])
@pytest.mark.parametrize("where", ["free", "table"])
@pytest.mark.parametrize("bad", ["first_too_large", "wraps_to_3", "tagged", "minus_one", "lowest", "largest"])
def test_plan_raises_for_page_ids_that_no_pool_holds(gpu, ps, where, bad):
    """Slots are page * page_size + offset in 32 bits: an id beyond them must not become another page's slot."""
    page = {"first_too_large": 2 ** 31 // ps, "wraps_to_3": 2 ** 32 // ps + 3,
            "tagged": -2 ** 31 + 3, "minus_one": -1, "lowest": -2 ** 31, "largest": 2 ** 31 - 1}[bad]
    assert page * ps >= 2 ** 31 or page < 0
    # request 0 goes on in its first page and takes a new one, request 1 is sound
    ctx, new, table, free = [5, 0], [ps, 3], [[4, -1], [-1, -1]], [6, 8]
    if where == "free":
        free[0] = page
    else:
        table[0][0] = page
    G.check()
    t = plan(gpu, ctx, new, free, table, ps + 4, ps)
    with pytest.raises(G.GtenError, match="status 5"):
        G.check()
    G.check()
    lost = range(ps - 5, ps) if where == "free" else range(0, ps - 5)  # the rows in the bad page
    sound = ([1, 8], [[4, -1], [-1, -1]]) if where == "free" else ([6, 8], [[1, -1], [-1, -1]])
    want = ref_plan(ctx, new, sound[0], 2, ps, sound[1], ps + 4)
    slots = [-1 if i in lost else s for i, s in enumerate(want[4])]
    assert t["slots"].tolist() == slots and t["pos"].tolist() == want[3]
    assert t["kv"].tolist() == want[2] and t["q_start"].tolist() == want[1] and t["used"].item() == 2


@pytest.mark.parametrize("ps", [16, 256])
def test_plan_takes_the_largest_page_id(gpu, ps):
    page = 2 ** 31 // ps - 1
    t = plan(gpu, [0], [ps], [page], [[-1]], ps, ps)
    G.check()
    assert t["slots"].tolist() == [page * ps + i for i in range(ps)]


def test_plan_ignores_bad_ids_that_it_does_not_use(gpu):
    """Free entries behind those taken, and the pages of requests that are not granted."""
    t = plan(gpu, [16, 16], [1, 40], [5, -1, 2 ** 30], [[2, -1], [2 ** 31 - 1, -1]], 41, 16)
    G.check()
    assert t["slots"].tolist() == [80] + [-1] * 40 and t["kv"].tolist() == [17, 0] and t["used"].item() == 1


def test_plan_then_append_leaves_other_pages_alone(gpu):
    """A wrapped id reaches no cell of another request."""
    ps, kvh, d = 16, 1, 64
    t = plan(gpu, [0], [3], [2 ** 28 + 2], [[-1]], 3, ps)
    pool = torch.zeros(4, ps * kvh * d * 2, dtype=torch.uint8, device=gpu)
    x = torch.ones(3, d, dtype=torch.float16, device=gpu)
    cache = G.PagedCache(pool, pool.clone(), F16, 4, ps, kvh, d)
    G.paged_append(gt(x, F16), gt(x, F16), gt(x, F16), gt(t["pos"]), gt(t["slots"]), cache, gt(torch.empty_like(x), F16))
    with pytest.raises(G.GtenError, match="status 5"):
        G.check()
    assert not bool(pool.any())


# ---- attention: table entries ---------------------------------------------------------------------------
#: every kernel: single rows over Q8, tiles of 8 and of 16 rows, chunks
KERNELS = [(2, 2, 1, 1), (4, 2, 1, 1), (16, 1, 1, 1), (4, 2, 40, 0), (32, 1, 9, 0)]


@pytest.mark.parametrize("cache,d", [(F16, 64), (F16, 128), (Q8, 64), (Q8, 128)])
@pytest.mark.parametrize("heads,kvh,n,max_new", KERNELS)
@pytest.mark.parametrize("entry", ["tagged", "minus_one", "n_pages", "largest"])
def test_bad_table_entries_raise(gpu, cache, d, heads, kvh, n, max_new, entry):
    """An entry whose low 31 bits name a page is as bad as any: no page of another request is read for it."""
    b = Batch(gpu, 90, [(200, n), (70, n)], heads, kvh, d, 16, cache, F16)
    pages = b.k.raw.shape[0]
    for col in (0, 5):
        b.table[0][col] = {"tagged": b.table[1][1] - 2 ** 31, "minus_one": -1, "n_pages": pages, "largest": 2 ** 31 - 1}[entry]
        G.check()
        b.run(max_new=max_new)
        with pytest.raises(G.GtenError, match="status 5"):
            G.check()
        # the other request is whole
        got = b.out.view(-1, heads, d).double()[n:2 * n]
        want, A, S = ref_attn(b.qv[n:2 * n], b.keys[1], b.values[1], 70 - n, d ** -0.5, 0, 0)
        assert bool(((got - want).abs() <= attn_bound(want, A, S, cache, F16)).all())


# ---- append: heads of several types in a warp ----------------------------------------------------------
@pytest.mark.parametrize("src", [F16, F32, Q8])
@pytest.mark.parametrize("cache,qdt", [(Q8, F16), (F16, Q8), (Q8, Q8), (F16, F16)])
@pytest.mark.parametrize("heads,kvh,d,rope_pct", [(36, 36, 64, 1.0), (28, 7, 64, 0.25), (16, 16, 128, 1.0), (20, 3, 128, 0.5),
                                                  (65, 1, 64, 1.0), (1, 1, 128, 1.0), (33, 33, 128, 0.0)])
def test_append_with_many_heads(gpu, src, cache, qdt, heads, kvh, d, rope_pct):
    """Rows of several turns of a CTA, and the border between queries, keys and values inside a warp, where some
    lanes quantize and others do not."""
    tp.test_append_matches(gpu, src, cache, qdt, heads, kvh, d, 16, rope_pct, 10000.0, 5000, False)


# ---- attention: values that are not finite, in long chunks --------------------------------------------
@pytest.mark.parametrize("d,heads,kvh", [(128, 32, 8), (64, 8, 8)])
@pytest.mark.parametrize("window,n_sink", [(0, 0), (9000, 5)])
def test_infinity_at_the_end_of_a_long_chunk(gpu, d, heads, kvh, window, n_sink):
    """An infinity that only the last token sees, in calls whose workers take many items: its row gets it, the others
    and other requests' are right, and looking for it costs milliseconds, not a walk over every key per item."""
    lens = [(30000, 1024), (700, 700), (29000, 300)]
    b = LongBatch(gpu, 91, lens, heads, kvh, d, 64, F16)
    kw = dict(window=window, n_sink=n_sink)
    keys, values = ([b.cells(p, i) for i in range(3)] for p in (b.k, b.v))

    def timed():
        G.check()
        e = [torch.cuda.Event(enable_timing=True) for _ in range(2)]
        e[0].record()
        b.run(**kw)
        e[1].record()
        G.check()
        return e[0].elapsed_time(e[1])

    clean = min(timed() for _ in range(3))
    b.set_row(b.v, 0, 29999, float("inf"))
    spoilt = timed()
    for r, i in [(0, 0), (0, 511), (0, 1022), (1, 0), (1, 300), (1, 699), (2, 0), (2, 299)]:
        want, A, S = b.want(r, i, keys[r], values[r], **kw)
        assert bool(((b.row(r, i) - want[0]).abs() <= long_bound(want, A, S)[0]).all()), (r, i)
    assert bool((b.row(0, 1023) == float("inf")).all())
    assert spoilt < clean + 20.0, (clean, spoilt)


def long_bound(want, A, S):
    """attn_bound for up to 30,000 keys: fp32 sums of n terms are off by at most n 2^-24 of the sum of magnitudes, here
    2^-9; the workers' shares of a few thousand keys at a time stay far below it."""
    return attn_bound(want, A, S, F16, F16) + A * 2.0 ** -9


# ---- attention: bounds on the new tokens over wide tables ---------------------------------------------
@pytest.mark.parametrize("heads,kvh,cache,pad", [(64, 8, F16, 0), (36, 36, Q8, 3072)])
def test_decode_steps_over_wide_tables(gpu, heads, kvh, cache, pad):
    """Single tokens of 1,024 requests whose tables have room for 2^19 keys: the bound on the new tokens chooses the
    kernels, not whether the call is taken."""
    n = 1024
    b = Batch(gpu, 92, [(1 + i % 2, 1) for i in range(n)], heads, kvh, 64, 16, cache, F16, pad=pad)
    table = torch.full((n, 1 << 15), -1, dtype=torch.int32, device=gpu)
    table[:, :b.mp] = i32(b.table, gpu)
    q, cache_, _, q_start, kv_lens, out = b.tensors()
    outs = []
    for max_new in (1, 0):
        b.out.fill_(3.0)
        G.paged_attn(q, cache_, gt(table), q_start, kv_lens, out, max_new=max_new)
        G.check()
        b.compare()


# ---- append and gtn_rotary_emb --------------------------------------------------------------------------
@pytest.mark.parametrize("d,rope_pct", [(64, 1.0), (64, 0.25), (64, 0.8), (64, 0.05), (128, 0.7), (128, 0.3), (128, 0.0),
                                        (64, 0.02)])
def test_append_rotates_as_rotary_emb(gpu, d, rope_pct):
    """The same rows at positions 0, 1, ... through both operators, rotated widths that are odd among them (0.8 of 64 is
    51: pairs 25 apart, exponents -2j / 51). rotary_emb forms its angle in fp32: the exponent 2j / rd is off by 2^-24 of
    itself and the power by some 2^-23, which ln(10000) < 10 and the position multiply; both cosines are then right to
    p * 12 * 2^-23 + 2^-22."""
    rows, heads, kvh = 40, 3, 1
    gen = torch.Generator(device=gpu).manual_seed(d)
    x = torch.randn(rows, heads * d, generator=gen, device=gpu)
    kv = torch.zeros(rows, kvh * d, device=gpu)
    pool = torch.zeros(3, 16 * kvh * d * 2, dtype=torch.uint8, device=gpu)
    cache = G.PagedCache(pool, pool.clone(), F16, 3, 16, kvh, d)
    out, want = torch.empty(rows, heads * d, dtype=torch.float16, device=gpu), torch.empty_like(x)
    G.rotary_emb(gt(x, F32), gt(want, F32), d, rope_pct)
    G.paged_append(gt(x, F32), gt(kv, F32), gt(kv, F32), gt(i32(range(rows), gpu)), gt(i32(range(rows), gpu)), cache, gt(out, F16),
                   rope_pct)
    G.check()
    p = torch.arange(rows, device=gpu, dtype=torch.float64)[:, None]
    mag = x.double().view(rows, heads, d).abs().amax(-1, keepdim=True).expand(-1, -1, d).reshape(rows, -1)
    err = 2 * mag * (p * 12 * 2.0 ** -23 + 2.0 ** -22)
    assert bool(((out.double() - want.double()).abs() <= err + (want.double().abs() + err) * 2.0 ** -11 + 2.0 ** -25).all())


# ---- column ranges of one buffer ------------------------------------------------------------------------
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("cache", [F16, Q8])
def test_rows_side_by_side(gpu, cache, in_place):
    """Queries, keys, values, rotated queries and outputs as columns of one buffer give what separate ones give."""
    heads, kvh, d, rows = 4, 2, 64, 37
    gen = torch.Generator(device=gpu).manual_seed(93)
    hd, kd = heads * d, kvh * d
    wide = torch.randn(rows, 3 * hd + 2 * kd, generator=gen, device=gpu).to(torch.float16)
    cuts = [0, hd, hd + kd, hd + 2 * kd, 2 * hd + 2 * kd, 3 * hd + 2 * kd]
    part = lambda w, i: gt(w[:, cuts[i]:cuts[i + 1]], F16, (rows, cuts[i + 1] - cuts[i]), (wide.shape[1], 1))  # noqa: E731
    own = [wide[:, a:b].contiguous() for a, b in zip(cuts, cuts[1:])]
    pos, lens, starts, table = i32(range(rows), gpu), i32([rows], gpu), i32([0, rows], gpu), i32([[2, 0, 1]], gpu)
    slots = i32([[2, 0, 1][t // 16] * 16 + t % 16 for t in range(rows)], gpu)
    got = []
    for q, k, v, qr, out in ([part(wide, i) for i in range(5)], [gt(x, F16) for x in own]):
        if in_place:
            qr = q
        kp, vp = (new_pool(cache, 3, 16, kvh, d, gpu) for _ in range(2))
        c = cache_of(kp, vp)
        G.paged_append(q, k, v, gt(pos), gt(slots), c, qr)
        G.paged_attn(qr, c, gt(table), gt(starts), gt(lens), out)
        G.check()
        got.append((kp.raw, vp.raw))
    for a, b in zip(*got):
        assert torch.equal(a, b)
    for i, x in enumerate(own):
        assert torch.equal(wide[:, cuts[i]:cuts[i + 1]], x), i


def test_plan_with_an_empty_free_list(gpu):
    """A server whose pages are all handed out goes on with the requests that need none."""
    t = plan(gpu, [5, 16, 31], [3, 1, 1], [], [[2, -1], [4, -1], [1, 3]], 6, 16)
    G.check()
    assert t["kv"].tolist() == [8, 0, 32] and t["used"].item() == 0 and t["q_start"].tolist() == [0, 3, 4, 5]
    assert t["slots"].tolist() == [37, 38, 39, -1, 63, -1] and t["table"].tolist() == [[2, -1], [4, -1], [1, 3]]

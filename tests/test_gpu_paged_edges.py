"""Calls of the paged serving operators that are allowed but rare: row ranges and windows at the ends of what
the arguments can say, pools past 4 GB, outputs in the queries' place, the decode kernels' own cases, and captured
calls of every kind of step. Bounds as in test_gpu_paged.py."""
import pytest
import torch

import gten_b200 as G
from paged_ref import F16, Q8, attn_bound, cache_of, gt, i32, new_pool, ref_attn, rows_of
from test_gpu_paged import Batch, generator, poison, rnd

pytestmark = pytest.mark.gpu


# ---- lengths --------------------------------------------------------------------------------------------
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 30, 161, 160, 159])
@pytest.mark.parametrize("max_new", [0, 5])
def test_window_of_the_table_and_more(gpu, window, max_new):
    """Windows around the table's length and the largest there is, with tokens before the first key."""
    b = Batch(gpu, 51, [(3, 5), (160, 5), (0, 4), (2, 3)], 4, 2, 64, 16, F16, F16)
    b.run(window=window, n_sink=1, max_new=max_new).compare(window=window, n_sink=1)
    G.check()


@pytest.mark.parametrize("max_new", [0, 1, 4])
@pytest.mark.parametrize("cache,heads,kvh", [(F16, 4, 1), (Q8, 2, 2)])
def test_row_ranges_that_overlap(gpu, cache, heads, kvh, max_new):
    """q_start that goes back and forth is an error (more rows than there are), not work without end."""
    b = Batch(gpu, 52, [(900, 60)] + [(900, 0)] * 7, heads, kvh, 64, 16, cache, F16)
    b.q_start = [0, 60] * 4 + [0]
    b.run(max_new=max_new)
    with pytest.raises(G.GtenError, match="status 5"):
        G.check()
    b = Batch(gpu, 53, [(90, 6), (40, 1)], heads, kvh, 64, 16, cache, F16)
    b.run().compare()
    G.check()


def test_rows_of_the_tensor_end_before_the_last_request(gpu):
    """A planner's refused requests keep their place in q_start: rows behind the tensor's end are not there."""
    b = Batch(gpu, 54, [(70, 33), (20, 1)], 4, 2, 64, 16, F16, F16)
    b.q_start += [60, 2 ** 31 - 1]
    b.kv_lens += [0, 0]
    b.table += [[-1] * b.mp] * 2
    for max_new in (0, 2, 40):
        b.out.fill_(9.0)
        b.run(max_new=max_new)
        got = b.out.view(-1, 4, 64).double()
        for s, n, kv, i in ((0, 33, 70, 0), (33, 1, 20, 1)):
            want, A, S = ref_attn(b.qv[s:s + n], b.keys[i], b.values[i], kv - n, 0.125, 0, 0)
            assert bool(((got[s:s + n] - want).abs() <= attn_bound(want, A, S, F16, F16)).all())
    G.check()


@pytest.mark.parametrize("n", [129, 400, 1100])
@pytest.mark.parametrize("cache", [F16, Q8])
def test_many_requests(gpu, n, cache):
    """More requests than a CTA has threads: single tokens, and some chunks between them."""
    lens = [(1 + i % 3, 1) for i in range(n)]
    b = Batch(gpu, 55, lens, 2, 2, 64, 16, cache, F16)
    b.run(max_new=1).compare()
    lens = [(1 + i % 3, 1) if i % 97 else (20, 9) for i in range(n)]
    b = Batch(gpu, 56, lens, 2, 1, 64, 16, cache, F16)
    b.run().compare()
    G.check()


def test_most_requests(gpu):
    n = 4096
    b = Batch(gpu, 57, [(i % 2, 1 if i % 64 == 1 else 0) for i in range(n)], 2, 1, 64, 16, F16, F16)
    for max_new in (1, 0):
        b.out.fill_(3.0)
        b.run(max_new=max_new).compare()
    G.check()


# ---- places ---------------------------------------------------------------------------------------------
@pytest.mark.parametrize("cache,d", [(F16, 64), (Q8, 128)])
def test_pools_past_4_gb(gpu, cache, d):
    """Page offsets beyond 32 bits (page_stride far above the page's bytes), read by every kernel."""
    extra = 64 << 20
    b = Batch(gpu, 58, [(700, 1), (300, 200), (500, 2)], 4, 2, d, 16, cache, F16, extra=extra)
    assert b.k.raw.shape[0] * extra > 6 << 30
    b.run().compare()
    b.out.fill_(3.0)
    b.run(max_new=200).compare()
    G.check()
    b = Batch(gpu, 59, [(700, 1), (500, 2)], 2, 2, d, 16, cache, F16, extra=extra)
    b.run(max_new=2).compare()
    G.check()


@pytest.mark.parametrize("cache", [F16, Q8])
def test_append_past_4_gb(gpu, cache):
    gen = generator(60, gpu)
    kp, vp = (new_pool(cache, 6, 16, 2, 64, gpu, 1 << 30, 0) for _ in range(2))
    q, k, v = (rnd(gen, 6, 128).to(torch.float16) for _ in range(3))
    out = torch.zeros_like(q)
    G.paged_append(gt(q, F16), gt(k, F16), gt(v, F16), gt(i32(range(6), gpu)), gt(i32([16 * i + 3 for i in range(6)], gpu)), cache_of(kp, vp),
                   gt(out, F16), 0.0)
    G.check()
    for i in range(6):
        for pool, x in ((kp, k), (vp, v)):
            want, got = x[i].double().view(2, 64), pool.get(i, 3)
            tol = 0.0 if cache == F16 else want.view(2, 2, 32).abs().amax(-1, keepdim=True).expand(2, 2, 32).reshape(2, 64) * (
                (1.0 / 254 + 2.0 ** -11) * (1 + 2.0 ** -10))
            assert bool(((got - want).abs() <= tol).all())


@pytest.mark.parametrize("io", [F16, Q8])
@pytest.mark.parametrize("cache", [F16, Q8])
@pytest.mark.parametrize("heads,kvh,lens,max_new", [(8, 2, [(900, 1), (500, 300), (40, 2)], 0), (8, 2, [(900, 2), (31, 1)], 2),
                                                    (3, 3, [(900, 1), (31, 1)], 1), (8, 2, [(600, 600)], 0)])
def test_output_in_the_queries_place(gpu, io, cache, heads, kvh, lens, max_new):
    b = Batch(gpu, 61, lens, heads, kvh, 64, 16, cache, io)
    b.run(max_new=max_new).compare()
    t = b.tensors()
    G.paged_attn(*t[:5], t[0], max_new=max_new)
    assert torch.equal(b.q[:b.q_start[-1]], b.out[:b.q_start[-1]])


def test_memory_of_the_host_is_refused(gpu):
    b = Batch(gpu, 62, [(40, 1)], 2, 1, 64, 16, F16, F16)
    t = b.tensors()
    host = torch.zeros(b.q.shape, dtype=torch.float16)
    for i in (0, 5):
        with pytest.raises(G.GtenError, match="not memory of the current device"):
            G.paged_attn(*t[:i], gt(host, F16), *t[i + 1:])
    with pytest.raises(G.GtenError, match="not memory of the current device"):
        G.paged_attn(*t[:2], gt(torch.zeros(1, b.mp, dtype=torch.int32)), *t[3:])
    kv = torch.zeros(1, 64, dtype=torch.float16, device=gpu)
    one = i32([0], gpu)
    for bad in (0, 1, 2):
        rows = [b.q[:1], kv, kv.clone()]
        rows[bad] = rows[bad].cpu()
        with pytest.raises(G.GtenError, match="not memory of the current device"):
            G.paged_append(*(gt(r, F16) for r in rows), gt(one), gt(one), t[1], gt(torch.empty_like(b.q[:1]), F16))
    b.run().compare()
    G.check()


# ---- the decode kernels ---------------------------------------------------------------------------------
@pytest.mark.parametrize("cache", [F16, Q8])
@pytest.mark.parametrize("heads,kvh,d,lens,max_new", [(32, 1, 64, [(300, 1), (50, 3)], 0), (24, 1, 128, [(300, 1), (50, 3)], 0),
                                                      (32, 1, 64, [(300, 1), (50, 1)], 1), (71, 1, 64, [(130, 2), (9, 1)], 2)])
def test_large_groups(gpu, cache, heads, kvh, d, lens, max_new):
    """More query heads per kv head than a decode tile has rows."""
    b = Batch(gpu, 63, lens, heads, kvh, d, 16, cache, F16)
    b.run(max_new=max_new).compare()


@pytest.mark.parametrize("io", [F16, Q8])
@pytest.mark.parametrize("d", [64, 128])
def test_single_rows_with_more_tokens_than_said(gpu, io, d):
    """max_new = 1 chooses the kernel of single rows; requests of many tokens come out right all the same."""
    b = Batch(gpu, 64, [(130, 65), (700, 1), (90, 5)], 3, 3, d, 16, Q8, io)
    b.run(max_new=1).compare()


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf"), -65504.0])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("cache", [F16, Q8])
@pytest.mark.parametrize("heads,kvh,n", [(4, 2, 1), (2, 2, 1), (2, 2, 3), (32, 2, 1)])
def test_masked_keys_in_decode_steps(gpu, value, which, cache, heads, kvh, n):
    kv, window, n_sink = 200, 60, 2
    b = Batch(gpu, 65, [(kv, n), (70, n)], heads, kvh, 64, 16, cache, F16)
    poison(b, 0, kv - n - 75, value, which)
    if n > 1:
        poison(b, 0, kv - 1, value, which)  # seen by the last row alone
    b.run(window=window, n_sink=n_sink, max_new=n)
    got = b.out.view(-1, heads, 64).double()
    want, A, S = ref_attn(b.qv[:n], b.keys[0], b.values[0], kv - n, 0.125, window, n_sink)
    rows = n - 1 if n > 1 else n
    assert bool(((got[:rows] - want[:rows]).abs() <= attn_bound(want, A, S, cache, F16)[:rows]).all())
    if n > 1 and (which == "v" and value != -65504.0 or which == "k" and value != value):
        assert not bool(torch.isfinite(got[n - 1]).any())
    want, A, S = ref_attn(b.qv[n:2 * n], b.keys[1], b.values[1], 70 - n, 0.125, window, n_sink)
    assert bool(((got[n:2 * n] - want).abs() <= attn_bound(want, A, S, cache, F16)).all())


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("cache", [F16, Q8])
@pytest.mark.parametrize("heads,kvh,n,max_new", [(2, 2, 1, 1), (4, 2, 1, 1), (4, 2, 70, 0)])
def test_queries_that_are_not_finite(gpu, value, cache, heads, kvh, n, max_new):
    """They spoil their own row and no other."""
    b = Batch(gpu, 66, [(90, n), (50, n if n == 1 else 40)], heads, kvh, 64, 16, cache, F16)
    b.q[0, 5] = value       # head 0 of the first row
    b.run(max_new=max_new)
    got = b.out.view(-1, heads, 64).double()
    assert not bool(torch.isfinite(got[0, 0]).any())
    for i, s in ((0, 0), (1, n)):
        m = b.new[i]
        want, A, S = ref_attn(b.qv[s:s + m], b.keys[i], b.values[i], b.kv_lens[i] - m, 0.125, 0, 0)
        ok = (got[s:s + m] - want).abs() <= attn_bound(want, A, S, cache, F16)
        if i == 0:
            ok[0, 0] = True
        assert bool(ok.all())


# ---- captured -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("cache,io", [(F16, F16), (Q8, Q8)])
def test_captured_mixed_steps_follow_the_lengths(gpu, cache, io):
    """One captured call without a bound on the new tokens, replayed for steps of single tokens, of chunks and of
    both, as the lengths on the device say."""
    heads, kvh, d, ps = 8, 2, 64, 16
    steps = [[(700, 1), (600, 1), (300, 1)], [(700, 1), (600, 250), (300, 1)], [(0, 0), (600, 300), (300, 100)],
             [(700, 1), (0, 0), (0, 0)], [(400, 400), (3, 3), (0, 0)]]
    kept = []
    for i, lens in enumerate(steps):
        pad = 420 - sum(n for _, n in lens)
        kept.append(Batch(gpu, 70 + i, lens, heads, kvh, d, ps, cache, io, pad=pad, more_cols=44 - max(-(-kv // ps) for kv, _ in lens)))
    pages = max(b.k.raw.shape[0] for b in kept)
    live = Batch(gpu, 80, [(16 * (pages // 3), 140)] * 3, heads, kvh, d, ps, cache, io)
    assert live.k.raw.shape[0] >= pages
    bufs = [i32([[0] * 44] * 3, gpu), i32([0] * 4, gpu), i32([0] * 3, gpu)]
    lt = live.tensors()
    t = (lt[0], lt[1], gt(bufs[0]), gt(bufs[1]), gt(bufs[2]), lt[5])
    ws = torch.empty(G.paged_attn_workspace(heads, d), dtype=torch.uint8, device=gpu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        G.paged_attn(*t, workspace=ws)
    for b in kept + kept[::-1]:
        for pool, src in ((live.k, b.k), (live.v, b.v)):
            pool.raw[:src.raw.shape[0]].copy_(src.raw)
        live.q.copy_(b.q)
        live.out.copy_(rows_of(io, torch.full((b.rows, heads * d), 3.0, device=gpu, dtype=torch.float64)))
        for dst, src in zip(bufs, (b.table, b.q_start, b.kv_lens)):
            dst.copy_(i32(src, gpu))
        graph.replay()
        b.out.copy_(live.out)
        b.compare()
    G.check()

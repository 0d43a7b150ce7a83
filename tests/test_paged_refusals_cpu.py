"""Refusals of the paged serving operators by their own messages: a base call that passes every check of its
arguments, and one change at a time. Without a GPU the base call ends at the first question to the device; the
pointers are never touched."""
import pytest

import gten_b200 as G

MB = 1 << 20
AT = [(i + 1) << 40 for i in range(16)]  # buffers that lie apart


def t(at, *shape, dtype=G.I32, strides=None):
    return G.GT(at, dtype, shape, strides)


def plan_args(**kw):
    a = dict(ctx_lens=t(AT[0], 3), new_lens=t(AT[1], 3), free_pages=t(AT[2], 9), n_free=t(AT[3], 1), page_size=16,
             block_table=t(AT[4], 3, 4), q_start=t(AT[5], 4), kv_lens=t(AT[6], 3), pos=t(AT[7], 7), slots=t(AT[8], 7),
             n_used=t(AT[9], 1), stream=0)
    a.update(kw)
    return a


def refusal(call, args):
    with pytest.raises(G.GtenError) as e:
        call(**args)
    return str(e.value)


#: what the base calls meet behind the checks of their arguments: no device, or one that does not own the pointers
PASSED = ("no CUDA-capable device", "driver version is insufficient", "not memory of the current device", "invalid argument",
          "error word", "initialization error")


def passed(msg):
    return any(p in msg for p in PASSED)


def test_plan_base_call_passes_the_checks():
    assert passed(refusal(G.paged_plan, plan_args()))


@pytest.mark.parametrize("page_size,max_pages", [(16, 1 << 26), (256, 1 << 22), (16, 2 ** 31 - 1), (64, 1 << 25)])
def test_plan_refuses_tables_of_2_30_keys(page_size, max_pages):
    """Lengths that such a row could hold would not fit 32 bits beside the new tokens."""
    msg = refusal(G.paged_plan, plan_args(page_size=page_size, block_table=t(AT[4], 3, max_pages)))
    assert "status 1" in msg and "block_table of" in msg


def test_plan_takes_tables_just_below_2_30_keys():
    assert passed(refusal(G.paged_plan, plan_args(block_table=t(AT[4], 3, (1 << 26) - 1))))


def attn_args(n=3, rows=5, heads=4, max_pages=4, page_size=16, kvh=2, dtype=G.F16, **kw):
    a = dict(q=t(AT[0], rows, heads * 64, dtype=G.F16), cache=G.PagedCache(AT[1], AT[2], dtype, 8, page_size, kvh, 64),
             block_table=t(AT[3], n, max_pages), q_start=t(AT[4], n + 1), kv_lens=t(AT[5], n),
             out=t(AT[6], rows, heads * 64, dtype=G.F16), workspace=Ws(AT[8], 64 * MB), stream=0)
    a.update(kw)
    return a


class Ws:
    def __init__(self, at, n):
        self.at, self.n = at, n

    def data_ptr(self):
        return self.at

    def numel(self):
        return self.n


def test_attn_base_call_passes_the_checks():
    assert passed(refusal(G.paged_attn, attn_args()))


#: calls whose tiles of 16 rows fit 32 bits of units and whose single rows do not
WIDE = [dict(n=1024, rows=1024, heads=64, kvh=8, max_pages=1 << 15),               # 8 query heads per kv head, 2^19 keys
        dict(n=1024, rows=1024, heads=128, kvh=8, max_pages=1 << 15),
        dict(n=1024, rows=4096, heads=36, kvh=36, max_pages=1 << 15, dtype=G.Q8),  # many more rows than requests
        dict(n=2, rows=1 << 20, heads=16, kvh=16, max_pages=1 << 13)]


@pytest.mark.parametrize("wide", WIDE, ids=str)
@pytest.mark.parametrize("max_new", [0, 1, 2, 8, 16, 17, 2 ** 31 - 1])
def test_attn_takes_with_a_bound_what_it_takes_without(wide, max_new):
    """max_new chooses the kernels, not whether a call is taken."""
    assert passed(refusal(G.paged_attn, attn_args(max_new=max_new, **wide)))


@pytest.mark.parametrize("max_new", [0, 1, 5])
def test_attn_refuses_units_beyond_32_bits(max_new):
    msg = refusal(G.paged_attn, attn_args(n=4096, rows=4096, heads=8, kvh=8, max_pages=1 << 16, max_new=max_new))
    assert "status 1" in msg and "too many for one call" in msg


def append_args(**kw):
    a = dict(q=t(AT[0], 5, 256, dtype=G.F16), k=t(AT[1], 5, 128, dtype=G.F16), v=t(AT[2], 5, 128, dtype=G.F16), pos=t(AT[3], 5),
             slots=t(AT[4], 5), cache=G.PagedCache(AT[5], AT[6], G.F16, 8, 16, 2, 64), q_out=t(AT[7], 5, 256, dtype=G.F16), stream=0)
    a.update(kw)
    return a


def test_append_base_call_passes_the_checks():
    assert passed(refusal(G.paged_append, append_args()))


INTS = [(G.paged_plan, plan_args, n) for n in ("ctx_lens", "new_lens", "free_pages", "n_free", "block_table", "q_start", "kv_lens",
                                               "pos", "slots", "n_used")]
INTS += [(G.paged_append, append_args, n) for n in ("pos", "slots")]
INTS += [(G.paged_attn, attn_args, n) for n in ("block_table", "q_start", "kv_lens")]


@pytest.mark.parametrize("off", [1, 2, 3])
@pytest.mark.parametrize("call,args,name", INTS, ids=lambda x: x if isinstance(x, str) else "")
def test_int_tensors_are_aligned(call, args, name, off):
    """A 4-byte load from another address faults."""
    a = args()
    a[name].buf += off
    msg = refusal(call, a)
    assert "status 1" in msg and f"{name} must be 4-byte aligned" in msg


# ---- overlaps -------------------------------------------------------------------------------------------
def f16(at, rows, cols, stride=None):
    return t(at, rows, cols, dtype=G.F16, strides=(stride, 1) if stride else None)


def pools(k=AT[5], v=AT[6], stride=0, n_pages=8):
    return G.PagedCache(k, v, G.F16, n_pages, 16, 2, 64, stride)  # pages of 4,096 bytes


@pytest.mark.parametrize("bad,what", [
    (dict(pos=t(AT[7] + 8, 5)), "q_out overlaps pos or slots"), (dict(slots=t(AT[7] + 2556, 5)), "q_out overlaps pos or slots"),
    (dict(cache=pools(AT[7])), "q_out overlaps the cache"), (dict(cache=pools(v=AT[7] - 7 * 4096)), "q_out overlaps the cache"),
    (dict(cache=pools(v=AT[5])), "pools of the cache overlap"), (dict(cache=pools(v=AT[5] + 7 * 4096)), "pools of the cache overlap"),
    (dict(cache=pools(v=AT[5] + 4080, stride=8192)), "pools of the cache overlap"),
    (dict(cache=pools(AT[0])), "cache overlaps an input"), (dict(cache=pools(v=AT[2] + 1264)), "cache overlaps an input"),
    (dict(pos=t(AT[6] + 8 * 4096 - 4, 5)), "cache overlaps an input"), (dict(slots=t(AT[5], 5)), "cache overlaps an input"),
    # in the queries' place, with keys or values that share rows with them
    (dict(q_out=f16(AT[0], 5, 256), k=f16(AT[0] + 256, 5, 128)), "q_out overlaps k or v"),
    (dict(q_out=f16(AT[0], 5, 256), v=f16(AT[0], 5, 128, 256)), "q_out overlaps k or v"),
    (dict(q=f16(AT[0], 5, 256, 512), q_out=f16(AT[0], 5, 256, 512), k=f16(AT[0] + 500, 5, 128, 512)), "q_out overlaps k or v"),
    (dict(q=f16(AT[0], 5, 256, 512), q_out=f16(AT[0], 5, 256, 512), k=f16(AT[0] + 512, 5, 128, 384)), "q_out overlaps k or v")],
    ids=str)
def test_append_refuses_overlaps(bad, what):
    msg = refusal(G.paged_append, append_args(**bad))
    assert "status 1" in msg and what in msg


@pytest.mark.parametrize("good", [
    dict(k=f16(AT[1], 5, 128), v=f16(AT[1], 5, 128)),                                     # read twice
    dict(cache=pools(v=AT[5] + 4096, stride=8192)),                                       # K and V pages in turns
    dict(cache=pools(v=AT[5] + 8192, stride=3 * 4096)), dict(cache=pools(n_pages=1, v=AT[5] + 4096)),
    dict(q_out=f16(AT[0], 5, 256)),                                                       # in the queries' place
    # column ranges of one buffer of 1,024 elements a row
    dict(q=f16(AT[0], 5, 256, 1024), k=f16(AT[0] + 512, 5, 128, 1024), v=f16(AT[0] + 768, 5, 128, 1024),
         q_out=f16(AT[0], 5, 256, 1024)),
    dict(q=f16(AT[0], 5, 256, 1024), k=f16(AT[0] + 512, 5, 128, 1024), v=f16(AT[0] + 768, 5, 128, 1024),
         q_out=f16(AT[0] + 1024, 5, 256, 1024)),
    dict(q=f16(AT[0] + 1024, 5, 256, 1024), q_out=f16(AT[0] + 512, 5, 256, 1024)),
    dict(q=f16(AT[0], 1, 256), k=f16(AT[0] + 512, 1, 128), v=f16(AT[0] + 768, 1, 128), q_out=f16(AT[0], 1, 256), pos=t(AT[3], 1),
         slots=t(AT[4], 1))], ids=str)
def test_append_takes_neighbours(good):
    assert passed(refusal(G.paged_append, append_args(**good)))


@pytest.mark.parametrize("bad,what", [
    (dict(block_table=t(AT[6] + 2556, 3, 4)), "out overlaps the lengths or the table"),
    (dict(q_start=t(AT[6], 4)), "out overlaps the lengths or the table"), (dict(kv_lens=t(AT[6] - 8, 3)), "out overlaps the lengths"),
    (dict(cache=pools(AT[6])), "out overlaps the cache"), (dict(cache=pools(v=AT[6] - 16)), "out overlaps the cache"),
    (dict(workspace=Ws(AT[6] + 16, 64 * MB)), "out overlaps workspace"),
    (dict(workspace=Ws(AT[0] - 64, 64 * MB)), "workspace overlaps q"),
    (dict(workspace=Ws(AT[3], 64 * MB)), "workspace overlaps the lengths or the table"),
    (dict(workspace=Ws(AT[4] - 1024, 64 * MB)), "workspace overlaps the lengths or the table"),
    (dict(workspace=Ws(AT[5] - 1024, 64 * MB)), "workspace overlaps the lengths or the table"),
    (dict(workspace=Ws(AT[1] + 4096, 64 * MB)), "workspace overlaps the cache"),
    (dict(workspace=Ws(AT[2] - 1024, 64 * MB)), "workspace overlaps the cache")], ids=str)
def test_attn_refuses_overlaps(bad, what):
    msg = refusal(G.paged_attn, attn_args(**bad))
    assert "status 1" in msg and what in msg


@pytest.mark.parametrize("good", [
    dict(out=f16(AT[0], 5, 256)), dict(q=f16(AT[0], 5, 256, 640), out=f16(AT[0] + 512, 5, 256, 640)),
    dict(q=f16(AT[0] + 1000 * 1280, 5, 256, 640), out=f16(AT[0] + 640, 5, 256, 640)),
    dict(cache=pools(AT[1], AT[1])), dict(cache=pools(AT[1], AT[1] + 4096, stride=8192)),
    dict(q=f16(AT[0], 1, 256), out=f16(AT[0] + 512, 1, 256))], ids=str)
def test_attn_takes_neighbours(good):
    assert passed(refusal(G.paged_attn, attn_args(**good)))


# ---- the device -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("call,args", [(G.paged_plan, plan_args), (G.paged_append, append_args), (G.paged_attn, attn_args)],
                         ids=["plan", "append", "attn"])
def test_without_an_error_word_nothing_is_launched(call, args):
    """The kernels write the device's error word without asking whether there is one."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("there is one")
    for _ in range(2):
        msg = refusal(call, args())
        assert "status 2" in msg and "no error word" in msg


def test_plan_takes_an_empty_free_list():
    assert passed(refusal(G.paged_plan, plan_args(free_pages=t(0, 0))))
    assert passed(refusal(G.paged_plan, plan_args(free_pages=t(AT[2], 0))))
    for bad in (t(0, 9), t(0, 0, dtype=G.F32), t(0, 0, 1), t(AT[2], -1)):
        assert "status 1" in refusal(G.paged_plan, plan_args(free_pages=bad))


# ---- every check of an argument by its own message -------------------------------------------------------
def check_refusal(call, args, bad, what):
    msg = refusal(call, args(**bad))
    assert "status 1" in msg and what in msg, msg


CACHE = dict(k=AT[11], v=AT[12], dtype=G.F16, n_pages=8, page_size=16, kv_heads=2, d_head=64, page_stride=0)


@pytest.mark.parametrize("call,args", [(G.paged_attn, attn_args), (G.paged_append, append_args)], ids=["attn", "append"])
@pytest.mark.parametrize("bad,what", [
    (dict(dtype=G.F32), "cache dtype 2"), (dict(dtype=G.Q4), "cache dtype 4"), (dict(dtype=G.I32), "cache dtype 0"),
    (dict(page_size=8), "page_size 8"), (dict(page_size=24), "page_size 24"), (dict(page_size=512), "page_size 512"),
    (dict(page_size=-16), "page_size -16"), (dict(d_head=96), "d_head 96"), (dict(d_head=0), "d_head 0"),
    (dict(kv_heads=0), "kv_heads 0"), (dict(kv_heads=1025), "kv_heads 1025"), (dict(n_pages=0), "n_pages 0"),
    (dict(n_pages=1 << 27), "n_pages 134217728"), (dict(k=0), "cache has no data"), (dict(v=0), "cache has no data"),
    (dict(k=AT[11] + 8), "pools must be 16-byte aligned"), (dict(v=AT[12] + 8), "pools must be 16-byte aligned"),
    (dict(page_stride=4080), "page_stride 4080"), (dict(page_stride=4104), "page_stride 4104"),
    (dict(page_stride=-16), "page_stride -16"), (dict(page_stride=1 << 31), "page_stride 2147483648")], ids=str)
def test_cache_messages(call, args, bad, what):
    assert passed(refusal(call, args(cache=G.PagedCache(**CACHE))))
    check_refusal(call, args, dict(cache=G.PagedCache(**{**CACHE, **bad})), what)


def x(name, *shape, **kw):
    """The attention call's tensor of that name in another shape."""
    at = {"q": AT[0], "out": AT[6], "block_table": AT[3], "q_start": AT[4], "kv_lens": AT[5]}[name]
    dtype = kw.pop("dtype", G.F16 if name in ("q", "out") else G.I32)
    return {name: t(at + kw.pop("off", 0), *shape, dtype=dtype, **kw)}


@pytest.mark.parametrize("bad,what", [
    ({**x("q", 5, 256, dtype=G.F32), **x("out", 5, 256, dtype=G.F32)}, "dtypes 2, 2"), (x("out", 5, 256, dtype=G.Q8), "dtypes 1, 3"),
    (x("out", 4, 256), "of one shape"), (x("out", 5, 128), "of one shape"), (x("q", 1280), "2-D, of one shape"),
    ({**x("q", 5, 96), **x("out", 5, 96)}, "q of 96 columns"), ({**x("q", 5, 192), **x("out", 5, 192)}, "heads 3 not a multiple"),
    (x("q", 5, 256, off=2), "16-byte aligned"), (x("q", 5, 256, strides=(260, 1)), "16-byte aligned"),
    (x("out", 5, 256, off=8), "16-byte aligned"), (x("q", 5, 256, strides=(128, 1)), "row strides"),
    (x("q", 5, 256, strides=(512, 2)), "row strides"), (x("out", 5, 256, strides=(248, 1)), "row strides"),
    ({**x("q", 5, 256, dtype=G.Q8, off=1), **x("out", 5, 256, dtype=G.Q8)}, "Q8 row alignment"),
    ({**x("q", 5, 256, dtype=G.Q8, strides=(260, 1)), **x("out", 5, 256, dtype=G.Q8)}, "Q8 row alignment"),
    (dict(q=t(0, 5, 256, dtype=G.F16)), "q has no data"), (dict(out=t(0, 5, 256, dtype=G.F16)), "out has no data"),
    (x("q", 0, 256), "q dim 0 is 0"), (x("block_table", 2, 4), "do not agree on 3 requests"),
    (x("block_table", 12), "block_table must be int32, 2-D"), (x("block_table", 3, 4, dtype=G.F32), "block_table must be int32"),
    (x("block_table", 3, 4, strides=(2, 1)), "block_table rows overlap"),
    (x("block_table", 3, 4, strides=(8, 2)), "block_table must be contiguous"), (x("block_table", 3, 1 << 26), "block_table of 67108864"),
    (x("q_start", 3), "do not agree"), (x("q_start", 4, dtype=G.F32), "q_start must be int32"),
    (x("q_start", 4, strides=(2,)), "q_start must be contiguous"), (x("kv_lens", 2), "do not agree on 2"),
    (x("kv_lens", 3, strides=(2,)), "kv_lens must be contiguous"), (x("kv_lens", 3, 1), "kv_lens must be int32, 1-D"),
    (dict(window=-1), "window -1"), (dict(n_sink=-1), "n_sink -1"), (dict(max_new=-1), "max_new"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(workspace=Ws(AT[8], 8)), "workspace of 8 bytes"),
    (dict(workspace=Ws(0, 64 * MB)), "workspace must be"), (dict(workspace=Ws(AT[8] + 4, 64 * MB)), "workspace must be 16-byte"),
    ({**x("block_table", 4097, 4), **x("q_start", 4098), **x("kv_lens", 4097)}, "4097 requests (at most 4096)"),
    ({**x("q", (1 << 20) + 1, 256), **x("out", (1 << 20) + 1, 256)}, "1048577 rows of 4 heads")], ids=str)
def test_attn_messages(bad, what):
    check_refusal(G.paged_attn, attn_args, bad, what)


def y(name, *shape, **kw):
    """The append call's tensor of that name in another shape."""
    at = dict(q=AT[0], k=AT[1], v=AT[2], pos=AT[3], slots=AT[4], q_out=AT[7])[name]
    dtype = kw.pop("dtype", G.I32 if name in ("pos", "slots") else G.F16)
    return {name: t(at + kw.pop("off", 0), *shape, dtype=dtype, **kw)}


@pytest.mark.parametrize("bad,what", [
    (y("k", 5, 128, dtype=G.F32), "dtypes differ"), (y("v", 5, 128, dtype=G.Q8), "dtypes differ"),
    ({**y("q", 5, 256, dtype=G.Q4), **y("k", 5, 128, dtype=G.Q4), **y("v", 5, 128, dtype=G.Q4)}, "q dtype 4"),
    (y("k", 4, 128), "k / v must be [5, 128]"), (y("v", 5, 64), "k / v must be [5, 128]"), (y("q", 5, 100), "q of 100 columns"),
    (y("q", 5), "2-D rows"), (y("q_out", 5, 256, dtype=G.F32), "q_out dtype 2"), (y("q_out", 5, 128), "q_out shape"),
    (y("q_out", 4, 256), "q_out shape"), (y("pos", 4), "must have 5 entries"), (y("slots", 6), "must have 5 entries"),
    (y("slots", 5, dtype=G.F32), "slots must be int32"), (y("pos", 5, 1), "pos must be int32, 1-D"),
    (y("q", 5, 256, strides=(100, 1)), "row strides"), (y("k", 5, 128, strides=(256, 2)), "row strides"),
    (y("q_out", 5, 256, strides=(255, 1)), "row strides"), (y("q", 5, 256, off=1), "row alignment"),
    (y("q_out", 5, 256, off=1), "row alignment"),
    ({**y("q", 5, 256, dtype=G.F32, off=2), **y("k", 5, 128, dtype=G.F32), **y("v", 5, 128, dtype=G.F32)}, "row alignment"),
    ({**y("q", 5, 256, dtype=G.Q8, strides=(272, 1)), **y("k", 5, 128, dtype=G.Q8), **y("v", 5, 128, dtype=G.Q8)}, "Q8 row stride 272"),
    (dict(q_out=t(AT[0] + 64, 5, 256, dtype=G.F16)), "q_out overlaps an input"),
    (dict(q_out=t(AT[0], 5, 256, dtype=G.Q8)), "q_out overlaps an input"), (dict(rope_pct=1.5), "rope_pct"),
    (dict(rope_pct=-0.1), "rope_pct"), (dict(rope_pct=float("nan")), "rope_pct"), (dict(rope_base=0.0), "rope_base"),
    (dict(rope_base=float("inf")), "rope_base"), (dict(rope_base=-1.0), "rope_base"), (dict(rope_base=float("nan")), "rope_base")],
    ids=str)
def test_append_messages(bad, what):
    check_refusal(G.paged_append, append_args, bad, what)


def z(name, *shape, **kw):
    """The planner call's tensor of that name in another shape."""
    names = ["ctx_lens", "new_lens", "free_pages", "n_free", "block_table", "q_start", "kv_lens", "pos", "slots", "n_used"]
    return {name: t(AT[names.index(name)], *shape, **kw)}


@pytest.mark.parametrize("bad,what", [
    (dict(page_size=0), "page_size 0"), (dict(page_size=8), "page_size 8"), (dict(page_size=48), "page_size 48"),
    (dict(page_size=512), "page_size 512"), (z("new_lens", 4), "do not agree on 3 requests"), (z("kv_lens", 4), "do not agree"),
    (z("q_start", 3), "do not agree"), (z("block_table", 4, 4), "do not agree"), (z("ctx_lens", 2), "do not agree on 2"),
    (z("block_table", 3, 4, strides=(3, 1)), "block_table rows overlap"), (z("block_table", 12), "block_table must be int32, 2-D"),
    (z("slots", 6), "pos and slots differ"), (z("pos", 8), "pos and slots differ"), (z("ctx_lens", 3, dtype=G.F32), "ctx_lens must be int32"),
    (z("free_pages", 9, 1), "free_pages must be int32, 1-D"), (z("n_used", 1, dtype=G.F16), "n_used must be int32"),
    (z("pos", 7, strides=(2,)), "pos must be contiguous"), (dict(n_used=t(0, 1)), "n_used has no data"),
    (dict(n_free=t(0, 1)), "n_free has no data"),
    ({**z("ctx_lens", 5000), **z("new_lens", 5000), **z("kv_lens", 5000), **z("q_start", 5001), **z("block_table", 5000, 4)},
     "5000 requests (at most 4096)"), (dict(slots=t(AT[7] + 24, 7)), "tensors that are written overlap others")], ids=str)
def test_plan_messages(bad, what):
    check_refusal(G.paged_plan, plan_args, bad, what)

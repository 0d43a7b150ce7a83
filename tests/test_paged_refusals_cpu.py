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

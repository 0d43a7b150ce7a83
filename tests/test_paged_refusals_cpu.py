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

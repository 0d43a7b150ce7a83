"""Refusals of the paged serving operators by their own messages: a base call that passes every check of its
arguments, and one change at a time. Without a GPU the base call ends at the first question to the device; the
pointers are never touched."""
import pytest

import gten_b200 as G

MB = 1 << 20
AT = [(64 + 64 * i) * MB for i in range(16)]  # buffers that lie apart


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
    msg = refusal(G.paged_plan, plan_args(page_size=page_size, block_table=t(1 << 40, 3, max_pages)))
    assert "status 1" in msg and "block_table of" in msg


def test_plan_takes_tables_just_below_2_30_keys():
    assert passed(refusal(G.paged_plan, plan_args(block_table=t(1 << 40, 3, (1 << 26) - 1))))

"""Refusals of the paged serving operators: every check of arguments runs before any device work, so
these need no GPU (the pointers are never touched); and the plain planner of the tests against small
cases worked out by hand."""
import pytest

import gten_b200 as G
from paged_ref import ref_plan

P = 1 << 20  # a 16-byte aligned address that nothing reads


def cache(**kw):
    a = dict(k=P, v=P, dtype=G.F16, n_pages=8, page_size=16, kv_heads=2, d_head=64, page_stride=0)
    a.update(kw)
    return G.PagedCache(**a)


def t(dtype, *shape, buf=P, strides=None):
    return G.GT(buf, dtype, shape, strides)


class Ws:
    def __init__(self, n=1 << 40, p=P):
        self.n, self.p = n, p

    def data_ptr(self):
        return self.p

    def numel(self):
        return self.n


def attn(**kw):
    a = dict(q=t(G.F16, 5, 256), cache=cache(), block_table=t(G.I32, 3, 4), q_start=t(G.I32, 4), kv_lens=t(G.I32, 3),
             out=t(G.F16, 5, 256), workspace=Ws(), stream=0)
    a.update(kw)
    G.paged_attn(**a)


def append(**kw):
    a = dict(q=t(G.F16, 5, 256), k=t(G.F16, 5, 128), v=t(G.F16, 5, 128), pos=t(G.I32, 5), slots=t(G.I32, 5), cache=cache(),
             q_out=t(G.F16, 5, 256, buf=P + 65536), stream=0)
    a.update(kw)
    G.paged_append(**a)


def plan(**kw):
    a = dict(ctx_lens=t(G.I32, 3), new_lens=t(G.I32, 3), free_pages=t(G.I32, 9), n_free=t(G.I32, 1), page_size=16,
             block_table=t(G.I32, 3, 4), q_start=t(G.I32, 4), kv_lens=t(G.I32, 3), pos=t(G.I32, 7), slots=t(G.I32, 7),
             n_used=t(G.I32, 1), stream=0)
    a.update(kw)
    G.paged_plan(**a)


BAD_CACHE = [dict(dtype=G.F32), dict(dtype=G.Q4), dict(page_size=8), dict(page_size=24), dict(page_size=512),
             dict(d_head=96), dict(d_head=0), dict(kv_heads=0), dict(n_pages=0), dict(n_pages=1 << 27), dict(k=0),
             dict(v=P + 8), dict(page_stride=4000), dict(page_stride=4096 + 8), dict(page_stride=-16)]


@pytest.mark.parametrize("call", [attn, append])
@pytest.mark.parametrize("bad", BAD_CACHE, ids=str)
def test_cache_descriptors(call, bad):
    with pytest.raises(G.GtenError, match="status 1"):
        call(cache=cache(**bad))


@pytest.mark.parametrize("bad", [
    dict(q=t(G.F32, 5, 256), out=t(G.F32, 5, 256)), dict(out=t(G.Q8, 5, 256)), dict(out=t(G.F16, 4, 256)),
    dict(q=t(G.F16, 5, 96), out=t(G.F16, 5, 96)), dict(q=t(G.F16, 5, 192), out=t(G.F16, 5, 192)),
    dict(q=t(G.F16, 5, 256, buf=P + 2)), dict(q=t(G.F16, 5, 256, strides=(260, 1))), dict(q=t(G.F16, 5, 256, strides=(128, 1))),
    dict(q=t(G.F16, 5, 256, strides=(512, 2))), dict(q=t(G.Q8, 5, 256, buf=P + 1), out=t(G.Q8, 5, 256)),
    dict(q=t(G.Q8, 5, 256, strides=(260, 1)), out=t(G.Q8, 5, 256)), dict(q=t(G.F16, 1280)), dict(q=t(G.F16, 5, 256, buf=0)),
    dict(block_table=t(G.I32, 2, 4)), dict(block_table=t(G.I32, 12)), dict(block_table=t(G.I32, 3, 4, strides=(2, 1))),
    dict(block_table=t(G.I32, 3, 1 << 28)), dict(q_start=t(G.I32, 3)), dict(q_start=t(G.F32, 4)),
    dict(kv_lens=t(G.I32, 2)), dict(kv_lens=t(G.I32, 3, strides=(2,))), dict(window=-1), dict(n_sink=-1), dict(max_new=-1),
    dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(workspace=Ws(8)), dict(workspace=Ws(p=0)),
    dict(workspace=Ws(p=P + 4)),
    dict(block_table=t(G.I32, 4097, 4), q_start=t(G.I32, 4098), kv_lens=t(G.I32, 4097))], ids=str)
def test_attn_arguments(bad):
    with pytest.raises(G.GtenError, match="status 1"):
        attn(**bad)


@pytest.mark.parametrize("bad", [
    dict(q=t(G.Q4, 5, 256)), dict(k=t(G.F32, 5, 128)), dict(k=t(G.F16, 4, 128)), dict(v=t(G.F16, 5, 64)),
    dict(q_out=t(G.F32, 5, 256, buf=P + 65536)), dict(q_out=t(G.F16, 5, 128, buf=P + 65536)),
    dict(q_out=t(G.F16, 5, 256, buf=P + 64)), dict(q_out=t(G.Q8, 5, 256)), dict(q=t(G.F16, 5, 100)),
    dict(pos=t(G.I32, 4)), dict(slots=t(G.F32, 5)), dict(q=t(G.F16, 5, 256, strides=(100, 1))),
    dict(q=t(G.F16, 5, 256, buf=P + 1)), dict(k=t(G.F16, 5, 128, strides=(256, 2))), dict(rope_pct=1.5), dict(rope_pct=-0.1),
    dict(rope_base=0.0), dict(rope_base=float("inf")), dict(rope_pct=float("nan"))], ids=str)
def test_append_arguments(bad):
    with pytest.raises(G.GtenError, match="status 1"):
        append(**bad)


@pytest.mark.parametrize("bad", [
    dict(page_size=0), dict(page_size=48), dict(page_size=512), dict(new_lens=t(G.I32, 4)), dict(kv_lens=t(G.I32, 4)),
    dict(q_start=t(G.I32, 3)), dict(block_table=t(G.I32, 4, 4)), dict(block_table=t(G.I32, 3, 4, strides=(3, 1))),
    dict(slots=t(G.I32, 6)), dict(ctx_lens=t(G.F32, 3)), dict(n_used=t(G.I32, 1, buf=0)), dict(free_pages=t(G.I32, 9, 1)),
    dict(ctx_lens=t(G.I32, 5000), new_lens=t(G.I32, 5000), kv_lens=t(G.I32, 5000), q_start=t(G.I32, 5001),
         block_table=t(G.I32, 5000, 4))], ids=str)
def test_plan_arguments(bad):
    with pytest.raises(G.GtenError, match="status 1"):
        plan(**bad)


def test_page_bytes():
    assert G.PagedCache.page_bytes(G.F16, 16, 4, 64) == 16 * 4 * 64 * 2
    assert G.PagedCache.page_bytes(G.Q8, 32, 36, 64) == 32 * 36 * 2 * 34
    with pytest.raises(G.GtenError):
        G.PagedCache.page_bytes(G.Q8, 20, 4, 64)


def test_reference_planner_by_hand():
    # request 0 has 3 of 4 rows of its page and takes 2 more tokens: one new page; request 1 starts: two;
    # request 2 would need one more than is free; request 3 needs none
    table, q_start, kv, pos, slots, used = ref_plan([3, 0, 4, 1], [2, 5, 1, 1], [10, 11, 12], 3, 4,
                                                    [[7, -1], [-1, -1], [8, -1], [9, -1]], 10)
    assert table == [[7, 10], [11, 12], [8, -1], [9, -1]]
    assert q_start == [0, 2, 7, 8, 9] and kv == [5, 5, 0, 2] and used == 3
    assert pos == [3, 4, 0, 1, 2, 3, 4, 4, 1, -1]
    assert slots == [31, 40, 44, 45, 46, 47, 48, -1, 37, -1]


FAR = [P + (i << 20) for i in range(12)]


def far_plan(**kw):
    """A plan whose tensors lie apart."""
    names = dict(ctx_lens=(3,), new_lens=(3,), free_pages=(9,), n_free=(1,), block_table=(3, 4), q_start=(4,), kv_lens=(3,),
                 pos=(7,), slots=(7,), n_used=(1,))
    a = {n: t(G.I32, *shape, buf=at) for (n, shape), at in zip(names.items(), FAR)}
    a.update({n: t(G.I32, *names[n], buf=FAR[list(names).index(o)] + 4 * at) for n, (o, at) in kw.items()})
    G.paged_plan(page_size=16, stream=0, **a)


@pytest.mark.parametrize("bad", [dict(kv_lens=("ctx_lens", 0)), dict(n_used=("n_free", 0)), dict(slots=("pos", 6)),
                                 dict(q_start=("new_lens", 2)), dict(block_table=("free_pages", 8)),
                                 dict(ctx_lens=("block_table", 11)), dict(pos=("kv_lens", 1))], ids=str)
def test_plan_outputs_lie_apart(bad):
    with pytest.raises(G.GtenError, match="overlap"):
        far_plan(**bad)


@pytest.mark.parametrize("bad", [
    dict(out=t(G.F16, 5, 256, buf=P + 512)), dict(out=t(G.F16, 5, 256, strides=(512, 1))),
    dict(q=t(G.F16, 5, 256, buf=P + 5 * 512 - 16)), dict(q=t(G.Q8, 5, 256, buf=P + 34), out=t(G.Q8, 5, 256))], ids=str)
def test_attn_output_lies_apart(bad):
    with pytest.raises(G.GtenError, match="overlap"):
        attn(**bad)


@pytest.mark.parametrize("bad", [dict(k=t(G.F16, 5, 128, buf=P + 65536 + 64)), dict(v=t(G.F16, 5, 128, buf=P + 65536 + 2304)),
                                 dict(k=t(G.F16, 5, 128, buf=P + 65536, strides=(256, 1)))], ids=str)
def test_append_output_lies_apart(bad):
    with pytest.raises(G.GtenError, match="status 1.*q_out"):
        append(**bad)


@pytest.mark.parametrize("bad", [
    dict(cache=cache(page_stride=1 << 31)), dict(cache=cache(page_stride=(1 << 40) + 16)),
    dict(q=t(G.F16, (1 << 20) + 1, 256), out=t(G.F16, (1 << 20) + 1, 256)),
    dict(block_table=t(G.I32, 3, 1 << 26)),                                                     # 2^30 keys a row
    dict(cache=cache(kv_heads=1024), q=t(G.F16, 1 << 20, 1 << 17), out=t(G.F16, 1 << 20, 1 << 17)),  # rows * heads
    dict(cache=cache(page_size=256, kv_heads=1, d_head=64), q=t(G.F16, 1 << 20, 2048), out=t(G.F16, 1 << 20, 2048),
         block_table=t(G.I32, 3, 1 << 15)),                                                     # rows * group units of keys
    dict(cache=cache(page_size=256, kv_heads=8), q=t(G.F16, 5, 512), out=t(G.F16, 5, 512), block_table=t(G.I32, 4096, 1 << 12),
         q_start=t(G.I32, 4097), kv_lens=t(G.I32, 4096))], ids=str)
def test_attn_calls_that_32_bits_cannot_count(bad):
    with pytest.raises(G.GtenError, match="status 1"):
        attn(**bad)

"""The binding's descriptors follow the objects they describe: fields that are set, shapes that change in place,
buffers that move; and objects that were used can be copied and pickled. No GPU: nothing reads the addresses."""
import copy
import pickle

import pytest

import gten_b200 as G


class Buf:
    """A buffer that can move."""

    def __init__(self, at):
        self.at = at

    def data_ptr(self):
        return self.at


def tensor(t) -> G.gtn_tensor:
    return G._d(t)._obj


def cache(c) -> G.gtn_paged_cache:
    return G._d(c)._obj


def new_cache(k=4096, v=8192, **kw):
    return G.PagedCache(k, v, G.F16, 8, 16, 2, 64, **kw)


def test_cache_follows_its_fields():
    c = new_cache()
    assert (cache(c).k, cache(c).v, cache(c).n_pages, cache(c).page_stride) == (4096, 8192, 8, 0)
    c.k = 1 << 20
    assert (cache(c).k, cache(c).v) == (1 << 20, 8192)
    c.v = Buf(1 << 21)
    assert cache(c).v == 1 << 21
    for name, value in (("dtype", G.Q8), ("n_pages", 3), ("page_size", 64), ("kv_heads", 5), ("d_head", 128), ("page_stride", 1 << 20)):
        setattr(c, name, value)
        assert getattr(cache(c), name) == value and getattr(c.desc(), name) == value


def test_cache_follows_a_buffer_that_moves():
    k, v = Buf(4096), Buf(8192)
    c = new_cache(k, v)
    assert (cache(c).k, cache(c).v) == (4096, 8192)
    k.at = 1 << 20
    assert (cache(c).k, cache(c).v) == (1 << 20, 8192)
    v.at = 1 << 21
    assert (cache(c).k, cache(c).v, c.desc().v) == (1 << 20, 1 << 21, 1 << 21)


def test_caches_stay_hashable_and_distinct():
    a, b = new_cache(), new_cache()
    assert a == a and a != b and len({a, b}) == 2


def test_tensor_follows_its_fields_and_buffer():
    b = Buf(4096)
    t = G.GT(b, G.F16, (3, 64))
    assert (tensor(t).data, list(tensor(t).shape)[:2], list(tensor(t).strides)[:2]) == (4096, [3, 64], [64, 1])
    assert G._d(t) is G._d(t)  # kept
    b.at = 8192
    assert tensor(t).data == 8192
    t.shape = (5, 32)
    assert list(tensor(t).shape)[:2] == [5, 32] and list(tensor(t).strides)[:2] == [32, 1]
    t.strides = (96, 1)
    assert list(tensor(t).strides)[:2] == [96, 1]
    t.dtype = G.F32
    assert tensor(t).dtype == G.F32


def test_tensor_whose_shape_changes_in_place():
    shape, strides = [3, 64], [96, 1]
    t = G.GT(4096, G.F16, shape, strides)
    assert list(tensor(t).shape)[:2] == [3, 64]
    shape[0] = 5
    strides[0] = 128
    assert list(tensor(t).shape)[:2] == [5, 64] and list(tensor(t).strides)[:2] == [128, 1]
    t = G.GT(4096, G.F16, (3, 64), strides)
    assert list(tensor(t).strides)[:2] == [128, 1]
    strides[0] = 64
    assert list(tensor(t).strides)[:2] == [64, 1]


def test_descriptors_of_other_classes():
    """Whatever has a desc() can be passed, and is asked every time."""
    class Mine:
        n = 3

        def desc(self):
            return G.GT(4096, G.F16, (self.n, 64)).desc()

    class Half(G.GT):
        def desc(self):
            d = super().desc()
            d.shape[0] //= 2
            return d

    m = Mine()
    assert tensor(m).shape[0] == 3
    m.n = 4
    assert tensor(m).shape[0] == 4
    assert tensor(Half(4096, G.F16, (6, 64))).shape[0] == 3


@pytest.mark.parametrize("used", [False, True])
@pytest.mark.parametrize("make", [lambda: G.GT(4096, G.F16, (3, 64)), new_cache], ids=["tensor", "cache"])
@pytest.mark.parametrize("again", [copy.copy, copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x))], ids=["copy", "deepcopy", "pickle"])
def test_copies(make, again, used):
    a = make()
    if used:
        G._d(a)
    b = again(a)
    assert type(b) is type(a) and bytes(b.desc()) == bytes(a.desc())
    name = "buf" if isinstance(a, G.GT) else "k"
    setattr(b, name, 1 << 20)
    first = tensor(b).data if isinstance(b, G.GT) else cache(b).k
    other = tensor(a).data if isinstance(a, G.GT) else cache(a).k
    assert (first, other) == (1 << 20, 4096)
    assert "_ref" not in a.__getstate__()


def test_equality_of_tensors_ignores_use():
    a, b = G.GT(4096, G.F16, (3, 64)), G.GT(4096, G.F16, (3, 64))
    G._d(a)
    assert a == b

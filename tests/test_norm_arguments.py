"""What the wrapper's norms of query and key heads hand to the library: every form the header has, on the CPU."""
import pytest

from ingot_amd import KvCache, KvTable, Session
from ingot_amd import _lib as L
from ingot_amd.host import DeviceTensor


def tensor(dtype, *shape):
    return DeviceTensor(None, dtype, shape, 4096, False)


@pytest.fixture
def append():
    """The descriptors of the norms of queries and keys, (weight, head stride, eps) or None."""
    s = Session.__new__(Session)
    s.lib, s.h = L.load(), None
    s._prepared = lambda fn, *a: a
    x, kv, pos, tab = tensor(L.DT_F32, 3, 2, 8), tensor(L.DT_F32, 3, 1, 8), tensor(L.DT_I32, 3), tensor(L.DT_F32, 5, 4)
    k = tensor(L.DT_BF16, 1, 2, 1, 4, 8)
    cache, table = KvCache(k, k), KvTable(tensor(L.DT_I32, 2, 2), tensor(L.DT_I32, 2))

    def of(q_weight, k_weight, **kw):
        a = s.prepare_norm_rotary_append(x, kv, kv, q_weight, k_weight, pos, tab, tab, x, cache, table, tensor(L.DT_I32, 3), **kw)
        return [n and (n._obj.d_weight, n._obj.head, round(n._obj.eps, 9)) for n in a[:2]]

    return of


def test_queries_and_keys_each_with_a_norm_of_their_own(append):
    w, per_head = tensor(L.DT_F32, 8), tensor(L.DT_F32, 2, 8)
    assert append(w, None) == [(4096, 0, 1e-6), None]
    assert append(None, 1, eps=1e-5) == [None, (None, 0, 1e-5)]
    assert append(1, w, eps=(1e-5, 1e-3)) == [(None, 0, 1e-5), (4096, 0, 1e-3)]
    assert append(per_head, 1.0, eps=[0.0, 0.5]) == [(4096, 8, 0.0), (None, 0, 0.5)]
    assert append(None, None) == [None, None]


def test_refusals(append):
    for q, k in ((2, None), (None, 0), (0.5, 1)):
        with pytest.raises(ValueError, match="norm weight"):
            append(q, k)
    with pytest.raises(ValueError):
        append(1, 1, eps=(1e-5, 1e-5, 1e-5))

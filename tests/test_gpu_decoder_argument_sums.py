"""Sizes whose sums pass 63 bits are refused like others that are too large."""
import ctypes as C

import numpy as np
import pytest

from helpers import announce
from ingot_amd import KvCache, KvTable
from ingot_amd import _lib as L

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("first,rows,rot", [(2 ** 63 - 1, 1, 4), (2 ** 63 - 1, 2 ** 63 - 1, 2), (1, 2 ** 63 - 1, 4),
                                            (2, 2 ** 62, 8), (2 ** 31 - 1, 1, 2), (0, 2 ** 31, 2)])
def test_tables(sess, first, rows, rot):
    announce(f"rotary table sizes {first} {rows} {rot}")
    t = sess.empty(L.DT_F32, (16,))
    args = L.RotaryTableArgs(first, rows, rot, L.ROTARY_PLAIN, 10000.0, 1.0, 0.0, 0.0, 0.0, 1.0, t.ptr, t.ptr)
    assert sess.lib.ingot_rocm_rotary_table(sess.h, C.byref(args)) == L.EINVAL
    t.free()


@pytest.mark.parametrize("heads", [2 ** 63 - 1, 2 ** 63 - 2, 2 ** 62, (1 << 20) - 1])
def test_heads_of_an_append(sess, heads):
    announce(f"rotary append heads {heads}")
    k = sess.empty(L.DT_F32, (1, 2, 1, 4, 8))
    cache = KvCache(k, k)
    table = KvTable(sess.to_device(np.zeros((1, 2), np.int32)), sess.to_device(np.zeros(1, np.int32)))
    ints = sess.to_device(np.array([0, 1], np.int32))
    view = L.HeadsDesc(k.ptr, 8, 8)
    rot = L.RotaryDesc(k.ptr, k.ptr, ints.ptr, 1, 8, 0)
    batch = L.KvBatchDesc(ints.ptr, None, 1, 1, 0)
    rc = sess.lib.ingot_rocm_rotary_append(sess.h, C.byref(rot), C.byref(cache.c), C.byref(table.c), C.byref(batch), heads,
                                           L.DT_F32, C.byref(view), C.byref(view), C.byref(view), C.byref(view))
    assert rc == L.EINVAL
    for t in (k, table.pages, table.lengths, ints):
        t.free()

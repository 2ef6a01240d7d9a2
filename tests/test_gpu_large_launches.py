"""Calls whose threads pass 2^32, which one launch does not take: long lists over large pages, tables of many angles."""
import numpy as np
import pytest

from decoder_reference import free_all, frequencies
from helpers import announce
from ingot_amd import DeviceTensor, IngotError, KvCache, KvTable
from ingot_amd import _lib as L
from test_gpu_kv_pages import Model, ints, same

pytestmark = pytest.mark.gpu

LIST = 1 << 20  # entries, nearly all of which name nothing


def padded(entries):
    """The entries at the beginning, over the middle and at the end of a list of −1."""
    out = np.full(LIST, -1, np.int32)
    n = len(entries)
    at = np.linspace(0, LIST - 1, n).astype(np.int64)
    out[at] = entries
    return out


def test_copy_of_a_long_list(sess):
    """Pages of 20 workgroups."""
    announce("kv_copy long list")
    rng = np.random.default_rng(1)
    m = Model(rng, 1, 1, 2, 10, 128, 64, L.DT_BF16, [0], spare=24)
    cache, table = m.upload(sess, refs=True)
    order = rng.permutation(24)
    src, dst = padded(order[:12]), padded(order[12:])
    ds, dd = ints(sess, src), ints(sess, dst)
    sess.kv_copy(cache, ds, dd)
    m.copy(order[:12], order[12:])
    same(m, cache, table, False)
    free_all(cache, table, ds, dd)


def test_fork_of_a_long_list(sess):
    announce("kv_fork long list")
    rng = np.random.default_rng(2)
    m = Model(rng, 1, 14, 3, 10, 128, 64, L.DT_BF16, [200, 140] + [0] * 12, spare=14)
    cache, table = m.upload(sess, refs=True)
    src, dst = np.arange(12) % 2, 2 + rng.permutation(12)
    ds, dd = ints(sess, padded(src)), ints(sess, padded(dst))
    sess.kv_fork(cache, table, ds, dd)
    same(m, cache, table, False, m.fork(src, dst))
    free_all(cache, table, ds, dd)


def test_compaction_of_a_long_list(sess):
    """Rows of 20 workgroups."""
    announce("kv_compact long list")
    rng = np.random.default_rng(3)
    m = Model(rng, 40, 9, 3, 8, 16, 64, L.DT_BF16, rng.integers(0, 20, 9), extra=12)
    cache, table = m.upload(sess, refs=True)
    rows = padded(rng.permutation(9))
    accept = np.sort(np.argsort(rng.random((LIST, 6)), axis=1)[:, :2], axis=1).astype(np.int32)
    counts = rng.integers(0, 3, LIST).astype(np.int32)
    new = np.full(9, -9, np.int32)
    ins = [ints(sess, a) for a in (rows, accept, counts, new)]
    sess.kv_compact(cache, table, *ins)
    used = rows >= 0
    m.compact(rows[used], accept[used], counts[used], new)
    assert np.array_equal(ins[3].numpy(), new)
    same(m, cache, table, False)
    free_all(cache, table, *ins)


def test_a_table_of_many_angles(sess):
    announce("rotary table of 2^32 angles")
    rot, rows = 65536, (1 << 17) + 3
    cos, sin = sess.rotary_table(rows, rot)
    f = frequencies(rot)
    for row in (0, 1, 4097, (1 << 17) - 1, 1 << 17, rows - 1):
        for t, want in ((cos, np.cos(row * f)), (sin, np.sin(row * f))):
            got = DeviceTensor(sess, L.DT_F32, (rot // 2,), t.ptr + row * rot * 2, False).numpy()
            assert np.abs(got - want).max() <= 2.0 ** -24 + 2.0 ** -30
    free_all(cos, sin)


def test_attention_of_too_many_tiles_is_declined(sess):
    """One sequence of 2^27 tokens that no launch has workgroups for; declined before anything is read."""
    announce("attention of too many tiles")
    k = sess.empty(L.DT_F32, (1, 2, 1, 4, 256))
    table = KvTable(ints(sess, [[0, 1]]), ints(sess, [0]))
    starts = ints(sess, [0, 1])
    q = DeviceTensor(sess, L.DT_F32, (1 << 27, 1, 256), k.ptr, False)
    with pytest.raises(IngotError, match="too many tiles") as e:
        sess.tree_attention(q, KvCache(k, k), table, starts, q)
    assert e.value.code == L.EDECLINED
    free_all(k, table, starts)

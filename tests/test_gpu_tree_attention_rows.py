"""Attention over a bf16 cache in its ring form (more than 16 rows to a key head, in waves of 16 or of 32 rows): missing pages,
empty rows, infinities, scales and far offsets."""
import numpy as np
import pytest

from decoder_reference import free_all, to_dtype, values
from helpers import announce
from ingot_amd import DeviceTensor, KvCache, KvTable
from ingot_amd import _lib as L
from test_gpu_tree_attention import Case
from test_gpu_tree_attention_windows import stand_in

pytestmark = pytest.mark.gpu

QUERIES = [L.DT_F32, L.DT_BF16]
# new tokens, query heads, key heads: 20 rows and 40 (16 to a wave), 90 (bf16 queries 32 to a wave), 132 (two row tiles)
DRAFTS = [(20, 2, 2), (10, 8, 2), (45, 4, 2), (66, 2, 1)]


@pytest.mark.parametrize("dtype", QUERIES)
@pytest.mark.parametrize("nodes,heads,kv", DRAFTS)
@pytest.mark.parametrize("dim,page", [(64, 1), (80, 16), (128, 40), (160, 7)])
def test_pages_that_are_not_there(sess, dtype, nodes, heads, kv, dim, page):
    announce(f"ring missing pages {dtype} {nodes} {heads} {kv} {dim} {page}")
    c = Case(dim + nodes, dtype, L.DT_BF16, [200, 90], [nodes, nodes - 3], heads, kv, dim, page)
    stand_in(c, 50.0)
    c.pages.pages[0, 1] = -1
    c.pages.pages[0, 120 // page] = c.pages.num
    c.pages.pages[1, (90 + 3) // page] = -5
    c.pages.pages[1, 0] = 2 ** 31 - 1
    c.check(c.run(sess))


@pytest.mark.parametrize("dtype", QUERIES)
@pytest.mark.parametrize("nodes,heads,kv", DRAFTS)
def test_rows_that_see_nothing(sess, dtype, nodes, heads, kv):
    announce(f"ring empty rows {dtype} {nodes} {heads} {kv}")
    c = Case(8, dtype, L.DT_BF16, [0, 45, 0, 12], [nodes, 0, 3, nodes, 5, 2], heads, kv, 64, 16, rows=[0, 1, 9, 2, 3, -1],
             hide=0.5)
    got = c.run(sess)
    c.check(got)
    empty = 0
    for b, r in enumerate(c.rows):
        for i in range(c.starts[b], c.starts[b + 1]):
            if not 0 <= r < 4 or (c.pages.len[r] == 0 and not c.tree[i].any()):
                empty += 1
                assert not got[i].any()
    assert empty > 5
    c.tree[:] = False
    c.check(c.run(sess))


@pytest.mark.parametrize("dtype", QUERIES)
@pytest.mark.parametrize("nodes,heads,kv", DRAFTS)
@pytest.mark.parametrize("bad", [np.inf, -np.inf])
def test_committed_values_that_are_infinite(sess, dtype, nodes, heads, kv, bad):
    """In blocks that every row sees whole and in the last committed block, which stands beside hidden nodes."""
    announce(f"ring infinite values {dtype} {nodes} {heads} {bad}")
    for pos in (100, 299):
        c = Case(11, dtype, L.DT_BF16, [300], [nodes], heads, kv, 64, 16, layers=1)
        pg, sl = c.pages.place(0, pos)
        c.pages.v[0, pg, kv - 1, sl, 9] = to_dtype(np.array(bad), L.DT_BF16).reshape(())
        got = c.run(sess, layer=0)
        reads = slice((kv - 1) * (heads // kv), heads)  # the query heads of the last key head
        assert (got[:, reads, 9] == bad).all()
        got[:, reads, 9] = 0
        assert np.isfinite(got).all()


@pytest.mark.parametrize("dtype", QUERIES)
@pytest.mark.parametrize("nodes", [20, 70])
def test_a_key_of_minus_infinity(sess, dtype, nodes):
    """A score of −Inf has no weight; one of +Inf makes its row NaN and no other."""
    announce(f"ring infinite key {dtype} {nodes}")
    c = Case(21, dtype, L.DT_BF16, [100], [nodes], 1, 1, 64, 16, layers=1)
    c.q[0::2, 0, 5] = to_dtype(np.array(0.5), dtype).reshape(())
    c.q[1::2, 0, 5] = to_dtype(np.array(-0.37), dtype).reshape(())
    pg, sl = c.pages.place(0, 60)
    c.pages.k[0, pg, 0, sl, 5] = to_dtype(np.array(-np.inf), L.DT_BF16).reshape(())
    got = c.run(sess, layer=0)
    c.check(got, layer=0, skip=range(1, nodes, 2))
    assert np.isnan(got[1::2]).all()


@pytest.mark.parametrize("dtype", QUERIES)
@pytest.mark.parametrize("nodes", [1, 20, 70])
@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_scales(sess, dtype, nodes, scale):
    announce(f"ring scale {dtype} {nodes} {scale}")
    c = Case(13, dtype, L.DT_BF16, [400], [nodes], 2, 1, 64, 16, scale=scale)
    c.check(c.run(sess))


@pytest.mark.parametrize("dtype", QUERIES)
@pytest.mark.parametrize("nodes,heads", [(20, 1), (40, 2)])
def test_offsets_past_32_bits(sess, dtype, nodes, heads):
    """Pages more than 2^31 elements into the cache (page stride of 2^24 elements; only the pages in use are filled)."""
    announce(f"ring far pages {dtype} {nodes} {heads}")
    rng = np.random.default_rng(19)
    page, dim, num, stride, held = 16, 64, 160, 1 << 24, 40
    ids = [158, 3, 140, 159, 150][:-(-(held + nodes) // page)]
    pool = sess.empty(L.DT_BF16, ((num - 1) * stride + page * dim,))
    data = to_dtype(rng.normal(0, 1, (len(ids), page, dim)), L.DT_BF16)  # keys, and values too
    for n, p in enumerate(ids):
        src = sess.to_device(data[n], L.DT_BF16)
        sess.copy_d2d(DeviceTensor(sess, L.DT_BF16, (page, dim), pool.ptr + 2 * p * stride, False), src)
        src.free()
    both = DeviceTensor(sess, L.DT_BF16, (1, num, 1, page, dim), pool.ptr, False)
    cache = KvCache(both, both)
    cache.c.stride_page, cache.c.stride_layer = stride, num * stride
    table = KvTable(sess.to_device(np.array([ids], np.int32)), sess.to_device(np.array([held], np.int32)))
    q = to_dtype(rng.normal(0, 1, (nodes, heads, dim)), dtype)
    dq, dy = sess.to_device(q, dtype), sess.empty(dtype, q.shape)
    starts = sess.to_device(np.array([0, nodes], np.int32))
    sess.tree_attention(dq, cache, table, starts, dy)
    got = values(dy.numpy())
    kk = values(data).reshape(-1, dim)
    for t in range(nodes):
        for h in range(heads):
            k = kk[:held + t + 1]
            s = k @ values(q)[t, h] / 8
            w = np.exp(s - s.max())
            want = (w[:, None] * k).sum(0) / w.sum()
            assert np.abs(got[t, h] - want).max() <= (1e-5 if dtype == L.DT_F32 else 2.0 ** -7) * np.abs(k).max()
    free_all(pool, table, dq, dy, starts)

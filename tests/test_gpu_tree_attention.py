"""Attention of drafted tokens over a paged cache on the GPU, against the definition in 64 bits."""
import numpy as np
import pytest

from decoder_reference import (Pages, attention, attention_bound, free_all, to_dtype, values)
from helpers import announce
from ingot_amd import Heads, IngotError, KvCache, KvTable
from ingot_amd import _lib as L

pytestmark = pytest.mark.gpu

KINDS = [(L.DT_F32, L.DT_BF16), (L.DT_BF16, L.DT_BF16), (L.DT_F32, L.DT_F32), (L.DT_BF16, L.DT_F32)]


def bits(seen):
    """Truth values [tokens, nodes] as int32 words."""
    t, n = seen.shape
    words = np.zeros((t, max(1, -(-n // 32))), np.uint32)
    for j in range(n):
        words[:, j // 32] |= seen[:, j].astype(np.uint32) << np.uint32(j % 32)
    return words.view(np.int32)


class Case:
    """Sequences on rows of a cache; the draft's masks are random trees (or a chain)."""

    def __init__(self, seed, dtype, cache, lengths, counts, heads, kv, dim, page, rows=None, tree=True, layers=2,
                 scale=None, hide=0.0):
        rng = self.rng = np.random.default_rng(seed)
        self.dtype, self.cache, self.dim, self.heads = dtype, cache, dim, heads
        self.rows = np.arange(len(counts), dtype=np.int32) if rows is None else np.asarray(rows, np.int32)
        n = max(counts)
        self.pages = Pages(rng, layers, len(lengths), -(-(max(lengths) + n) // page) + 1, kv, page, dim, cache, lengths, extra=n)
        self.starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        self.total, self.max_nodes = int(self.starts[-1]), n
        self.q = to_dtype(rng.normal(0, 1, (self.total, heads, dim)), dtype)
        self.scale = dim ** -0.5 if scale is None else scale
        self.tree = None
        if tree:
            self.tree = np.zeros((self.total, n), bool)
            for b, c in enumerate(counts):
                for i in range(c):
                    t = self.starts[b] + i
                    if i:
                        self.tree[t] = self.tree[self.starts[b] + rng.integers(max(0, i - 4), i)]
                    self.tree[t, i] = True
                for i in range(c):
                    if rng.random() < hide:
                        self.tree[self.starts[b] + i] = False

    def seen(self, b, i, j):
        return j <= i if self.tree is None else bool(self.tree[self.starts[b] + i, j])

    def run(self, sess, slot_major=False, max_tokens=None, layer=1, mask=None, max_nodes=None, in_place=False, strided=False):
        cache, table = self.pages.upload(sess, slot_major)
        if strided:
            width = self.heads * self.dim + 5
            wide = np.zeros((self.total, width), self.q.dtype)
            wide[:, 3:3 + self.heads * self.dim] = self.q.reshape(self.total, -1)
            dq = sess.to_device(wide, self.dtype)
            dy = sess.empty(self.dtype, (self.heads, self.total + 1, self.dim + 3))
            q = Heads(dq, self.total, self.heads, self.dim, 3, width, self.dim)
            y = Heads(dy, self.total, self.heads, self.dim, 1, self.dim + 3, (self.total + 1) * (self.dim + 3))
        else:
            q = dq = sess.to_device(self.q, self.dtype)
            y = dy = dq if in_place else sess.empty(self.dtype, self.q.shape)
        if not in_place:
            dy_fill = to_dtype(np.full(dy.shape, 7.0), self.dtype)
            fill = sess.to_device(dy_fill, self.dtype)
            sess.copy_d2d(dy, fill)
            fill.free()
        starts, rows = sess.to_device(self.starts), sess.to_device(self.rows)
        m = bits(self.tree) if mask is None and self.tree is not None else mask
        dm = sess.to_device(m) if m is not None else None
        most = int(self.pages.len.max()) + self.max_nodes if max_tokens is None else max_tokens
        kw = dict(rows=rows, layer=layer, max_nodes=self.max_nodes if max_nodes is None else max_nodes, max_tokens=most,
                  mask=dm, scale=self.scale)
        sess.tree_attention(q, cache, table, starts, y, **kw)
        out = dy.numpy()
        if not in_place:
            sess.tree_attention(q, cache, table, starts, y, **kw)
            assert dy.numpy().tobytes() == out.tobytes(), "a second call differs"
        if strided:
            out = np.stack([out[h].reshape(-1)[1:][:self.total * (self.dim + 3)].reshape(self.total, -1)[:, :self.dim]
                            for h in range(self.heads)], axis=1)
        free_all(cache, table, dq, starts, rows, *([dm] if dm is not None else []), *([] if in_place else [dy]))
        return values(out)

    def check(self, got, layer=1, max_nodes=None, max_tokens=0, skip=()):
        nodes = self.max_nodes if max_nodes is None else max_nodes
        want, mass, size = attention(self.pages, layer, values(self.q), self.starts, self.rows, self.seen, self.scale, nodes,
                                     max_tokens)
        for b in range(len(self.rows)):  # tokens past max_nodes are not written
            over = slice(self.starts[b] + nodes, max(self.starts[b] + nodes, self.starts[b + 1]))
            want[over] = 7.0
            mass[over] = 0
        bound = attention_bound(want, mass, size, self.dim, int(self.pages.len.max()) + nodes, self.dtype, self.cache)
        with np.errstate(invalid="ignore"):
            off = np.abs(got - want)
        keep = np.ones(self.total, bool)
        keep[list(skip)] = False
        assert np.isfinite(got[keep]).all(), "not finite"
        assert (off[keep] <= bound[keep]).all(), f"over the bound by {(off / bound)[keep].max():.3g}, off by {off[keep].max():.3g}"


@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("lengths,counts,heads,kv,dim,page,tree", [
    ([0], [1], 1, 1, 64, 16, False),
    ([1], [1], 4, 4, 128, 16, True),
    ([517], [1], 16, 16, 128, 16, False),
    ([31, 32, 33, 0, 127], [1, 1, 1, 1, 1], 8, 2, 64, 8, False),
    ([100, 7, 64, 0], [5, 16, 1, 7], 8, 2, 80, 24, True),
    ([700, 3], [9, 33], 6, 2, 128, 1, True),
    ([260, 0], [40, 70], 4, 1, 96, 7, True),
    ([130, 600], [17, 3], 5, 1, 256, 32, True),
    ([90], [65], 8, 8, 160, 100, False),
    ([300, 20], [64, 50], 10, 2, 8, 64, False),
    ([1500], [3], 2, 1, 40, 3, True),
    ([70, 33], [130, 97], 2, 1, 128, 24, True)])
def test_attention(sess, dtype, cache, lengths, counts, heads, kv, dim, page, tree):
    announce(f"attention {dtype} {cache} {lengths} {counts} {heads} {kv} {dim} {page}")
    c = Case(len(lengths) + dim, dtype, cache, lengths, counts, heads, kv, dim, page, tree=tree)
    c.check(c.run(sess, slot_major=page == 24, in_place=False))


@pytest.mark.parametrize("dtype,cache", KINDS)
def test_long_contexts_are_cut_and_joined(sess, dtype, cache):
    """Positions in many pieces, sequences far shorter than max_tokens (pieces without a position), pages of one slot:
    more pages than one table of offsets holds."""
    announce(f"attention long {dtype} {cache}")
    c = Case(5, dtype, cache, [9001, 40, 2600], [2, 3, 1], 2, 1, 64, 1)
    c.check(c.run(sess))
    c = Case(6, dtype, cache, [20011], [4], 8, 1, 128, 16, layers=1)
    c.check(c.run(sess, layer=0), layer=0)


@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("lengths,counts,heads,kv,dim,page,tree,rows", [
    ([17000, 40, 2600, 0, 9000], [1, 3, 2, 0, 4], 8, 8, 8, 16, True, None),
    ([12000, 900, 5000], [20, 33, 1], 16, 16, 16, 64, False, [2, 0, 1]),
    ([9000, 130, 4000, 77], [70, 9, 40, 5], 16, 4, 24, 32, True, [0, 3, -1, 2]),
    ([30000, 64], [2, 1], 256, 64, 8, 48, False, None)])
def test_pieces_cut_by_lengths(sess, dtype, cache, lengths, counts, heads, kv, dim, page, tree, rows):
    """Sequences of very different lengths whose pieces are long: one without tokens, one without a row."""
    announce(f"attention cut {dtype} {cache} {lengths}")
    c = Case(9 + dim, dtype, cache, lengths, counts, heads, kv, dim, page, tree=tree, layers=1, rows=rows)
    c.check(c.run(sess, layer=0), layer=0)


@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("batch,longest,most", [(70, 6000, 3), (300, 1500, 2), (64, 4000, 30)])
def test_many_sequences_in_pieces(sess, dtype, cache, batch, longest, most):
    """More sequences than the cut by lengths takes, tiles for more than half of the card, and as many as it takes."""
    announce(f"attention many {dtype} {cache} {batch}")
    rng = np.random.default_rng(batch)
    lengths = rng.integers(0, 40, batch)
    lengths[rng.integers(0, batch, 3)] = [longest, longest // 2, longest - 1]
    c = Case(batch, dtype, cache, lengths.tolist(), rng.integers(0, most + 1, batch - 1).tolist() + [most], 1, 1, 8, 64,
             rows=rng.permutation(batch), layers=1)
    c.check(c.run(sess, layer=0), layer=0)


@pytest.mark.parametrize("dtype,cache", KINDS)
def test_one_piece_over_many_pages(sess, dtype, cache):
    """So many sequences that nothing is cut, one of them past one table of offsets (1024 pages)."""
    announce(f"attention one piece {dtype} {cache}")
    lengths = [3] * 700
    lengths[333] = 2500
    c = Case(7, dtype, cache, lengths, [1] * 700, 1, 1, 64, 2, layers=1, tree=False)
    c.check(c.run(sess, layer=0), layer=0)


@pytest.mark.parametrize("dtype,cache", KINDS)
def test_rows_that_see_nothing(sess, dtype, cache):
    """Empty mask rows without a context, sequences without tokens, without a row, on rows out of range."""
    announce(f"attention empty rows {dtype} {cache}")
    c = Case(8, dtype, cache, [0, 45, 0, 12], [6, 0, 3, 4, 5, 2], 4, 2, 64, 16, rows=[0, 1, 9, 2, 3, -1], hide=0.5)
    got = c.run(sess)
    c.check(got)
    for b, r in enumerate(c.rows):
        for i in range(c.starts[b], c.starts[b + 1]):
            if not 0 <= r < 4 or (c.pages.len[r] == 0 and not c.tree[i].any()):
                assert not got[i].any()
    c.tree[:] = False
    got = c.run(sess)
    c.check(got)


@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("page", [1, 16, 40])
def test_pages_that_are_not_there(sess, dtype, cache, page):
    announce(f"attention missing pages {dtype} {cache} {page}")
    c = Case(9, dtype, cache, [200, 90], [4, 4], 4, 2, 64, page)
    c.pages.pages[0, 1] = -1
    c.pages.pages[0, 120 // page] = c.pages.num
    c.pages.pages[1, (90 + 3) // page] = -5
    c.pages.pages[1, 0] = 2 ** 31 - 1
    c.check(c.run(sess))


@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 3e38])
def test_values_in_hidden_places(sess, dtype, cache, bad):
    """NaN, infinities and the largest numbers in slots that nobody sees (past the last token, in page 0, which stands in
    for pages that are not there) and in nodes that some rows see: those rows take them, the others do not."""
    announce(f"attention hidden {bad} {dtype} {cache}")
    c = Case(10, dtype, cache, [50, 20], [12, 40], 4, 2, 80, 16, layers=1)
    p = c.pages
    used = np.zeros((p.num, p.page), bool)
    for r in range(2):
        for pos in range(int(p.len[r]) + int(c.starts[r + 1] - c.starts[r])):
            used[p.place(r, pos)] = True
    fill = to_dtype(np.array(bad), cache).reshape(())
    for a in (p.k, p.v):
        a[0][np.broadcast_to(~used[:, None, :, None], a[0].shape)] = fill
    c.check(c.run(sess, layer=0), layer=0)
    # a node's value, then its key
    for a, nodes in ((p.v, [(0, 5), (1, 33)]), (p.k, [(0, 7)])):
        for b, i in nodes:
            pg, sl = p.place(b, int(p.len[b]) + i)
            a[0, pg, :, sl, 3] = fill
    see = [t for b in range(2) for t in range(c.starts[b], c.starts[b + 1])
           if c.tree[t, 5 if b == 0 else 33] or (b == 0 and c.tree[t, 7])]
    got = c.run(sess, layer=0)
    assert 0 < len(see) < c.total
    c.check(got, layer=0, skip=see)
    if not np.isfinite(bad):
        for t in see:
            only_value = c.starts[1] <= t or not c.tree[t, 7]
            if only_value:
                assert (np.isnan(got[t, :, 3]) if np.isnan(bad) else got[t, :, 3] == bad).all()
                others = np.delete(got[t], 3, axis=1)
                assert np.isfinite(others).all()


@pytest.mark.parametrize("dtype,cache", KINDS)
def test_committed_values_that_are_not_finite(sess, dtype, cache):
    """An infinity among the committed values reaches every row, in its dimension only."""
    announce(f"attention inf {dtype} {cache}")
    c = Case(11, dtype, cache, [300], [3], 2, 2, 64, 16, layers=1)
    pg, sl = c.pages.place(0, 100)
    c.pages.v[0, pg, 1, sl, 9] = to_dtype(np.array(np.inf), cache).reshape(())
    got = c.run(sess, layer=0)
    assert (got[:, 1, 9] == np.inf).all()
    got[:, 1, 9] = 0
    assert np.isfinite(got).all()


@pytest.mark.parametrize("dtype,cache", KINDS)
def test_a_key_of_minus_infinity(sess, dtype, cache):
    """A committed key whose score is −Inf for a query has no weight there; where it is +Inf the row is NaN, as the
    formula has it. Zeros among the terms of a split query must not turn either into NaN."""
    announce(f"attention infinite key {dtype} {cache}")
    c = Case(21, dtype, cache, [100], [6], 1, 1, 64, 16, layers=1)
    c.q[0::2, 0, 5] = to_dtype(np.array(0.5), dtype).reshape(())  # one bit: the lower terms of it are zero
    c.q[1::2, 0, 5] = to_dtype(np.array(-0.37), dtype).reshape(())
    pg, sl = c.pages.place(0, 60)
    c.pages.k[0, pg, 0, sl, 5] = to_dtype(np.array(-np.inf), cache).reshape(())
    c.check(c.run(sess, layer=0), layer=0, skip=[1, 3, 5])
    assert np.isnan(c.run(sess, layer=0)[1::2]).all()


def test_a_row_of_minus_infinity(sess):
    """Visible scores that are all −Inf give zeros; NaN in a query gives NaN in its row alone."""
    announce("attention -inf scores")
    c = Case(12, L.DT_F32, L.DT_F32, [20], [3], 1, 1, 64, 16, layers=1)
    c.pages.k[:] = np.abs(c.pages.k)
    c.q[1] = -np.inf
    c.q[2, 0, 7] = np.nan
    got = c.run(sess, layer=0)
    assert not got[1].any() and np.isnan(got[2]).all() and np.isfinite(got[0]).all()


@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_scales(sess, scale):
    """No scale, a negative one, and scores over a wide range (a running maximum that keeps rising)."""
    announce(f"attention scale {scale}")
    c = Case(13, L.DT_F32, L.DT_BF16, [400], [5], 4, 2, 64, 16, scale=scale)
    c.check(c.run(sess))


@pytest.mark.parametrize("dtype,cache", KINDS)
def test_strided_heads(sess, dtype, cache):
    """q inside wider rows at an odd offset, y head by head with gaps: nothing is aligned."""
    announce(f"attention strided {dtype} {cache}")
    c = Case(14, dtype, cache, [70, 5], [4, 9], 6, 3, 72, 16)
    c.check(c.run(sess, strided=True))
    c = Case(15, dtype, cache, [3000], [2], 2, 1, 72, 16, tree=False, layers=1)
    c.check(c.run(sess, strided=True, layer=0), layer=0)


def test_in_place(sess):
    announce("attention in place")
    for lengths in ([60, 9], [6000, 9]):
        c = Case(16, L.DT_BF16, L.DT_BF16, lengths, [4, 20], 4, 2, 64, 16)
        c.check(c.run(sess, in_place=True))


def test_limits(sess):
    """max_nodes and max_tokens below what is there; a mask of fewer words than nodes; no limit given."""
    announce("attention limits")
    c = Case(17, L.DT_F32, L.DT_BF16, [40, 50], [9, 6], 4, 2, 64, 16)
    got = c.run(sess, max_nodes=7)
    c.check(got, max_nodes=7)
    c.check(c.run(sess, max_tokens=0))
    c.check(c.run(sess, max_tokens=44), max_tokens=44)
    c = Case(18, L.DT_F32, L.DT_BF16, [40], [50], 4, 2, 64, 16)
    c.tree[:, 32:] = False
    c.check(c.run(sess, mask=bits(c.tree[:, :32])))


def test_offsets_past_32_bits(sess):
    """Pages more than 2^31 elements into the cache (page stride of 2^24 elements; only the pages in use are filled)."""
    announce("attention far pages")
    rng = np.random.default_rng(19)
    page, dim, num, stride = 16, 64, 160, 1 << 24
    pool = sess.empty(L.DT_BF16, ((num - 1) * stride + page * dim,))
    k, v = (to_dtype(rng.normal(0, 1, (3, page, dim)), L.DT_BF16) for _ in range(2))
    from ingot_amd import DeviceTensor

    ids = [159, 3, 140]
    for n, p in enumerate(ids):
        for a, off in ((k, 0), (v, page * dim)):
            part = DeviceTensor(sess, L.DT_BF16, (page, dim), pool.ptr + 2 * (p * stride + (off if p < num - 1 else 0)), False)
            if p == num - 1 and off:
                continue  # the last page holds keys only: values are read from the same place
            src = sess.to_device(a[n], L.DT_BF16)
            sess.copy_d2d(part, src)
            src.free()
    both = DeviceTensor(sess, L.DT_BF16, (1, num, 1, page, dim), pool.ptr, False)
    cache = KvCache(both, both)
    cache.c.stride_page, cache.c.stride_layer = stride, num * stride
    table = KvTable(sess.to_device(np.array([ids], np.int32)), sess.to_device(np.array([40], np.int32)))
    q = rng.normal(0, 1, (1, 1, dim)).astype(np.float32)
    dq, dy, starts = sess.to_device(q), sess.empty(L.DT_F32, q.shape), sess.to_device(np.array([0, 1], np.int32))
    sess.tree_attention(dq, cache, table, starts, dy)
    kk = values(k).reshape(-1, dim)[:41]
    s = kk @ q[0, 0].astype(np.float64) / 8
    w = np.exp(s - s.max())
    want = (w[:, None] * kk).sum(0) / w.sum()
    assert np.abs(dy.numpy()[0, 0] - want).max() <= 1e-5 * np.abs(kk).max()
    free_all(pool, table, dq, dy, starts)


def test_nothing_to_do(sess):
    announce("attention of nothing")
    k = sess.empty(L.DT_BF16, (1, 2, 1, 4, 8))
    table = KvTable(sess.to_device(np.zeros((1, 2), np.int32)), sess.to_device(np.zeros(1, np.int32)))
    q = sess.empty(L.DT_F32, (0, 2, 8))
    sess.tree_attention(q, KvCache(k, k), table, sess.to_device(np.zeros(2, np.int32)), q)
    sess.sync()


def test_refusals(sess):
    announce("attention refusals")
    table = KvTable(sess.to_device(np.zeros((1, 2), np.int32)), sess.to_device(np.zeros(1, np.int32)))
    starts = sess.to_device(np.array([0, 3], np.int32))

    def refused(code, text, shape=(1, 2, 1, 4, 16), heads=2, cache_dtype=L.DT_BF16, dtype=L.DT_F32, change=None, **kw):
        k = sess.empty(cache_dtype, shape)
        c = KvCache(k, k)
        q, y = sess.empty(dtype, (3, heads, shape[4])), sess.empty(dtype, (3, heads, shape[4]))
        if change:
            q, y = change(q, y)
        with pytest.raises(IngotError, match=text) as e:
            sess.tree_attention(q, c, table, starts, y, **kw)
        assert e.value.code == code

    refused(L.EDECLINED, "head_dim 264 > 256", shape=(1, 2, 1, 4, 264))
    refused(L.EDECLINED, "multiples of 8", shape=(1, 2, 1, 4, 12))
    refused(L.EINVAL, "3 heads over 2", shape=(1, 2, 2, 4, 16), heads=3)
    refused(L.EINVAL, "f32 or bf16", dtype=L.DT_I32)
    refused(L.EINVAL, "cache must be", cache_dtype=L.DT_F16)
    refused(L.EINVAL, "layer 2 of 1", layer=2)
    refused(L.EINVAL, "scale", scale=float("nan"))
    refused(L.EINVAL, "bad sizes", max_nodes=-1)
    refused(L.EINVAL, "bad sizes", max_tokens=2 ** 31)
    refused(L.EINVAL, "no words", mask=sess.empty(L.DT_I32, (3, 0)))
    refused(L.EINVAL, "overlap", change=lambda q, y: (q, Heads(y, 3, 2, 16, token=32, head=8)))
    refused(L.EINVAL, "in place", heads=1, change=lambda q, y: (Heads(q, 2, 1, 16, token=16), Heads(q, 2, 1, 16, token=32)))
    k = sess.empty(L.DT_BF16, (1, 2, 1, 4, 16))
    with pytest.raises(ValueError, match="mask"):
        q = sess.empty(L.DT_F32, (3, 2, 16))
        sess.tree_attention(q, KvCache(k, k), table, starts, q, mask=sess.empty(L.DT_I32, (2, 1)))
    sess.sync()

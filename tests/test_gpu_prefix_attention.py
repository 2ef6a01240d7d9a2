"""Attention of sequences that share prefixes on the GPU, against the definition in 64 bits and the attention of each alone."""
import ctypes as C

import numpy as np
import pytest

from decoder_reference import Pages, attention, attention_bound, free_all, to_dtype, values
from helpers import announce
from ingot_amd import Heads, IngotError, KvCache, KvTable
from ingot_amd import _lib as L

pytestmark = pytest.mark.gpu


@pytest.fixture
def sess(env_session):
    """A session that reads every prefix once, however small (INGOT_PREFIX_PATH, read when the session opens)."""
    return env_session(INGOT_PREFIX_PATH=2)


def shared_pages(rng, first, shared, lengths, counts, kv, page, dim, dtype, layers=1, slack=2):
    """Pages whose rows hold the prefixes of their groups in common: the full pages are the same, the part of a page behind
    them has the same keys and values in the rows' own pages. Row b is sequence b."""
    batch = len(lengths)
    most = max(-(-(int(n) + int(c)) // page) for n, c in zip(lengths, counts)) + slack
    p = Pages(rng, layers, batch, most, kv, page, dim, dtype, lengths, extra=max(counts) if len(counts) else 0)
    for g in range(len(shared)):
        for b in range(first[g] + 1, first[g + 1]):
            full, part = shared[g] // page, shared[g] % page
            p.pages[b, :full] = p.pages[first[g], :full]
            if part:
                src, dst = p.pages[first[g], full], p.pages[b, full]
                for pool in (p.k, p.v):
                    pool[:, dst, :, :part] = pool[:, src, :, :part]
    return p


def call(sess, p, q, dtype, starts, first, shared, mask=None, scale=None, layer=0, rows=None, slot_major=False, plain=False, **kw):
    cache, table = p.upload(sess, slot_major)
    dq, y = sess.to_device(q, dtype), sess.to_device(to_dtype(np.full(q.shape, 7.0), dtype), dtype)
    ins = [sess.to_device(np.asarray(a, np.int32)) for a in (starts, first, shared)]
    extra = [] if mask is None else [sess.to_device(mask.view(np.int32))]
    if rows is not None:
        extra.append(sess.to_device(np.asarray(rows, np.int32)))
        kw["rows"] = extra[-1]
    if mask is not None:
        kw["mask"] = extra[0]
    if plain:
        kw.pop("max_shared", None)
        sess.tree_attention(dq, cache, table, ins[0], y, scale=scale, layer=layer, **kw)
    else:
        sess.prefix_attention(dq, cache, table, ins[0], y, ins[1], ins[2], scale=scale, layer=layer, **kw)
    out = values(y.numpy())
    free_all(cache, table, dq, y, *ins, *extra)
    return out


def tree_mask(rng, counts):
    """Words of random ancestor masks; one node in eight sees committed tokens only."""
    words = -(-max(max(counts), 1) // 32)
    mask = np.zeros((int(sum(counts)), words), np.uint32)
    t = 0
    for n in counts:
        for i in range(n):
            if i:
                mask[t + i] = mask[t + int(rng.integers(max(0, i - 3), i))]
            if rng.random() > 1 / 8:
                mask[t + i, i // 32] |= np.uint32(1 << (i % 32))
        t += n
    return mask


def seen_by(mask, starts):
    if mask is None:
        return lambda b, i, o: o <= i
    return lambda b, i, o: o < 32 * mask.shape[1] and bool((mask[starts[b] + i, o // 32] >> np.uint32(o % 32)) & 1)


TYPES = [(L.DT_F32, L.DT_BF16), (L.DT_BF16, L.DT_BF16), (L.DT_F32, L.DT_F32), (L.DT_BF16, L.DT_F32)]


@pytest.mark.parametrize("dtype,cdtype", TYPES)
@pytest.mark.parametrize("heads,kv,dim,page,groups,shared,own,nodes,masked", [
    (2, 2, 64, 16, [4], [40], 9, 1, False), (8, 2, 128, 16, [3, 5], [160, 33], 40, 1, False),
    (4, 1, 80, 24, [2, 1, 4], [100, 0, 77], 30, 5, True), (12, 3, 64, 7, [6], [300], 20, 9, True),
    (16, 2, 128, 64, [9], [700], 100, 3, False), (6, 6, 256, 8, [3, 3], [60, 130], 10, 4, True),
    (1, 1, 8, 1, [2, 2], [5, 1], 3, 2, False), (5, 1, 96, 32, [7], [513], 1, 40, True),
    (8, 1, 64, 16, [40], [260], 12, 2, False)])
def test_groups(sess, dtype, cdtype, heads, kv, dim, page, groups, shared, own, nodes, masked):
    """Groups of several sizes; a sequence before them and one behind them share nothing; lengths of none and more."""
    announce(f"prefix {dtype} {cdtype} {heads} {kv} {dim} {page} {groups} {shared} {nodes} {masked}")
    rng = np.random.default_rng(heads * 1000 + dim + page + nodes)
    batch = sum(groups) + 2
    first = np.concatenate([[1], 1 + np.cumsum(groups)])
    base = np.zeros(batch, np.int64)
    for g, n in enumerate(groups):
        base[first[g]:first[g] + n] = shared[g]
    lengths = base + rng.integers(0, own + 1, batch)
    counts = rng.integers(1, nodes + 1, batch)
    counts[rng.integers(0, batch)] = 0 if nodes > 1 else 1
    counts[1] = nodes
    starts = np.concatenate([[0], np.cumsum(counts)])
    p = shared_pages(rng, first, shared, lengths, counts, kv, page, dim, cdtype)
    q = to_dtype(rng.normal(0, 1, (int(starts[-1]), heads, dim)), dtype)
    mask = tree_mask(rng, counts) if masked else None
    scale = dim ** -0.5
    got = call(sess, p, q, dtype, starts, first, shared, mask, scale, max_nodes=nodes,
               max_tokens=int((lengths + counts).max()), max_shared=max(shared))
    want, mass, size = attention(p, 0, values(q), starts, range(batch), seen_by(mask, starts), scale, nodes)
    bound = attention_bound(want, mass, size, dim, int((lengths + counts).max()), dtype, cdtype)
    assert (np.abs(got - want) <= bound).all(), np.abs(got - want).max()
    loose = call(sess, p, q, dtype, starts, first, shared, mask, scale)  # no limits given
    assert (np.abs(loose - want) <= bound).all()
    again = call(sess, p, q, dtype, starts, first, shared, mask, scale)
    assert np.array_equal(loose, again)


@pytest.mark.parametrize("dtype,cdtype", TYPES[:3])
@pytest.mark.parametrize("batch,groups,shared,nodes", [(5, 2, 3000, 3), (70, 66, 40, 1), (130, 3, 500, 1), (1100, 5, 20, 1)])
def test_many(sess, dtype, cdtype, batch, groups, shared, nodes):
    """Long prefixes in many pieces, more groups than a wave has lanes, more sequences than a workgroup has threads: against
    each sequence's attention by itself, whose errors have the same bound."""
    announce(f"prefix many {dtype} {cdtype} {batch} {groups} {shared}")
    rng = np.random.default_rng(batch + groups)
    heads, kv, dim, page = 4, 2, 64, 16
    cut = np.sort(rng.permutation(np.arange(1, batch))[:groups - 1])
    first = np.concatenate([[0], cut, [batch]])
    common = rng.integers(shared // 2, shared + 1, groups)
    base = np.repeat(common, np.diff(first))
    lengths, counts = base + rng.integers(0, 50, batch), rng.integers(1, nodes + 1, batch)
    starts = np.concatenate([[0], np.cumsum(counts)])
    p = shared_pages(rng, first, common, lengths, counts, kv, page, dim, cdtype)
    q = to_dtype(rng.normal(0, 1, (int(starts[-1]), heads, dim)), dtype)
    kw = dict(max_nodes=nodes, max_tokens=int((lengths + counts).max()))
    got = call(sess, p, q, dtype, starts, first, common, max_shared=shared, **kw)
    alone = call(sess, p, q, dtype, starts, first, common, plain=True, **kw)
    # |y| and the mass of |v| are below max |v|, the scores' terms below 6 for these sizes (64 products of normal numbers / 8)
    top = np.abs(values(p.v)).max()
    rel = 4 * (dim + 8) * 2.0 ** -24 * 8 + (lengths.max() + 64) * 2.0 ** -24
    if dtype == L.DT_BF16:
        rel += 2 * 2.0 ** -8
    assert np.abs(got - alone).max() <= 2 * rel * top
    assert np.abs(got - alone).mean() <= rel * top / 4


@pytest.mark.parametrize("dtype,cdtype", TYPES[:3])
def test_what_is_not_seen(sess, dtype, cdtype):
    """NaN and infinities in slots past the committed tokens, on pages of nobody and in nodes the mask hides do not reach a
    result; a page that is missing in the prefix hides its tokens, for the whole group; rows that see nothing give zeros."""
    announce(f"prefix unseen {dtype} {cdtype}")
    rng = np.random.default_rng(3)
    heads, kv, dim, page = 8, 2, 64, 16
    first, shared = np.array([0, 3, 5]), np.array([70, 0])
    lengths, counts = np.array([70, 90, 75, 0, 0]), np.array([3, 2, 4, 2, 1])
    starts = np.concatenate([[0], np.cumsum(counts)])
    p = shared_pages(rng, first, shared, lengths, counts, kv, page, dim, cdtype)
    p.pages[:3, 2] = -1  # of the prefix
    p.pages[1, 80 // page] = p.num + 3  # of row 1's own
    mask = tree_mask(rng, counts)
    mask[-1] = 0  # the last sequence has no committed tokens and its node sees nothing
    mask[:, 0] &= ~np.uint32(2)  # nobody sees node 1
    bad = to_dtype(np.array([np.nan, np.inf, -np.inf]), cdtype)
    k, v = values(p.k), values(p.v)
    used = np.zeros((p.num, page), bool)
    for b, n in enumerate(lengths + counts):
        for pos in range(n):
            at = p.place(b, pos)
            if at and pos != lengths[b] + 1:
                used[at] = True
    for pg in range(p.num):
        for s in range(page):
            if not used[pg, s]:
                p.k[0, pg, :, s], p.v[0, pg, :, s] = bad[(pg + s) % 3], bad[(pg + s + 1) % 3]
    q = to_dtype(rng.normal(0, 1, (int(starts[-1]), heads, dim)), dtype)
    got = call(sess, p, q, dtype, starts, first, shared, mask, 0.125, max_nodes=4, max_tokens=120)
    want, mass, size = attention(p, 0, values(q), starts, range(5), seen_by(mask, starts), 0.125, 4)
    assert np.isfinite(want).all() and (want[-1] == 0).all()
    assert (np.abs(got - want) <= attention_bound(want, mass, size, dim, 120, dtype, cdtype)).all()


def test_infinities_that_are_seen(sess):
    """An infinity or a NaN in a value of the prefix reaches every row of the group, one in a rest its own rows only; a key
    of −Inf hides its token."""
    announce("prefix infinities")
    rng = np.random.default_rng(4)
    heads, kv, dim, page = 6, 1, 64, 8
    first, shared, lengths, counts = np.array([0, 4]), np.array([50]), np.array([55, 60, 50, 52]), np.array([1, 2, 1, 1])
    starts = np.concatenate([[0], np.cumsum(counts)])
    for dtype, cdtype in TYPES[:3]:
        p = shared_pages(rng, first, shared, lengths, counts, kv, page, dim, cdtype)
        for pos, d, x in ((7, 3, np.inf), (20, 5, -np.inf), (33, 5, np.inf), (41, 60, np.nan)):
            pg, s = p.place(0, pos)
            p.v[0, pg, 0, s, d] = to_dtype(np.array([x]), cdtype)[0]
        pg, s = p.place(1, 57)
        p.v[0, pg, 0, s, 11] = to_dtype(np.array([np.inf]), cdtype)[0]
        q = to_dtype(rng.normal(0, 1, (int(starts[-1]), heads, dim)), dtype)
        got = call(sess, p, q, dtype, starts, first, shared, None, 0.125)
        want, mass, size = attention(p, 0, values(q), starts, range(4), seen_by(None, starts), 0.125, 9)
        fine = np.isfinite(want)
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
        assert not fine[:, :, [3, 5, 60]].any() and not fine[1:3, :, 11].any() and fine[[0, 3, 4], :, 11].all()
        with np.errstate(invalid="ignore"):
            off = np.abs(got - want) <= attention_bound(want, np.where(np.isfinite(mass), mass, 1.0), size, dim, 64, dtype, cdtype)
        assert off[fine].all()


@pytest.mark.parametrize("scale", [0.0, -0.3, 40.0])
def test_scales_layers_rows_and_strides(sess, scale):
    """Rows of the table in any order (and one it does not have), a layer past the first, heads in columns of a wider matrix
    in place, slots of all heads together."""
    announce(f"prefix scales {scale}")
    rng = np.random.default_rng(5)
    heads, kv, dim, page = 4, 2, 64, 16
    batch = 6
    order = np.array([3, 0, 5, 1, 2, 4])
    first, shared = np.array([1, 4, 6]), np.array([48, 21])
    base = np.array([0, 48, 48, 48, 21, 21])
    lengths, counts = base + rng.integers(0, 20, batch), rng.integers(1, 4, batch)
    starts = np.concatenate([[0], np.cumsum(counts)])
    p = shared_pages(rng, first, shared, lengths, counts, kv, page, dim, L.DT_BF16, layers=2)
    pages, lens = p.pages.copy(), p.len.copy()
    p.pages[order], p.len[order] = pages, lens
    total = int(starts[-1])
    wide = to_dtype(rng.normal(0, 1, (total, heads * dim + 24)), L.DT_F32)
    q = np.ascontiguousarray(wide[:, 8:8 + heads * dim]).reshape(total, heads, dim)
    rows = order.copy()
    rows[0] = 9  # not in the table: zeros
    cache, table = p.upload(sess, True)
    dq = sess.to_device(wide)
    ins = [sess.to_device(np.asarray(a, np.int32)) for a in (starts, first, shared, rows)]
    view = Heads(dq, total, heads, dim, 8, heads * dim + 24, dim)
    sess.prefix_attention(view, cache, table, ins[0], view, ins[1], ins[2], rows=ins[3], layer=1, scale=scale)
    out = dq.numpy()
    want, mass, size = attention(p, 1, values(q), starts, rows, seen_by(None, starts), np.float64(np.float32(scale)), 9)
    got = out[:, 8:8 + heads * dim].reshape(total, heads, dim).astype(np.float64)
    assert (np.abs(got - want) <= attention_bound(want, mass, size, dim, 80, L.DT_F32, L.DT_BF16)).all()
    assert np.array_equal(out[:, :8], wide[:, :8]) and np.array_equal(out[:, 8 + heads * dim:], wide[:, 8 + heads * dim:])
    free_all(cache, table, dq, *ins)


def test_limits(sess):
    """Nodes past max_nodes give no output, positions past max_tokens are not seen, tokens in common past max_shared are not
    shared but seen all the same; tokens outside all sequences keep their output."""
    announce("prefix limits")
    rng = np.random.default_rng(6)
    heads, kv, dim, page = 4, 1, 64, 16
    first, shared = np.array([0, 3]), np.array([100])
    lengths, counts = np.array([110, 100, 130]), np.array([4, 2, 3])
    starts = np.concatenate([[2], 2 + np.cumsum(counts)])
    p = shared_pages(rng, first, shared, lengths, counts, kv, page, dim, L.DT_F32)
    q = rng.normal(0, 1, (int(starts[-1]) + 3, heads, dim)).astype(np.float32)
    for limits in (dict(max_nodes=2), dict(max_tokens=105), dict(max_tokens=60), dict(max_shared=40), dict(max_shared=1)):
        got = call(sess, p, q, L.DT_F32, starts, first, shared, None, 0.1, **limits)
        want, mass, size = attention(p, 0, q.astype(np.float64), starts, range(3), seen_by(None, starts), np.float64(np.float32(0.1)),
                                     limits.get("max_nodes", 9), limits.get("max_tokens", 0))
        bound = attention_bound(want, mass, size, dim, 140, L.DT_F32, L.DT_F32)
        out = np.ones(len(q), bool)
        for b in range(3):
            n = min(counts[b], limits.get("max_nodes", 9))
            out[starts[b]:starts[b] + n] = False
        assert (got[out] == 7).all()
        assert (np.abs(got - want) <= bound)[~out].all(), limits


def test_sequences_that_have_ended(sess):
    """A padded batch: sequences without tokens, with an empty row or none, at the head of a group and in its middle."""
    announce("prefix padded")
    rng = np.random.default_rng(9)
    heads, kv, dim, page = 4, 2, 64, 16
    first, shared = np.array([0, 5, 8]), np.array([90, 40])
    lengths, counts = np.array([90, 95, 100, 90, 97, 40, 44, 41]), np.array([0, 0, 2, 0, 1, 0, 3, 1])
    starts = np.concatenate([[0], np.cumsum(counts)])
    p = shared_pages(rng, first, shared, lengths, counts, kv, page, dim, L.DT_BF16)
    q = to_dtype(rng.normal(0, 1, (int(starts[-1]), heads, dim)), L.DT_F32)
    rows = np.array([-1, 1, 2, 99, 4, 5, 6, 7])
    for b in (1, 5):  # freed rows
        p.len[b], p.pages[b] = 0, -1
    got = call(sess, p, q, L.DT_F32, starts, first, shared, None, 0.125, rows=rows)
    want, mass, size = attention(p, 0, values(q), starts, rows, seen_by(None, starts), 0.125, 9)
    assert (np.abs(want) > 0).all()
    assert (np.abs(got - want) <= attention_bound(want, mass, size, dim, 110, L.DT_F32, L.DT_BF16)).all()


def test_bad_groups_stay_within_the_buffers(sess):
    """Bounds that do not rise or lie outside the batch, negative counts: whatever the result, sequences of no bad group keep
    theirs."""
    announce("prefix bad groups")
    rng = np.random.default_rng(7)
    heads, kv, dim, page = 4, 2, 64, 16
    lengths, counts = np.full(6, 64), np.full(6, 2)
    starts = np.arange(7) * 2
    p = shared_pages(rng, [0, 6], [64], lengths, counts, kv, page, dim, L.DT_BF16)
    q = to_dtype(rng.normal(0, 1, (12, heads, dim)), L.DT_F32)
    alone = call(sess, p, q, L.DT_F32, starts, [0, 6], [64], plain=True)
    for first, shared in (([-5, 3, 9], [64, 64]), ([4, 2, 6], [10, 64]), ([2 ** 31 - 1, -2 ** 31, 6], [64, 64]),
                          ([0, 3, 6], [-7, 2 ** 31 - 1]), ([6, 6, 6], [3, 3])):
        call(sess, p, q, L.DT_F32, starts, first, shared)
    got = call(sess, p, q, L.DT_F32, starts, [0, 3, 6], [-7, 32])
    assert np.abs(got - alone).max() <= 2.0 ** -16


@pytest.mark.parametrize("batch,shared", [(3, 200), (40, 3000)])
def test_routes(env_session, batch, shared):
    """Prefixes once, each sequence alone, and whichever the sizes choose: few short ones alone, many long ones once."""
    announce(f"prefix routes {batch} {shared}")
    rng = np.random.default_rng(8)
    heads, kv, dim, page = 8, 8, 128, 16
    first, common = np.array([0, batch]), np.array([shared])
    lengths, counts = shared + rng.integers(0, 20, batch), np.ones(batch, int)
    starts = np.arange(batch + 1)
    p = shared_pages(rng, first, common, lengths, counts, kv, page, dim, L.DT_BF16)
    q = to_dtype(rng.normal(0, 1, (batch, heads, dim)), L.DT_F32)
    kw = dict(max_nodes=1, max_tokens=shared + 21, max_shared=shared)
    once, alone, chosen = (call(env_session(INGOT_PREFIX_PATH=i), p, q, L.DT_F32, starts, first, common, **kw) for i in (2, 1, 0))
    plain = call(env_session(INGOT_PREFIX_PATH=0), p, q, L.DT_F32, starts, first, common, plain=True, **kw)
    assert np.array_equal(alone, plain) and not np.array_equal(once, alone)
    assert np.array_equal(chosen, alone if batch == 3 else once)
    top = np.abs(values(p.v)).max()
    assert np.abs(once - alone).max() <= 2 * (4 * (dim + 8) * 2.0 ** -24 * 12 + (shared + 90) * 2.0 ** -24) * top


def test_nothing_to_do_and_refusals(sess):
    announce("prefix refusals")
    z = sess.empty(L.DT_F32, (0, 2, 8))
    k = sess.empty(L.DT_BF16, (1, 2, 1, 4, 8))
    cache = KvCache(k, k)
    table = KvTable(sess.to_device(np.zeros((2, 2), np.int32)), sess.to_device(np.zeros(2, np.int32)))
    i = {n: sess.to_device(np.zeros(n, np.int32)) for n in (1, 2, 3, 4)}
    sess.prefix_attention(z, cache, table, i[3], z, i[2], i[1])
    q = sess.to_device(np.ones((3, 2, 8), np.float32))
    none = sess.empty(L.DT_I32, (0,))
    starts = sess.to_device(np.array([0, 2, 3], np.int32))
    sess.prefix_attention(q, cache, table, starts, q, i[1], none)  # no groups: the attention of each alone
    sess.sync()

    def refused(code, text, *a, **kw):
        with pytest.raises(IngotError, match=text) as e:
            sess.prefix_attention(*a, **kw)
        assert e.value.code == code

    refused(L.EINVAL, "groups=3 of 2", q, cache, table, starts, q, i[4], i[3])
    refused(L.EINVAL, "bad sizes", q, cache, table, starts, q, i[2], i[1], max_shared=-1)
    refused(L.EINVAL, "layer", q, cache, table, starts, q, i[2], i[1], layer=1)
    refused(L.EINVAL, "scale", q, cache, table, starts, q, i[2], i[1], scale=float("nan"))
    refused(L.EINVAL, "max_tokens=-1", q, cache, table, starts, q, i[2], i[1], max_tokens=-1)
    with pytest.raises(ValueError, match="first"):
        sess.prefix_attention(q, cache, table, starts, q, i[1], i[1])
    with pytest.raises(ValueError, match="differ"):
        sess.prefix_attention(q, cache, table, starts, z, i[2], i[1])
    hq = Heads(q)
    args = L.TreeAttentionArgs(2, 3, 0, None, 0, hq.c, hq.c, L.DT_F32, 0.5)
    batch = L.KvBatchDesc(starts.ptr, None, 2, 3, 0)
    for prefix, text in ((None, "nil prefix"), (L.KvPrefixDesc(None, i[1].ptr, 1, 0), "nil groups"),
                         (L.KvPrefixDesc(i[2].ptr, None, 1, 0), "nil groups"), (L.KvPrefixDesc(i[2].ptr, i[1].ptr, -1, 0), "bad sizes")):
        with pytest.raises(IngotError, match=text):
            L.check(sess.lib.ingot_rocm_prefix_attention(sess.h, C.byref(cache.c), C.byref(table.c), C.byref(batch),
                                                         None if prefix is None else C.byref(prefix), C.byref(args)))

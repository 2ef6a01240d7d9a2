"""Attention over shared prefixes where starts or groups do not rise and the items of their spans would pass 2^31: nothing is
read or written outside the buffers, and what is sound keeps its result."""
import numpy as np
import pytest

from decoder_reference import free_all, to_dtype, values
from helpers import announce
from ingot_amd import KvCache, KvTable
from ingot_amd import _lib as L

pytestmark = pytest.mark.gpu


def setting(sess, rng, batch, tokens):
    """Rows of 9 committed tokens on one of 64 pages of 16 slots; one head of 8 dimensions."""
    pages = [sess.to_device(to_dtype(rng.normal(0, 1, (1, 64, 1, 16, 8)), L.DT_BF16), L.DT_BF16) for _ in range(2)]
    cache = KvCache(*pages)
    table = KvTable(sess.to_device((np.arange(batch) % 64).astype(np.int32)[:, None]),
                    sess.to_device(np.full(batch, 9, np.int32)))
    q = sess.to_device(to_dtype(rng.normal(0, 1, (tokens, 1, 8)), L.DT_BF16), L.DT_BF16)
    return cache, table, q


def test_groups_that_do_not_rise(env_session):
    """2^18 bounds that are 0 and nearly the batch in turn: half of the groups have all tokens, 2^33 items. The sequences behind
    them have what they have alone."""
    announce("prefix bad groups of many items")
    s, rng = env_session(INGOT_PREFIX_PATH=2), np.random.default_rng(51)
    batch, tokens = 1 << 18, 1 << 20
    cache, table, q = setting(s, rng, batch, tokens)
    starts = s.to_device((np.arange(batch + 1) * 4).astype(np.int32))
    bounds = np.zeros(batch + 1, np.int32)
    bounds[1::2] = batch - 6
    first, shared = s.to_device(bounds), s.to_device(np.full(batch, 5, np.int32))
    y, alone = (s.to_device(np.zeros((tokens, 1, 8), np.uint16), L.DT_BF16) for _ in range(2))
    limits = dict(max_nodes=4, max_tokens=13)
    s.prefix_attention(q, cache, table, starts, y, first, shared, max_shared=5, **limits)
    s.tree_attention(q, cache, table, starts, alone, **limits)
    got, want = values(y.numpy())[-24:], values(alone.numpy())[-24:]
    # each rounds its probabilities to bf16 (2^-8 of the mass of |v|, at most its largest) and its result (2^-8 of itself)
    top = np.abs(values(cache.v.numpy())).max()
    assert (np.abs(want) > 0).all() and (np.abs(got - want) <= 2 * 2.0 ** -8 * (top + np.maximum(np.abs(got), np.abs(want)))).all()
    free_all(cache, table, q, starts, first, shared, y, alone)


def test_starts_that_do_not_rise(env_session):
    """2^18 starts that are 0 and all tokens in turn: half of the sequences have all tokens, 2^32 items of 128 rows. What comes of
    them is not specified; a sound call after it has its result."""
    announce("prefix bad starts of many items")
    s, rng = env_session(INGOT_PREFIX_PATH=2), np.random.default_rng(52)
    batch, tokens = 1 << 18, 1 << 22
    cache, table, q = setting(s, rng, batch, tokens)
    bad = np.zeros(batch + 1, np.int32)
    bad[1::2] = tokens
    ends = np.minimum(np.arange(batch + 1) * 2, 64)
    group = s.to_device(np.array([0, 8], np.int32)), s.to_device(np.array([0], np.int32))
    y = s.to_device(np.zeros((tokens, 1, 8), np.uint16), L.DT_BF16)
    results = []
    for starts in (ends, bad, ends):
        d = s.to_device(starts.astype(np.int32))
        s.prefix_attention(q, cache, table, d, y, *group, max_shared=1)
        results.append(values(y.numpy())[:64])
        d.free()
    assert np.isfinite(results[0]).all() and (np.abs(results[0]) > 0).all() and np.array_equal(results[0], results[2])
    free_all(cache, table, q, y, *group)

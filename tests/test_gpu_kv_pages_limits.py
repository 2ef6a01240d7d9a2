"""Pages asked for at the ends of the ranges: the count of what is missing past 31 bits."""
import numpy as np
import pytest

from decoder_reference import free_all
from helpers import announce
from ingot_amd import KvCache, KvTable
from ingot_amd import _lib as L
from test_gpu_kv_pages import Model, ints, same

pytestmark = pytest.mark.gpu

INT_MAX = 2 ** 31 - 1


@pytest.mark.parametrize("rows,page", [(3, 4), (4, 4), (7, 4), (8, 4), (12, 4), (16, 4), (1, 1), (2, 1), (3, 1)])
@pytest.mark.parametrize("wide", [False, True])
def test_what_is_missing_past_31_bits(sess, rows, page, wide):
    """Every row asks for 2^31 − 1 tokens: the sum of what they lack passes 31 and 32 bits (8 rows with pages of 4 lack
    2^32 pages) and stops at 2^31 − 1. `wide`: the first row asks for what it has room for and the pool has not."""
    announce(f"kv_reserve missing {rows} {page} {wide}")
    k = sess.empty(L.DT_BF16, (1, 6, 1, page, 8))
    most = 64 if wide else 2
    lengths = np.zeros(rows, np.int32)
    table = KvTable(ints(sess, np.full((rows, most), -1)), ints(sess, lengths), ints(sess, [0] * 6), ints(sess, [5]))
    asks = np.full(rows, INT_MAX)
    lacking = rows * -(-INT_MAX // page)
    if wide:
        asks[0] = 60 * page  # within its row, more than the pool
        lacking += 60 - -(-INT_MAX // page)
    dr, dt = ints(sess, np.arange(rows)), ints(sess, asks)
    sess.kv_reserve(KvCache(k, k), table, dr, dt)
    assert int(table.missing.numpy()[0]) == min(lacking, INT_MAX)
    assert (table.pages.numpy() == -1).all() and not table.references.numpy().any()
    free_all(k, table, dr, dt)


def test_reserve_of_all_there_could_be(sess):
    """The request for 2^31 − 1 tokens of test_reserve, with the sum compared."""
    announce("kv_reserve missing many")
    rng = np.random.default_rng(40)
    m = Model(rng, 1, 40, 16, 1, 4, 8, L.DT_BF16, rng.integers(0, 20, 40), spare=87)
    cache, table = m.upload(sess, refs=True)
    rows = rng.permutation(40).astype(np.int32)
    tokens = np.full(40, INT_MAX, np.int32)
    tokens[::3] = 5
    dr, dt = ints(sess, rows), ints(sess, tokens)
    sess.kv_reserve(cache, table, dr, dt)
    missing = m.reserve(rows, tokens)
    assert missing > 2 ** 32
    same(m, cache, table, False, INT_MAX)
    free_all(cache, table, dr, dt)


@pytest.mark.parametrize("length,tokens,page", [(5, INT_MAX, 4), (INT_MAX, INT_MAX, 16), (1, INT_MAX, 1 << 20),
                                                (INT_MAX - 6, 6, 16), (INT_MAX - 6, 7, 24)])
def test_lengths_past_31_bits(sess, length, tokens, page):
    """A row of more tokens than 31 bits count lacks their pages, not 2^31 of them."""
    announce(f"kv_reserve length {length} {tokens} {page}")
    k = sess.empty(L.DT_BF16, (1, 2, 1, 16, 8))
    cache = KvCache(k, k)
    cache.c.page_size = page  # the call reads and writes the table alone
    table = KvTable(ints(sess, [[0, -1, -1]]), ints(sess, [length]), ints(sess, [1, 0]), ints(sess, [5]))
    dr, dt = ints(sess, [0]), ints(sess, [tokens])
    sess.kv_reserve(cache, table, dr, dt)
    assert int(table.missing.numpy()[0]) == -(-(length + tokens) // page) - 1
    assert table.pages.numpy().tolist() == [[0, -1, -1]] and table.references.numpy().tolist() == [1, 0]
    free_all(k, table, dr, dt)

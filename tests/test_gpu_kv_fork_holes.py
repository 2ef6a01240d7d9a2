"""Forks of rows whose part-filled page is not there."""
import numpy as np
import pytest

from decoder_reference import free_all
from helpers import announce
from test_gpu_kv_pages import DTYPES, Model, ints, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("children", [1, 300])
@pytest.mark.parametrize("hole", [-1, -7, "past"])
def test_fork_of_a_row_with_a_hole(sess, dtype, children, hole):
    """A source whose part-filled page is not there: its copies have none there either (and take none from the pool),
    whatever the free pages still hold."""
    announce(f"kv_fork hole {dtype} {children} {hole}")
    rng = np.random.default_rng(children)
    lengths = [11, 9] + [0] * (2 * children)
    m = Model(rng, 1, 2 + 2 * children, 4, 1, 4, 8, dtype, lengths, spare=2 * children + 3)
    lost = m.pages[0, 2]
    m.pages[0, 2] = m.num if hole == "past" else hole
    m.refs[lost] = 0
    cache, table = m.upload(sess, refs=True)
    src, dst = np.arange(2 * children) % 2, 2 + rng.permutation(2 * children)
    ds, dd = ints(sess, src), ints(sess, dst)
    sess.kv_fork(cache, table, ds, dd)
    kept = m.len.copy()
    m.len[0] = 8  # forked as if the row ended before its hole
    missing = m.fork(src, dst)
    m.len[:] = kept
    m.len[dst] = m.len[src]
    same(m, cache, table, False, missing)
    assert missing == 0
    free_all(cache, table, ds, dd)

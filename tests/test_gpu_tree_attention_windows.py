"""Attention over more pages than one table of offsets (1024 of them) holds, in both forms of the kernel, with pages that are
not there in some of the tables' windows and not in others."""
import numpy as np
import pytest

from decoder_reference import to_dtype
from helpers import announce
from ingot_amd import _lib as L
from test_gpu_tree_attention import KINDS, Case

pytestmark = pytest.mark.gpu


def stand_in(c, value):
    """Page 0, which is read in place of pages that are not there, leaves the table and holds `value`."""
    p = c.pages
    spare = np.setdiff1d(np.arange(1, p.num), p.pages[p.pages >= 0])
    p.pages[p.pages == 0] = spare[0]
    p.k[:, 0] = p.v[:, 0] = to_dtype(np.array(value), p.dtype).reshape(())


@pytest.mark.parametrize("dtype,cache", KINDS)
@pytest.mark.parametrize("page,length", [(1, 5000), (2, 6500)])
def test_windows_of_shared_rows(sess, dtype, cache, page, length):
    """One sequence among so many that nothing is cut, over five and four tables of offsets; pages are missing in the
    second and the last but one, none in the others."""
    announce(f"shared-row windows {dtype} {cache} {page} {length}")
    lengths = [3] * 1100
    lengths[333] = length
    c = Case(3 + page, dtype, cache, lengths, [1] * 1100, 1, 1, 64, page, layers=1, tree=False)
    stand_in(c, 50.0)
    c.pages.pages[333, [1100, 2047, (length // page // 1024 - 1) * 1024 + 30]] = -1
    c.check(c.run(sess, layer=0), layer=0)


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("tree", [False, True])
def test_windows_of_the_ring(sess, dtype, dim, tree):
    """So many sequences that nothing is cut, one of 80 rows over 3200 pages of one slot: four tables of offsets; pages are
    missing in the second and the last."""
    nodes = 40
    announce(f"ring windows {dtype} {dim} {tree}")
    lengths = [2] * 1100
    lengths[777] = 3200 - nodes
    counts = [1] * 1100
    counts[777] = nodes
    c = Case(dim, dtype, L.DT_BF16, lengths, counts, 2, 1, dim, 1, layers=1, tree=tree)
    stand_in(c, 50.0)
    c.pages.pages[777, [1500, 3100]] = -1
    c.check(c.run(sess, layer=0), layer=0)

"""NaN queries of every bit pattern in the attention over a paged cache: the rows they stand in are NaN."""
import numpy as np
import pytest

from helpers import announce
from ingot_amd import _lib as L
from test_gpu_tree_attention import Case

pytestmark = pytest.mark.gpu

NAN_F32 = [0x7F800001, 0x7F80FFFF, 0xFF800001, 0xFF80FFFF, 0x7F810000, 0xFFBFFFFF, 0x7FC00000, 0xFFFFFFFF]
NAN_BF16 = [0x7F81, 0xFF81, 0x7FC0, 0xFFFF]


@pytest.mark.parametrize("cache", [L.DT_BF16, L.DT_F32])
@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("nodes", [8, 20, 70])
@pytest.mark.parametrize("scale", [0.125, -0.125])
def test_queries_that_are_nan(sess, cache, dtype, nodes, scale):
    """All keys of the dimension are positive: were the NaN an infinity instead, some of the rows' scores would all be
    −Inf and the rows zeros."""
    announce(f"attention NaN queries {cache} {dtype} {nodes} {scale}")
    c = Case(31, dtype, cache, [50], [nodes], 1, 1, 64, 16, layers=1, tree=False, scale=scale)
    k = c.pages.k[..., 5]
    c.pages.k[..., 5] = k & 0x7FFF if k.dtype == np.uint16 else np.abs(k)
    patterns = NAN_F32 if dtype == L.DT_F32 else NAN_BF16
    bits = c.q.view(np.uint32) if dtype == L.DT_F32 else c.q
    odd = range(1, nodes, 2)
    for n, t in enumerate(odd):
        bits[t, 0, 5] = patterns[n % len(patterns)]
    got = c.run(sess, layer=0)
    assert np.isnan(got[list(odd)]).all()
    c.check(got, layer=0, skip=odd)

"""Attention over shared prefixes for sequences of a group that have tokens and no row of the table: the same on both routes."""
import numpy as np
import pytest

from decoder_reference import attention, attention_bound, to_dtype, values
from helpers import announce
from ingot_amd import _lib as L
from test_gpu_prefix_attention import call, seen_by, shared_pages

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,cdtype", [(L.DT_F32, L.DT_BF16), (L.DT_BF16, L.DT_BF16), (L.DT_F32, L.DT_F32)])
@pytest.mark.parametrize("path", [1, 2])
def test_tokens_without_a_row_give_zeros(env_session, path, dtype, cdtype):
    """Slots of a fixed batch whose request has ended, at the head of a group, in its middle and at its end, and a group of
    nothing else."""
    announce(f"prefix row-less {path} {dtype} {cdtype}")
    rng = np.random.default_rng(31)
    heads, kv, dim, page = 8, 2, 64, 16
    first, shared = np.array([0, 4, 6, 9]), np.array([90, 33, 50])
    lengths = np.repeat(shared, np.diff(first)) + rng.integers(0, 20, 9)
    counts = np.array([1, 2, 1, 3, 1, 1, 1, 1, 2])
    starts = np.concatenate([[0], np.cumsum(counts)])
    rows = np.array([-1, 1, 9, 3, -1, 2 ** 31 - 1, 6, 7, -2 ** 31])
    p = shared_pages(rng, first, shared, lengths, counts, kv, page, dim, cdtype)
    q = to_dtype(rng.normal(0, 1, (int(starts[-1]), heads, dim)), dtype)
    got = call(env_session(INGOT_PREFIX_PATH=path), p, q, dtype, starts, first, shared, None, 0.125, rows=rows, max_nodes=3,
               max_tokens=130, max_shared=90)
    want, mass, size = attention(p, 0, values(q), starts, rows, seen_by(None, starts), 0.125, 3)
    for b in (0, 2, 4, 5, 8):
        assert (want[starts[b]:starts[b + 1]] == 0).all() and (got[starts[b]:starts[b + 1]] == 0).all(), b
    assert (np.abs(got - want) <= attention_bound(want, mass, size, dim, 130, dtype, cdtype)).all()

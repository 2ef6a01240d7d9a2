"""The route of attention over shared prefixes where the host does not say how long they are at most."""
import numpy as np
import pytest

from decoder_reference import to_dtype
from helpers import announce
from ingot_amd import _lib as L
from test_gpu_prefix_attention import call, shared_pages

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shared", [16, 2000])
def test_prefixes_of_unknown_length_are_not_taken_for_all_of_the_cache(env_session, shared):
    """Sequences of 2000 positions that have 16 in common, or all: without max_shared each is taken alone, with it whichever is
    faster."""
    announce(f"prefix unknown {shared}")
    rng = np.random.default_rng(41)
    heads, kv, dim, page, batch = 8, 8, 128, 16, 40
    first, common = np.array([0, batch]), np.array([shared])
    lengths, counts = np.full(batch, 2000), np.ones(batch, int)
    starts = np.arange(batch + 1)
    p = shared_pages(rng, first, common, lengths, counts, kv, page, dim, L.DT_BF16)
    q = to_dtype(rng.normal(0, 1, (batch, heads, dim)), L.DT_F32)
    s = env_session(INGOT_PREFIX_PATH=0)
    limits = dict(max_nodes=1, max_tokens=2001)
    alone = call(s, p, q, L.DT_F32, starts, first, common, plain=True, **limits)
    once = call(env_session(INGOT_PREFIX_PATH=2), p, q, L.DT_F32, starts, first, common, **limits)
    assert not np.array_equal(once, alone)
    assert np.array_equal(call(s, p, q, L.DT_F32, starts, first, common, **limits), alone)
    known = call(s, p, q, L.DT_F32, starts, first, common, max_shared=shared, **limits)
    assert np.array_equal(known, alone) == (shared == 16)

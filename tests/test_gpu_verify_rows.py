"""Verification through the wrapper over rows of logits that are longer than the vocabulary."""
import numpy as np
import pytest

from decoder_reference import free_all, to_dtype, values
from helpers import announce
from ingot_amd import _lib as L
from test_gpu_verify_drafts import definition, peaked

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("vocab,wide,draft_wide", [(2500, 2560, None), (2500, 2503, 2500), (2047, 2048, 2051), (7, 64, 9)])
def test_padded_rows(sess, dtype, vocab, wide, draft_wide):
    """What lies past the vocabulary would be the largest logit of every row."""
    announce(f"verify padded rows {dtype} {vocab} {wide} {draft_wide}")
    rng = np.random.default_rng(vocab + wide)
    batch, nodes = 5, 4
    total = batch * nodes
    logits = to_dtype(np.full((total, wide), 99.0), dtype)
    logits[:, :vocab] = peaked(rng, total, vocab, dtype)
    draft = None
    if draft_wide:
        draft = to_dtype(np.full((total, draft_wide), 99.0), dtype)
        draft[:, :vocab] = to_dtype(values(logits[:, :vocab]) + rng.normal(0, 0.7, (total, vocab)), dtype)
    tokens, starts = rng.integers(0, 7, total).astype(np.int32), (np.arange(batch + 1) * nodes).astype(np.int32)
    heat = np.array([0.8, 0, 1.2, 1, 0], np.float32)
    au, su = rng.random(total).astype(np.float32), rng.random(batch).astype(np.float32)
    want, near, near_draw = definition(values(logits[:, :vocab]), tokens, starts, None,
                                       None if draft is None else values(draft[:, :vocab]), heat, au, su, nodes)
    assert not near_draw
    dev = [sess.to_device(logits, dtype), sess.to_device(starts), sess.to_device(tokens)]
    out = [sess.empty(L.DT_I32, s) for s in ((batch, nodes), (batch,), (batch,))]
    kw = dict(temperature=sess.to_device(heat), accept_u=sess.to_device(au), sample_u=sess.to_device(su))
    if draft is not None:
        kw["draft"] = sess.to_device(draft, dtype)
    sess.verify_drafts(*dev, *out, vocab=vocab, **kw)
    for o, w in zip(out, want):
        assert np.array_equal(o.numpy(), w)
    free_all(*dev, *out, *kw.values())

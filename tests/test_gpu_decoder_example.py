"""The speculative decoding example on the GPU: the operators between a layer's projections together."""
import importlib.util
import os

import numpy as np
import pytest

from decoder_reference import frequencies, rotate, to_dtype, values
from helpers import announce
from ingot_amd import _lib as L

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "speculative_decoding.py")
    spec = importlib.util.spec_from_file_location("speculative_decoding", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def build(example, sess, seed, **kw):
    """A decoder and its weights as 64-bit matrices (what the device holds: rounded to bf16)."""
    kept = []
    upload = sess.upload_weight

    def spy(w, **k):
        kept.append(values(to_dtype(w, L.DT_BF16)))
        return upload(w, **k)

    sess.upload_weight = spy
    try:
        return example.Decoder(sess, np.random.default_rng(seed), **kw), kept
    finally:
        del sess.upload_weight


def plain_logits(model, weights, text):
    """The decoder in 64 bits, keys and values rounded to the cache's type."""
    h, kv, d, n = model.heads, model.kv, model.dim, len(text)
    x = model.embed[text].astype(np.float64)
    pos = np.arange(n)
    f = pos[:, None] * frequencies(d, 10000.0, L.ROTARY_PLAIN)[None, :]
    for i in range(len(model.layers)):
        qkv, out, up, down = weights[4 * i:4 * i + 4]
        m = (x @ qkv.T).reshape(n, h + 2 * kv, d)
        q, k = (rotate(m[:, a:b], np.cos(f), np.sin(f), pos, False) for a, b in ((0, h), (h, h + kv)))
        k, v = (values(to_dtype(a, L.DT_BF16)) for a in (k, m[:, h + kv:]))
        att = np.zeros((n, h, d))
        for j in range(h):
            s = q[:, j] @ k[:, j * kv // h].T / np.sqrt(d)
            s[np.triu_indices(n, 1)] = -np.inf
            p = np.exp(s - s.max(1, keepdims=True))
            att[:, j] = (p / p.sum(1, keepdims=True)) @ v[:, j * kv // h]
        x = x + att.reshape(n, -1) @ out.T
        u = x @ up.T
        x = x + (u / (1 + np.exp(-u))) @ down.T
    return x @ weights[-1].T


def test_logits_are_the_decoders(example, sess):
    """A key or value next to a rounding boundary may round the other way (2^-8 of itself): through attention, the layers'
    gains of about 1 and the head that moves a logit by a few 2^-8 of the logits' size; a wrong position, page or head
    moves it by all of it."""
    announce("example logits")
    model, weights = build(example, sess, 3, layers=2, rows=3, pages=40, max_tokens=128)
    text = np.random.default_rng(8).integers(0, model.vocab, 45).tolist()
    want = plain_logits(model, weights, text)
    size = np.sqrt((want ** 2).mean())
    parts = [model.step([1], [example.chain(text[:20])])[0]]
    model.accept([1], [list(range(20))])
    model.fork([1], [2])
    # the text's tokens as one branch of a tree, others beside them
    rng = np.random.default_rng(9)
    tree, node = [], {}
    for i, t in enumerate(text[20:]):
        parent = node.get(i - 1, -1)
        if i:
            tree.append((int(rng.integers(0, model.vocab)), parent, i))
        node[i] = len(tree)
        tree.append((t, parent, i))
    path = [node[i] for i in range(25)]
    drafted = model.step([2], [tree])[0]
    parts.append(drafted[path])
    assert np.abs(np.concatenate(parts) - want).max() <= 2.0 ** -4 * size
    # accepted in part, the rest of the text goes on behind what was kept; the forked row is as it was
    model.accept([2], [path[:9]])
    again = model.step([2, 1], [example.chain(text[29:]), example.chain(text[20:])])
    assert np.abs(again[0] - want[29:]).max() <= 2.0 ** -4 * size
    assert np.abs(again[1] - want[20:]).max() <= 2.0 ** -4 * size
    model.drop([1, 2, 0])
    assert not model.table.references.numpy().any() and not model.table.lengths.numpy().any()


@pytest.mark.parametrize("continuations,page", [(1, 16), (4, 16), (3, 5)])
def test_drafts_give_the_same_texts(example, sess, continuations, page):
    announce(f"example texts {continuations} {page}")
    model, _ = build(example, sess, 1, rows=continuations, page_size=page, pages=continuations * (160 // page + 2),
                     max_tokens=160)
    prompt = np.random.default_rng(2).integers(0, model.vocab, 33).tolist()
    single, many = example.generate(model, prompt, continuations, 64, depth=0)
    texts, steps = example.generate(model, prompt, continuations, 64)
    assert texts == single
    assert many == 63 and steps < many
    assert not model.table.references.numpy().any()


def test_too_few_pages_are_reported(example, sess):
    announce("example pages")
    model, _ = build(example, sess, 1, layers=1, rows=1, pages=2, max_tokens=160)
    with pytest.raises(MemoryError, match="pages"):
        model.step([0], [example.chain(list(range(33)))])

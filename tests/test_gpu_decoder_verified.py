"""The speculative decoding example with normed heads, a prompt read once for all rows and drafts verified on the device."""
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
    """A decoder with norms and its weights as 64-bit matrices (what the device holds: rounded to bf16)."""
    kept = []
    upload = sess.upload_weight

    def spy(w, **k):
        kept.append(values(to_dtype(w, L.DT_BF16)))
        return upload(w, **k)

    sess.upload_weight = spy
    try:
        return example.Decoder(sess, np.random.default_rng(seed), norms=True, **kw), kept
    finally:
        del sess.upload_weight


def plain_logits(model, weights, text):
    """The decoder in 64 bits, keys and values rounded to the cache's type."""
    h, kv, d, n = model.heads, model.kv, model.dim, len(text)
    x = model.embed[text].astype(np.float64)
    pos = np.arange(n)
    f = pos[:, None] * frequencies(d, 10000.0, L.ROTARY_PLAIN)[None, :]
    for i, layer in enumerate(model.layers):
        qkv, out, up, down = weights[4 * i:4 * i + 4]
        m = (x @ qkv.T).reshape(n, h + 2 * kv, d)
        wq, wk = (w.numpy().astype(np.float64) for w in layer["norms"])
        q, k = (rotate(a * w / np.sqrt((a * a).mean(-1, keepdims=True) + 1e-6), np.cos(f), np.sin(f), pos, False)
                for a, w in ((m[:, :h], wq), (m[:, h:h + kv], wk)))
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


@pytest.mark.parametrize("path", [0, 2])
def test_texts_are_the_models(example, env_session, path):
    """Greedy texts, verified on the device and by the host, with prompts read once (path 2) and as the sizes choose, are
    the argmax of the decoder in 64 bits, given the same text before, wherever that leads by 2^-5 of the logits' size (a key
    or value next to a rounding boundary moves a logit by a few 2^-8 of it). Drafts save steps."""
    announce(f"verified decoding {path}")
    sess = env_session(INGOT_PREFIX_PATH=path)
    model, weights = build(example, sess, 5, layers=2, rows=3, pages=60, max_tokens=160)
    prompt = np.random.default_rng(6).integers(0, model.vocab, 33).tolist()
    rng = np.random.default_rng(7)
    texts, steps = example.generate(model, prompt, 3, 60, temperature=0.0, rng=rng)
    host, host_steps = example.generate(model, prompt, 3, 60)
    assert steps < 45 and all(len(t) == 93 for t in texts)
    checked = 0
    for found in (texts, host):
        for t in found:
            want = plain_logits(model, weights, t)
            size = np.sqrt((want ** 2).mean())
            order = np.sort(want, axis=1)
            sure = order[:, -1] - order[:, -2] > 2.0 ** -5 * size
            follows = np.argmax(want, axis=1)[33:-1] == np.array(t[34:])
            assert follows[sure[33:-1]].all()
            checked += int(sure[33:-1].sum())
    assert checked > 200
    assert model.table.references.numpy().sum() == 0 and (model.table.lengths.numpy() == 0).all()


@pytest.mark.parametrize("heat", [0.8, 15.0, 60.0])
def test_drawn_texts(example, sess, heat):
    """Texts that are drawn: the same numbers give the same texts; every token has a probability. A token's logit is
    its row of the head, whose one part is the embedding of the token before, times what the layers make of that embedding:
    about 256 (256 squares of normal numbers) for the one that follows in the cycle, against a deviation of 16 · 2.2 times
    the size of a value, 40 to 60, for the 96 others. So at 0.8 and 15 the likeliest nearly always follows; at 60, where it
    leads by some 2 nats, other numbers give another text."""
    announce(f"drawn decoding {heat}")
    model, weights = build(example, sess, 5, layers=1, rows=2, pages=40, max_tokens=160)
    prompt = np.random.default_rng(6).integers(0, model.vocab, 20).tolist()
    runs = [example.generate(model, prompt, 2, 40, temperature=heat, rng=np.random.default_rng(s))[0] for s in (1, 1, 2)]
    assert runs[0] == runs[1]
    assert heat < 60 or runs[0] != runs[2]
    for t in runs[0]:
        want = plain_logits(model, weights, t)[20:-1] / heat
        p = np.exp(want - want.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        assert p[np.arange(len(p)), t[21:]].min() > 1e-7  # 40 draws: such a token has a chance of less than 97 · 40 · 1e-7

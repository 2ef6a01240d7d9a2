"""Verification where a random number lies next to the border of a decision, or nothing is left after one: candidates that have
all of the mass between them, drafts that have the target's probabilities but for a last bit."""
import numpy as np
import pytest

from decoder_reference import free_all, to_dtype, values
from helpers import announce
from ingot_amd import _lib as L

pytestmark = pytest.mark.gpu

BELOW_ONE = np.float32(0.99999994)  # the largest f32 below 1


def weights(row, heat):
    """exp((x − max) / heat) in 64 bits."""
    with np.errstate(under="ignore"):
        return np.exp((row - row.max()) / np.float64(np.float32(heat)))


def child_kept(w, tokens, numbers):
    """The first of the candidates that is kept (their place, or None), each against the sum of what its predecessors left: a
    sum over those tokens and not a difference, so that the last one with a weight is compared with itself."""
    w = w.copy()
    for i, (t, u) in enumerate(zip(tokens, numbers)):
        left = w.sum()
        if w[t] > 0:
            # every sum here is off by less than 10^-14 of itself
            assert left == w[t] or abs(np.float64(u) * left - w[t]) > 1e-12 * w[t], "a number on the border"
            if np.float64(u) * left < w[t]:
                return i
        w[t] = 0.0
    return None


def run(sess, logits, dtype, tokens, starts, heat, au, su, max_accept, parents=None, draft=None):
    batch = len(starts) - 1
    ins = [sess.to_device(logits, dtype)] + [sess.to_device(np.asarray(a, np.int32)) for a in (starts, tokens)]
    out = [sess.to_device(np.full(s, 77, np.int32)) for s in ((batch, max_accept), (batch,), (batch,))]
    kw = {k: sess.to_device(np.asarray(a, np.float32)) for k, a in (("temperature", heat), ("accept_u", au), ("sample_u", su))}
    if parents is not None:
        kw["parents"] = sess.to_device(np.asarray(parents, np.int32))
    if draft is not None:
        kw["draft"] = sess.to_device(draft, dtype)
    sess.verify_drafts(*ins, *out, **kw)
    got = [t.numpy() for t in out]
    free_all(*ins, *out, *kw.values())
    return got


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("vocab,places", [(3, (0, 1, 2)), (40, (3, 30, 17)), (70001, (9, 2048, 70000))])
def test_the_last_candidate_with_a_weight_is_kept(sess, dtype, vocab, places):
    """Three tokens that are not masked, all proposed, the last of 6e-6: two are turned down, so the third is kept whatever its
    number below 1, and its own row says what follows. The same in a batch that a launch of its own walks."""
    announce(f"verify last candidate {dtype} {vocab}")
    x = np.full((4, vocab), -np.inf, np.float32)
    x[:, places] = [3.83, 5.97, -5.99]
    x[3] = -np.inf
    x[3, places[1]] = 1.0
    logits = to_dtype(x, dtype)
    w = weights(values(logits)[0], 1.0)
    for last in (0.5, 0.985, 0.99, BELOW_ONE):
        numbers = np.array([0.2, 0.999995, last], np.float32)
        assert child_kept(w, places, numbers) == 2
        for batch in (1, 1100 if vocab < 100 else 30):
            got = run(sess, np.tile(logits, (batch, 1)), dtype, np.tile([0, *places], batch), np.arange(batch + 1) * 4,
                      np.ones(batch), np.tile([0, *numbers], batch), np.full(batch, 0.5), 3, np.tile([-1, 0, 0, 0], batch))
            assert (got[0] == [0, 3, -1]).all() and (got[1] == 2).all() and (got[2] == places[1]).all(), (last, batch)


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
def test_all_tokens_proposed(sess, dtype):
    """Rows of 2 to 8 tokens that are not masked, all proposed in any order (some twice, others of nothing among them), with
    numbers next to 1: one of them is always kept, the one that the definition keeps."""
    announce(f"verify all proposed {dtype}")
    rng = np.random.default_rng(21)
    seqs, vocab, nodes = 1500, 2100, 12
    x = np.full((seqs * nodes, vocab), -np.inf, np.float32)
    tokens, au, heat = np.zeros(seqs * nodes, int), np.zeros(seqs * nodes, np.float32), np.ones(seqs, np.float32)
    want = []
    for b in range(seqs):
        root = b * nodes
        m = int(rng.integers(2, 9))
        allowed = rng.permutation(vocab)[:m]
        x[root, allowed] = values(to_dtype(rng.normal(0, 4, m), dtype))
        order = np.concatenate([allowed, rng.integers(0, vocab, 3)])
        order = np.concatenate([rng.permutation(order), np.full(nodes - 1 - len(order), vocab)])
        tokens[root + 1:root + nodes] = order
        au[root + 1:root + nodes] = np.where(rng.random(nodes - 1) < 0.7, BELOW_ONE, rng.uniform(0.999, 1, nodes - 1).astype(np.float32))
        au[root + 1:root + nodes] = np.minimum(au[root + 1:root + nodes], BELOW_ONE)
        heat[b] = rng.uniform(0.5, 2)
        x[root + 1:root + nodes, 5] = 0.0  # what follows a child
        inside = order < vocab
        w = weights(x[root].astype(np.float64), heat[b])
        want.append(1 + np.flatnonzero(inside)[child_kept(w, order[inside], au[root + 1:root + nodes][inside])])
    got = run(sess, to_dtype(x, dtype), dtype, tokens, np.arange(seqs + 1) * nodes, heat, au, np.full(seqs, 0.5), 2,
              np.tile([-1] + [0] * (nodes - 1), seqs))
    assert np.array_equal(got[0][:, 1], want) and (got[1] == 2).all() and (got[2] == 5).all(), (
        np.flatnonzero(got[0][:, 1] != want)[:20].tolist())


@pytest.mark.parametrize("children,vocab", [(63, 100), (64, 2048), (200, 5000), (700, 2500)])
def test_more_candidates_than_lanes(sess, children, vocab):
    """All tokens that are not masked proposed in hundreds of nodes, many twice, grandchildren between them; numbers next to 1:
    the one that is kept may be in any of the rounds of 64 nodes."""
    announce(f"verify many candidates {children} {vocab}")
    rng = np.random.default_rng(children)
    seqs, n = 12, children + 1
    x = np.full((seqs * n, vocab), -np.inf, np.float32)
    x[:, 3] = 1.0
    tokens, parents = np.zeros((seqs, n), int), np.zeros((seqs, n), int)
    au = np.full((seqs, n), BELOW_ONE, np.float32)
    want = []
    for b in range(seqs):
        parents[b, 0] = -1
        for i in range(5, n, 5):  # every fifth node is a child of another
            parents[b, i] = rng.integers(1, i)
        of_root = np.flatnonzero(parents[b] == 0)
        allowed = rng.permutation(vocab)[:len(of_root) * 2 // 3]
        x[b * n], x[b * n, allowed] = -np.inf, rng.normal(0, 3, len(allowed))
        tokens[b] = rng.integers(0, vocab, n)
        tokens[b, of_root] = rng.permutation(np.concatenate([allowed, rng.choice(allowed, len(of_root) - len(allowed))]))
        want.append(of_root[child_kept(weights(x[b * n].astype(np.float64), 1.0), tokens[b, of_root], au[b, of_root])])
    got = run(sess, x, L.DT_F32, tokens.ravel(), np.arange(seqs + 1) * n, np.ones(seqs), au.ravel(), np.full(seqs, 0.5), 2,
              parents.ravel())
    assert np.array_equal(got[0][:, 1], want) and (got[1] == 2).all(), (got[0][:, 1].tolist(), want)
    assert (got[2] == 3).all()


@pytest.mark.parametrize("heat,size", [(1e-42, 1e-42), (1e-39, 1e-39), (1e38, 3.3e38), (3e37, 1e38)])
def test_temperatures_past_the_range_of_32_bits(sess, heat, size):
    """Factors that f32 does not hold, and logits whose differences it does not hold though both have a weight."""
    announce(f"verify range {heat}")
    rng = np.random.default_rng(24)
    seqs, n, vocab = 200, 6, 1000
    x = np.full((seqs * n, vocab), -np.inf)
    tokens, au = np.zeros((seqs, n), int), rng.random((seqs, n)).astype(np.float32)
    want = []
    for b in range(seqs):
        allowed = rng.permutation(vocab)[:9]
        x[b * n, allowed] = rng.uniform(-1, 1, 9) * size
        tokens[b, 1:] = allowed[:n - 1]
        x[b * n + 1:b * n + n, 4] = 0.0
    x = x.astype(np.float32)
    for b in range(seqs):
        kept = child_kept(weights(x[b * n].astype(np.float64), heat), tokens[b, 1:], au[b, 1:])
        want.append(-1 if kept is None else kept + 1)
    assert want.count(-1) > 5 and len(set(want)) == n
    got = run(sess, x, L.DT_F32, tokens.ravel(), np.arange(seqs + 1) * n, np.full(seqs, heat), au.ravel(), np.full(seqs, 0.5), 2,
              np.tile([-1] + [0] * (n - 1), seqs))
    assert np.array_equal(got[0][:, 1], want), np.flatnonzero(got[0][:, 1] != want).tolist()
    assert (got[2][np.array(want) > 0] == 4).all()


@pytest.mark.parametrize("vocab", [50, 2049, 30011])
def test_drafts_that_differ_by_a_last_bit(sess, vocab):
    """The draft's logits are the target's, the target's with another last bit, or those 8 higher: every decision falls as in
    the definition, and where a token is turned down what follows comes from what the draft leaves."""
    announce(f"verify near drafts {vocab}")
    rng = np.random.default_rng(22)
    seqs, nodes = 300, 3
    logits = (rng.integers(-4096, 4096, (seqs * nodes, vocab)) / 1024).astype(np.float32)
    draft = logits.copy()
    draft[0::3] += 8
    some = rng.random(logits.shape) < 0.5
    draft[1::3] = np.where(some, np.nextafter(logits, np.float32(9)), logits)[1::3]
    tokens = rng.integers(0, vocab, seqs * nodes)
    starts = np.arange(seqs + 1) * nodes
    au = np.where(rng.random(seqs * nodes) < 0.5, BELOW_ONE, 1 - rng.integers(1, 16, seqs * nodes) * 2.0 ** -24).astype(np.float32)
    su = np.zeros(seqs, np.float32)
    accepted, after = np.full((seqs, nodes), -1), np.full(seqs, -1)
    for b in range(seqs):
        path = [0]
        while True:
            r = b * nodes + path[-1]
            p, q = (weights(a[r].astype(np.float64), 1.0) for a in (logits, draft))
            p, q = p / p.sum(), q / q.sum()
            rest = p
            if path[-1] + 1 < nodes:
                t, u = tokens[r + 1], np.float64(au[r + 1])
                assert abs(u * q[t] - p[t]) > 1e-12 * p[t], "a number on the border"
                if u * q[t] < p[t]:
                    path.append(path[-1] + 1)
                    continue
                rest = np.where(p - q > 1e-12 * p, p - q, 0.0)
            run_sum = np.cumsum(rest)
            # differences of 10^-7 of p, each off by 10^-15 of p: borders are known to 10^-7 of the sum
            while True:
                su[b] = rng.random()
                if np.abs(run_sum - np.float64(su[b]) * run_sum[-1]).min() > 1e-6 * run_sum[-1]:
                    break
            after[b] = np.argmax(run_sum > np.float64(su[b]) * run_sum[-1])
            break
        accepted[b, :len(path)] = path
    turned_down = (accepted[:, -1] < 0).sum()
    assert 10 < turned_down < seqs - 10
    got = run(sess, logits, L.DT_F32, tokens, starts, np.ones(seqs), au, su, nodes, draft=draft)
    assert np.array_equal(got[0], accepted), np.flatnonzero((got[0] != accepted).any(1))[:20].tolist()
    assert np.array_equal(got[2], after), np.flatnonzero(got[2] != after)[:20].tolist()


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
def test_a_draft_that_leaves_nothing(sess, dtype):
    """Where p is nowhere above q the next token is drawn from p: a draft with the target's logits whose token a number of 1 turns
    down, and one that has e^-60 of a token that the target masks."""
    announce(f"verify draft leaves nothing {dtype}")
    rng = np.random.default_rng(23)
    vocab, seqs = 5003, 60
    x = to_dtype(rng.normal(0, 2, (2 * seqs, vocab)), dtype)
    masked = values(x)
    masked[::4, 4100] = -np.inf
    x = to_dtype(masked, dtype)
    y = values(x)
    y[::4, 4100] = -60.0
    tokens = np.full(2 * seqs, 4100)
    au = np.tile(np.array([0, 0.5, 0, 1.0], np.float32), seqs // 2)
    su = rng.random(seqs).astype(np.float32)
    want = []
    for b in range(seqs):
        run_sum = np.cumsum(weights(values(x)[2 * b], 0.8))
        assert np.abs(run_sum - np.float64(su[b]) * run_sum[-1]).min() > 1e-9 * run_sum[-1]
        want.append(np.argmax(run_sum > np.float64(su[b]) * run_sum[-1]))
    got = run(sess, x, dtype, tokens, np.arange(seqs + 1) * 2, np.full(seqs, 0.8), au, su, 2, draft=to_dtype(y, dtype))
    assert (got[1] == 1).all() and np.array_equal(got[2], want), np.flatnonzero(got[2] != want).tolist()

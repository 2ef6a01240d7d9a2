"""Verification of drafted tokens on the GPU, against the definition in 64 bits."""
import ctypes as C

import numpy as np
import pytest

from decoder_reference import free_all, to_dtype, values
from helpers import announce
from ingot_amd import IngotError
from ingot_amd import _lib as L

pytestmark = pytest.mark.gpu


def probabilities(row, heat):
    """softmax(row / heat) in 64 bits, None where the row cannot be used."""
    if np.isnan(row).any() or not np.isfinite(row.max()):
        return None
    with np.errstate(over="ignore", under="ignore"):
        e = np.exp((row - row.max()) / heat)
    return e / e.sum()


def drawn(w, u):
    """(index drawn, distance of the target from the nearest border, relative to the whole)."""
    run = np.cumsum(w)
    if not run[-1] > 0:
        return -1, 1.0
    target = np.float64(u) * run[-1]
    past = np.flatnonzero((run > target) & (w > 0))
    at = past[0] if past.size else np.flatnonzero(w > 0)[-1]
    return int(at), float(np.abs(run - target).min() / run[-1])


def definition(logits, tokens, starts, parents=None, draft=None, heat=None, au=None, su=None, max_accept=1):
    """accepted, counts, next of the definition, and the nodes and sequences whose number lies near a border (an acceptance
    within 2^-18 of p, a draw within 1e-11 of the whole)."""
    batch, total = len(starts) - 1, len(logits)
    accepted, counts, after = np.full((batch, max_accept), -1, np.int32), np.zeros(batch, np.int32), np.full(batch, -1, np.int32)
    near, near_draw = [], []
    for b in range(batch):
        lo, n = int(starts[b]), max(0, min(int(starts[b + 1]), total) - int(starts[b]))
        if lo < 0 or n == 0:
            continue
        t = 0.0 if heat is None else np.float64(heat[b])
        path, usable = [0], t >= 0 and np.isfinite(t)
        while usable:
            row, cur = logits[lo + path[-1]], path[-1]
            p = probabilities(row, t if t > 0 else 1.0)
            children = [i for i in range(1, n) if (parents[lo + i] if parents is not None else i - 1) == cur and i > cur]
            if p is None:
                break
            if t == 0:
                best = int(np.argmax(row))
                kept = next((i for i in children if tokens[lo + i] == best), None) if len(path) < max_accept else None
                if kept is None:
                    after[b] = best
                    break
                path.append(kept)
                continue
            w, gone, kept = p.copy(), 0.0, None
            if len(path) < max_accept:
                for i in children:
                    k = tokens[lo + i]
                    pk = w[k] if 0 <= k < len(p) else 0.0
                    u = np.float64(0 if au[lo + i] < 0 else au[lo + i])
                    if draft is not None:
                        q = probabilities(draft[lo + cur], t)
                        left = u * q[k] if q is not None and 0 <= k < len(p) else np.nan
                    else:
                        left = u * max(1.0 - gone, 0.0)
                    if pk > 0 and abs(left - pk) <= 2.0 ** -18 * pk:
                        near.append(lo + i)
                    if left < pk:
                        kept = i
                        break
                    if draft is not None:
                        w = np.full(len(p), np.nan) if q is None else np.maximum(p - q, 0.0)
                    elif 0 <= k < len(p):
                        gone += w[k]
                        w[k] = 0.0
            if kept is None:
                if not np.isnan(w).any():
                    after[b], gap = drawn(w, su[b])
                    if gap < 1e-11:
                        near_draw.append(b)
                break
            path.append(kept)
        accepted[b, :len(path)], counts[b] = path, len(path)
    return (accepted, counts, after), near, near_draw


def run(sess, logits, dtype, tokens, starts, parents, draft, heat, au, su, max_accept):
    batch = len(starts) - 1
    dev = [sess.to_device(logits, dtype), sess.to_device(starts.astype(np.int32)), sess.to_device(tokens.astype(np.int32))]
    out = [sess.to_device(np.full(s, 77, np.int32)) for s in ((batch, max_accept), (batch,), (batch,))]
    kw = {}
    if parents is not None:
        kw["parents"] = sess.to_device(parents.astype(np.int32))
    if draft is not None:
        kw["draft"] = sess.to_device(draft, dtype)
    for name, a in (("temperature", heat), ("accept_u", au), ("sample_u", su)):
        if a is not None:
            kw[name] = sess.to_device(a.astype(np.float32))
    sess.verify_drafts(*dev, *out, **kw)
    got = [t.numpy() for t in out]
    free_all(*dev, *out, *kw.values())
    return got


def check(sess, logits, dtype, tokens, starts, parents=None, draft=None, heat=None, au=None, su=None, max_accept=4, rng=None):
    """The kernels against the definition. Numbers that lie near a border are drawn again (with `rng`) before the run."""
    for _ in range(20):
        want, near, near_draw = definition(values(logits), tokens, starts, parents, None if draft is None else values(draft),
                                           heat, au, su, max_accept)
        if rng is None or not (near or near_draw):
            break
        au[near], su[near_draw] = rng.random(len(near)), rng.random(len(near_draw))
    got = run(sess, logits, dtype, tokens, starts, parents, draft, heat, au, su, max_accept)
    for g, w, name in zip(got, want, ("accepted", "counts", "next")):
        assert np.array_equal(g, w), f"{name}: {g.tolist()} but {w.tolist()}"[:2000]
    return want


def trees(rng, counts, vocab):
    """Parents and tokens of random trees, children among the first tokens of the vocabulary (which `logits` favours)."""
    parents, tokens = [], []
    for n in counts:
        parents += [-1][:n] + [int(rng.integers(max(0, i - 6), i)) for i in range(1, n)]
        tokens += [int(x) for x in rng.integers(0, min(vocab, 7), n)]
    return np.array(parents, np.int32), np.array(tokens, np.int32)


def peaked(rng, rows, vocab, dtype):
    x = rng.normal(0, 1.5, (rows, vocab))
    x[:, :7] += np.log(vocab) + rng.normal(0, 2, (rows, min(vocab, 7)))
    return to_dtype(x, dtype)


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("kind", ["tree", "chain", "draft"])
@pytest.mark.parametrize("batch,nodes,vocab", [
    (1, 1, 1), (1, 1, 33), (3, 5, 7), (2, 9, 2048), (5, 4, 2049), (1, 3, 20011), (1, 1, 70001), (4, 17, 4096), (7, 2, 5000),
    (130, 3, 50), (6, 70, 300), (2, 200, 64), (3, 6, 40003), (2, 2, 140001), (1, 1, 300007), (700, 2, 9)])
def test_verify(sess, dtype, kind, batch, nodes, vocab):
    """Sequences of all lengths from none on, one of four greedy; rows before the first and behind the last sequence."""
    announce(f"verify {dtype} {kind} {batch} {nodes} {vocab}")
    rng = np.random.default_rng(batch * 100000 + nodes * 1000 + vocab)
    counts = rng.integers(0 if batch > 1 else 1, nodes + 1, batch)
    counts[0] = nodes
    starts = np.concatenate([[0], np.cumsum(counts)]) + 2
    total = int(starts[-1]) + 3
    parents, tokens = trees(rng, [2, *counts, 3], vocab)
    heat = rng.uniform(0.3, 1.5, batch).astype(np.float32)
    heat[1::4] = 0
    au, su = rng.random(total).astype(np.float32), rng.random(batch).astype(np.float32)
    logits = peaked(rng, total, vocab, dtype)
    draft = None
    if kind == "draft":
        draft = to_dtype(values(logits) + rng.normal(0, 0.7, logits.shape), dtype)
    want = check(sess, logits, dtype, tokens, starts, parents if kind == "tree" else None, draft, heat, au, su, nodes, rng)
    assert vocab < 7 or batch < 100 or len(set(want[1].tolist())) > 2  # paths of several lengths


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
def test_greedy_takes_the_first_of_equal_ones(sess, dtype):
    """Ties between places of one chunk, of two chunks and of many; no random numbers are given."""
    announce(f"verify greedy {dtype}")
    rng = np.random.default_rng(1)
    vocab, n = 9001, 12
    logits = rng.integers(-3, 3, (n, vocab)).astype(np.float32)
    logits[:, [4000, 4001, 8999]] = 5
    logits[3, 17] = logits[5, 9000] = 6
    logits[7] = 2
    tokens = np.array([0, 4000, 4000, 4001, 17, 4000, 9000, 4000, 0, 4000, 4000, 8999])
    want = check(sess, to_dtype(logits, dtype), dtype, tokens, np.array([0, 3, 6, 10, 12]), max_accept=5)
    # row 3 gives 17, row 4 the first of 4000, 4001, 8999; row 6 that too, row 7 (all alike) 0; row 10 gives 4000 and not 8999
    assert want[1].tolist() == [3, 3, 4, 1]


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("greedy", [False, True])
def test_rows_that_cannot_be_used(sess, dtype, greedy):
    """A NaN, an infinity, a row of −Inf, as the first row of a sequence and as a later one; temperatures that are none.
    Logits of −Inf otherwise: their tokens never follow, and their children are never kept."""
    announce(f"verify bad rows {dtype} {greedy}")
    rng = np.random.default_rng(2)
    vocab, seqs = 3000, 9
    x = np.full((2 * seqs, vocab), -np.inf, np.float32)
    x[:, 5:20] = rng.normal(0, 1, (2 * seqs, 15))
    x[0::2, 7] = 30  # the first child (token 7) is kept
    x[0, 2999], x[3, 2048] = np.nan, np.nan
    x[4, 9], x[7, 2999] = np.inf, np.inf
    x[8], x[11] = -np.inf, -np.inf
    tokens = np.tile([3, 7], seqs)
    tokens[13] = 2000  # −Inf
    heat = np.full(seqs, 0.0 if greedy else 0.8, np.float32)
    heat[7], heat[8] = -1.0, np.nan
    au, su = np.full(2 * seqs, 0.5, np.float32), np.linspace(0.1, 0.9, seqs).astype(np.float32)
    starts = np.arange(seqs + 1) * 2
    want = check(sess, to_dtype(x, dtype), dtype, tokens, starts, None, None, heat, au, su, 2)
    assert want[1].tolist() == [1, 2, 1, 2, 1, 2, 1, 1, 1]
    assert [v < 0 for v in want[2].tolist()] == [True, True, True, True, True, True, False, True, True]
    heat[7] = np.inf
    check(sess, to_dtype(x, dtype), dtype, tokens, starts, None, None, heat, au, su, 2)
    draft = to_dtype(np.where(np.arange(vocab)[None, :] < 30, 0.0, -np.inf) + np.zeros(x.shape), dtype)
    draft[2] = to_dtype(np.full(vocab, np.nan), dtype)  # a draft row that cannot be used: turned down, nothing follows
    check(sess, to_dtype(x, dtype), dtype, tokens, starts, None, draft, heat, au, su, 2)


@pytest.mark.parametrize("heat", [1e-40, 1e-3, 50.0, 3e38])
def test_extreme_temperatures(sess, heat):
    """From one that leaves only the largest logit to one that leaves all tokens alike."""
    announce(f"verify temperature {heat}")
    rng = np.random.default_rng(3)
    vocab, n = 5003, 4
    logits = rng.normal(0, 3, (n, vocab)).astype(np.float32)
    tokens = np.array([0, int(np.argmax(logits[0])), 17, 18])
    au, su = rng.random(n).astype(np.float32), np.array([0.73, 0.2], np.float32)
    check(sess, logits, L.DT_F32, tokens, np.array([0, 2, 4]), None, None, np.full(2, heat, np.float32), au, su, 2, rng)


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
def test_logits_at_the_ends_of_their_type(sess, dtype):
    """Tokens masked by the type's lowest value instead of −Inf never follow; where all have it, or the largest one, they are
    alike."""
    announce(f"verify lowest {dtype}")
    rng = np.random.default_rng(10)
    vocab, n = 3001, 5
    low = -3.3895313892515355e38  # the lowest bf16, and no f32's lowest by far less than a step of bf16
    x = np.full((n, vocab), low, np.float32)
    x[0, 100:120] = rng.normal(0, 2, 20)
    x[2, 50] = -low
    x[3] = -low
    tokens, heat = np.array([0, 110, 0, 0, 0]), np.full(5, 0.7, np.float32)
    su = rng.random(5).astype(np.float32)
    want = check(sess, to_dtype(x, dtype), dtype, tokens, np.arange(6), None, None, heat, su, su, 1, rng)
    assert 100 <= want[2][0] < 120 and want[2][2] == 50
    x[:] = np.finfo(np.float32).min if dtype == L.DT_F32 else low
    x[1, 7] = 3.0
    want = check(sess, to_dtype(x, dtype), dtype, tokens, np.arange(6), None, None, heat, su, su, 1, rng)
    assert want[2][1] == 7


def test_bad_tokens_and_parents(sess):
    """Tokens outside the vocabulary and parents that do not come before their child are never kept, and repeated tokens of
    one parent have nothing left; across more than 64 children too."""
    announce("verify bad nodes")
    rng = np.random.default_rng(4)
    vocab, n = 600, 150
    logits = rng.normal(0, 0.3, (2 * n, vocab)).astype(np.float32)
    logits[:, 11] += 7  # nearly all of p
    parents = np.zeros(2 * n, np.int32)
    parents[[0, n]] = -1
    tokens = np.tile(rng.permutation(vocab)[:n], 2)
    tokens[tokens == 11] = 12
    parents[5], parents[6], parents[7], parents[8] = 5, 9, -3, 2 ** 31 - 1
    tokens[[5, 6, 7, 8, 9]] = 11
    parents[9] = -2 ** 31
    tokens[10], tokens[20], tokens[30] = vocab, -1, -2 ** 31
    tokens[n + 2], tokens[n + 70], tokens[n + 140], tokens[n + 141] = 11, 11, 11, 44
    au = np.full(2 * n, 0.9, np.float32)
    au[[n + 2, n + 70, n + 140]] = 0.9999999  # turned down: its mass is 0.99 or less
    for u in (0.0, 0.3, 0.999):
        want = check(sess, logits, L.DT_F32, tokens, np.array([0, n, 2 * n]), parents, None, np.ones(2, np.float32), au,
                     np.full(2, u, np.float32), 4)
        assert want[1].tolist()[0] == 1 and want[2][1] != 11


def test_nothing_left_is_never_kept(sess):
    """Numbers below 0, and children whose parents' mass is all turned down: a token outside the vocabulary, one of −Inf and
    one that came before have nothing, and are not kept."""
    announce("verify nothing left")
    vocab = 40
    x = np.full((8, vocab), -np.inf, np.float32)
    x[:, [3, 4, 5]] = 0.0
    tokens = np.array([0, vocab, 17, -1, 3, 3, 4, 5])
    parents = np.array([-1, 0, 0, 0, 0, 0, 0, 0])
    heat = np.ones(1, np.float32)
    au = np.array([-1, -1, -1, -np.inf, 0.9, -3, 0.6, 0.7], np.float32)
    # thirds: 3 is turned down (0.9 > 1/3), then 3 again has nothing; 4 of two thirds: 0.4 > 1/3; 5 of one third: 0.23 < 1/3
    want = check(sess, x, L.DT_F32, tokens, np.array([0, 8]), parents, None, heat, au, np.array([0.5], np.float32), 2)
    assert want[0].tolist() == [[0, 7]]
    au[[6, 7]] = 1.0
    for more in (0.99999994, 1.0, 5.0):
        au[4] = more
        got = run(sess, x, L.DT_F32, np.array([0, 3, 4, 5, 3, 4, 5, 3]), np.array([0, 8]), parents, None, heat,
                  np.full(8, more, np.float32), np.array([0.5], np.float32), 2)
        if more > 1:
            assert got[1].tolist() == [1] and got[2].tolist() == [-1]
        else:  # of what is left a child has all or nothing
            assert all(int(i) in (-1, 1, 2, 3) for i in got[0][0, 1:])


def test_max_accept(sess):
    """At max_accept nodes the walk stops, and the next token is drawn from all of p."""
    announce("verify max accept")
    rng = np.random.default_rng(5)
    vocab, n = 300, 6
    logits = np.full((n, vocab), 0, np.float32)
    logits[:, 9] = 40
    tokens = np.full(n, 9)
    for m in (1, 2, 5, 6, 9):
        want = check(sess, logits, L.DT_F32, tokens, np.array([0, n]), None, None, np.ones(1, np.float32),
                     rng.random(n).astype(np.float32), np.array([0.5], np.float32), m)
        assert want[1][0] == min(m, n) and want[2][0] == 9


def test_random_numbers_at_and_past_their_ends(sess):
    """0 keeps a child of any mass and draws the first token with a weight; 1 or more draws the last; NaN keeps nothing."""
    announce("verify ends")
    vocab = 5000
    x = np.full((10, vocab), -np.inf, np.float32)
    x[:, 4200:4300] = 0
    tokens = np.full(10, 4250)
    heat = np.ones(5, np.float32)
    au = np.repeat(np.array([0, 0.99999994, 1, -1, np.nan], np.float32), 2)
    su = np.array([0, 0.99999994, 1, -1, np.nan], np.float32)
    got = run(sess, x, L.DT_F32, tokens, np.arange(6) * 2, None, None, heat, au, su, 2)
    assert got[1].tolist() == [2, 1, 1, 2, 1]
    assert got[2].tolist() == [4200, 4299, 4299, 4200, 4299]


@pytest.mark.parametrize("kind", ["tree", "chain", "draft"])
def test_the_next_token_has_the_targets_distribution(sess, kind):
    """40000 sequences with the same logits: what follows the root (the first child kept, or the token drawn) has the
    target's probabilities, each within 5 standard deviations."""
    announce(f"verify distribution {kind}")
    rng = np.random.default_rng(6)
    seqs, vocab, n = 40000, 8, 3
    row, temp = rng.normal(0, 1, vocab), 0.9
    logits = np.tile(row, (seqs * n, 1)).astype(np.float32)
    heat = np.full(seqs, temp, np.float32)
    p = probabilities(logits[0].astype(np.float64), np.float64(heat[0]))
    draft = None
    parents = np.tile([-1, 0, 0], seqs) if kind == "tree" else None
    tokens = np.tile([0, 2, 5], seqs)
    if kind == "draft":
        q_row = (row + rng.normal(0, 1, vocab)).astype(np.float32)
        draft = np.tile(q_row, (seqs * n, 1))
        tokens = rng.choice(vocab, seqs * n, p=probabilities(q_row.astype(np.float64), np.float64(heat[0])))
    au, su = rng.random(seqs * n).astype(np.float32), rng.random(seqs).astype(np.float32)
    accepted, counts, after = run(sess, logits, L.DT_F32, tokens, np.arange(seqs + 1) * n, parents, draft, heat, au, su, n)
    first = np.where(counts > 1, tokens[np.arange(seqs) * n + np.maximum(accepted[:, 1], 0)], after)
    share = np.bincount(first, minlength=vocab) / seqs
    assert (np.abs(share - p) <= 5 * np.sqrt(p * (1 - p) / seqs)).all(), (share, p)
    # a child is kept with the candidates' whole mass, or with the mass that p and q have in common
    rate = {"tree": p[2] + p[5], "chain": p[2]}.get(kind)
    if kind == "draft":
        rate = np.minimum(p, probabilities(q_row.astype(np.float64), np.float64(heat[0]))).sum()
    assert abs((counts > 1).mean() - rate) <= 5 * np.sqrt(rate * (1 - rate) / seqs)


def test_repeated_calls_and_no_rows(sess):
    announce("verify repeated")
    rng = np.random.default_rng(7)
    vocab, n = 30000, 20
    logits = rng.normal(0, 2, (n, vocab)).astype(np.float32)
    args = (logits, L.DT_F32, np.argmax(logits[np.maximum(np.arange(n) - 1, 0)], 1), np.arange(5) * 5, None, None,
            np.full(4, 0.5, np.float32), rng.random(n).astype(np.float32), rng.random(4).astype(np.float32), 5)
    first = run(sess, *args)
    for _ in range(3):
        assert all(np.array_equal(a, b) for a, b in zip(first, run(sess, *args)))
    got = run(sess, np.zeros((0, 9), np.float32), L.DT_F32, np.zeros(0), np.zeros(4), None, None, None, None, None, 2)
    assert got[0].tolist() == [[-1, -1]] * 3 and got[1].tolist() == [0] * 3 and got[2].tolist() == [-1] * 3
    # rows that the logits do not have make a sequence empty
    got = run(sess, logits[:4, :9].copy(), L.DT_F32, np.zeros(4), np.array([-2, 3, 3, 9]), None, None, None, None, None, 2)
    assert got[1].tolist() == [0, 0, 1] and got[2].tolist()[:2] == [-1, -1]


def test_rows_apart(sess):
    """Rows of logits farther apart than the vocabulary, beginning at an odd element."""
    announce("verify rows apart")
    rng = np.random.default_rng(8)
    vocab, ld, n = 2500, 2503, 5
    for dtype in (L.DT_F32, L.DT_BF16):
        flat = to_dtype(rng.normal(0, 3, 1 + n * ld), dtype)
        logits = flat[1:].reshape(n, ld)[:, :vocab]
        tokens, starts = np.argmax(values(logits), 1)[np.maximum(np.arange(n) - 1, 0)].astype(np.int32), np.array([0, n], np.int32)
        dev = [sess.to_device(a, d) for a, d in ((flat, dtype), (tokens, L.DT_I32), (starts, L.DT_I32))]
        out = [sess.empty(L.DT_I32, s) for s in ((1, n), (1,), (1,))]
        args = L.VerifyArgs(1, n, vocab, dev[0].ptr + flat.itemsize, None, ld, 0, dev[2].ptr, dev[1].ptr, None, None, None, None,
                            n, out[0].ptr, out[1].ptr, out[2].ptr, dtype)
        L.check(sess.lib.ingot_rocm_verify_drafts(sess.h, C.byref(args)))
        want, _, _ = definition(values(logits), tokens, starts, max_accept=n)
        assert all(np.array_equal(o.numpy(), w) for o, w in zip(out, want)) and want[1][0] == n
        free_all(*dev, *out)


def test_refusals(sess):
    announce("verify refusals")
    z = sess.empty(L.DT_F32, (4, 8))
    i4, i2, i3, acc = (sess.empty(L.DT_I32, s) for s in ((4,), (2,), (3,), (2, 3)))
    f4, f2 = sess.empty(L.DT_F32, (4,)), sess.empty(L.DT_F32, (2,))

    def refused(code, text, *a, **kw):
        with pytest.raises(IngotError, match=text) as e:
            sess.verify_drafts(*a, **kw)
        assert e.value.code == code

    refused(L.EINVAL, "chain", z, i3, i4, acc, i2, i2, parents=i4, draft=z)
    refused(L.EINVAL, "random numbers", z, i3, i4, acc, i2, i2, temperature=f2)
    refused(L.EINVAL, "random numbers", z, i3, i4, acc, i2, i2, temperature=f2, sample_u=f2)
    refused(L.EINVAL, "f32 or bf16", sess.empty(L.DT_I32, (4, 8)), i3, i4, acc, i2, i2)
    refused(L.EINVAL, "bad sizes", z, i3, i4, sess.empty(L.DT_I32, (2, 0)), i2, i2)
    refused(L.EINVAL, "bad sizes", sess.empty(L.DT_F32, (4, 0)), i3, i4, acc, i2, i2)
    many = [sess.empty(L.DT_I32, s) for s in ((9_000_001,), (9_000_000, 1), (9_000_000,))]
    refused(L.EDECLINED, "too many", sess.empty(L.DT_F32, (0, 8)), many[0], sess.empty(L.DT_I32, (0,)), many[1], many[2], many[2])
    free_all(*many)
    refused(L.EDECLINED, "2\\^24", sess.empty(L.DT_BF16, (4, (1 << 24) + 1)), i3, i4, acc, i2, i2)
    for bad in (dict(parents=i3), dict(draft=sess.empty(L.DT_F32, (4, 9))), dict(temperature=f4), dict(accept_u=f2),
                dict(sample_u=f4), dict(draft=sess.empty(L.DT_BF16, (4, 8)))):
        with pytest.raises(ValueError, match="verify_drafts"):
            sess.verify_drafts(z, i3, i4, acc, i2, i2, **bad)
    with pytest.raises(ValueError, match="tokens"):
        sess.verify_drafts(z, i3, i3, acc, i2, i2)
    for field, value, text in (("logits_ld", 7, "rows of"), ("d_starts", None, "nil"), ("d_next", None, "nil"),
                               ("d_logits", None, "nil"), ("tokens", -1, "bad sizes"), ("batch", 1 << 40, "bad sizes"),
                               ("logits_ld", 1 << 31, "2\\^30")):
        args = L.VerifyArgs(2, 4, 8, z.ptr, None, 8, 8, i3.ptr, i4.ptr, None, None, None, None, 3, acc.ptr, i2.ptr, i2.ptr,
                            L.DT_F32)
        setattr(args, field, value)
        with pytest.raises(IngotError, match=text):
            L.check(sess.lib.ingot_rocm_verify_drafts(sess.h, C.byref(args)))
    with pytest.raises(IngotError, match="nil arguments"):
        L.check(sess.lib.ingot_rocm_verify_drafts(sess.h, None))

"""The decoder step's newer calls in captured graphs, and in two sessions at once."""
import ctypes as C

import numpy as np
import pytest

from decoder_reference import free_all, to_dtype, values
from helpers import announce
from ingot_amd import IngotError, KvCache, KvTable
from ingot_amd import _lib as L

pytestmark = pytest.mark.gpu


class Step:
    """Norm, rotation and append of one new token of each of `batch` sequences that share a prefix, their attention, and the
    draw of a token from given logits; inputs from a seed, into the same buffers."""

    def __init__(self, sess, batch=6, shared=200, heads=8, kv=2, dim=64, page=16, vocab=5000):
        self.s, self.batch, self.shared, self.heads, self.kv, self.dim, self.vocab = sess, batch, shared, heads, kv, dim, vocab
        most, full = shared // page + 3, shared // page
        pages = np.full((batch, most), -1, np.int32)
        pages[:, :full] = np.arange(full)
        for b in range(batch):
            pages[b, full:] = full + b * (most - full) + np.arange(most - full)
        self.num = full + batch * (most - full)
        self.shape = (1, self.num, kv, page, dim)
        e, i = sess.empty, lambda *s: sess.empty(L.DT_I32, s)
        self.cache = KvCache(e(L.DT_BF16, self.shape), e(L.DT_BF16, self.shape))
        self.table = KvTable(sess.to_device(pages), i(batch))
        self.q, self.k, self.v = (e(L.DT_F32, (batch, n, dim)) for n in (heads, kv, kv))
        self.y, self.logits = e(L.DT_F32, (batch, heads, dim)), e(L.DT_F32, (batch, vocab))
        self.w = sess.to_device(np.linspace(0.5, 1.5, dim).astype(np.float32))
        self.cos, self.sin = sess.rotary_table(shared + 64, dim)
        self.pos, self.tokens, self.counts, self.next, self.accepted = i(batch), i(batch), i(batch), i(batch), i(batch, 1)
        self.heat, self.au, self.su = (e(L.DT_F32, (batch,)) for _ in range(3))
        self.starts = sess.to_device(np.arange(batch + 1).astype(np.int32))
        self.first, self.common = sess.to_device(np.array([0, batch], np.int32)), sess.to_device(np.array([full * page], np.int32))

    def fill(self, seed):
        rng = np.random.default_rng(seed)
        s, b = self.s, self.batch
        lengths = self.shared // 16 * 16 + rng.integers(0, 30, b)
        new = [(self.cache.k, rng.normal(0, 1, self.shape)), (self.cache.v, rng.normal(0, 1, self.shape)),
               (self.table.lengths, lengths), (self.pos, lengths), (self.tokens, np.zeros(b)),
               (self.heat, rng.uniform(0.5, 1, b)), (self.au, rng.random(b)), (self.su, rng.random(b)),
               (self.logits, rng.normal(0, 2, (b, self.vocab)))]
        new += [(t, rng.normal(0, 1, t.shape)) for t in (self.q, self.k, self.v)]
        for t, a in new:
            h = s.to_device(to_dtype(a, L.DT_BF16) if t.dtype == L.DT_BF16 else np.asarray(
                a, np.int32 if t.dtype == L.DT_I32 else np.float32), t.dtype)
            s.copy_d2d(t, h)
            h.free()

    def run(self):
        s = self.s
        s.norm_rotary_append(self.q, self.k, self.v, self.w, self.w, self.pos, self.cos, self.sin, self.q, self.cache,
                             self.table, self.starts)
        s.prefix_attention(self.q, self.cache, self.table, self.starts, self.y, self.first, self.common, max_nodes=1,
                           max_tokens=self.shared + 32, max_shared=self.shared)
        s.verify_drafts(self.logits, self.starts, self.tokens, self.accepted, self.counts, self.next, temperature=self.heat,
                        accept_u=self.au, sample_u=self.su)

    def results(self):
        return [t.numpy() for t in (self.q, self.cache.k, self.cache.v, self.y, self.accepted, self.counts, self.next)]

    def free(self):
        free_all(self.cache, self.table, self.q, self.k, self.v, self.y, self.logits, self.w, self.cos, self.sin, self.pos,
                 self.tokens, self.counts, self.next, self.accepted, self.heat, self.au, self.su, self.starts, self.first,
                 self.common)


def runtime():
    with open("/proc/self/maps") as f:
        return C.CDLL(next(ln.split()[-1] for ln in f if "libamdhip64" in ln))


@pytest.mark.parametrize("path", [1, 2])
def test_captured_and_replayed(env_session, path):
    """A capture before the workspace has grown is refused and leaves the capture usable; afterwards every replay, with other
    inputs each time, gives the eager results; also after the session's workspace has grown past the captured one."""
    announce(f"decoder capture {path}")
    s, hip = env_session(INGOT_PREFIX_PATH=path), runtime()
    step = Step(s)
    step.fill(0)
    st, graph, ex = C.c_void_p(), C.c_void_p(), C.c_void_p()
    L.check(s.lib.ingot_rocm_stream(s.h, C.byref(st)))
    s.sync()
    assert s.workspace_bytes() == 0
    assert hip.hipStreamBeginCapture(st, 2) == 0  # relaxed
    with pytest.raises(IngotError, match="before the capture") as e:
        step.run()
    assert e.value.code == L.EINVAL
    assert hip.hipStreamEndCapture(st, C.byref(graph)) == 0
    hip.hipGraphDestroy(graph)
    step.run()
    s.sync()
    step.fill(0)
    assert hip.hipStreamBeginCapture(st, 2) == 0
    step.run()
    assert hip.hipStreamEndCapture(st, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(ex), graph, None, None, C.c_size_t(0)) == 0
    held = s.workspace_bytes()
    for seed in (1, 2, 3):
        step.fill(seed)
        step.run()
        want = step.results()
        if seed == 3:  # another call makes the workspace grow
            w = s.upload_weight(np.ones((256, 2048), np.float32), trans=True, pack_dtype=L.DT_BF16)
            big = [s.empty(L.DT_F32, shape) for shape in ((8192, 2048), (8192, 256))]
            s.gemm(big[0], w, big[1], 8192)  # packs its activations
            w.free()
            assert s.workspace_bytes() > held
            free_all(*big)
        step.fill(seed)
        for t in (step.y, step.next, step.counts):
            s.memset(t, 0)
        assert hip.hipGraphLaunch(ex, st) == 0
        assert all(np.array_equal(a, b) for a, b in zip(step.results(), want)), seed
        step.fill(seed)  # eager work between replays
        step.run()
        assert all(np.array_equal(a, b) for a, b in zip(step.results(), want)), seed
    hip.hipGraphExecDestroy(ex)
    hip.hipGraphDestroy(graph)
    step.free()


def test_two_sessions_at_once(env_session):
    """Calls of two sessions, on streams of their own, in flight together: each has its own workspace."""
    announce("decoder two sessions")
    steps = [Step(env_session(INGOT_PREFIX_PATH=2), batch=20, shared=1000) for _ in range(2)]
    want = []
    for i, step in enumerate(steps):
        step.fill(i)
        step.run()
        want.append(step.results())
    for _ in range(3):
        for i, step in enumerate(steps):
            step.fill(i)
        for step in steps:
            step.run()
        for step, w in zip(steps, want):
            assert all(np.array_equal(a, b) for a, b in zip(step.results(), w))
    for step in steps:
        step.free()

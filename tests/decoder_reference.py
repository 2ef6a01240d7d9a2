"""The decoder-step operators from their definitions, in 64 bits on the CPU (numpy), for the GPU tests."""
import numpy as np

import oracle
from ingot_amd import _lib as L


def to_dtype(a, dtype):
    """f32 values as the array the library takes for `dtype` (bf16: bit patterns)."""
    a = np.ascontiguousarray(a, np.float32)
    return oracle.f32_to_bf16(a) if dtype == L.DT_BF16 else a


def values(a):
    """The values an array of to_dtype's kind stands for, in 64 bits."""
    return oracle.bf16_to_f32(a).astype(np.float64) if a.dtype == np.uint16 else a.astype(np.float64)


def upload(sess, a, dtype):
    return sess.to_device(to_dtype(a, dtype), dtype)


def rotate(x, cos, sin, positions, interleaved, inverse=False):
    """x [tokens, heads, dim] (64 bits) turned; positions outside the tables give NaN."""
    half = cos.shape[1]
    y = np.array(x, np.float64)
    for t, p in enumerate(positions):
        inside = 0 <= p < cos.shape[0]
        c = cos[p].astype(np.float64) if inside else np.full(half, np.nan)
        s = sin[p].astype(np.float64) if inside else np.full(half, np.nan)
        if inverse:
            s = -s
        ia = np.arange(half) * 2 if interleaved else np.arange(half)
        ib = ia + 1 if interleaved else ia + half
        a, b = x[t][:, ia], x[t][:, ib]
        y[t][:, ia], y[t][:, ib] = a * c - b * s, b * c + a * s
    return y


def rotate_bound(x, cos, sin, positions, interleaved, dtype):
    """Rounding bound of rotate in f32 (two products, one sum, each within 2^-24 of the terms) and one store."""
    y = np.abs(rotate(np.abs(x), np.abs(cos), -np.abs(sin), positions, interleaved, False))
    lim = np.abs(rotate(np.abs(x), np.abs(cos), np.abs(sin), positions, interleaved, False))
    terms = np.maximum(y, lim)
    return terms * (3 * 2.0 ** -24 + (2.0 ** -9 if dtype == L.DT_BF16 else 0.0)) * 2 + 1e-30


def frequencies(rot, base=10000.0, scaling=L.ROTARY_PLAIN, factor=1.0, trained=0.0, low=1.0, high=32.0):
    j = np.arange(rot // 2, dtype=np.float64)
    if scaling == L.ROTARY_BASE and rot > 2:
        base = base * factor ** (rot / (rot - 2))
    f = base ** (-2.0 * j / rot)
    if scaling == L.ROTARY_LINEAR:
        f = f / factor
    if scaling == L.ROTARY_BY_PARTS:
        turns = trained * f / (2 * np.pi)
        g = np.clip((turns - low) / (high - low), 0, 1)
        f = (1 - g) * f / factor + g * f
    return f


class Pages:
    """A cache and its table on the host: k, v [layers, pages, heads, page, dim] as stored, pages [rows, max_pages]."""

    def __init__(self, rng, layers, rows, max_pages, heads, page, dim, dtype, lengths, extra=0, spare=3):
        self.dtype, self.page, self.dim, self.heads, self.layers = dtype, page, dim, heads, layers
        self.len = np.asarray(lengths, np.int32)
        need = [-(-(int(n) + extra) // page) for n in self.len]
        self.num = sum(need) + spare
        order = rng.permutation(self.num).astype(np.int32)
        self.pages = np.full((rows, max_pages), -1, np.int32)
        at = 0
        for r, n in enumerate(need):
            self.pages[r, :n] = order[at:at + n]
            at += n
        self.refs = np.zeros(self.num, np.int32)
        for p in self.pages[self.pages >= 0]:
            self.refs[p] += 1
        shape = (layers, self.num, heads, page, dim)
        self.k = to_dtype(rng.normal(0, 1, shape), dtype)
        self.v = to_dtype(rng.normal(0, 1, shape), dtype)

    def upload(self, sess, slot_major=False, refs=False):
        from ingot_amd import KvCache, KvTable

        order = (lambda a: np.ascontiguousarray(a.transpose(0, 1, 3, 2, 4))) if slot_major else (lambda a: a)
        cache = KvCache(sess.to_device(order(self.k), self.dtype), sess.to_device(order(self.v), self.dtype), slot_major)
        table = KvTable(sess.to_device(self.pages), sess.to_device(self.len),
                        sess.to_device(self.refs) if refs else None,
                        sess.to_device(np.full(1, 77, np.int32)) if refs else None)
        return cache, table

    @staticmethod
    def read(cache, slot_major=False):
        k, v = cache.k.numpy(), cache.v.numpy()
        if slot_major:
            k, v = k.transpose(0, 1, 3, 2, 4), v.transpose(0, 1, 3, 2, 4)
        return k, v

    def place(self, row, pos):
        """(page, slot) of a position of a row, None where the table has none."""
        if not 0 <= row < self.pages.shape[0] or pos < 0 or pos // self.page >= self.pages.shape[1]:
            return None
        p = self.pages[row, pos // self.page]
        return (p, pos % self.page) if 0 <= p < self.num else None


def attention(pages, layer, q, starts, rows, seen, scale, max_nodes, max_tokens=0):
    """Attention of q [tokens, heads, dim] (64 bits) from its definition. seen(b, node, other) says which nodes a node sees.
    Returns y, the same with |v| for v (the scale of roundings of p), and the largest sum of |scale·q·k| terms of a row."""
    tokens, heads, dim = q.shape
    k, v = values(pages.k[layer]), values(pages.v[layer])
    y, mass, size = np.zeros(q.shape), np.zeros(q.shape), np.zeros((tokens, heads))
    group = heads // pages.heads
    for b, r in enumerate(rows):
        n = min(int(starts[b + 1] - starts[b]), max_nodes)
        if not 0 <= r < len(pages.len):
            continue
        held = int(pages.len[r])
        for i in range(n):
            t = starts[b] + i
            at = [p for p in range(held + n) if (p < held or seen(b, i, p - held)) and (not max_tokens or p < max_tokens)]
            at = [x for x in (pages.place(r, p) for p in at) if x]
            if not at:
                continue
            pg, sl = np.array([x[0] for x in at]), np.array([x[1] for x in at])
            for h in range(heads):
                kk, vv = k[pg, h // group, sl], v[pg, h // group, sl]
                with np.errstate(invalid="ignore", over="ignore"):
                    s = scale * (kk @ q[t, h])
                    top = s.max()
                    if top == -np.inf:
                        continue
                    p = np.exp(s - top)
                    y[t, h] = (p[:, None] * vv).sum(0) / p.sum()
                    mass[t, h] = (p[:, None] * np.abs(vv)).sum(0) / p.sum()
                    size[t, h] = (abs(scale) * np.abs(kk) @ np.abs(q[t, h])).max()
    return y, mass, size


def attention_bound(y, mass, size, dim, keys, dtype, cache):
    """Error bound of one pass in f32: a score is off by (dim + 8)·2^-24 of its terms' sizes, which p takes over as a
    relative error (twice: in the sum too); sums over `keys` terms; exp2 and the quotient. bf16 queries round p and y."""
    rel = 4 * (dim + 8) * 2.0 ** -24 * size[..., None] + (keys + 64) * 2.0 ** -24
    if dtype == L.DT_BF16:
        if cache == L.DT_BF16:
            rel = rel + 2.0 ** -8
        return mass * rel + np.abs(y) * 2.0 ** -8 + 1e-30
    return mass * rel + 1e-30


def free_all(*things):
    for t in things:
        for x in ((t.k, t.v) if hasattr(t, "k") and hasattr(t, "kv_heads") else
                  (t.pages, t.lengths, t.references, t.missing) if hasattr(t, "references") else (t,)):
            if x is not None:
                x.free()

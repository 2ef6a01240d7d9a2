"""Norms of heads with their rotation, and their append to cache pages, on the GPU against the definition in 64 bits."""
import numpy as np
import pytest

from decoder_reference import Pages, free_all, rotate, to_dtype, values
from helpers import announce
from ingot_amd import Heads, IngotError, KvCache, KvTable
from ingot_amd import _lib as L

pytestmark = pytest.mark.gpu


def tables(rows, half, rng):
    a = rng.uniform(-4, 4, (rows, half))
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def normed(x, weight, eps):
    """x [tokens, heads, dim] in 64 bits; weight [dim], [heads, dim] or None."""
    with np.errstate(invalid="ignore", divide="ignore"):
        y = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps)))
        return y if weight is None else y * weight.astype(np.float64)


def definition(x, weight, eps, cos, sin, pos, interleaved, dtype):
    """The result and a bound of its roundings. The sum of dim squares is off by at most (dim + 8) · 2^-24 of itself in any
    order, which the root halves; the mean, eps, root and quotient add 2^-24 each (a root and a quotient in f32 are within
    one step, 2^-23), the two products 2^-24 each: n is off by (dim / 2 + 12) · 2^-24 of itself. The turn adds three
    roundings of its terms |a·cos| + |b·sin|, the store half a step (2^-8 in bf16)."""
    n = normed(x, weight, eps)
    y = rotate(n, cos, sin, pos, interleaved)
    c, s = np.abs(cos), np.abs(sin)
    terms = np.maximum(np.abs(rotate(np.abs(n), c, s, pos, interleaved)), np.abs(rotate(np.abs(n), c, -s, pos, interleaved)))
    bound = terms * (x.shape[-1] / 2 + 16) * 2.0 ** -24 + np.abs(y) * (2.0 ** -8 if dtype == L.DT_BF16 else 2.0 ** -24)
    return y, bound * 1.01 + 1e-37  # second order; values below the smallest normal number


def check(got, want, bound, what):
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN elsewhere"
    bad = np.abs(got - want) > bound
    assert not bad[~np.isnan(want)].any(), f"{what}: {np.nanmax(np.abs(got - want) - bound)} over the bound"


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,rot,weights", [
    (1, 1, 64, 64, 1), (1, 16, 128, 128, 1), (5, 3, 80, 80, 2), (7, 4, 80, 20, 0), (33, 2, 64, 0, 1), (3, 5, 33, 14, 2),
    (65, 1, 2, 2, 1), (257, 7, 128, 32, 2), (9, 2, 256, 128, 1), (4, 3, 96, 90, 1), (5, 3, 20, 8, 2), (3, 2, 1, 0, 1),
    (2, 3, 1100, 600, 2), (3, 2, 331, 330, 1), (2, 1, 4096, 128, 1), (1200, 7, 64, 64, 2), (2100, 5, 96, 24, 1)])
def test_norm_rotary(sess, dtype, interleaved, tokens, heads, dim, rot, weights):
    """weights: none, one for all heads, one for each."""
    announce(f"norm rotary {dtype} {interleaved} {tokens} {heads} {dim} {rot} {weights}")
    rng = np.random.default_rng(tokens * 1000 + dim + rot)
    cos, sin = tables(50, rot // 2, rng)
    pos = rng.integers(0, 50, tokens).astype(np.int32)
    x = to_dtype(rng.normal(0, 1, (tokens, heads, dim)) * np.exp(rng.normal(0, 2, (tokens, heads, 1))), dtype)
    w = None if not weights else rng.normal(1, 0.3, (heads, dim) if weights == 2 else (dim,)).astype(np.float32)
    dx, dy = sess.to_device(x, dtype), sess.empty(dtype, x.shape)
    ins = [sess.to_device(a) for a in (pos, cos, sin)]
    dw = None if w is None else sess.to_device(w)
    sess.norm_rotary(dx, dw, *ins, dy, eps=1e-5, interleaved=interleaved)
    check(values(dy.numpy()), *definition(values(x), w, 1e-5, cos, sin, pos, interleaved, dtype), "norm rotary")
    sess.norm_rotary(dx, dw, *ins, dx, eps=1e-5, interleaved=interleaved)  # in place
    assert np.array_equal(dx.numpy(), dy.numpy())
    free_all(dx, dy, *ins, *([] if dw is None else [dw]))


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("offset,gap", [(1, 0), (2, 0), (4, 0), (8, 0), (0, 1), (0, 2), (0, 4), (2, 4), (8, 6)])
def test_views_of_every_alignment(sess, dtype, offset, gap):
    """Heads that begin `offset` elements into a buffer and lie dim + gap apart, in place; what lies between them stays."""
    announce(f"norm rotary views {dtype} {offset} {gap}")
    rng = np.random.default_rng(offset * 10 + gap)
    t, h, d, rot = 5, 3, 48, 32
    cos, sin = tables(9, rot // 2, rng)
    pos = rng.integers(0, 9, t).astype(np.int32)
    w = rng.normal(1, 0.3, d).astype(np.float32)
    flat = to_dtype(rng.normal(0, 1, offset + t * h * (d + gap)), dtype)
    x = flat[offset:].reshape(t, h, d + gap)[..., :d]
    dx, ins = sess.to_device(flat, dtype), [sess.to_device(a) for a in (w, pos, cos, sin)]
    view = Heads(dx, t, h, d, offset, h * (d + gap), d + gap)
    sess.norm_rotary(view, *ins, view)
    out = dx.numpy()
    check(values(out[offset:].reshape(t, h, d + gap)[..., :d]), *definition(values(x), w, 1e-6, cos, sin, pos, False, dtype),
          "a view")
    assert out[:offset].tobytes() == flat[:offset].tobytes()
    assert out[offset:].reshape(t, h, -1)[..., d:].tobytes() == flat[offset:].reshape(t, h, -1)[..., d:].tobytes()
    free_all(dx, *ins)


def test_weights_at_odd_addresses(sess):
    """A weight that begins one element into its buffer, and weights of heads an odd number of elements apart."""
    announce("norm rotary odd weights")
    rng = np.random.default_rng(5)
    t, h, d = 4, 3, 64
    cos, sin = tables(9, 32, rng)
    pos = rng.integers(0, 9, t).astype(np.int32)
    x = rng.normal(0, 1, (t, h, d)).astype(np.float32)
    flat = rng.normal(1, 0.3, 1 + h * (d + 1)).astype(np.float32)
    dx, dw, dy = sess.to_device(x), sess.to_device(flat), sess.empty(L.DT_F32, x.shape)
    ins = [sess.to_device(a) for a in (pos, cos, sin)]
    for stride in (0, d + 1):
        import ctypes as C
        rot = L.RotaryDesc(ins[1].ptr, ins[2].ptr, ins[0].ptr, 9, d, 0)
        norm = L.HeadNormDesc(dw.ptr + 4, stride, 1e-6)
        hx, hy = Heads(dx), Heads(dy)
        L.check(sess.lib.ingot_rocm_norm_rotary_apply(sess.h, C.byref(norm), C.byref(rot), t, h, d, L.DT_F32, C.byref(hx.c),
                                                      C.byref(hy.c)))
        w = np.stack([flat[1 + i * stride:1 + i * stride + d] for i in range(h)])
        check(dy.numpy().astype(np.float64), *definition(x.astype(np.float64), w, 1e-6, cos, sin, pos, False, L.DT_F32),
              f"stride {stride}")
    free_all(dx, dw, dy, *ins)


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
def test_special_values(sess, dtype):
    """Zeros stay zeros (eps > 0) and are NaN without it; an infinity or a NaN spoils its own head only, as in the formula;
    a position outside the tables gives NaN in the rotated dimensions only."""
    announce(f"norm rotary special values {dtype}")
    rng = np.random.default_rng(3)
    cos, sin = tables(4, 4, rng)
    pos = np.array([0, -1, 4, 3, 2 ** 31 - 1, -2 ** 31, 1, 2], np.int32)
    x = rng.normal(0, 1, (8, 3, 12)).astype(np.float32)
    x[0, 0] = 0
    x[3, 1, 5], x[6, 2, 0], x[7, 0, 11] = np.inf, np.nan, -np.inf
    x = to_dtype(x, dtype)
    dx, y = sess.to_device(x, dtype), sess.empty(dtype, x.shape)
    ins = [sess.to_device(a) for a in (pos, cos, sin)]
    for eps in (1e-6, 0.0):
        sess.norm_rotary(dx, None, *ins, y, eps=eps)
        with np.errstate(invalid="ignore"):
            want, bound = definition(values(x), None, eps, cos, sin, np.clip(pos, 0, 3), False, dtype)
        out = (pos < 0) | (pos > 3)
        want[out, :, :8] = np.nan
        check(values(y.numpy()), want, bound, f"eps {eps}")
    free_all(dx, y, *ins)


@pytest.mark.parametrize("dtype,cdtype", [(L.DT_F32, L.DT_BF16), (L.DT_BF16, L.DT_BF16), (L.DT_F32, L.DT_F32),
                                          (L.DT_BF16, L.DT_F32)])
@pytest.mark.parametrize("heads,kv,dim,rot,page,slot_major,fused,weights,many", [
    (4, 2, 64, 64, 16, False, False, (1, 1), 1), (3, 3, 80, 20, 24, True, True, (2, 2), 1),
    (1, 1, 128, 128, 1, False, True, (1, 0), 1), (8, 2, 32, 8, 7, True, False, (0, 2), 1),
    (5, 3, 64, 32, 16, False, True, (2, 1), 60), (3, 1, 1040, 16, 8, False, False, (1, 1), 1)])
def test_append(sess, dtype, cdtype, heads, kv, dim, rot, page, slot_major, fused, weights, many):
    """Rows in any order, a sequence without tokens, one whose page is missing in the table, and one without a row: their
    tokens are not written, everything else of the cache stays as it was. `many` times as many tokens in the last
    sequences; weights 0: not normed."""
    announce(f"norm append {dtype} {cdtype} {heads} {kv} {dim} {rot} {page} {many}")
    rng = np.random.default_rng(heads * 100 + dim + page)
    lengths = [5, 0, 2 * page, 3 * page + 1, 9]
    p = Pages(rng, 2, 5, 9 + 10 * many, kv, page, dim, cdtype, lengths, extra=9 * many)
    p.pages[3, lengths[3] // page] = -1  # a page that is not there
    p.pages[4, lengths[4] // page] = p.num  # and one that the cache does not have
    rows = np.array([2, 3, 1, 0, 7, -1, 4], np.int32)
    counts = [4 * many, 2, 9 * many, 0, 3, 2 * many, 1]
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    total = int(starts[-1])
    cos, sin = tables(40, rot // 2, rng)
    pos = rng.integers(0, 40, total).astype(np.int32)
    cache, table = p.upload(sess, slot_major)
    interleaved = page == 24
    if fused:  # q, k, v as columns of one matrix, as a QKV projection leaves them, with more columns between rows
        width = (heads + 2 * kv) * dim + (3 if dim == 80 else 8)
        qkv = to_dtype(rng.normal(0, 1, (total, width)), dtype)
        dq = sess.to_device(qkv, dtype)
        q, k, v = (Heads(dq, total, n, dim, off * dim, width, dim)
                   for n, off in ((heads, 0), (kv, heads), (kv, heads + kv)))
        m = values(qkv)
        hq, hk, hv = (m[:, a * dim:(a + n) * dim].reshape(total, n, dim)
                      for n, a in ((heads, 0), (kv, heads), (kv, heads + kv)))
        used = [dq]
    else:
        arrays = [to_dtype(rng.normal(0, 1, (total, n, dim)), dtype) for n in (heads, kv, kv)]
        used = [sess.to_device(a, dtype) for a in arrays]
        q, k, v = used
        hq, hk, hv = (values(a) for a in arrays)
    wq, wk = (None if not w else rng.normal(1, 0.3, (n, dim) if w == 2 else (dim,)).astype(np.float32)
              for w, n in zip(weights, (heads, kv)))
    dw = [None if w is None else sess.to_device(w) for w in (wq, wk)]
    y = q if fused else sess.empty(dtype, (total, heads, dim))  # fused: in place
    ins = [sess.to_device(a) for a in (pos, cos, sin, starts, rows)]
    sess.norm_rotary_append(q, k, v, *dw, *ins[:3], y, cache, table, ins[3], rows=ins[4], layer=1, interleaved=interleaved)

    def wanted(x, w, dt):
        if w is not None:
            return definition(x, w, 1e-6, cos, sin, pos, interleaved, dt)
        n = np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(1e-6)))  # not normed: n cancels, its roundings cover
        r, b = definition(x, None, 1e-6, cos, sin, pos, interleaved, dt)
        return r * n, b * n

    if fused:
        out = values(dq.numpy())
        got_q = out[:, :heads * dim].reshape(total, heads, dim)
        assert np.array_equal(out[:, heads * dim:], m[:, heads * dim:]), "keys and values in place change"
    else:
        got_q = values(y.numpy())
    check(got_q, *wanted(hq, wq, dtype), "queries")
    want_k, want_v = values(p.k), values(p.v)
    bound_k = np.zeros_like(want_k)
    turned, bound = wanted(hk, wk, cdtype)
    for b, r in enumerate(rows):
        for i in range(counts[b]):
            t = starts[b] + i
            at = p.place(r, lengths[r] + i) if 0 <= r < 5 else None
            if at:
                want_k[1, at[0], :, at[1]] = turned[t]
                bound_k[1, at[0], :, at[1]] = bound[t]
                want_v[1, at[0], :, at[1]] = values(to_dtype(hv[t], cdtype))
    got_k, got_v = Pages.read(cache, slot_major)
    check(values(got_k), want_k, bound_k, "keys")
    assert np.array_equal(values(got_v), want_v), "values"
    free_all(cache, table, *([] if fused else [y]), *used, *ins, *[w for w in dw if w is not None])


def test_nothing_to_do(sess):
    announce("norm rotary of nothing")
    z = sess.empty(L.DT_F32, (0, 2, 8))
    tab, pos = sess.empty(L.DT_F32, (3, 4)), sess.empty(L.DT_I32, (0,))
    sess.norm_rotary(z, None, pos, tab, tab, z)
    k = sess.empty(L.DT_BF16, (1, 2, 1, 4, 8))
    table = KvTable(sess.to_device(np.zeros((1, 2), np.int32)), sess.to_device(np.zeros(1, np.int32)))
    kv = sess.empty(L.DT_F32, (0, 1, 8))
    sess.norm_rotary_append(z, kv, kv, None, None, pos, tab, tab, z, KvCache(k, k), table,
                            sess.to_device(np.zeros(2, np.int32)))
    sess.sync()


def test_refusals(sess):
    announce("norm rotary refusals")
    x, y = sess.empty(L.DT_F32, (3, 2, 8)), sess.empty(L.DT_F32, (3, 2, 8))
    pos, tab, w = sess.empty(L.DT_I32, (3,)), sess.empty(L.DT_F32, (5, 4)), sess.empty(L.DT_F32, (8,))

    def refused(code, text, f, *a, **kw):
        with pytest.raises(IngotError, match=text) as e:
            f(*a, **kw)
        assert e.value.code == code

    odd = sess.empty(L.DT_F32, (5, 5))
    refused(L.EINVAL, "rot_dim", sess.norm_rotary, x, w, pos, odd, odd, y)
    for eps in (-1e-6, float("nan"), float("inf")):
        refused(L.EINVAL, "eps", sess.norm_rotary, x, w, pos, tab, tab, y, eps=eps)
    ints = sess.empty(L.DT_I32, (3, 2, 8))
    refused(L.EINVAL, "f32 or bf16", sess.norm_rotary, ints, w, pos, tab, tab, ints)
    refused(L.EINVAL, "overlap", sess.norm_rotary, x, w, pos, tab, tab, Heads(y, 3, 2, 8, token=16, head=4))
    refused(L.EINVAL, "in place", sess.norm_rotary, Heads(x, 3, 1, 8, token=8), w, pos, tab, tab, Heads(x, 3, 1, 8, token=16))
    import ctypes as C
    rot, hx = L.RotaryDesc(tab.ptr, tab.ptr, pos.ptr, 5, 8, 0), Heads(x)
    for norm, text in ((None, "nil norm"), (C.byref(L.HeadNormDesc(w.ptr, 4, 1e-6)), "elements apart"),
                       (C.byref(L.HeadNormDesc(w.ptr, -8, 1e-6)), "elements apart")):
        rc = sess.lib.ingot_rocm_norm_rotary_apply(sess.h, norm, C.byref(rot), 3, 2, 8, L.DT_F32, C.byref(hx.c), C.byref(hx.c))
        assert rc == L.EINVAL and text in sess.lib.ingot_rocm_last_error().decode()
    for bad in (sess.empty(L.DT_F32, (7,)), sess.empty(L.DT_F32, (3, 8)), sess.empty(L.DT_BF16, (8,))):
        with pytest.raises(ValueError, match="norm weight"):
            sess.norm_rotary(x, bad, pos, tab, tab, y)
    k = sess.empty(L.DT_BF16, (1, 2, 1, 4, 8))
    table = KvTable(sess.to_device(np.zeros((1, 2), np.int32)), sess.to_device(np.zeros(1, np.int32)))
    kv, starts = sess.empty(L.DT_F32, (3, 1, 8)), sess.to_device(np.array([0, 3], np.int32))
    refused(L.EINVAL, "layer 1 of 1", sess.norm_rotary_append, x, kv, kv, w, w, pos, tab, tab, y, KvCache(k, k), table, starts,
            layer=1)
    refused(L.EINVAL, "eps of k", sess.norm_rotary_append, x, kv, kv, None, w, pos, tab, tab, y, KvCache(k, k), table, starts,
            eps=-1.0)

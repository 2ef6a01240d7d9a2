"""Rotary positions and their append to cache pages on the GPU, against the definition in 64 bits."""
import numpy as np
import pytest

from decoder_reference import (Pages, free_all, frequencies, rotate, rotate_bound, to_dtype, upload, values)
from helpers import announce
from ingot_amd import Heads, IngotError, KvCache, KvTable
from ingot_amd import _lib as L

pytestmark = pytest.mark.gpu


def tables(rows, half, rng):
    a = rng.uniform(-4, 4, (rows, half))
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


def check(got, want, bound, what):
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN elsewhere"
    bad = np.abs(got - want) > bound
    assert not bad[~np.isnan(want)].any(), f"{what}: {np.nanmax(np.abs(got - want) - bound)} over the bound"


@pytest.mark.parametrize("scaling,kw", [
    (L.ROTARY_PLAIN, {}), (L.ROTARY_LINEAR, dict(factor=4.0)), (L.ROTARY_BASE, dict(factor=8.0)),
    (L.ROTARY_BY_PARTS, dict(factor=16.0, trained=4096.0, low=1.0, high=32.0)),
    (L.ROTARY_BY_PARTS, dict(factor=8.0, trained=8192.0, low=1.0, high=4.0))])
@pytest.mark.parametrize("first,rows,rot", [(0, 300, 128), (1 << 20, 65, 64), (0, 1, 2)])
def test_tables(sess, scaling, kw, first, rows, rot):
    """Angles in 64 bits: each entry within one rounding to f32 of the definition, at positions past a million too (the
    64-bit angle itself is off by 2^20 · 2^-52)."""
    announce(f"rotary table {scaling} {first} {rows} {rot}")
    cos, sin = sess.rotary_table(rows, rot, base=50000.0, first=first, scaling=scaling, amplitude=1.25, **kw)
    a = np.arange(first, first + rows)[:, None] * frequencies(rot, 50000.0, scaling, **kw)[None, :]
    for got, want in ((cos.numpy(), np.cos(a)), (sin.numpy(), np.sin(a))):
        assert np.abs(got - 1.25 * want).max() <= 1.25 * (2.0 ** -24 + 2.0 ** -30)
    free_all(cos, sin)


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,dim,rot", [
    (1, 1, 64, 64), (1, 16, 128, 128), (5, 3, 80, 80), (7, 4, 80, 20), (33, 2, 64, 0), (3, 5, 33, 14), (65, 1, 2, 2),
    (257, 7, 128, 32), (9, 2, 256, 128), (4, 3, 96, 90), (6, 2, 96, 24), (5, 3, 20, 8)])
def test_rotary(sess, dtype, interleaved, tokens, heads, dim, rot):
    announce(f"rotary {dtype} {interleaved} {tokens} {heads} {dim} {rot}")
    rng = np.random.default_rng(tokens * 1000 + dim + rot)
    cos, sin = tables(50, rot // 2, rng)
    pos = rng.integers(0, 50, tokens).astype(np.int32)
    x = to_dtype(rng.normal(0, 1, (tokens, heads, dim)), dtype)
    dx, dy = sess.to_device(x, dtype), sess.empty(dtype, x.shape)
    dp, dc, ds = sess.to_device(pos), sess.to_device(cos), sess.to_device(sin)
    sess.rotary(dx, dp, dc, ds, dy, interleaved=interleaved)
    want = rotate(values(x), cos, sin, pos, interleaved)
    bound = rotate_bound(values(x), cos, sin, pos, interleaved, dtype)
    got = values(dy.numpy())
    check(got, want, bound, "rotary")
    assert np.array_equal(got[..., rot:], values(x)[..., rot:]), "dimensions past rot_dim change"
    sess.rotary(dx, dp, dc, ds, dx, interleaved=interleaved)  # in place
    assert np.array_equal(dx.numpy(), dy.numpy())
    sess.rotary(dy, dp, dc, ds, dy, interleaved=interleaved, inverse=True)
    back = values(dy.numpy())
    assert np.abs(back - values(x)).max() <= (2.0 ** -6 if dtype == L.DT_BF16 else 2.0 ** -20) * np.abs(values(x)).max()
    free_all(dx, dy, dp, dc, ds)


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("offset,gap", [(1, 0), (2, 0), (4, 0), (8, 0), (0, 1), (0, 2), (0, 4), (2, 4), (8, 6)])
def test_views_of_every_alignment(sess, dtype, offset, gap):
    """Heads that begin `offset` elements into a buffer and lie dim + gap apart."""
    announce(f"rotary views {dtype} {offset} {gap}")
    rng = np.random.default_rng(offset * 10 + gap)
    t, h, d, rot = 5, 3, 48, 32
    cos, sin = tables(9, rot // 2, rng)
    pos = rng.integers(0, 9, t).astype(np.int32)
    flat = to_dtype(rng.normal(0, 1, offset + t * h * (d + gap)), dtype)
    x = flat[offset:].reshape(t, h, d + gap)[..., :d]
    dx, ins = sess.to_device(flat, dtype), [sess.to_device(a) for a in (pos, cos, sin)]
    view = Heads(dx, t, h, d, offset, h * (d + gap), d + gap)
    sess.rotary(view, *ins, view)
    out = dx.numpy()
    check(values(out[offset:].reshape(t, h, d + gap)[..., :d]), rotate(values(x), cos, sin, pos, False),
          rotate_bound(values(x), cos, sin, pos, False, dtype), "a view")
    assert out[:offset].tobytes() == flat[:offset].tobytes()
    assert out[offset:].reshape(t, h, -1)[..., d:].tobytes() == flat[offset:].reshape(t, h, -1)[..., d:].tobytes()
    free_all(dx, *ins)


@pytest.mark.parametrize("interleaved", [False, True])
def test_inverse_is_the_gradient(sess, interleaved):
    """The inverse turn of dy is the gradient of <dy, rotary(x)>: against differences of the kernel's own outputs (the
    operator is linear in x, so a difference of 1 is exact but for roundings)."""
    announce(f"rotary gradient {interleaved}")
    rng = np.random.default_rng(11)
    t, h, d, rot = 3, 2, 16, 12
    cos, sin = tables(9, rot // 2, rng)
    pos = np.array([0, 8, 3], np.int32)
    dp, dc, ds = sess.to_device(pos), sess.to_device(cos), sess.to_device(sin)
    x, dy = rng.normal(0, 1, (2, t, h, d)).astype(np.float32)
    dev_dy, dev_dx = sess.to_device(dy), sess.empty(L.DT_F32, dy.shape)
    sess.rotary(dev_dy, dp, dc, ds, dev_dx, interleaved=interleaved, inverse=True)
    grad = dev_dx.numpy().astype(np.float64)
    check(grad, rotate(dy.astype(np.float64), cos, sin, pos, interleaved, True),
          rotate_bound(dy, cos, sin, pos, interleaved, L.DT_F32), "gradient")

    def loss(v):
        dv, out = sess.to_device(v), sess.empty(L.DT_F32, v.shape)
        sess.rotary(dv, dp, dc, ds, out, interleaved=interleaved)
        r = float((out.numpy().astype(np.float64) * dy).sum())
        free_all(dv, out)
        return r

    for i in [(0, 0, 0), (1, 1, 5), (1, 0, 7), (2, 1, 11), (2, 0, 15)]:
        up, down = x.copy(), x.copy()
        up[i] += 0.5
        down[i] -= 0.5
        step = float(up[i]) - float(down[i])
        assert abs((loss(up) - loss(down)) / step - grad[i]) <= 64 * 2.0 ** -24 * np.abs(dy).sum()
    free_all(dp, dc, ds, dev_dy, dev_dx)


def test_position_outside_the_tables(sess):
    announce("rotary positions outside")
    rng = np.random.default_rng(3)
    cos, sin = tables(4, 4, rng)
    pos = np.array([0, -1, 4, 3, 2 ** 31 - 1, -2 ** 31], np.int32)
    x = rng.normal(0, 1, (6, 2, 12)).astype(np.float32)
    ins = [sess.to_device(a) for a in (x, pos, cos, sin)]
    y = sess.empty(L.DT_F32, x.shape)
    sess.rotary(*ins, y)
    check(y.numpy().astype(np.float64), rotate(x.astype(np.float64), cos, sin, pos, False),
          rotate_bound(x, cos, sin, np.clip(pos, 0, 3), False, L.DT_F32), "outside")
    free_all(y, *ins)


@pytest.mark.parametrize("dtype,cdtype", [(L.DT_F32, L.DT_BF16), (L.DT_BF16, L.DT_BF16), (L.DT_F32, L.DT_F32),
                                          (L.DT_BF16, L.DT_F32)])
@pytest.mark.parametrize("heads,kv,dim,rot,page,slot_major,fused", [
    (4, 2, 64, 64, 16, False, False), (3, 3, 80, 20, 24, True, True), (1, 1, 128, 128, 1, False, True),
    (8, 2, 32, 8, 7, True, False)])
def test_append(sess, dtype, cdtype, heads, kv, dim, rot, page, slot_major, fused):
    """Rows in any order, a sequence without tokens, one whose page is missing in the table, and one without a row:
    their tokens are not written, everything else of the cache stays as it was."""
    announce(f"append {dtype} {cdtype} {heads} {kv} {dim} {rot} {page}")
    rng = np.random.default_rng(heads * 100 + dim + page)
    lengths = [5, 0, 2 * page, 3 * page + 1, 9]
    p = Pages(rng, 2, 5, 20, kv, page, dim, cdtype, lengths, extra=9)
    p.pages[3, lengths[3] // page] = -1  # a page that is not there
    p.pages[4, lengths[4] // page] = p.num  # and one that the cache does not have
    rows = np.array([2, 3, 1, 0, 7, -1, 4], np.int32)
    counts = [4, 2, 9, 0, 3, 2, 1]
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    total = int(starts[-1])
    cos, sin = tables(40, rot // 2, rng)
    pos = rng.integers(0, 40, total).astype(np.int32)
    cache, table = p.upload(sess, slot_major)
    interleaved = page == 24
    if fused:  # q, k, v as columns of one matrix, as a QKV projection leaves them, with three more columns between rows
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
    y = sess.empty(dtype, (total, heads, dim))
    ins = [sess.to_device(a) for a in (pos, cos, sin, starts, rows)]
    before = [a.copy() for a in (p.k, p.v)]
    sess.rotary_append(q, k, v, ins[0], ins[1], ins[2], y, cache, table, ins[3], rows=ins[4], layer=1,
                       interleaved=interleaved)
    check(values(y.numpy()), rotate(hq, cos, sin, pos, interleaved),
          rotate_bound(hq, cos, sin, pos, interleaved, dtype), "queries")
    want_k, want_v = values(before[0]), values(before[1])
    bound_k = np.zeros_like(want_k)
    turned, bound = rotate(hk, cos, sin, pos, interleaved), rotate_bound(hk, cos, sin, pos, interleaved, cdtype)
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
    free_all(cache, table, y, *used, *ins)


def test_nothing_to_do(sess):
    announce("rotary of nothing")
    z = sess.empty(L.DT_F32, (0, 2, 8))
    tab, pos = sess.empty(L.DT_F32, (3, 4)), sess.empty(L.DT_I32, (0,))
    sess.rotary(z, pos, tab, tab, z)
    k = sess.empty(L.DT_BF16, (1, 2, 1, 4, 8))
    table = KvTable(sess.to_device(np.zeros((1, 2), np.int32)), sess.to_device(np.zeros(1, np.int32)))
    kv = sess.empty(L.DT_F32, (0, 1, 8))
    sess.rotary_append(z, kv, kv, pos, tab, tab, z, KvCache(k, k), table, sess.to_device(np.zeros(2, np.int32)))
    sess.sync()


def test_refusals(sess):
    announce("rotary refusals")
    x, y = sess.empty(L.DT_F32, (3, 2, 8)), sess.empty(L.DT_F32, (3, 2, 8))
    pos, tab = sess.empty(L.DT_I32, (3,)), sess.empty(L.DT_F32, (5, 4))

    def refused(code, text, f, *a, **kw):
        with pytest.raises(IngotError, match=text) as e:
            f(*a, **kw)
        assert e.value.code == code

    refused(L.EINVAL, "rot_dim", sess.rotary, x, pos, sess.empty(L.DT_F32, (5, 5)), sess.empty(L.DT_F32, (5, 5)), y)
    refused(L.EINVAL, "f32 or bf16", sess.rotary, sess.empty(L.DT_I32, (3, 2, 8)), pos, tab, tab,
            sess.empty(L.DT_I32, (3, 2, 8)))
    refused(L.EINVAL, "overlap", sess.rotary, x, pos, tab, tab, Heads(y, 3, 2, 8, token=16, head=4))
    refused(L.EINVAL, "in place", sess.rotary, Heads(x, 3, 1, 8, token=8), pos, tab, tab, Heads(x, 3, 1, 8, token=16))
    refused(L.EINVAL, "nil", sess.rotary, x, pos, tab, tab, Heads(type(x)(sess, L.DT_F32, (3, 2, 8), 0, False)))
    with pytest.raises(ValueError, match="positions"):
        sess.rotary(x, sess.empty(L.DT_I32, (2,)), tab, tab, y)
    with pytest.raises(ValueError, match="view"):
        Heads(x, 3, 2, 8, token=17)
    for kw in (dict(scaling=9), dict(base=0.0), dict(scaling=L.ROTARY_LINEAR, factor=0.0),
               dict(scaling=L.ROTARY_BY_PARTS, factor=2.0, trained=100.0, low=4.0, high=4.0), dict(first=-1)):
        refused(L.EINVAL, "rotary_table", sess.rotary_table, 4, 8, **kw)
    refused(L.EINVAL, "bad sizes", sess.rotary_table, 4, 7)
    table = KvTable(sess.to_device(np.zeros((1, 2), np.int32)), sess.to_device(np.zeros(1, np.int32)))
    starts = sess.to_device(np.array([0, 3], np.int32))

    def append(shape, dtype=L.DT_BF16, layer=0, ptr_off=0):
        k = sess.empty(dtype, shape)
        c = KvCache(k, k)
        c.c.d_k += ptr_off
        h = sess.empty(L.DT_F32, (3, shape[2], shape[4]))
        t = sess.empty(L.DT_F32, (5, 2))
        sess.rotary_append(h, h, h, pos, t, t, sess.empty(L.DT_F32, h.shape), c, table, starts, layer=layer)

    refused(L.EDECLINED, "multiple", append, (1, 2, 1, 4, 12))
    refused(L.EDECLINED, "aligned", append, (1, 2, 1, 4, 16), ptr_off=2)
    refused(L.EINVAL, "layer 1 of 1", append, (1, 2, 1, 4, 16), layer=1)
    refused(L.EINVAL, "cache must be", append, (1, 2, 1, 4, 16), dtype=L.DT_I8)

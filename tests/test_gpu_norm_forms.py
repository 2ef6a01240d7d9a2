"""Norms of queries and keys with weights of one, and with an eps each, in the append to cache pages on the GPU."""
import numpy as np
import pytest

from decoder_reference import Pages, free_all, to_dtype, values
from helpers import announce
from ingot_amd import _lib as L
from test_gpu_norm_rotary import check, definition, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [L.DT_F32, L.DT_BF16])
@pytest.mark.parametrize("ones", [(True, True), (True, False), (False, True)])
def test_weights_of_one_and_an_eps_each(sess, dtype, ones):
    announce(f"norm forms {dtype} {ones}")
    rng = np.random.default_rng(61)
    heads, kv, dim, page, rot = 4, 2, 64, 8, 32
    lengths, counts, eps = np.array([5, 0, 13]), np.array([2, 3, 1]), (0.03, 0.4)
    starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    p = Pages(rng, 1, 3, 4, kv, page, dim, L.DT_F32, lengths, extra=3)
    cos, sin = tables(20, rot // 2, rng)
    pos = (np.repeat(lengths - starts[:-1], counts) + np.arange(starts[-1])).astype(np.int32)
    x = [to_dtype(rng.normal(0, 0.5, (int(starts[-1]), n, dim)), dtype) for n in (heads, kv, kv)]
    w = [None if one else rng.normal(1, 0.3, dim).astype(np.float32) for one in ones]
    cache, table = p.upload(sess)
    dx = [sess.to_device(a, dtype) for a in x]
    ins = [sess.to_device(a) for a in (pos, cos, sin, starts)]
    dw = [1 if a is None else sess.to_device(a) for a in w]
    sess.norm_rotary_append(*dx, *dw, *ins[:3], dx[0], cache, table, ins[3], eps=eps)
    check(values(dx[0].numpy()), *definition(values(x[0]), w[0], eps[0], cos, sin, pos, False, dtype), "queries")
    want, bound = definition(values(x[1]), w[1], eps[1], cos, sin, pos, False, L.DT_F32)
    k = Pages.read(cache)[0]
    for b in range(3):
        for i in range(counts[b]):
            pg, sl = p.place(b, int(lengths[b]) + i)
            t = starts[b] + i
            check(k[0, pg, :, sl].astype(np.float64), want[t], bound[t], f"key {t}")
    free_all(cache, table, *dx, *ins, *[a for a in dw if not isinstance(a, int)])

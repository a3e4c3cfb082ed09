"""Attention over a paged cache where its numbers could go wrong and the element-wise bounds of a plain comparison would not show it:
values that are no numbers behind weights that vanish, large values behind them, sums over many keys, terms that are left out."""
import numpy as np
import pytest

import paged_model as pm
from raster_b200 import _lib as L
from test_paged_attention import DT, NP, Pool, close, normal
from test_paged_calls import Prompts


def at(pool, b, pos):
    page = pool.k.shape[1]
    return pool.table[b, pos // page], pos % page


# ---- a NaN behind weights that vanish ------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d,rows,n", [("bf16", 64, 3, 2600), ("bf16", 128, 20, 1500), ("bf16", 256, 2, 2600), ("bf16", 64, 70, 300),
                                            ("f32", 64, 3, 2600), ("f32", 128, 2, 1500)])
def test_a_key_that_is_no_number_far_below_the_largest_score(ctx, dtype, d, rows, n):
    """Its own score is not below anything: every row that sees it is NaN, in whatever part of the keys it lies.  (Keys in parts, and one
    case that is not cut.)"""
    n_q, page = 4, 32
    x = Prompts(ctx, dtype, n_q, 1, d, page, [n], [rows])
    p = x.pool
    k = p.k.copy()
    q = x.q[:, :, :]
    x.q = np.abs(q)
    x.bq.upload(pm.encode(x.q, dtype))
    k[at(p, 0, n - rows - 20)] = 60.0                     # a score of 60 sum(q) / sqrt(d), hundreds above all others
    p.bk.upload(pm.encode(k, dtype))
    x.call()
    ctx.sync()
    got = pm.decode(x.raw(), dtype).reshape(rows, n_q, d)
    want = pm.decode(pm.encode(p.v[at(p, 0, n - rows - 20)], dtype), dtype)[0]
    # that key's value alone: rounded with its weight and in the end (2 h, in bf16); 3 additions of its terms and the reciprocal, cut
    # (2 u each), a product and the exponential (4 u)
    h, u = pm.HALF[dtype], 2.0 ** -24
    assert (np.abs(got - want) <= ((2 * h if dtype == "bf16" else 0) + 12 * u) * np.abs(want)).all()
    for pos in (3, 100, n // 2, n - rows - 1):
        spoiled = k.copy()
        spoiled[at(p, 0, pos)][0, 5] = np.nan
        p.bk.upload(pm.encode(spoiled, dtype))
        x.call()
        ctx.sync()
        got = pm.decode(x.raw(), dtype).reshape(rows, n_q, d)
        assert np.isnan(got).all(), (pos, np.isnan(got).mean())
    x.free()


# ---- large values behind weights that vanish -----------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n_q,n_kv,d,lens", [(2, 1, 64, [40, 500]), (16, 1, 128, [100, 33]), (8, 2, 256, [300])])
def test_decode_of_large_values_whose_weights_vanish(ctx, dtype, n_q, n_kv, d, lens):
    """Weights of 2^-150 and less come to nothing, times 10^38 too."""
    p = Pool(ctx, lens, n_kv, d, 16, dtype, seed=d)
    q = np.abs(pm.decode(pm.encode(normal(d, len(lens), n_q, d), dtype), dtype)) + 1
    k, v = p.k.copy(), p.v.copy()
    keys, values = [a.copy() for a in p.keys], [a.copy() for a in p.values]
    for b, n in enumerate(lens):
        for pos in (0, 17, n - 2):
            k[at(p, b, pos)] = keys[b][pos] = -60.0        # a score of -60 sum(q) / sqrt(d) or less: -480 and below
            v[at(p, b, pos)] = values[b][pos] = pm.decode(pm.encode(np.array(2e38 if pos else -2e38), dtype), dtype)
    p.bk.upload(pm.encode(k, dtype))
    p.bv.upload(pm.encode(v, dtype))
    bq, bo = ctx.array_to_buffer(pm.encode(q, dtype)), ctx.make_buffer(len(lens) * n_q * d, NP[dtype])
    ctx.paged_decode_attention(bq, p.bk, p.bv, bo, p.bt, p.bl, len(lens), n_q, n_q // n_kv, n_kv, d, 16, p.n_pages, p.width, d ** -0.5, DT[dtype])
    ctx.sync()
    got = pm.decode(bo.download(), dtype).reshape(len(lens), n_q, d)
    for b, n in enumerate(lens):
        # the model in f64 keeps such weights; what is left of them in f32 is nothing, so these positions do not count
        keep = [i for i in range(n) if i not in (0, 17, n - 2)]
        want, tol = pm.attention(q[b:b + 1], keys[b][keep], values[b][keep], d ** -0.5, False, dtype)
        close(got[b:b + 1], want, tol, f"sequence {b}")
    for b in (bq, bo):
        b.free()
    p.free()

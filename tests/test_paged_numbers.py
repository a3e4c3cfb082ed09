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

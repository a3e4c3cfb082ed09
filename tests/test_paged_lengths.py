"""Lengths at their ends: sequences that hold nothing, and lengths beyond what a table has room for, in every call over a paged cache."""
import numpy as np
import pytest

import paged_model as pm
from raster_b200 import _lib as L
from test_paged_attention import DT, NP, Pool, close, normal


# ---- slots of a batch that nobody uses ------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_an_idle_slot_is_no_error(ctx, dtype):
    """A decode step of a batch some of whose sequences hold nothing (length 0, no page): their rows are left out and rstq_sync has nothing to
    say.  A sequence of length 0 that does hold a page, or one of some length that does not, is an error as before."""
    n_q, n_kv, d, page, lens = 4, 2, 64, 16, [16, 0, 17, 0, 0, 5]
    B = len(lens)
    p = Pool(ctx, lens, n_kv, d, page, dtype)
    table = np.where(p.table >= p.n_pages, -1, p.table).astype(np.int32)
    q, k, v = normal(1, B, n_q, d), normal(2, B, n_kv, d), normal(3, B, n_kv, d)
    up = ctx.array_to_buffer
    bq, bk, bv = up(q), up(k), up(v)
    bqt, bo = up(np.full(B * n_q * d, 7, NP[dtype])), ctx.make_buffer(B * n_q * d, NP[dtype])
    before = p.bk.download()

    def step():
        ctx.paged_rope_append(bq, bk, bv, bqt, p.bk, p.bv, p.bt, p.bl, None, B, B, n_q, n_kv, d, page, p.n_pages, p.width, 1e4, L.F32, DT[dtype])
        ctx.paged_decode_attention(bqt, p.bk, p.bv, bo, p.bt, p.bl, B, n_q, n_q // n_kv, n_kv, d, page, p.n_pages, p.width, 0.125, DT[dtype])

    def rows_written():
        pool = p.bk.download()
        return int((pool.view(np.uint8).reshape(-1, n_kv * d * pool.itemsize) != before.view(np.uint8).reshape(-1, n_kv * d * pool.itemsize)).any(1).sum())

    for empty in (0, -3):                                     # (a negative length counts as none)
        p.bt.upload(table)
        p.bl.upload(np.array([n or empty for n in lens], np.int32))
        p.bk.upload(before)
        step()
        ctx.sync()                                            # nothing to say
        raw = bqt.download().reshape(B, n_q, d)
        out = pm.decode(bo.download(), dtype).reshape(B, n_q, d)
        for b, n in enumerate(lens):
            if n:
                want = pm.rope(q[b], n - 1, 1e4)
                assert np.abs(pm.decode(raw[b], dtype) - want).max() <= (pm.HALF[dtype] + 2.0 ** -20) * np.abs(want).max()
                assert np.isfinite(out[b]).all() and out[b].any()
            else:
                assert (raw[b] == 7).all() and not out[b].any()
        assert rows_written() == 3
    for b, entry, n in ((1, 0, 0), (3, -1, 1), (4, p.n_pages, 0), (1, -2, 0)):
        p.bt.upload(table)
        tab = table.copy()
        tab[b, 0] = entry
        p.bt.upload(tab)
        some = np.array(lens, np.int32)
        some[b] = n
        p.bl.upload(some)
        ctx.paged_rope_append(bq, bk, bv, bqt, p.bk, p.bv, p.bt, p.bl, None, B, B, n_q, n_kv, d, page, p.n_pages, p.width, 1e4, L.F32, DT[dtype])
        with pytest.raises(L.RstqError) as e:
            ctx.sync()
        assert e.value.code == L.E_RANGE
        ctx.sync()
    for b in (bq, bk, bv, bqt, bo):
        b.free()
    p.free()

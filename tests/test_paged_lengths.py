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


# ---- lengths beyond the table ----------------------------------------------------------------------------
BEYOND = [
    # dtype, n_q, n_kv, d, page, pages of a sequence, lengths, new rows
    ("bf16", 4, 2, 64, 16, 6, [100, 96, 130, 97, 1000], [30, 96, 20, 5, 3]),
    ("bf16", 8, 1, 128, 32, 5, [170, 2000, 161], [150, 40, 170]),
    ("bf16", 4, 1, 128, 256, 8, [2051, 2100], [4, 60]),            # keys in parts
    ("bf16", 2, 1, 256, 16, 6, [100, 130], [30, 20]),
    ("f32", 4, 2, 64, 16, 6, [100, 96, 130, 97], [30, 96, 20, 5]),
    ("f32", 4, 1, 128, 256, 8, [2051, 2100], [4, 60]),
    ("f32", 2, 1, 256, 16, 6, [100, 130], [30, 20]),               # row by row
    ("bf16", 2, 2, 64, 16, 2, [40 + i % 3 for i in range(150)], [10] * 150),
    ("bf16", 1, 1, 64, 16, 2, [(1 << 31) - 1, 33], [50, 2]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n_q,n_kv,d,page,width,lens,new", BEYOND)
def test_rows_keep_their_places_where_lengths_go_beyond_the_table(ctx, dtype, n_q, n_kv, d, page, width, lens, new):
    """Row t stands at lens - (cu[b + 1] - t) in every call: rows whose position has a page are written there and see what is before them, the
    others are not written and see all that there is."""
    room = width * page
    p = Pool(ctx, [min(n, room) for n in lens], n_kv, d, page, dtype, seed=d, width=width)
    p.bl.upload(np.array(lens, np.int32))
    rows, cu = sum(new), np.cumsum([0] + new).astype(np.int32)
    up = ctx.array_to_buffer
    q = pm.decode(pm.encode(normal(4, rows, n_q, d), dtype), dtype)
    bq, bo, bcu = up(pm.encode(q, dtype)), ctx.make_buffer(rows * n_q * d, NP[dtype]), up(cu)
    ctx.paged_prompt_attention(bq, p.bk, p.bv, bo, p.bt, bcu, p.bl, rows, len(lens), n_q, n_q // n_kv, n_kv, d, page, p.n_pages, width, d ** -0.5, True,
                               DT[dtype])
    ctx.sync()
    got = pm.decode(bo.download(), dtype).reshape(rows, n_q, d)
    for b in range(len(lens)) if len(lens) < 20 else (0, 1, 77, 149):
        for r in sorted({0, new[b] // 2, new[b] - 1, min(max(room - lens[b] + new[b] - 1, 0), new[b] - 1)}):
            m = min(max(lens[b] - new[b] + r + 1, 0), room)
            want, tol = pm.attention(q[cu[b] + r][None], p.keys[b][:m], p.values[b][:m], d ** -0.5, False, dtype)
            close(got[cu[b] + r][None], want, tol, f"sequence {b} row {r} of {m} keys")
    # the same rows written
    k, v = normal(5, rows, n_kv, d), normal(6, rows, n_kv, d)
    x, bk, bv = up(normal(7, rows, n_q, d)), up(k), up(v)
    before = p.bv.download().reshape(-1, n_kv * d)
    ctx.paged_rope_append(x, bk, bv, bo, p.bk, p.bv, p.bt, p.bl, bcu, rows, len(lens), n_q, n_kv, d, page, p.n_pages, width, 1e4, L.F32, DT[dtype])
    if any(n > room for n in lens):
        with pytest.raises(L.RstqError) as e:
            ctx.sync()
        assert e.value.code == L.E_RANGE
    ctx.sync()
    want = before.copy()
    for b, n in enumerate(lens):
        for r in range(new[b]):
            pos = n - new[b] + r
            if 0 <= pos < room:
                want[p.table[b, pos // page] * page + pos % page] = pm.encode(v[cu[b] + r].reshape(-1), dtype)
    after = p.bv.download().reshape(-1, n_kv * d)
    assert np.array_equal(after.view(np.uint8), want.view(np.uint8))
    for b in (bq, bo, bcu, x, bk, bv):
        b.free()
    p.free()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_of_lengths_beyond_the_table_sees_all_of_it(ctx, dtype):
    n_q, n_kv, d, page, width, lens = 4, 2, 64, 16, 3, [49, (1 << 31) - 1, 48, 5]
    p = Pool(ctx, [min(n, 48) for n in lens], n_kv, d, page, dtype, width=width)
    p.bl.upload(np.array(lens, np.int32))
    q = pm.decode(pm.encode(normal(3, 4, n_q, d), dtype), dtype)
    bq, bo = ctx.array_to_buffer(pm.encode(q, dtype)), ctx.make_buffer(4 * n_q * d, NP[dtype])
    ctx.paged_decode_attention(bq, p.bk, p.bv, bo, p.bt, p.bl, 4, n_q, 2, n_kv, d, page, p.n_pages, width, 0.125, DT[dtype])
    ctx.sync()
    got = pm.decode(bo.download(), dtype).reshape(4, n_q, d)
    for b in range(4):
        want, tol = pm.attention(q[b:b + 1], p.keys[b], p.values[b], 0.125, False, dtype)
        close(got[b:b + 1], want, tol, f"sequence {b}")
    bq.free()
    bo.free()
    p.free()


# ---- arrays that begin on 16 bytes and on no more ---------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n_q,n_kv,d", [("bf16", 4, 2, 64), ("bf16", 7, 1, 8), ("bf16", 2, 2, 136), ("bf16", 3, 1, 128), ("f32", 4, 2, 64), ("f32", 3, 1, 40),
                                              ("f32", 2, 1, 256)])
def test_arrays_on_16_bytes(ctx, dtype, n_q, n_kv, d):
    """Every array 16 bytes behind a boundary of 256, rows a multiple of 16 bytes long and of nothing more."""
    page, lens, new = 16, [40, 150, 3], [40, 20, 1]
    p = Pool(ctx, lens, n_kv, d, page, dtype, seed=d)
    B, rows, cu = 3, sum(new), np.cumsum([0] + new).astype(np.int32)
    made = []

    def up(a):
        a = np.ascontiguousarray(a)
        base = ctx.make_buffer(a.nbytes + 272, np.uint8)
        base.fill_bytes(0xFF)
        b = ctx.wrap_buffer(base.device_ptr + 16, a.size, a.dtype.type)
        b.upload(a.reshape(-1))
        made.extend((b, base))
        return b

    item = NP[dtype]().itemsize
    step = n_q * d + 16 // item * (1 if (n_q * d * item // 16) % 2 == 0 else 2)        # an odd number of 16 bytes
    full = pm.encode(normal(4, rows, step), dtype)
    q = pm.decode(full, dtype)[:, :n_q * d].reshape(rows, n_q, d)
    bk, bv, bt, bl, bcu, bq = up(pm.encode(p.k, dtype)), up(pm.encode(p.v, dtype)), up(p.table), up(np.array(lens, np.int32)), up(cu), up(full)
    bo = up(np.full(rows * n_q * d, 7, NP[dtype]))
    heads, scale = (n_q, n_q // n_kv, n_kv, d, page, p.n_pages, p.width), d ** -0.5
    ctx.paged_prompt_attention(bq, bk, bv, bo, bt, bcu, bl, rows, B, *heads, scale, True, DT[dtype], ldq=step)
    ctx.sync()
    got = pm.decode(bo.download(), dtype).reshape(rows, n_q, d)
    for b in range(B):
        s = slice(cu[b], cu[b + 1])
        close(got[s], *pm.attention(q[s], p.keys[b], p.values[b], scale, True, dtype), f"prompt {b}")
    keys, values, ku = np.concatenate(p.keys), np.concatenate(p.values), np.cumsum([0] + lens).astype(np.int32)
    kstep = n_kv * d + 16 // item * (1 if (n_kv * d * item // 16) % 2 == 0 else 2)
    pad = lambda x: np.concatenate([pm.encode(x.reshape(len(x), -1), dtype), np.full((len(x), kstep - n_kv * d), 9, NP[dtype])], 1)  # noqa: E731
    ctx.prompt_attention(bq, up(pad(keys)), up(pad(values)), bo, bcu, up(ku), rows, len(keys), B, n_q, n_q // n_kv, n_kv, d, scale, True, DT[dtype], ldq=step,
                         ldk=kstep)
    ctx.sync()
    assert np.abs(pm.decode(bo.download(), dtype).reshape(rows, n_q, d) - got).max() <= 4 * pm.HALF[dtype] * np.abs(got).max()
    ctx.paged_decode_attention(bq, bk, bv, bo, bt, bl, B, *heads, scale, DT[dtype], ldq=step)
    ctx.sync()
    got = pm.decode(bo.download(n=B * n_q * d), dtype).reshape(B, n_q, d)
    for b in range(B):
        close(got[b:b + 1], *pm.attention(q[b:b + 1], p.keys[b], p.values[b], scale, False, dtype), f"decode {b}")
    x, k, v = normal(7, rows, n_q, d), normal(8, rows, n_kv, d), normal(9, rows, n_kv, d)
    ctx.paged_rope_append(up(x), up(k), up(v), bo, bk, bv, bt, bl, bcu, rows, B, n_q, n_kv, d, page, p.n_pages, p.width, 1e4, L.F32, DT[dtype])
    ctx.sync()
    got, pool = pm.decode(bo.download(), dtype).reshape(rows, n_q, d), bv.download().reshape(p.v.shape)
    for b in range(B):
        for t in range(cu[b], cu[b + 1]):
            pos = lens[b] - (cu[b + 1] - t)
            want = pm.rope(x[t], pos, 1e4)
            assert np.abs(got[t] - want).max() <= (pm.HALF[dtype] + 2.0 ** -20) * np.abs(want).max()
            assert np.array_equal(pool[p.table[b, pos // page], pos % page], pm.encode(v[t], dtype))
    refs, info, gone = np.zeros(p.n_pages, np.int32), up(np.zeros(4, np.int32)), up(np.array([1], np.int32))
    for b, n in enumerate(lens):
        refs[p.table[b, :-(-n // page)]] = 1
    br = up(refs)
    before = bk.download().reshape(p.k.shape)
    ctx.pages_free(bt, bl, br, gone, info, 1, B, p.n_pages, p.width, page)
    ctx.pages_compact(bk, bv, bt, bl, br, bt, br, info, B, p.n_pages, p.width, page, 1, n_kv * d * item)
    ctx.sync()
    assert info.download()[:2].tolist() == [0, sum(-(-n // page) for b, n in enumerate(lens) if b != 1)]
    after, table = bk.download().reshape(p.k.shape), bt.download().reshape(p.table.shape)
    for b in (0, 2):
        for j in range(-(-lens[b] // page)):
            assert np.array_equal(after[table[b, j]].view(np.uint8), before[p.table[b, j]].view(np.uint8))
    for b in made:
        b.free()
    p.free()

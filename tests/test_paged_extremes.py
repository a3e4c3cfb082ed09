"""The operators over a paged cache at the largest numbers of sequences and heads that they take."""
import numpy as np
import pytest

import paged_model as pm
from raster_b200 import _lib as L
from test_paged_attention import DT, NP, Pool, close, normal
from test_pages import Cache


def heads_of(q, k, v, scale, dtype, pick):
    """pm.attention of some heads alone: q [rows, n_q, d], k, v [n, n_kv, d]."""
    group = q.shape[1] // k.shape[1]
    outs = [pm.attention(q[:, h:h + 1], k[:, h // group:h // group + 1], v[:, h // group:h // group + 1], scale, True, dtype) for h in pick]
    return np.concatenate([o for o, _ in outs], 1), np.concatenate([t for _, t in outs], 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n_q,n_kv", [(65536, 1), (65536, 65536), (40000, 8)])
def test_as_many_heads_as_there_can_be(ctx, dtype, n_q, n_kv):
    d, page, lens, new = 8, 16, [17, 3], [2, 1]
    p = Pool(ctx, lens, n_kv, d, page, dtype, seed=1)
    rows, scale, cu = 3, d ** -0.5, np.array([0, 2, 3], np.int32)
    q = pm.decode(pm.encode(normal(2, rows, n_q, d), dtype), dtype)
    up = ctx.array_to_buffer
    bq, bo, bcu = up(pm.encode(q, dtype)), ctx.make_buffer(rows * n_q * d, NP[dtype]), up(cu)
    pick = sorted({0, 1, 15, 16, 17, n_q // 2, n_q - 17, n_q - 1})
    ctx.paged_prompt_attention(bq, p.bk, p.bv, bo, p.bt, bcu, p.bl, rows, 2, n_q, n_q // n_kv, n_kv, d, page, p.n_pages, p.width, scale, True, DT[dtype])
    ctx.sync()
    got = pm.decode(bo.download(), dtype).reshape(rows, n_q, d)
    for b in range(2):
        s = slice(cu[b], cu[b + 1])
        close(got[s][:, pick], *heads_of(q[s], p.keys[b], p.values[b], scale, dtype, pick), f"prompt {b}")
    ctx.paged_decode_attention(bq, p.bk, p.bv, bo, p.bt, p.bl, 2, n_q, n_q // n_kv, n_kv, d, page, p.n_pages, p.width, scale, DT[dtype])
    ctx.sync()
    got = pm.decode(bo.download(n=2 * n_q * d), dtype).reshape(2, n_q, d)
    for b in range(2):
        close(got[b:b + 1][:, pick], *heads_of(q[b:b + 1], p.keys[b], p.values[b], scale, dtype, pick), f"decode {b}")
    # and their rows written
    k, v = normal(3, rows, n_kv, d), normal(4, rows, n_kv, d)
    x = normal(5, rows, n_q, d)
    bx, bk, bv = up(x), up(k), up(v)
    ctx.paged_rope_append(bx, bk, bv, bo, p.bk, p.bv, p.bt, p.bl, bcu, rows, 2, n_q, n_kv, d, page, p.n_pages, p.width, 1e4, L.F32, DT[dtype])
    ctx.sync()
    got, pool = pm.decode(bo.download(), dtype).reshape(rows, n_q, d), p.bv.download().reshape(p.v.shape)
    for t, b in ((0, 0), (1, 0), (2, 1)):
        pos = lens[b] - (cu[b + 1] - t)
        want = pm.rope(x[t], pos, 1e4)
        assert np.abs(got[t] - want).max() <= (pm.HALF[dtype] + 2.0 ** -20) * np.abs(want).max()
        assert np.array_equal(pool[p.table[b, pos // page], pos % page], pm.encode(v[t], dtype))
    for b in (bq, bo, bcu, bx, bk, bv):
        b.free()
    p.free()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_as_many_sequences_as_there_can_be(ctx, dtype):
    n_q, n_kv, d, page, B = 2, 1, 8, 16, 65536
    rng = np.random.default_rng(1)
    lens = rng.integers(0, 21, B).astype(np.int32)
    lens[[0, B // 2, B - 1]] = 0, 0, 20
    new = np.where(lens > 0, rng.integers(0, 3, B), 0).astype(np.int32)
    new = np.minimum(new, lens)
    need = (lens + page - 1) // page
    n_pages = int(need.sum()) + 1
    order = rng.permutation(n_pages)[:need.sum()].astype(np.int32)
    table = np.full((B, 2), -1, np.int32)
    ends = np.cumsum(need)
    for j in range(2):
        has = need > j
        table[has, j] = order[(ends - need)[has] + j]
    k, v = (pm.decode(pm.encode(normal(s, n_pages, page, n_kv, d), dtype), dtype) for s in (2, 3))
    rows, cu = int(new.sum()), np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = pm.decode(pm.encode(normal(4, max(rows, B), n_q, d), dtype), dtype)
    up = ctx.array_to_buffer
    bq, bk, bv, bt, bl, bcu = up(pm.encode(q, dtype)), up(pm.encode(k, dtype)), up(pm.encode(v, dtype)), up(table), up(lens), up(cu)
    bo = ctx.make_buffer(len(q) * n_q * d, NP[dtype])
    heads, scale = (n_q, n_q // n_kv, n_kv, d, page, n_pages, 2), d ** -0.5
    some = [0, 1, 1023, 1024, B // 2, B - 2, B - 1] + rng.integers(0, B, 300).tolist()
    mine = lambda pool, b: np.concatenate([pool[i] for i in table[b, :need[b]]])[:lens[b]]  # noqa: E731

    ctx.paged_decode_attention(bq, bk, bv, bo, bt, bl, B, *heads, scale, DT[dtype])
    ctx.sync()
    got = pm.decode(bo.download(n=B * n_q * d), dtype).reshape(B, n_q, d)
    assert np.isfinite(got).all() and not got[lens == 0].any()
    for b in some:
        if lens[b]:
            close(got[b:b + 1], *pm.attention(q[b:b + 1], mine(k, b), mine(v, b), scale, False, dtype), f"decode {b}")
    ctx.paged_prompt_attention(bq, bk, bv, bo, bt, bcu, bl, rows, B, *heads, scale, True, DT[dtype])
    ctx.sync()
    got = pm.decode(bo.download(n=rows * n_q * d), dtype).reshape(rows, n_q, d)
    assert np.isfinite(got).all()
    for b in some:
        if new[b]:
            s = slice(cu[b], cu[b + 1])
            close(got[s], *pm.attention(q[s], mine(k, b), mine(v, b), scale, True, dtype), f"prompt {b}")
    # rows written: with their sequences, and one for each (those that hold nothing are idle)
    for per in (True, False):
        n = rows if per else B
        x, kk, vv = normal(5, n, n_q, d), normal(6, n, n_kv, d), normal(7, n, n_kv, d)
        bx, bkk, bvv = up(x), up(kk), up(vv)
        ctx.paged_rope_append(bx, bkk, bvv, bo, bk, bv, bt, bl, bcu if per else None, n, B, n_q, n_kv, d, page, n_pages, 2, 1e4, L.F32, DT[dtype])
        ctx.sync()
        pool = bv.download().reshape(n_pages, page, n_kv, d)
        for b in some:
            for t in range(cu[b], cu[b + 1]) if per else [b] * int(lens[b] > 0):
                pos = lens[b] - (cu[b + 1] - t) if per else lens[b] - 1
                assert np.array_equal(pool[table[b, pos // page], pos % page], pm.encode(vv[t], dtype))
        for b in (bx, bkk, bvv):
            b.free()
    for b in (bq, bk, bv, bt, bl, bcu, bo):
        b.free()


@pytest.mark.gpu
def test_pages_of_as_many_sequences_as_there_can_be(ctx):
    B = 65536
    rng = np.random.default_rng(3)
    c = Cache(ctx, B, 60000, 2, 16, layers=1, row=1, seed=3)
    half = rng.permutation(B).tolist()
    c.extend(half[:B // 2], [int(x) for x in rng.integers(0, 25, B // 2)])
    c.fork(half[:B // 2], half[B // 2:])
    c.extend(half, [0] * B)
    c.free(half[::2])
    c.compact()
    c.free(half)
    assert c.m.used() == 0
    c.close()

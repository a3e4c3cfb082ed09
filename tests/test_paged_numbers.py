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


# ---- f32 prompts: all the terms, and sums over many keys -------------------------------------------------
def f32_bound(d, n):
    """Relative 2-norm of an f32 prompt's error, for scores of about 1 (2 at the most where the weight is).  An addition of the tensor core
    cuts off at most 2^-23 of its sum, always towards zero:
      * four of them in a row for the first terms of a tile's P V (the small terms' are 2^-8 of that);
      * d / 16 of them for the first terms of a score, and five for the rest of it (the small terms, the exponential, the scale), times
        the score, which moves a weight by that much;
      * a tile's result is added to the row's in f32 to nearest, and so are the sums of weights: 2^-24 each, n / 64 of them, which
        go either way."""
    return 2.0 ** -23 * (4 + 2 * (d / 16 + 5) + (n / 64) ** 0.5)


def f64_rows(q, k, v, rows, scale, causal=False):
    """[len(rows), n_q, d] of one KV head in 64 bits; causal: q's last row is k's last."""
    out = []
    for r in rows:
        m = len(k) - len(q) + r + 1 if causal else len(k)
        s = q[r].astype(np.float64) @ k[:m, 0].astype(np.float64).T * scale
        w = np.exp(s - s.max(-1, keepdims=True))
        out.append(w / w.sum(-1, keepdims=True) @ v[:m, 0].astype(np.float64))
    return np.array(out)


def off(got, want):
    return np.linalg.norm(got - want) / np.linalg.norm(want)


def three_terms(x):
    out = []
    for _ in range(3):
        t = (x.view(np.uint32) & 0xFFFF0000).view(np.float32)
        out.append(t.astype(np.float64))
        x = x - t
    return out


@pytest.mark.parametrize("d,n", [(64, 40), (64, 500), (128, 130)])
def test_the_f32_bound_tells_terms_that_are_left_out(d, n):
    """Of the six products of terms, three alone miss it (planted in a model here), all six hold it by far."""
    q, k, v = normal(1, 4, d), normal(2, n, d), normal(3, n, d)
    kept = [(0, 0), (0, 1), (1, 0), (1, 1), (0, 2), (2, 0)]

    def product(a, b, pairs):
        ta, tb = three_terms(a.astype(np.float32)), three_terms(b.astype(np.float32))
        return sum(ta[i] @ tb[j] for i, j in pairs)

    want = f64_rows(q[:, None], k[:, None], v[:, None], range(4), d ** -0.5)[:, 0]
    for s_pairs, p_pairs, holds in ((kept, kept, True), (kept[:3], kept, False), (kept, kept[:3], False), (kept[:3], kept[:3], False)):
        s = product(q, np.ascontiguousarray(k.T), s_pairs) * d ** -0.5
        w = np.exp(s - s.max(-1, keepdims=True))
        got = product(w, v, p_pairs) / w.sum(-1, keepdims=True)
        if holds:
            assert off(got, want) < f32_bound(d, n) / 10
        else:
            assert off(got, want) > 2 * f32_bound(d, n)


@pytest.mark.gpu
@pytest.mark.parametrize("d,rows,n,values", [
    (64, 40, 40, "normal"), (64, 500, 500, "normal"), (128, 130, 130, "normal"), (96, 300, 300, "normal"), (128, 1300, 1300, "normal"),
    (64, 1300, 4000, "positive"), (128, 1300, 4000, "positive"), (64, 1300, 16000, "positive"), (128, 1300, 16000, "positive"),
    (64, 20, 16000, "positive"), (128, 20, 16000, "positive"), (64, 1300, 16000, "normal")])      # (20 rows: keys in parts)
def test_f32_prompts_hold_f32(ctx, d, rows, n, values):
    n_q = 16
    q, k, v = normal(1, rows, n_q, d), normal(2, n, 1, d), normal(3, n, 1, d)
    if values == "positive":
        v = np.abs(v) + 0.5
    up = ctx.array_to_buffer
    bq, bk, bv, cq, ck = up(q), up(k), up(v), up(np.array([0, rows], np.int32)), up(np.array([0, n], np.int32))
    bo = ctx.make_buffer(rows * n_q * d, np.float32)
    ctx.prompt_attention(bq, bk, bv, bo, cq, ck, rows, n, 1, n_q, n_q, 1, d, d ** -0.5, True, L.F32)
    ctx.sync()
    pick = sorted({0, 1, rows // 2, rows - 2, rows - 1})
    got, want = bo.download().reshape(rows, n_q, d)[pick], f64_rows(q, k, v, pick, d ** -0.5, True)
    for i, r in enumerate(pick):
        assert off(got[i], want[i]) <= f32_bound(d, n), (r, off(got[i], want[i]))
    for b in (bq, bk, bv, bo, cq, ck):
        b.free()


# ---- bf16 over a million positions -----------------------------------------------------------------------
class Repeated:
    """A cache of 2^20 positions a sequence, whose pages are the same 64 over and over, in other orders: attention over all of it is attention
    over those 64.  V is 1 or somewhat more or less, so that what is lost of a sum is lost of the result."""
    n, page = 1 << 20, 256

    def __init__(self, ctx, seqs, d):
        rng = np.random.default_rng(seqs + d)
        some = 64 * self.page
        self.k = pm.decode(pm.encode(normal(7, some, 1, d), "bf16"), "bf16")
        self.v = pm.decode(pm.encode(0.5 + rng.random((some, 1, d)).astype(np.float32), "bf16"), "bf16")
        self.width = self.n // self.page
        order = np.concatenate([rng.permutation(64) for _ in range(self.width // 64)]).astype(np.int32)
        self.bufs = [ctx.array_to_buffer(x) for x in (pm.encode(self.k, "bf16"), pm.encode(self.v, "bf16"), np.stack([np.roll(order, 64 * b) for b in range(seqs)]),
                                                      np.full(seqs, self.n, np.int32))]
        self.bk, self.bv, self.bt, self.bl = self.bufs

    def check(self, got, q, d):
        """A step of the result's own (h), and 2^-11 of it: a thousand additions that cut off 2^-23 of a growing sum, over and over (2^-14), the
        scores' rounding and, of prompts, that of the weights, whose mean over so many is far below that."""
        for i in range(len(q)):
            want = f64_rows(q[i:i + 1], self.k, self.v, [0], d ** -0.5)[0]
            assert (np.abs(got[i] - want) <= (pm.HALF["bf16"] + 2.0 ** -11) * want).all(), (i, (got[i] / want - 1).mean(), np.abs(got[i] / want - 1).max())

    def free(self):
        for b in self.bufs:
            b.free()


@pytest.mark.gpu
@pytest.mark.parametrize("n_q,d,seqs", [(4, 128, 300), (16, 64, 296), (12, 256, 150)])
def test_decode_over_a_million_positions(ctx, n_q, d, seqs):
    """As many sequences as there are blocks of threads: each sums one by itself."""
    x = Repeated(ctx, seqs, d)
    q = pm.decode(pm.encode(normal(5, seqs, n_q, d), "bf16"), "bf16")
    bq, bo = ctx.array_to_buffer(pm.encode(q, "bf16")), ctx.make_buffer(seqs * n_q * d, np.uint16)
    ctx.paged_decode_attention(bq, x.bk, x.bv, bo, x.bt, x.bl, seqs, n_q, n_q, 1, d, x.page, 64, x.width, d ** -0.5, L.BF16)
    ctx.sync()
    got = pm.decode(bo.download(), "bf16").reshape(seqs, n_q, d)
    pick = [0, seqs // 3, seqs - 1]
    x.check(got[pick], q[pick], d)
    bq.free()
    bo.free()
    x.free()


@pytest.mark.gpu
@pytest.mark.parametrize("n_q,d,rows", [(16, 128, 1300), (16, 64, 1300), (8, 256, 2500), (4, 64, 5), (16, 128, 40), (2, 256, 130)])
def test_prompts_over_a_million_positions(ctx, n_q, d, rows):
    """Enough rows that the keys are not cut into parts, and few, whose parts are 2^16 keys and more."""
    x = Repeated(ctx, 1, d)
    q = pm.decode(pm.encode(normal(5, rows, n_q, d), "bf16"), "bf16")
    bq, bo, cu = ctx.array_to_buffer(pm.encode(q, "bf16")), ctx.make_buffer(rows * n_q * d, np.uint16), ctx.array_to_buffer(np.array([0, rows], np.int32))
    ctx.paged_prompt_attention(bq, x.bk, x.bv, bo, x.bt, cu, x.bl, rows, 1, n_q, n_q, 1, d, x.page, 64, x.width, d ** -0.5, False, L.BF16)
    ctx.sync()
    got = pm.decode(bo.download(), "bf16").reshape(rows, n_q, d)
    pick = sorted({0, rows // 2, rows - 1})
    x.check(got[pick], q[pick], d)
    for b in (bq, bo, cu):
        b.free()
    x.free()


@pytest.mark.gpu
def test_one_row_of_many_keys_taken_by_itself(ctx):
    """An infinity above the diagonal of one of many sequences of 2^23 keys: its rows by themselves take longer than any wait in the kernel
    may, one row alone does, and the block has its next rows in hand meanwhile."""
    n, page, d, seqs, rows, distinct = 1 << 23, 256, 64, 300, 2, 64
    width = n // page
    k = pm.decode(pm.encode(normal(1, (distinct + 1) * page, 1, d), "bf16"), "bf16")
    v = pm.decode(pm.encode(np.random.default_rng(2).random(((distinct + 1) * page, 1, d)).astype(np.float32) + 0.5, "bf16"), "bf16")
    v[-1, 0, 5] = np.inf                                      # the last position of the last page, which ends one sequence
    table = np.tile(np.arange(width, dtype=np.int32) % distinct, (seqs, 1))
    table[-1, -1] = distinct                                  # (the last sequence's rows come first)
    up = ctx.array_to_buffer
    q = pm.decode(pm.encode(normal(3, seqs * rows, 1, d), "bf16"), "bf16")
    bq, bk, bv, bt = up(pm.encode(q, "bf16")), up(pm.encode(k, "bf16")), up(pm.encode(v, "bf16")), up(table)
    bl, cu, bo = up(np.full(seqs, n, np.int32)), up(np.arange(seqs + 1, dtype=np.int32) * rows), ctx.make_buffer(seqs * rows * d, np.uint16)
    ctx.paged_prompt_attention(bq, bk, bv, bo, bt, cu, bl, seqs * rows, seqs, 1, 1, 1, d, page, distinct + 1, width, d ** -0.5, True, L.BF16)
    ctx.sync()
    got = pm.decode(bo.download(), "bf16").reshape(seqs * rows, d)
    assert np.isposinf(got[-1, 5]) and np.isfinite(np.delete(got[-1], 5)).all() and np.isfinite(got[:-1]).all()
    for r in (0, seqs, 2 * seqs - 2):                         # first rows of theirs, which do not see the last key
        b = r // rows
        times = np.bincount(table[b], minlength=distinct + 1).repeat(page)
        times[table[b, -1] * page + page - 1] -= 1
        s = k[:, 0].astype(np.float64) @ q[r, 0].astype(np.float64) * d ** -0.5
        w = np.exp(s - s.max()) * times
        want = (w / w.sum()) @ np.where(np.isinf(v[:, 0]), 0, v[:, 0]).astype(np.float64)
        assert (np.abs(got[r] - want) <= (pm.HALF["bf16"] + 2.0 ** -11) * want).all(), (r, np.abs(got[r] / want - 1).max())
    for b in (bq, bk, bv, bt, bl, cu, bo):
        b.free()


# ---- the second term of a decode weight --------------------------------------------------------------------
def cancelling(seed, n, heads, d, scale):
    """q [heads, d], k and v [n, heads, d], all bf16, whose weighted values cancel but for the last value's rounding: what the weights are
    rounded by stands alone in the result."""
    q, k, v = (pm.decode(pm.encode(normal(seed + i, *shape), "bf16"), "bf16") for i, shape in enumerate(((heads, d), (n, heads, d), (n, heads, d))))
    for h in range(heads):
        w = np.exp(k[:, h].astype(np.float64) @ q[h].astype(np.float64) * scale)
        v[n - 1, h] = pm.decode(pm.encode((-(w[:-1] @ v[:-1, h]) / w[-1]).astype(np.float32), "bf16"), "bf16")
    return q, k, v


def test_the_tolerance_tells_a_weight_of_one_term():
    """A weight rounded or cut to bf16 misses what two terms hold (planted in a model here)."""
    d, heads = 64, 4
    q, k, v = cancelling(5, 64, heads, d, d ** -0.5)
    want, tol = pm.attention(q[None], k, v, d ** -0.5, False, "bf16", p_terms=2)
    up = lambda x: pm.from_bf16(pm.to_bf16(x))  # noqa: E731
    cut = lambda x: (x.view(np.uint32) & 0xFFFF0000).view(np.float32)  # noqa: E731
    for form, holds in ((lambda w: cut(w).astype(np.float64) + up(w - cut(w)), True), (up, False), (cut, False)):
        got = np.zeros((heads, d))
        for h in range(heads):
            s = k[:, h].astype(np.float64) @ q[h].astype(np.float64) * d ** -0.5
            w = np.exp(s - s.max()).astype(np.float32)
            got[h] = up((form(w) @ v[:, h].astype(np.float64) / w.astype(np.float64).sum()).astype(np.float32))
        over = np.abs(got - want[0]) / tol[0]
        assert (over.max() <= 1) == holds and (holds or over.max() > 3), over.max()


@pytest.mark.gpu
@pytest.mark.parametrize("group,n_kv,d,lens", [(1, 4, 64, [64, 40, 17]), (4, 2, 128, [64, 100]), (8, 1, 64, [33, 64]), (16, 1, 128, [64]), (12, 2, 256, [64, 50])])
def test_decode_weights_have_two_terms(ctx, group, n_kv, d, lens):
    p = Pool(ctx, lens, n_kv, d, 16, "bf16")
    k, v, q = p.k.copy(), p.v.copy(), np.zeros((len(lens), n_kv * group, d), np.float32)
    some = []
    for b, n in enumerate(lens):
        qq, kk, vv = cancelling(10 * b + d, n, n_kv, d, d ** -0.5)
        q[b] = np.repeat(qq, group, 0)
        some.append((kk, vv))
        for pos in range(n):
            k[at(p, b, pos)], v[at(p, b, pos)] = kk[pos], vv[pos]
    p.bk.upload(pm.encode(k, "bf16"))
    p.bv.upload(pm.encode(v, "bf16"))
    bq, bo = ctx.array_to_buffer(pm.encode(q, "bf16")), ctx.make_buffer(q.size, np.uint16)
    ctx.paged_decode_attention(bq, p.bk, p.bv, bo, p.bt, p.bl, len(lens), n_kv * group, group, n_kv, d, 16, p.n_pages, p.width, d ** -0.5, L.BF16)
    ctx.sync()
    got = pm.decode(bo.download(), "bf16").reshape(q.shape)
    for b in range(len(lens)):
        want, tol = pm.attention(q[b:b + 1], *some[b], d ** -0.5, False, "bf16", p_terms=2)
        close(got[b:b + 1], want, tol, f"sequence {b}")
    bq.free()
    bo.free()
    p.free()


# ---- scales that are not positive --------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("scale", [0.0, -0.125, -1.0, 1e-30])
@pytest.mark.parametrize("n_q,n_kv,d,page,lens,new", [(4, 2, 64, 16, [70, 0, 33], [70, 0, 5]), (8, 1, 128, 32, [1500, 40], [3, 40]), (2, 1, 256, 16, [50, 20], [50, 2])])
def test_scales_that_are_not_positive(ctx, dtype, scale, n_q, n_kv, d, page, lens, new):
    """The largest score is then the smallest product, or all of them are the same."""
    x = Prompts(ctx, dtype, n_q, n_kv, d, page, lens, new, seed=d)
    x.scale = scale
    x.call()
    ctx.sync()
    x.check()
    p, B = x.pool, len(lens)
    q = pm.decode(pm.encode(normal(9, B, n_q, d), dtype), dtype)
    bq, bo = ctx.array_to_buffer(pm.encode(q, dtype)), ctx.make_buffer(B * n_q * d, NP[dtype])
    ctx.paged_decode_attention(bq, p.bk, p.bv, bo, p.bt, p.bl, B, n_q, n_q // n_kv, n_kv, d, page, p.n_pages, p.width, scale, DT[dtype])
    ctx.sync()
    got = pm.decode(bo.download(), dtype).reshape(B, n_q, d)
    for b in range(B):
        want, tol = pm.attention(q[b:b + 1], p.keys[b], p.values[b], scale, False, dtype)
        close(got[b:b + 1], want, tol, f"sequence {b}")
    # packed, without causality
    keys, values = np.concatenate(p.keys), np.concatenate(p.values)
    up = ctx.array_to_buffer
    bk, bv, bku = up(pm.encode(keys, dtype)), up(pm.encode(values, dtype)), up(np.cumsum([0] + lens).astype(np.int32))
    ctx.prompt_attention(x.bq, bk, bv, x.bo, x.bcu, bku, x.rows, len(keys), B, n_q, n_q // n_kv, n_kv, d, scale, False, DT[dtype])
    ctx.sync()
    got = pm.decode(x.raw(), dtype).reshape(x.rows, n_q, d)
    for b in range(B):
        if new[b]:
            r = x.cu[b + 1] - 1
            want, tol = pm.attention(x.q[r][None], p.keys[b], p.values[b], scale, False, dtype)
            close(got[r][None], want, tol, f"sequence {b}, packed")
    for b in (bq, bo, bk, bv, bku):
        b.free()
    x.free()


# ---- values near the type's largest -------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,lens,new", [(64, [400, 90], [40, 90]), (128, [2600], [3]), (128, [300], [300]), (256, [200], [30])])
def test_values_near_the_largest_there_are(ctx, dtype, d, lens, new):
    """A weight is never more than 1, so a value of 3e38 stays one where its score goes beyond the earlier ones by a few."""
    n_q, page = 2, 16
    x = Prompts(ctx, dtype, n_q, 1, d, page, lens, new, seed=d)
    p = x.pool
    k, v = p.k.copy(), p.v.copy()
    x.q = np.broadcast_to(pm.decode(pm.encode(np.abs(normal(1, 1, 1, d)) + 0.5, dtype), dtype), x.q.shape).copy()      # (a row's scores are a key's, whatever the row)
    x.bq.upload(pm.encode(x.q, dtype))
    for b, n in enumerate(lens):
        for i, (pos, score) in enumerate(((n // 2, 4.0), (n - new[b] // 2 - 1, 5.0))):
            key = score * d ** 0.5 * x.q[0, 0] / (x.q[0, 0] ** 2).sum() + 0.5 * p.keys[b][pos]
            k[at(p, b, pos)] = p.keys[b][pos] = pm.decode(pm.encode(key.astype(np.float32), dtype), dtype)
            v[at(p, b, pos)][0, ::2] = p.values[b][pos][0, ::2] = pm.decode(pm.encode(np.array(-3e38 if i else 3e38), dtype), dtype)
    p.bk.upload(pm.encode(k, dtype))
    p.bv.upload(pm.encode(v, dtype))
    x.call()
    ctx.sync()
    x.check()
    q = pm.encode(x.q[:len(lens)], dtype)
    bq, bo = ctx.array_to_buffer(q), ctx.make_buffer(q.size, NP[dtype])
    ctx.paged_decode_attention(bq, p.bk, p.bv, bo, p.bt, p.bl, len(lens), n_q, n_q, 1, d, page, p.n_pages, p.width, d ** -0.5, DT[dtype])
    ctx.sync()
    got = pm.decode(bo.download(), dtype).reshape(len(lens), n_q, d)
    for b in range(len(lens)):
        want, tol = pm.attention(x.q[b:b + 1], p.keys[b], p.values[b], d ** -0.5, False, dtype)
        close(got[b:b + 1], want, tol, f"decode {b}")
    bq.free()
    bo.free()
    x.free()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n_q,d", [("f32", 2, 128), ("f32", 7, 128), ("bf16", 7, 128), ("f32", 4, 96), ("bf16", 4, 256)])
def test_rows_taken_by_themselves(ctx, dtype, n_q, d):
    """Infinities above the diagonal of blocks that share a tile with other heads, or have registers moved between their warps."""
    x = Prompts(ctx, dtype, n_q, 1, d, 16, [300, 150], [300, 150], seed=d)
    p = x.pool
    k, v = p.k.copy(), p.v.copy()
    v[at(p, 0, 200)][0, 7] = np.inf
    k[at(p, 1, 100)][0, 3] = np.nan
    p.bk.upload(pm.encode(k, dtype))
    p.bv.upload(pm.encode(v, dtype))
    x.call()
    ctx.sync()
    got = pm.decode(x.raw(), dtype).reshape(x.rows, n_q, d)
    assert np.isposinf(got[200:300, :, 7]).all() and np.isnan(got[400:]).all()
    for b, rows in ((0, (0, 127, 128, 199)), (1, (0, 64, 99))):
        for r in rows:
            i = x.cu[b] + r
            close(got[i][None], *pm.attention(x.q[i][None], p.keys[b][:r + 1], p.values[b][:r + 1], x.scale, False, dtype), f"sequence {b} row {r}")
    for r in (200, 299):
        keep = [i for i in range(d) if i != 7]
        want, tol = pm.attention(x.q[r][None], p.keys[0][:r + 1], p.values[0][:r + 1], x.scale, False, dtype)
        close(got[r][None][..., keep], want[..., keep], tol[..., keep], f"row {r}")
    x.free()

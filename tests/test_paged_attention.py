"""Attention and appends over a paged cache against plain forms in 64 bits (tests/paged_model.py, which derives the
tolerances), at the sizes and masks where they can go wrong."""
import ctypes as C

import numpy as np
import pytest

import paged_model as pm
from raster_b200 import _lib as L

DT = {"f32": L.F32, "bf16": L.BF16}
NP = {"f32": np.float32, "bf16": np.uint16}


def normal(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


class Pool:
    """Random pages in random places; what no sequence holds is NaN."""

    def __init__(self, ctx, lens, n_kv, d, page, dtype, seed=0, spare=3, width=None):
        rng = np.random.default_rng(seed + 99)
        need = [-(-n // page) for n in lens]
        self.n_pages, self.width = sum(need) + spare, width or max(max(need), 1)
        order = rng.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((len(lens), self.width), 1 << 29, np.int32)       # behind the pages: never read
        self.k = np.full((self.n_pages, page, n_kv, d), np.nan, np.float32)
        self.v = self.k.copy()
        self.keys, self.values, at = [], [], 0
        for b, n in enumerate(lens):
            self.table[b, :need[b]] = order[at:at + need[b]]
            at += need[b]
            k, v = (pm.decode(pm.encode(normal(seed + 2 * b + i + 7, n, n_kv, d), dtype), dtype) for i in (0, 1))
            for j in range(need[b]):
                part = slice(j * page, min(n, (j + 1) * page))
                self.k[self.table[b, j], :part.stop - part.start] = k[part]
                self.v[self.table[b, j], :part.stop - part.start] = v[part]
            self.keys.append(k)
            self.values.append(v)
        self.bufs = [ctx.array_to_buffer(pm.encode(self.k, dtype)), ctx.array_to_buffer(pm.encode(self.v, dtype)),
                     ctx.array_to_buffer(self.table), ctx.array_to_buffer(np.array(lens, np.int32))]
        self.bk, self.bv, self.bt, self.bl = self.bufs

    def free(self):
        for b in self.bufs:
            b.free()


def close(got, want, tol, what=""):
    assert np.isfinite(got).all(), what
    over = np.abs(got.astype(np.float64) - want) - tol
    assert over.max() <= 0, f"{what}: {over.max()} beyond the tolerance at {np.unravel_index(over.argmax(), over.shape)}"


# ---- the models themselves ------------------------------------------------------------------------
def test_models_known_answers():
    x = normal(1, 3, 8)
    assert np.allclose(pm.rope(x, 0, 1e4), x)
    assert np.allclose(pm.rope(np.array([[1.0, 0.0]]), 1, 1e4), [[np.cos(1), np.sin(1)]])
    q, k, v = np.zeros((2, 1, 4)), normal(2, 3, 1, 4), normal(3, 3, 1, 4)
    out, _ = pm.attention(q, k, v, 1.0, True, "f32")
    assert np.allclose(out[0, 0], v[:2, 0].mean(0)) and np.allclose(out[1, 0], v[:, 0].mean(0))
    out, _ = pm.attention(np.ones((3, 1, 4)), k[:2], v[:2], 1.0, True, "f32")     # more rows than keys: the first sees none
    assert not out[0].any() and np.allclose(out[1, 0], v[0, 0])
    assert list(pm.from_bf16(pm.to_bf16(np.array([1.0, 1.00390625, 1.01171875], np.float32)))) == [1.0, 1.0, 1.015625]


# ---- refusals ----------------------------------------------------------------------------------------
def test_null_handles_are_status_codes():
    lib = L.load()
    for name in ("rstq_paged_rope_append", "rstq_paged_decode_attention", "rstq_prompt_attention", "rstq_paged_prompt_attention",
                 "rstq_pages_free", "rstq_pages_extend", "rstq_pages_fork", "rstq_pages_compact", "rstq_pages_copy"):
        args = [None if a is C.c_void_p else a(1) for a in L.SIGNATURES[name]]
        assert getattr(lib, name)(*args) == L.E_INVALID


@pytest.mark.gpu
def test_refusals(ctx):
    lens, heads = [20, 5], (4, 2, 2, 64)
    p = Pool(ctx, lens, 2, 64, 16, "f32")
    rows = 2
    q, out = ctx.make_buffer(rows * 256, np.float32), ctx.make_buffer(rows * 256, np.float32)
    cu = ctx.array_to_buffer(np.array([0, 1, 2], np.int32))
    n_q, group, n_kv, d = heads

    def decode(**kw):
        a = dict(q=q, kcache=p.bk, vcache=p.bv, out=out, table=p.bt, lens=p.bl, seqs=2, n_q=n_q, group=group, n_kv=n_kv, head_dim=d,
                 page=16, n_pages=p.n_pages, max_pages=p.width, scale=0.125, dtype=L.F32)
        ctx.paged_decode_attention(**{**a, **kw})

    def prompt(**kw):
        a = dict(q=q, k=p.bk, v=p.bv, out=out, cu_q=cu, cu_k=cu, rows=rows, kv_rows=2, seqs=2, n_q=n_q, group=group, n_kv=n_kv,
                 head_dim=d, scale=0.125)
        ctx.prompt_attention(**{**a, **kw})

    def append(**kw):
        a = dict(q=q, k=q, v=q, qout=out, kcache=p.bk, vcache=p.bv, table=p.bt, lens=p.bl, cu=None, rows=2, seqs=2, n_q=n_q, n_kv=n_kv,
                 head_dim=d, page=16, n_pages=p.n_pages, max_pages=p.width, theta=1e4)
        ctx.paged_rope_append(**{**a, **kw})

    small = ctx.make_buffer(16, np.float32)
    cases = [(decode, dict(head_dim=60), L.E_SHAPE), (decode, dict(head_dim=264), L.E_SHAPE), (decode, dict(group=3), L.E_SHAPE),
             (decode, dict(page=24), L.E_SHAPE), (decode, dict(page=8), L.E_SHAPE), (decode, dict(dtype=7), L.E_INVALID),
             (decode, dict(seqs=0), L.E_LIMIT), (decode, dict(n_pages=p.n_pages + 1), L.E_INVALID),
             (decode, dict(ldq=128), L.E_SHAPE), (decode, dict(ldq=257), L.E_ALIGN), (decode, dict(out=small), L.E_INVALID),
             (decode, dict(scale=float("nan")), L.E_SHAPE), (decode, dict(max_pages=1 << 21), L.E_LIMIT),
             (prompt, dict(causal=2), L.E_INVALID), (prompt, dict(rows=-1), L.E_SHAPE), (prompt, dict(cu_k=small, seqs=40), L.E_INVALID),
             (prompt, dict(ldk=64), L.E_SHAPE), (prompt, dict(kv_rows=1 << 20), L.E_INVALID),
             (append, dict(rows=1), L.E_SHAPE), (append, dict(theta=0.0), L.E_SHAPE), (append, dict(in_dtype=5), L.E_INVALID),
             (append, dict(ldkv=129), L.E_ALIGN), (append, dict(n_q=0), L.E_SHAPE)]
    for fn, kw, code in cases:
        with pytest.raises(L.RstqError) as e:
            fn(**kw)
        assert e.value.code == code, (fn.__name__, kw, e.value)
    ctx.sync()
    for b in (q, out, cu, small):
        b.free()
    p.free()


# ---- rope + append ---------------------------------------------------------------------------------
APPENDS = [
    # in, stored, n_q, n_kv, d, page, lengths, new rows (None: one each, no cu)
    ("f32", "bf16", 4, 2, 64, 16, [1, 16, 17, 33], None),
    ("f32", "f32", 8, 8, 128, 32, [5, 100, 64], None),
    ("bf16", "bf16", 7, 1, 96, 16, [40, 1, 9], [40, 1, 3]),
    ("bf16", "f32", 2, 2, 8, 64, [70], [70]),
    ("f32", "bf16", 6, 3, 256, 128, [300, 0, 130], [200, 0, 1]),
    ("f32", "bf16", 1, 1, 16, 256, [100000], [2]),          # far positions
    ("f32", "f32", 4, 1, 64, 16, [1300], [1290]),           # enough rows for four to a block
]


@pytest.mark.gpu
@pytest.mark.parametrize("tin,tout,n_q,n_kv,d,page,lens,new", APPENDS)
@pytest.mark.parametrize("fused", [False, True])
def test_rope_append(ctx, tin, tout, n_q, n_kv, d, page, lens, new, fused):
    theta, pad = 1e4, 3 if new else 0
    counts = new or [1] * len(lens)
    rows = sum(counts) + pad
    p = Pool(ctx, lens, n_kv, d, page, tout, seed=5)
    qkv = pm.encode(normal(11, rows, (n_q + 2 * n_kv) * d), tin)
    x = pm.decode(qkv, tin)
    q, k, v = x[:, :n_q * d].reshape(rows, n_q, d), x[:, n_q * d:(n_q + n_kv) * d].reshape(rows, n_kv, d), x[:, (n_q + n_kv) * d:].reshape(rows, n_kv, d)
    if fused:       # q, k and v as slices of one matrix
        base = ctx.array_to_buffer(qkv)
        step, item = (n_q + 2 * n_kv) * d, NP[tin]().itemsize
        total = rows * step
        bq, bk, bv = (ctx.wrap_buffer(base.device_ptr + o * item, total - o, NP[tin]) for o in (0, n_q * d, (n_q + n_kv) * d))
        ld = dict(ldq=step, ldkv=step)
    else:
        base, ld = None, {}
        bq, bk, bv = (ctx.array_to_buffer(pm.encode(t, tin)) for t in (q, k, v))
    bo = ctx.array_to_buffer(np.full(rows * n_q * d, 7, NP[tout]))
    cu = ctx.array_to_buffer(np.cumsum([0] + counts).astype(np.int32)) if new else None
    ctx.paged_rope_append(bq, bk, bv, bo, p.bk, p.bv, p.bt, p.bl, cu, rows, len(lens), n_q, n_kv, d, page, p.n_pages, p.width, theta,
                          DT[tin], DT[tout], **ld)
    ctx.sync()
    raw = bo.download().reshape(rows, n_q, d)
    got_q = pm.decode(raw, tout)
    gk, gv = pm.decode(p.bk.download(), tout).reshape(p.k.shape), pm.decode(p.bv.download(), tout).reshape(p.v.shape)
    wk, wv = p.k.copy(), p.v.copy()
    # cos and sin to 2 * 2^-24, two products and a sum in f32, then the stored type
    def tol(want, a):
        h = np.abs(a)
        pair = np.concatenate([h[..., :d // 2] + h[..., d // 2:]] * 2, -1)
        return pm.HALF[tout] * np.abs(want) + 6 * 2.0 ** -24 * pair + 1e-38
    t = 0
    tk = np.zeros(wk.shape)
    for b, n in enumerate(counts):
        for i in range(n):
            pos = lens[b] - n + i
            want = pm.rope(q[t], pos, theta)
            close(got_q[t], want, tol(want, q[t]), f"q row {t}")
            pg, s = p.table[b, pos // page], pos % page
            wk[pg, s], wv[pg, s] = pm.rope(k[t], pos, theta), pm.decode(pm.encode(v[t], tout), tout)
            tk[pg, s] = tol(wk[pg, s], k[t])
            t += 1
    assert (raw[t:] == 7).all()                        # rows behind the last sequence
    assert np.array_equal(np.isnan(gk), np.isnan(wk)) and np.array_equal(gv, wv, equal_nan=True)
    assert (np.nan_to_num(np.abs(gk - wk) - tk) <= 0).all()
    for o in (bq, bk, bv, bo, base, cu):
        if o is not None:
            o.free()
    p.free()


@pytest.mark.gpu
def test_rope_append_in_place_and_rows_without_a_page(ctx):
    """qout may be q; a row whose position lies behind its pages, or before the sequence, or whose table entry names no page is
    left out and rstq_sync says so."""
    n_q, n_kv, d, page = 4, 2, 64, 16
    p = Pool(ctx, [16, 17, 16], n_kv, d, page, "f32")
    q, k, v = normal(1, 3, n_q, d), normal(2, 3, n_kv, d), normal(3, 3, n_kv, d)
    bq, bk, bv = ctx.array_to_buffer(q), ctx.array_to_buffer(k), ctx.array_to_buffer(v)
    before = p.bk.download()
    for lens, table, done in (([16, 17, 0], None, [0, 1]), ([33, 17, 16], None, [1, 2]), ([16, 17, 16], (0, 0, p.n_pages), [1, 2])):
        bq.upload(q)
        p.bk.upload(before)
        p.bl.upload(np.array(lens, np.int32))
        tab = p.table.copy()
        if table:
            tab[table[0], table[1]] = table[2]
        p.bt.upload(tab)
        ctx.paged_rope_append(bq, bk, bv, bq, p.bk, p.bv, p.bt, p.bl, None, 3, 3, n_q, n_kv, d, page, p.n_pages, p.width, 1e4)
        with pytest.raises(L.RstqError) as e:
            ctx.sync()
        assert e.value.code == L.E_RANGE
        ctx.sync()
        got = bq.download().reshape(q.shape)
        for b in range(3):
            want = pm.rope(q[b], lens[b] - 1, 1e4) if b in done else q[b]
            assert np.abs(got[b] - want).max() <= 1e-5 * (b in done)
        pool = p.bk.download()
        moved = int((pool.view(np.uint32) != before.view(np.uint32)).reshape(-1, n_kv * d).any(1).sum())
        assert moved == len(done)
    for b in (bq, bk, bv):
        b.free()
    p.free()


# ---- decode ----------------------------------------------------------------------------------------
DECODES = [
    # dtype, n_q, n_kv, d, page, lengths
    ("bf16", 8, 2, 128, 16, [1, 15, 16, 17, 0, 63, 64, 65]),
    ("bf16", 32, 8, 128, 16, [300]),
    ("bf16", 28, 4, 128, 32, [1000, 3, 129]),
    ("bf16", 4, 4, 64, 64, [200, 1, 700]),
    ("bf16", 16, 1, 64, 128, [513, 128]),
    ("bf16", 24, 1, 128, 16, [50, 260]),           # more heads in the group than a block serves at once
    ("bf16", 4, 2, 96, 16, [70, 31]),
    ("bf16", 3, 1, 8, 16, [20]),
    ("bf16", 2, 1, 256, 16, [40, 100]),
    ("bf16", 8, 8, 128, 256, [2500, 255, 257]),
    ("f32", 8, 2, 128, 16, [1, 15, 16, 17, 0, 33, 64]),
    ("f32", 32, 32, 128, 32, [700, 40]),
    ("f32", 7, 1, 64, 16, [333, 2]),
    ("f32", 20, 1, 128, 64, [130]),
    ("f32", 2, 2, 40, 16, [77]),
    ("f32", 4, 1, 256, 16, [65]),
    ("bf16", 4, 1, 128, 16, list(range(0, 200, 2))),     # many short sequences
    ("f32", 2, 1, 64, 16, [6000]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n_q,n_kv,d,page,lens", DECODES)
def test_decode(ctx, dtype, n_q, n_kv, d, page, lens):
    p = Pool(ctx, lens, n_kv, d, page, dtype, seed=n_q + d)
    B = len(lens)
    step = n_q * d + 16
    full = pm.encode(normal(3, B, step) * 2, dtype)             # q in rows that are longer than q
    q = pm.decode(full, dtype)[:, :n_q * d].reshape(B, n_q, d)
    bq, bo = ctx.array_to_buffer(full), ctx.array_to_buffer(np.full(B * n_q * d, 7, NP[dtype]))
    scale = d ** -0.5

    def run():
        ctx.paged_decode_attention(bq, p.bk, p.bv, bo, p.bt, p.bl, B, n_q, n_q // n_kv, n_kv, d, page, p.n_pages, p.width, scale,
                                   DT[dtype], ldq=step)
        ctx.sync()
        return bo.download()
    raw = run()
    got = pm.decode(raw, dtype).reshape(B, n_q, d)
    for b in range(B):
        want, tol = pm.attention(q[b:b + 1], p.keys[b], p.values[b], scale, False, dtype)
        close(got[b:b + 1], want, tol, f"sequence {b} of {lens[b]}")
    assert np.array_equal(run(), raw)                           # the same again, bit for bit
    bq.free()
    bo.free()
    p.free()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_decode_lengths_and_pages_that_say_too_much(ctx, dtype):
    """A length beyond the pages counts as their end, a negative one as none; an entry that names no page leaves its positions
    out, and rstq_sync says so."""
    n_q, n_kv, d, page = 4, 2, 64, 16
    p = Pool(ctx, [48, 20, 30], n_kv, d, page, dtype)
    p.bl.upload(np.array([1000, 20, -5], np.int32))
    tab = p.table.copy()
    tab[1, 0] = -1
    tab[2] = 1 << 28
    p.bt.upload(tab)
    q = pm.decode(pm.encode(normal(3, 3, n_q, d), dtype), dtype)
    bq, bo = ctx.array_to_buffer(pm.encode(q, dtype)), ctx.make_buffer(3 * n_q * d, NP[dtype])
    ctx.paged_decode_attention(bq, p.bk, p.bv, bo, p.bt, p.bl, 3, n_q, 2, n_kv, d, page, p.n_pages, p.width, 0.125, DT[dtype])
    with pytest.raises(L.RstqError) as e:
        ctx.sync()
    assert e.value.code == L.E_RANGE
    ctx.sync()
    got = pm.decode(bo.download(), dtype).reshape(3, n_q, d)
    want, tol = pm.attention(q[:1], p.keys[0], p.values[0], 0.125, False, dtype)
    close(got[:1], want, tol)
    want, tol = pm.attention(q[1:2], p.keys[1][16:], p.values[1][16:], 0.125, False, dtype)
    close(got[1:2], want, tol)
    assert not got[2].any()
    bq.free()
    bo.free()
    p.free()


@pytest.mark.gpu
def test_decode_scores_that_are_not_numbers(ctx):
    """Infinities and NaN in positions that a row sees come out as softmax says, in other sequences' rows not at all."""
    n_q, n_kv, d, page = 2, 1, 64, 16
    for dtype in ("f32", "bf16"):
        p = Pool(ctx, [40, 40, 40], n_kv, d, page, dtype)
        k, v = p.bk.download().reshape(p.k.shape), p.bv.download().reshape(p.v.shape)
        nan, inf = pm.encode(np.array([np.nan, np.inf], np.float32), dtype)
        k[p.table[0, 1], 3, 0, 5] = nan
        v[p.table[1, 2], 1, 0, 9] = inf
        p.bk.upload(k)
        p.bv.upload(v)
        q = pm.decode(pm.encode(normal(3, 3, n_q, d), dtype), dtype)
        bq, bo = ctx.array_to_buffer(pm.encode(q, dtype)), ctx.make_buffer(3 * n_q * d, NP[dtype])
        ctx.paged_decode_attention(bq, p.bk, p.bv, bo, p.bt, p.bl, 3, n_q, 2, n_kv, d, page, p.n_pages, p.width, 0.125, DT[dtype])
        ctx.sync()
        got = pm.decode(bo.download(), dtype).reshape(3, n_q, d)
        assert np.isnan(got[0]).all()
        assert np.isposinf(got[1, :, 9]).all() and np.isfinite(np.delete(got[1], 9, -1)).all()
        want, tol = pm.attention(q[2:], p.keys[2], p.values[2], 0.125, False, dtype)
        close(got[2:], want, tol)
        for b in (bq, bo):
            b.free()
        p.free()


# ---- prompts ---------------------------------------------------------------------------------------
PROMPTS = [
    # dtype, n_q, n_kv, d, page (0: packed), key lengths, new rows (None: all), causal
    ("bf16", 4, 2, 128, 0, [1, 2, 127, 0, 128, 129], None, True),
    ("bf16", 2, 2, 64, 0, [300, 17], None, True),
    ("bf16", 7, 1, 128, 0, [260], None, True),
    ("bf16", 2, 1, 96, 0, [140, 33], None, True),
    ("bf16", 2, 1, 128, 0, [200, 64], None, False),
    ("bf16", 2, 1, 64, 0, [50, 10, 400], [70, 10, 130], True),      # more rows than keys; fewer
    ("bf16", 2, 1, 64, 0, [50, 0, 300], [70, 10, 13], False),
    ("bf16", 1, 1, 256, 0, [90], None, True),
    ("bf16", 1, 1, 8, 0, [90], None, True),
    ("bf16", 4, 1, 128, 16, [300, 40, 17], [130, 40, 1], True),
    ("bf16", 2, 2, 64, 32, [129, 260, 0], [2, 200, 0], True),
    ("bf16", 2, 1, 128, 64, [700], [300], True),
    ("bf16", 2, 1, 128, 128, [500, 200], [500, 60], True),
    ("bf16", 2, 1, 128, 256, [600, 255, 257], [257, 1, 129], True),
    ("bf16", 2, 1, 128, 16, [100, 30], [20, 30], False),
    ("f32", 4, 2, 64, 0, [1, 2, 63, 0, 64, 65, 150], None, True),
    ("f32", 2, 2, 128, 0, [130, 33], None, True),
    ("f32", 3, 1, 40, 0, [70], None, False),
    ("f32", 2, 1, 256, 0, [60], None, True),
    ("f32", 2, 1, 128, 16, [200, 40], [100, 40], True),
    ("f32", 2, 1, 64, 0, [50, 10], [70, 10], True),
]


def prompt_case(ctx, dtype, n_q, n_kv, d, page, lens, new, causal, spoil=None, scale=None):
    """Runs a prompt call in rows that are longer than they need be, with rows behind the last sequence; returns
    [(got, q, k, v) per sequence]."""
    new = new or lens
    rows, pad = sum(new), 5
    step = n_q * d + 8
    full = pm.encode(normal(4, rows + pad, step) * 2, dtype)
    q = pm.decode(full, dtype)[:, :n_q * d].reshape(rows + pad, n_q, d)
    bq, bo = ctx.array_to_buffer(full), ctx.array_to_buffer(np.full((rows + pad) * n_q * d, 7, NP[dtype]))
    cu = np.cumsum([0] + list(new)).astype(np.int32)
    bcu = ctx.array_to_buffer(cu)
    scale = scale or d ** -0.5
    extra = []
    if page:
        p = Pool(ctx, lens, n_kv, d, page, dtype, seed=n_q + d)
        keys, values = p.keys, p.values
        ctx.paged_prompt_attention(bq, p.bk, p.bv, bo, p.bt, bcu, p.bl, rows + pad, len(lens), n_q, n_q // n_kv, n_kv, d, page,
                                   p.n_pages, p.width, scale, causal, DT[dtype], ldq=step)
        ctx.sync()
        p.free()
    else:
        ku = np.cumsum([0] + list(lens)).astype(np.int32)
        kstep = n_kv * d + 16
        k, v = (pm.decode(pm.encode(normal(s, ku[-1] + 4, kstep), dtype), dtype) for s in (5, 6))
        k[ku[-1]:], v[ku[-1]:] = np.nan, np.nan                 # keys behind the last sequence
        if spoil:
            spoil(k, v, ku)
        bk, bv, bku = ctx.array_to_buffer(pm.encode(k, dtype)), ctx.array_to_buffer(pm.encode(v, dtype)), ctx.array_to_buffer(ku)
        extra = [bk, bv, bku]
        ctx.prompt_attention(bq, bk, bv, bo, bcu, bku, rows + pad, ku[-1] + 4, len(lens), n_q, n_q // n_kv, n_kv, d, scale, causal,
                             DT[dtype], ldq=step, ldk=kstep)
        ctx.sync()
        cut = lambda x, b: x[ku[b]:ku[b + 1], :n_kv * d].reshape(-1, n_kv, d)  # noqa: E731
        keys, values = [cut(k, b) for b in range(len(lens))], [cut(v, b) for b in range(len(lens))]
    raw = bo.download().reshape(rows + pad, n_q, d)
    assert (raw[rows:] == 7).all()
    got = pm.decode(raw, dtype)
    for b in [bq, bo, bcu] + extra:
        b.free()
    return [(got[cu[b]:cu[b + 1]], q[cu[b]:cu[b + 1]], keys[b], values[b]) for b in range(len(lens))], scale


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n_q,n_kv,d,page,lens,new,causal", PROMPTS)
def test_prompt(ctx, dtype, n_q, n_kv, d, page, lens, new, causal):
    seqs, scale = prompt_case(ctx, dtype, n_q, n_kv, d, page, lens, new, causal)
    for b, (got, q, k, v) in enumerate(seqs):
        if len(q):
            want, tol = pm.attention(q, k, v, scale, causal, dtype)
            close(got, want, tol, f"sequence {b}")


# few rows behind many keys, which are cut into parts; groups of heads that share a tile and that do not; many blocks of rows
LONG = [
    ("bf16", 8, 2, 128, 32, [2500, 1100, 7, 1500], [2, 40, 7, 1], True),
    ("bf16", 6, 2, 64, 16, [3000, 0, 1030], [5, 0, 30], True),
    ("bf16", 2, 2, 128, 0, [1500, 200], [3, 200], True),
    ("bf16", 16, 1, 96, 64, [1200], [20], False),
    ("bf16", 4, 1, 128, 256, [4000], [1], True),
    ("bf16", 8, 1, 64, 0, [700, 600, 650], None, True),
    ("f32", 4, 1, 128, 32, [1500, 70], [3, 70], True),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n_q,n_kv,d,page,lens,new,causal", LONG)
def test_prompt_of_few_rows_behind_many_keys(ctx, dtype, n_q, n_kv, d, page, lens, new, causal):
    seqs, scale = prompt_case(ctx, dtype, n_q, n_kv, d, page, lens, new, causal)
    for b, (got, q, k, v) in enumerate(seqs):
        pick = sorted({0, len(q) // 2, len(q) - 1}) if len(q) > 64 else range(len(q))       # (the model is slow)
        for r in pick:
            if len(q):
                m = len(k) - len(q) + r + 1 if causal else len(k)
                want, tol = pm.attention(q[r:r + 1], k[:m], v[:m], scale, False, dtype)
                close(got[r:r + 1], want, tol, f"sequence {b} row {r}")


@pytest.mark.gpu
def test_prompt_parts_with_values_that_are_not_numbers(ctx):
    """Keys cut into parts: an infinity above the diagonal, in the last part, is not seen; one below it is."""
    n_q, n_kv, d, page, n, rows = 4, 1, 64, 32, 2600, 3
    p = Pool(ctx, [n], n_kv, d, page, "bf16")
    v = p.bv.download().reshape(p.v.shape)
    at = lambda pos: (p.table[0, pos // page], pos % page)  # noqa: E731
    v[at(n - 1)][0, 5] = pm.encode(np.array([np.inf], np.float32), "bf16")[0]        # the last row's own
    v[at(100)][0, 6] = pm.encode(np.array([-np.inf], np.float32), "bf16")[0]         # everybody's
    p.bv.upload(v)
    q = pm.decode(pm.encode(normal(4, rows, n_q, d), "bf16"), "bf16")
    bq, bo, cu = ctx.array_to_buffer(pm.encode(q, "bf16")), ctx.make_buffer(rows * n_q * d, np.uint16), ctx.array_to_buffer(np.array([0, rows], np.int32))
    ctx.paged_prompt_attention(bq, p.bk, p.bv, bo, p.bt, cu, p.bl, rows, 1, n_q, n_q, n_kv, d, page, p.n_pages, p.width, 0.125, True, L.BF16)
    ctx.sync()
    got = pm.decode(bo.download(), "bf16").reshape(rows, n_q, d)
    assert np.isneginf(got[:, :, 6]).all() and np.isposinf(got[2, :, 5]).all() and np.isfinite(got[:2, :, 5]).all()
    for r in range(rows):
        m = n - rows + r + 1
        want, tol = pm.attention(q[r:r + 1], p.keys[0][:m], p.values[0][:m], 0.125, False, "bf16")
        keep = [i for i in range(d) if i not in (5, 6)]
        close(got[r:r + 1][..., keep], want[..., keep], tol[..., keep], f"row {r}")
    tab = p.table.copy()
    tab[0, 40] = p.n_pages
    p.bt.upload(tab)                                                                   # a page that is none: its positions are left out
    ctx.paged_prompt_attention(bq, p.bk, p.bv, bo, p.bt, cu, p.bl, rows, 1, n_q, n_q, n_kv, d, page, p.n_pages, p.width, 0.125, True, L.BF16)
    with pytest.raises(L.RstqError) as e:
        ctx.sync()
    assert e.value.code == L.E_RANGE
    got = pm.decode(bo.download(), "bf16").reshape(rows, n_q, d)
    k, w = (np.delete(x[0], np.s_[40 * page:41 * page], 0) for x in (p.keys, p.values))
    want, tol = pm.attention(q[:1], k[:len(k) - 2], w[:len(k) - 2], 0.125, False, "bf16")
    close(got[:1][..., keep], want[..., keep], tol[..., keep])
    for b in (bq, bo, cu):
        b.free()
    p.free()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,d", [("bf16", 128), ("bf16", 64), ("bf16", 256), ("f32", 64)])
def test_prompt_rows_do_not_see_what_comes_after_them(ctx, dtype, d):
    """NaN and infinities in keys and values that a row does not see (later ones of its own sequence, other sequences') leave it
    as it is; rows that see them show them."""
    lens = [40, 150, 130]

    def spoil(k, v, ku):
        k[ku[1] + 100, 3] = np.nan
        v[ku[1] + 90, 7] = np.inf
        v[ku[2] + 128, 2] = np.nan

    seqs, scale = prompt_case(ctx, dtype, 2, 1, d, 0, lens, None, True, spoil)
    for b, clean in ((0, 40), (1, 90), (2, 128)):
        got, q, k, v = seqs[b]
        want, tol = pm.attention(q[:clean], k[:clean], v[:clean], scale, True, dtype)
        close(got[:clean], want, tol, f"sequence {b}")
    assert np.isposinf(seqs[1][0][90:100, :, 7]).all() and np.isfinite(np.delete(seqs[1][0][90:100], 7, -1)).all()
    assert np.isnan(seqs[1][0][100:]).all()
    assert np.isnan(seqs[2][0][128:, :, 2]).all() and np.isfinite(np.delete(seqs[2][0][128:], 2, -1)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prompt_large_scores(ctx, dtype):
    """Scores of some hundreds, growing along the keys and falling along them: the running maximum moves all the time."""
    seqs, scale = prompt_case(ctx, dtype, 2, 1, 64, 0, [400], None, True, lambda k, v, ku: k.__imul__(
        np.linspace(0.1, 20, len(k), dtype=np.float32)[:, None]) if dtype == "f32" else k.__imul__(2.0 ** (np.arange(len(k)) // 64)[:, None]))
    got, q, k, v = seqs[0]
    want, tol = pm.attention(q, k, v, scale, True, dtype)
    close(got, want, tol)
    seqs, scale = prompt_case(ctx, dtype, 2, 1, 64, 0, [400], None, False, lambda k, v, ku: k.__imul__(2.0 ** -(np.arange(len(k)) // 64)[:, None] * 16))
    got, q, k, v = seqs[0]
    want, tol = pm.attention(q, k, v, scale, False, dtype)
    close(got, want, tol)

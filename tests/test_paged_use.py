"""The operators over a paged cache as a program has them: by their registered names, and between the quantized matmuls."""
import numpy as np
import pytest

import paged_model as pm
from oracle import oracle as orc
from raster_b200 import _lib as L
from raster_b200 import cuda_runtime as rt
from raster_b200 import synth
from test_paged_attention import DT, NP, Pool, close, normal
from test_pages import Cache

NAMES = {"paged-rope-append!": 9, "paged-decode-attention!": 6, "prompt-attention!": 6, "paged-prompt-attention!": 7, "pages-free!": 5, "pages-extend!": 6,
         "pages-fork!": 8, "pages-compact!": 8, "pages-copy!": 5}


def test_registered_names_and_numbers_of_arrays():
    for name, arrays in NAMES.items():
        assert rt.kernel_registry_entry(name)["kernel_name"] == name
        for wrong in (arrays - 1, arrays + 1):
            with pytest.raises(ValueError):
                rt.bind_registered_map_void_kernel(name, [None] * wrong, [])
    with pytest.raises(ValueError):
        rt.bind_registered_map_void_kernel("pages-free!", [None] * 5, [1, 2, 3, 4])
    with pytest.raises(TypeError):
        rt.bind_registered_map_void_kernel("pages-copy!", [np.zeros(4)] * 5, [1, 2, 3, 4])


@pytest.fixture
def session():
    ctx = rt.init(("cuda:0",))
    yield ctx
    rt.shutdown()


@pytest.mark.gpu
def test_pages_by_their_registered_names(session):
    c = Cache(session, 6, 30, 5, 16)
    state = [c.bt, c.bl, c.br]

    def ints(*v):
        return c.ints(v)

    a, b = ints(0, 1, 2), ints(33, 16, 5)
    rt.invoke_registered_map_void_kernel("pages-extend!", [*state, a, b, c.bi], [3, *c.sizes])
    c.after(c.m.extend([0, 1, 2], [33, 16, 5]), 0, a, b)
    a, b = ints(0, 1), ints(3, 4)
    rt.invoke_registered_map_void_kernel("pages-fork!", [c.bk, c.bv, *state, a, b, c.bi], [2, *c.sizes, c.layers, c.row])
    status, pairs = c.m.fork([0, 1], [3, 4])
    c.move(pairs)
    c.after(status, len(pairs), a, b)
    a = ints(1, 0)
    rt.invoke_registered_map_void_kernel("pages-free!", [*state, a, c.bi], [2, *c.sizes])
    c.after(c.m.free([1, 0]), 0, a)
    bound = rt.bind_registered_map_void_kernel("pages-compact!", [c.bk, c.bv, *state, c.bt, c.br, c.bi], [*c.sizes, c.layers, c.row])
    rt.launch_registered_bound(bound)
    pairs = c.m.compact()
    c.move(pairs)
    c.after(0, len(pairs))
    a, b = ints(0, 1), ints(28, 29)
    rt.invoke_registered_map_void_kernel("pages-copy!", [c.bk, c.bv, a, b, c.bi], [2, c.n_pages, c.layers, c.page * c.row])
    assert c.info() == [0, 0, 2, 0]
    c.move([(0, 28), (1, 29)])
    assert np.array_equal(c.bk.download().reshape(c.k.shape), c.k) and np.array_equal(c.bv.download().reshape(c.v.shape), c.v)
    a.free()
    b.free()
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_step_by_registered_names_in_a_graph(session, dtype):
    """Rope and append, decode and prompt attention bound once, run by themselves and then as one graph."""
    n_q, n_kv, d, page, lens, new = 4, 2, 64, 16, [40, 17, 5], [3, 17, 1]
    ctx, B, rows, scale = session, 3, 21, d ** -0.5
    p = Pool(ctx, lens, n_kv, d, page, dtype)
    q, k, v = normal(1, rows, n_q, d), normal(2, rows, n_kv, d), normal(3, rows, n_kv, d)
    up = ctx.array_to_buffer
    cu = np.cumsum([0] + new).astype(np.int32)
    bq, bk, bv, bcu, bku = up(q), up(k), up(v), up(cu), up(np.cumsum([0] + lens).astype(np.int32))
    bqt, bo, bd, bp = (ctx.make_buffer(n * n_q * d, NP[dtype]) for n in (rows, rows, B, rows))
    keys, values = (up(pm.encode(np.concatenate(x), dtype)) for x in (p.keys, p.values))
    t, pages = DT[dtype], [page, p.n_pages, p.width]
    bind = lambda name, arrays, scalars: rt.bind_registered_map_void_kernel(name, arrays, scalars, async_=True)  # noqa: E731
    bounds = [bind("paged-rope-append!", [bq, bk, bv, bqt, p.bk, p.bv, p.bt, p.bl, bcu], [rows, B, n_q, n_kv, d, *pages, 1e4, L.F32, t]),
              bind("paged-prompt-attention!", [bqt, p.bk, p.bv, bo, p.bt, bcu, p.bl], [rows, B, n_q, n_q // n_kv, n_kv, d, *pages, scale, True, t]),
              bind("paged-decode-attention!", [bqt, p.bk, p.bv, bd, p.bt, p.bl], [B, n_q, n_q // n_kv, n_kv, d, *pages, scale, t]),
              bind("prompt-attention!", [bqt, keys, values, bp, bcu, bku], [rows, sum(lens), B, n_q, n_q // n_kv, n_kv, d, scale, True, t])]

    def check():
        qt = pm.decode(bqt.download(), dtype).reshape(rows, n_q, d)
        pk, pv = (pm.decode(x.download(), dtype).reshape(p.k.shape) for x in (p.bk, p.bv))
        got, dec, packed = (pm.decode(x.download(), dtype).reshape(-1, n_q, d) for x in (bo, bd, bp))
        for b, n in enumerate(lens):
            kk, vv = (np.concatenate([x[i] for i in p.table[b, :-(-n // page)]])[:n] for x in (pk, pv))
            for r in range(new[b]):
                want = pm.rope(q[cu[b] + r], n - new[b] + r, 1e4)
                assert np.abs(qt[cu[b] + r] - want).max() <= (pm.HALF[dtype] + 2.0 ** -20) * np.abs(want).max()
            close(got[cu[b]:cu[b + 1]], *pm.attention(qt[cu[b]:cu[b + 1]], kk, vv, scale, True, dtype), f"prompt {b}")
            close(dec[b:b + 1], *pm.attention(qt[b:b + 1], kk, vv, scale, False, dtype), f"decode {b}")
            close(packed[cu[b]:cu[b + 1]], *pm.attention(qt[cu[b]:cu[b + 1]], p.keys[b], p.values[b], scale, True, dtype), f"packed {b}")

    for b in bounds:
        rt.launch_registered_bound(b)
    rt.synchronize_async()
    check()
    graph = rt.record_graph(bounds)
    for b in (bqt, bo, bd, bp):
        b.fill_bytes(0xFF)
    rt.replay_graph(graph)
    check()
    rt.destroy_graph(graph)
    for b in (bq, bk, bv, bcu, bku, bqt, bo, bd, bp, keys, values):
        b.free()
    p.free()


# ---- between the matmuls -------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("counts", [[70, 1, 33, 0], [1, 1, 1, 1], [300, 129, 2, 64]])
def test_between_the_matmuls(ctx, dtype, counts):
    """A layer's attention as it is used: hidden rows through the fused q|k|v matmul, whose rows (f32, slices of one matrix) are turned and written
    to their pages, attention in the cache's type, and its rows, as they are, into the output matmul; the first step a prompt, the second one
    token for every sequence that has any.  Each stage against a model of it on what the stage before left."""
    n_q, n_kv, d, page, width, H = 4, 2, 64, 16, 24, 256
    n_qkv, scale, B, t = (n_q + 2 * n_kv) * d, d ** -0.5, 4, DT[dtype]
    wqkv, sqkv = orc.quantize_weight(synth.normal(1, n_qkv * H, 0.08), 8)
    wo, so = orc.quantize_weight(synth.normal(2, H * n_q * d, 0.05), 4)
    bqkv = ctx.bind_weight(wqkv, sqkv, n_qkv, H, L.FMT_Q8_0, L.LAYOUT_ROWMAJOR)
    bwo = ctx.bind_weight(wo, so, H, n_q * d, L.FMT_Q4_0, L.LAYOUT_ROWMAJOR)
    dense = [orc.matmul_dq_f64(w, sc, fmt, np.eye(k, dtype=np.float32), k, k, n).reshape(k, n) for w, sc, fmt, k, n in
             ((wqkv, sqkv, 1, H, n_qkv), (wo, so, 0, n_q * d, H))]

    def product(got, x, w):
        """Of several rows: both operands are rounded to 16 bits, 2^-8 at most each, the sums in f32 to (H + 8) 2^-23."""
        want, most = x.astype(np.float64) @ w, np.abs(x.astype(np.float64)) @ np.abs(w)
        assert (np.abs(got - want) <= (2.0 ** -7 + 2.0 ** -16 + (H + 8) * 2.0 ** -23) * most).all(), (np.abs(got - want) / most).max()
    n_pages = 64
    m = pm.Pages(B, n_pages, width, page)
    up, mk = ctx.array_to_buffer, ctx.make_buffer
    bt, bl, br, bi = up(m.table), up(m.lens), up(m.refs), mk(4, np.int32)
    bk, bv = mk(n_pages * page * n_kv * d, NP[dtype]), mk(n_pages * page * n_kv * d, NP[dtype])
    bk.fill_bytes(0xFF)
    bv.fill_bytes(0xFF)
    everyone = up(np.arange(B, dtype=np.int32))

    def step(new, seed):
        decode = new == [1 if n else 0 for n in new] and seed > 1
        rows = B if decode else sum(new)
        x = normal(seed, rows, H)
        bx, by, bqt, bo, bz = up(x), mk(rows * n_qkv, np.float32), mk(rows * n_q * d, NP[dtype]), mk(rows * n_q * d, NP[dtype]), mk(rows * H, np.float32)
        counts, cu = up(np.array(new, np.int32)), np.cumsum([0] + new).astype(np.int32)
        bcu = up(cu)
        parts = [ctx.wrap_buffer(by.device_ptr + 4 * o, rows * n_qkv - o, np.float32) for o in (0, n_q * d, (n_q + n_kv) * d)]
        ctx.pages_extend(bt, bl, br, everyone, counts, bi, B, B, n_pages, width, page)
        ctx.qmatmul(bqkv, bx, by, rows, L.F32, L.F32, L.MODE_F)
        ctx.paged_rope_append(*parts, bqt, bk, bv, bt, bl, None if decode else bcu, rows, B, n_q, n_kv, d, page, n_pages, width, 1e4, L.F32, t,
                              ldq=n_qkv, ldkv=n_qkv)
        if decode:
            ctx.paged_decode_attention(bqt, bk, bv, bo, bt, bl, B, n_q, n_q // n_kv, n_kv, d, page, n_pages, width, scale, t)
        else:
            ctx.paged_prompt_attention(bqt, bk, bv, bo, bt, bcu, bl, rows, B, n_q, n_q // n_kv, n_kv, d, page, n_pages, width, scale, True, t)
        ctx.qmatmul(bwo, bo, bz, rows, t, L.F32, L.MODE_F)
        ctx.sync()
        assert bi.download()[0] == 0 and m.extend(list(range(B)), new) == 0
        y, z = by.download().reshape(rows, n_qkv), bz.download().reshape(rows, H)
        product(y, x, dense[0])
        qt = pm.decode(bqt.download(), dtype).reshape(rows, n_q, d)
        o = pm.decode(bo.download(), dtype).reshape(rows, n_q, d)
        pk, pv = (pm.decode(b.download(), dtype).reshape(n_pages, page, n_kv, d) for b in (bk, bv))
        for b in range(B):
            n, place = int(m.lens[b]), [b] if decode else list(range(cu[b], cu[b + 1]))
            if not new[b]:
                assert not decode or not o[b].any()
                continue
            kk, vv = (np.concatenate([p[i] for i in m.table[b, :-(-n // page)]])[:n] for p in (pk, pv))
            for i, r in enumerate(place):
                pos = n - len(place) + i
                for got, x0, heads in ((qt[r], 0, n_q), (kk[pos], n_q * d, n_kv)):
                    turned = pm.rope(y[r, x0:x0 + heads * d].reshape(heads, d), pos, 1e4)
                    assert np.abs(got - turned).max() <= (pm.HALF[dtype] + 2.0 ** -20) * np.abs(turned).max()
                assert np.array_equal(vv[pos], pm.decode(pm.encode(y[r, (n_q + n_kv) * d:].reshape(n_kv, d), dtype), dtype))
            pick = sorted({0, len(place) // 2, len(place) - 1})
            for i in pick:
                seen = n - len(place) + i + 1
                close(o[place[i]][None], *pm.attention(qt[place[i]][None], kk[:seen], vv[:seen], scale, False, dtype), f"sequence {b} row {i}")
        product(z, o.reshape(rows, n_q * d), dense[1])
        for b in (bx, by, bqt, bo, bz, counts, bcu, *parts):
            b.free()

    step(counts, 1)
    for i in range(3):
        step([1 if n else 0 for n in counts], 2 + i)
    for b in (bt, bl, br, bi, bk, bv, everyone):
        b.free()
    for w in (bqkv, bwo):
        w.free()

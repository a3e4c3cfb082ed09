"""Calls over a paged cache as programs make them beyond the plain one: arrays that lie over one another (refused), graphs replayed
after their arrays have changed, two contexts at once, a lent stream, pages that are none in every kind of attention, long lists."""
import numpy as np
import pytest

import paged_model as pm
from raster_b200 import Context
from raster_b200 import _lib as L
from test_paged_attention import DT, NP, Pool, close, normal
from test_pages import Cache


class Prompts:
    """New rows of sequences in a paged cache, with room for `rows` of them and for any lengths up to lens; keeps what a call needs."""

    def __init__(self, ctx, dtype, n_q, n_kv, d, page, lens, new, seed=0):
        self.ctx, self.dtype, self.sizes, self.page = ctx, dtype, (n_q, n_q // n_kv, n_kv, d), page
        self.pool = Pool(ctx, lens, n_kv, d, page, dtype, seed=seed)
        self.lens, self.new, self.rows, self.scale = list(lens), list(new), sum(new), d ** -0.5
        self.bq, self.bo = ctx.make_buffer(self.rows * n_q * d, NP[dtype]), ctx.make_buffer(self.rows * n_q * d, NP[dtype])
        self.bcu = ctx.make_buffer(len(lens) + 1, np.int32)
        self.fill(seed)

    def fill(self, seed, lens=None, new=None):
        """Other queries; other lengths and rows, no more of them than there were."""
        self.lens, self.new = lens or self.lens, new or self.new
        n_q, _, _, d = self.sizes
        self.q = pm.decode(pm.encode(normal(seed + 50, self.rows, n_q, d), self.dtype), self.dtype)
        self.cu = np.cumsum([0] + self.new).astype(np.int32)
        self.bq.upload(pm.encode(self.q, self.dtype))
        self.bcu.upload(self.cu)
        self.pool.bl.upload(np.array(self.lens, np.int32))
        self.bo.upload(np.zeros(self.bo.n_elements, NP[self.dtype]))

    def call(self):
        p = self.pool
        self.ctx.paged_prompt_attention(self.bq, p.bk, p.bv, self.bo, p.bt, self.bcu, p.bl, self.rows, len(self.lens), *self.sizes, self.page,
                                        p.n_pages, p.width, self.scale, True, DT[self.dtype])

    def raw(self):
        return self.bo.download()

    def check(self):
        n_q, _, _, d = self.sizes
        got = pm.decode(self.raw(), self.dtype).reshape(self.rows, n_q, d)
        for b, n in enumerate(self.lens):
            rows = self.cu[b + 1] - self.cu[b]
            for r in sorted({0, rows // 2, rows - 1}) if rows else []:
                m, at = n - rows + r + 1, self.cu[b] + r
                want, tol = pm.attention(self.q[at:at + 1], self.pool.keys[b][:m], self.pool.values[b][:m], self.scale, False, self.dtype)
                close(got[at:at + 1], want, tol, f"sequence {b} row {r}")

    def free(self):
        for b in (self.bq, self.bo, self.bcu):
            b.free()
        self.pool.free()


# one launch; keys cut into parts and joined; f32; any shape
CALLS = [("bf16", 8, 2, 128, 32, [300, 257, 40], [300, 130, 1]),
         ("bf16", 8, 2, 64, 16, [2600, 900, 1300], [3, 40, 2]),
         ("f32", 4, 2, 64, 16, [200, 130], [70, 130]),
         ("f32", 8, 2, 128, 32, [1500, 700, 900], [3, 60, 2]),
         ("bf16", 2, 1, 256, 16, [90, 33], [20, 33])]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n_q,n_kv,d,page,lens,new", CALLS)
def test_a_prompt_call_in_a_graph(ctx, dtype, n_q, n_kv, d, page, lens, new):
    """Recorded once and replayed for other queries, lengths and numbers of rows: what an eager call gives, bit for bit, every time."""
    x = Prompts(ctx, dtype, n_q, n_kv, d, page, lens, new)
    ctx.graph_begin()
    x.call()
    graph = ctx.graph_end()
    for seed, ls, ns in ((1, None, None), (2, [n - 7 for n in lens], [max(n - 30, 0) for n in new]), (3, lens, new)):
        x.fill(seed, ls, ns)
        graph.replay()
        ctx.sync()
        x.check()
        first = x.raw().copy()
        graph.replay()
        ctx.sync()
        assert np.array_equal(x.raw(), first)
        x.bo.upload(np.zeros(x.bo.n_elements, NP[dtype]))
        x.call()
        ctx.sync()
        assert np.array_equal(x.raw(), first)
    graph.destroy()
    x.free()


@pytest.mark.gpu
@pytest.mark.parametrize("case", [1, 3])
def test_two_contexts_at_once(case):
    """Each with scratch of its own: calls under way together give what each gives alone."""
    both = [Context(("cuda:0",)) for _ in range(2)]
    work = [Prompts(c, *CALLS[case], seed=s) for s, c in enumerate(both)]
    alone = []
    for x in work:
        x.call()
        x.ctx.sync()
        x.check()
        alone.append(x.raw().copy())
    for _ in range(5):
        for _ in range(4):
            for x in work:
                x.call()
        for x, a in zip(work, alone):
            x.ctx.sync()
            assert np.array_equal(x.raw(), a)
    for x in work:
        x.free()
    for c in both:
        c.close()


@pytest.mark.gpu
def test_on_a_lent_stream(ctx):
    import torch
    x = Prompts(ctx, *CALLS[1])
    x.call()
    ctx.sync()
    want = x.raw().copy()
    s = torch.cuda.Stream()
    ctx.set_stream(s.cuda_stream)
    try:
        x.bo.upload(np.zeros(x.bo.n_elements, np.uint16))
        x.call()
        ctx.sync()
        assert np.array_equal(x.raw(), want)
    finally:
        ctx.set_stream(None)
    x.free()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n_q,n_kv,d,page,lens,new", CALLS)
def test_prompts_with_a_page_that_is_none(ctx, dtype, n_q, n_kv, d, page, lens, new):
    """Its positions are left out, the other sequences are as they were, rstq_sync says so once."""
    x = Prompts(ctx, dtype, n_q, n_kv, d, page, lens, new)
    tab, gone = x.pool.table.copy(), 1
    tab[0, gone] = -3
    x.pool.bt.upload(tab)
    x.call()
    with pytest.raises(L.RstqError) as e:
        ctx.sync()
    assert e.value.code == L.E_RANGE
    ctx.sync()
    got = pm.decode(x.raw(), dtype).reshape(x.rows, n_q, d)
    for r in (0, new[0] - 1):
        m = lens[0] - new[0] + r + 1
        keep = [i for i in range(m) if i // page != gone]
        want, tol = pm.attention(x.q[r:r + 1], x.pool.keys[0][keep], x.pool.values[0][keep], x.scale, False, dtype)
        close(got[r:r + 1], want, tol, f"row {r}")
    at = new[0] + new[1] - 1
    want, tol = pm.attention(x.q[at:at + 1], x.pool.keys[1], x.pool.values[1], x.scale, False, dtype)
    close(got[at:at + 1], want, tol, "the next sequence's last row")
    x.free()


@pytest.mark.gpu
def test_launches_are_counted(ctx):
    for case, launches in ((CALLS[0], 1), (CALLS[1], 2), (CALLS[2], 1), (CALLS[3], 2), (CALLS[4], 1)):
        x = Prompts(ctx, *case)
        n = ctx.launch_count()
        x.call()
        assert ctx.launch_count() - n == launches
        ctx.sync()
        x.free()


# ---- arrays over one another ------------------------------------------------------------------------
@pytest.mark.gpu
def test_attention_does_not_write_over_what_it_reads(ctx):
    x = Prompts(ctx, *CALLS[2])
    p, (n_q, group, n_kv, d) = x.pool, x.sizes
    over = ctx.wrap_buffer(x.bq.device_ptr + 64, x.bq.n_elements - 16, np.float32)
    n = ctx.launch_count()

    def prompt(**kw):
        a = dict(q=x.bq, kcache=p.bk, vcache=p.bv, out=x.bo, table=p.bt, cu_q=x.bcu, lens=p.bl, rows=x.rows - 1, seqs=2, n_q=n_q, group=group,
                 n_kv=n_kv, head_dim=d, page=x.page, n_pages=p.n_pages, max_pages=p.width, scale=0.1)
        ctx.paged_prompt_attention(**{**a, **kw})

    def packed(**kw):
        a = dict(q=x.bq, k=p.bk, v=p.bv, out=x.bo, cu_q=x.bcu, cu_k=x.bcu, rows=x.rows - 1, kv_rows=100, seqs=2, n_q=n_q, group=group, n_kv=n_kv,
                 head_dim=d, scale=0.1)
        ctx.prompt_attention(**{**a, **kw})

    def decode(**kw):
        a = dict(q=x.bq, kcache=p.bk, vcache=p.bv, out=x.bo, table=p.bt, lens=p.bl, seqs=2, n_q=n_q, group=group, n_kv=n_kv, head_dim=d, page=x.page,
                 n_pages=p.n_pages, max_pages=p.width, scale=0.1)
        ctx.paged_decode_attention(**{**a, **kw})

    def append(**kw):
        a = dict(q=x.bq, k=x.bo, v=x.bo, qout=x.bq, kcache=p.bk, vcache=p.bv, table=p.bt, lens=p.bl, cu=None, rows=2, seqs=2, n_q=n_q, n_kv=n_kv,
                 head_dim=d, page=x.page, n_pages=p.n_pages, max_pages=p.width, theta=1e4)
        ctx.paged_rope_append(**{**a, **kw})

    for fn, kw in ((prompt, dict(out=x.bq)), (prompt, dict(out=over)), (prompt, dict(out=p.bk)), (prompt, dict(out=p.bv)),
                   (packed, dict(out=over)), (packed, dict(out=p.bk)), (decode, dict(out=x.bq)), (decode, dict(out=over)), (decode, dict(out=p.bv)),
                   (append, dict(qout=over)), (append, dict(ldq=n_q * d + 4)),                         # in place, but not where they were
                   (append, dict(in_dtype=L.BF16)), (append, dict(dtype=L.BF16)), (append, dict(k=x.bq)), (append, dict(vcache=p.bk)),
                   (append, dict(qout=p.bk)), (append, dict(q=p.bk, qout=x.bq, k=x.bo))):
        with pytest.raises(L.RstqError) as e:
            fn(**kw)
        assert e.value.code == L.E_INVALID, (fn.__name__, kw, e.value)
    for fn, kw in ((append, dict(theta=float("inf"))), (decode, dict(scale=1e31)), (prompt, dict(scale=-float("inf")))):
        with pytest.raises(L.RstqError) as e:
            fn(**kw)
        assert e.value.code == L.E_SHAPE
    assert ctx.launch_count() == n
    x.free()


@pytest.mark.gpu
def test_pages_calls_do_not_write_over_what_they_read(ctx):
    c = Cache(ctx, 4, 8, 4, 16)
    one, other, S = c.ints([0]), c.ints([1]), c.sizes
    part = ctx.wrap_buffer(c.bt.device_ptr + 16, c.bt.n_elements, np.int32)          # (never read: refused before)
    n = ctx.launch_count()
    for i, fn in enumerate([
            lambda: ctx.pages_free(c.bt, c.bl, c.br, c.bl, c.bi, 1, *S),
            lambda: ctx.pages_free(c.bt, c.bl, c.br, c.bi, c.bi, 1, *S),
            lambda: ctx.pages_free(c.bt, c.bt, c.br, one, c.bi, 1, *S),
            lambda: ctx.pages_extend(c.bt, c.bl, c.br, one, c.bt, c.bi, 1, *S),
            lambda: ctx.pages_extend(c.bt, c.bl, c.bt, one, other, c.bi, 1, *S),
            lambda: ctx.pages_fork(c.bk, c.bk, c.bt, c.bl, c.br, one, other, c.bi, 1, *S, 2, 16),
            lambda: ctx.pages_fork(c.bk, c.bv, c.bt, c.bl, c.br, one, c.br, c.bi, 1, *S, 2, 16),
            lambda: ctx.pages_compact(c.bk, c.bv, c.bt, c.bl, c.br, part, c.br, c.bi, *S, 2, 16),
            lambda: ctx.pages_compact(c.bk, c.bv, c.bt, c.bl, c.br, c.bt, c.bt, c.bi, *S, 2, 16),
            lambda: ctx.pages_compact(c.bk, c.bv, c.bt, c.bl, c.br, c.bk, c.br, c.bi, *S, 2, 16),
            lambda: ctx.pages_copy(c.bk, c.bv, one, c.bk, c.bi, 1, 8, 2, 256),
            lambda: ctx.pages_copy(c.bk, c.bk, one, other, c.bi, 1, 8, 2, 256)]):
        with pytest.raises(L.RstqError) as e:
            fn()
        assert e.value.code == L.E_INVALID, (i, e.value)
    assert ctx.launch_count() == n
    one.free()
    other.free()
    c.close()


# ---- pages ------------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_pages_calls_in_a_graph(ctx):
    """A round of all calls, recorded once and replayed: lists and counts in device memory say who ends, branches and grows."""
    c = Cache(ctx, 12, 60, 5, 16, layers=2, row=24, seed=3)
    c.extend(list(range(6)), [70, 16, 33, 1, 48, 20])
    gone, src, dst, who, more = (c.ints([0] * k) for k in (1, 2, 2, 3, 3))
    infos = [ctx.make_buffer(4, np.int32) for _ in range(4)]

    def calls():
        ctx.pages_free(c.bt, c.bl, c.br, gone, infos[0], 1, *c.sizes)
        ctx.pages_fork(c.bk, c.bv, c.bt, c.bl, c.br, src, dst, infos[1], 2, *c.sizes, c.layers, c.row)
        ctx.pages_extend(c.bt, c.bl, c.br, who, more, infos[2], 3, *c.sizes)
        ctx.pages_compact(c.bk, c.bv, c.bt, c.bl, c.br, c.bt, c.br, infos[3], *c.sizes, c.layers, c.row)

    ctx.graph_begin()
    calls()
    graph = ctx.graph_end()
    rounds = [([0], [2, 5], [6, 7], [6, 7, 3], [5, 20, 16]), ([4], [3, 6], [0, 8], [8, 0, 9], [1, 2, 80]),
              ([7], [1, 1], [10, 11], [9, 3, 5], [0, 1, 0]), ([9], [9, 0], [7, 4], [7, 4, 2], [1, 1, 1])]
    for g, s, d, w, m in rounds:
        for b, v in ((gone, g), (src, s), (dst, d), (who, w), (more, m)):
            b.upload(np.array(v + [0], np.int32))
        graph.replay()
        status, pairs = c.m.free(g), []
        want = [status]
        status, pairs = c.m.fork(s, d)
        c.move(pairs)
        want.append(status)
        want.append(c.m.extend(w, m))
        moves = c.m.compact()
        c.move(moves)
        want.append(0)
        ctx.sync()
        got = [b.download().tolist() for b in infos]
        assert [i[0] for i in got] == want, (got, want)
        assert got[1][2] == len(pairs) and got[3][1:3] == [c.m.used(), len(moves)]
        assert np.array_equal(c.bt.download().reshape(c.m.table.shape), c.m.table)
        assert np.array_equal(c.bl.download(), c.m.lens) and np.array_equal(c.br.download(), c.m.refs)
        assert np.array_equal(c.bk.download().reshape(c.k.shape), c.k) and np.array_equal(c.bv.download().reshape(c.v.shape), c.v)
    graph.destroy()
    for b in (gone, src, dst, who, more, *infos):
        b.free()
    c.close()


@pytest.mark.gpu
def test_long_sequences_and_long_lists(ctx):
    """Sequences of thousands of pages and lists of more than a block has threads."""
    c = Cache(ctx, 2100, 9000, 5000, 16, layers=1, row=1, seed=4)
    c.extend([7, 3], [16 * 4700 + 5, 16 * 900])
    c.fork([7, 3], [8, 9])
    c.extend([8, 7], [16 * 200, 30])
    c.free([7, 3])
    c.compact()
    many = [s for s in range(2100) if s not in (7, 3, 8, 9)][:1500]
    c.extend(many, [1 + s % 17 for s in range(1500)])
    c.free(many[::2])
    c.fork(many[1::2], many[::2])
    c.compact(in_place=False)
    c.free([8, 9] + many)
    assert c.m.used() == 0
    c.close()


# ---- offsets beyond 32 bits -------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("d", [128, 256])
def test_a_pool_of_more_than_2_32_elements(ctx, d):
    """Rows written to, read from and moved out of the last pages of a pool whose elements no 32-bit offset reaches."""
    n_q, n_kv, page, theta, scale = 16, 1024 // d, 256, 1e4, d ** -0.5
    size = page * n_kv * d
    n_pages, lens = (1 << 32) // size + 6, [300, 513]                  # two pages and three, of the last six
    table = np.array([[n_pages - 1, n_pages - 5, -1], [n_pages - 2, n_pages - 6, n_pages - 3]], np.int32)
    rows = sum(lens)
    bk, bv = ctx.make_buffer(n_pages * size, np.uint16), ctx.make_buffer(n_pages * size, np.uint16)
    at = lambda b, i: ctx.wrap_buffer(b.device_ptr + 2 * size * i, size, np.uint16)  # noqa: E731
    for i in range(n_pages - 6, n_pages):
        for b in (bk, bv):
            w = at(b, i)
            w.fill_bytes(0xFF)
            w.free()
    q, k, v = (normal(s, rows, h, d) for s, h in ((1, n_q), (2, n_kv), (3, n_kv)))
    up = ctx.array_to_buffer
    bq, bkn, bvn, bt, bl = up(q), up(k), up(v), up(table), up(np.array(lens, np.int32))
    cu = np.cumsum([0] + lens).astype(np.int32)
    bcu, bqt, bo = up(cu), ctx.make_buffer(rows * n_q * d, np.uint16), ctx.make_buffer(rows * n_q * d, np.uint16)
    ctx.paged_rope_append(bq, bkn, bvn, bqt, bk, bv, bt, bl, bcu, rows, 2, n_q, n_kv, d, page, n_pages, 3, theta, L.F32, L.BF16)
    ctx.sync()

    def pages(pool, tab):
        out = []
        for b, n in enumerate(lens):
            parts = []
            for j in range(-(-n // page)):
                w = at(pool, int(tab[b, j]))
                parts.append(pm.from_bf16(w.download()).reshape(page, n_kv, d))
                w.free()
            out.append(np.concatenate(parts)[:n])
        return out
    kk, vv = pages(bk, table), pages(bv, table)
    for b, n in enumerate(lens):
        assert np.array_equal(vv[b], pm.from_bf16(pm.to_bf16(v[cu[b]:cu[b + 1]])))
        for i in (0, n // 2, n - 1):       # (rounded once; the angle's sine and cosine to 2^-22 of a row's largest)
            want = pm.rope(k[cu[b] + i], i, theta)
            assert (np.abs(kk[b][i] - want) <= pm.HALF["bf16"] * np.abs(want) + 2.0 ** -20 * np.abs(k[cu[b] + i]).max()).all()
    qt = pm.from_bf16(bqt.download()).reshape(rows, n_q, d)
    heads = (n_q, n_q // n_kv, n_kv, d, page, n_pages, 3, scale)

    def check(got, b, r):
        m = r + 1
        want, tol = pm.attention(qt[cu[b] + r][None], kk[b][:m], vv[b][:m], scale, False, "bf16")
        close(got[None], want, tol, f"sequence {b} row {r}")
    ctx.paged_prompt_attention(bqt, bk, bv, bo, bt, bcu, bl, rows, 2, *heads, True, L.BF16)
    ctx.sync()
    got = pm.from_bf16(bo.download()).reshape(rows, n_q, d)
    for b, n in enumerate(lens):
        for r in (0, 255, 256, n - 1):
            check(got[cu[b] + r], b, r)
    last = up(pm.to_bf16(qt[cu[1:] - 1]))
    ctx.paged_decode_attention(last, bk, bv, bo, bt, bl, 2, *heads, L.BF16)
    ctx.sync()
    got = pm.from_bf16(bo.download(n=2 * n_q * d)).reshape(2, n_q, d)
    for b, n in enumerate(lens):
        check(got[b], b, n - 1)
    # to the first pages
    refs = np.zeros(n_pages, np.int32)
    refs[table[table >= 0]] = 1
    br, bi = up(refs), ctx.make_buffer(4, np.int32)
    ctx.pages_compact(bk, bv, bt, bl, br, bt, br, bi, 2, n_pages, 3, page, 1, n_kv * d * 2)
    ctx.sync()
    moved = bt.download().reshape(2, 3)
    assert bi.download().tolist() == [0, 5, 5, 0] and sorted(moved[table >= 0]) == list(range(5))
    assert all(np.array_equal(a, b) for a, b in zip(kk + vv, pages(bk, moved) + pages(bv, moved)))
    for b in (bk, bv, bq, bkn, bvn, bt, bl, bcu, bqt, bo, last, br, bi):
        b.free()


# ---- many sequences -----------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,n_q,n_kv,d,page,lens,new", [
    ("f32", 8, 2, 128, 32, [2500, 1100, 7, 1500], [2, 40, 7, 1]),
    ("f32", 6, 2, 64, 16, [3000, 0, 1030], [5, 0, 30]),
    ("f32", 2, 2, 96, 16, [1500, 200], [130, 3]),
    ("f32", 4, 1, 128, 256, [4000], [1]),
])
def test_few_rows_behind_many_keys_in_f32(ctx, dtype, n_q, n_kv, d, page, lens, new):
    x = Prompts(ctx, dtype, n_q, n_kv, d, page, lens, new)
    x.call()
    ctx.sync()
    x.check()
    x.free()


@pytest.mark.gpu
def test_parts_in_f32_with_values_that_are_not_numbers(ctx):
    """An infinity that only the last row sees, one that all see, and nothing of the first in the others."""
    n_q, d, page, n, rows = 4, 64, 32, 2600, 3
    x = Prompts(ctx, "f32", n_q, 1, d, page, [n], [rows])
    p = x.pool
    v = p.v.copy()
    at = lambda pos: (p.table[0, pos // page], pos % page)  # noqa: E731
    v[at(n - 1)][0, 5] = np.inf
    v[at(100)][0, 6] = -np.inf
    p.bv.upload(v)
    x.call()
    ctx.sync()
    got = x.raw().reshape(rows, n_q, d)
    assert np.isneginf(got[:, :, 6]).all() and np.isposinf(got[2, :, 5]).all() and np.isfinite(got[:2, :, 5]).all()
    keep = [i for i in range(d) if i not in (5, 6)]
    for r in range(rows):
        m = n - rows + r + 1
        want, tol = pm.attention(x.q[r:r + 1], p.keys[0][:m], p.values[0][:m], x.scale, False, "f32")
        close(got[r:r + 1][..., keep], want[..., keep], tol[..., keep], f"row {r}")
    x.free()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,seqs", [("bf16", 65), ("bf16", 128), ("bf16", 129), ("bf16", 700), ("f32", 129), ("f32", 1100)])
def test_prompts_of_many_sequences(ctx, dtype, seqs):
    """Empty ones among them, at the ends too; some of several blocks of rows."""
    n_q, n_kv, d, page = 4, 2, 64, 16
    rng = np.random.default_rng(seqs)
    lens = [int(x) for x in rng.integers(0, 40, seqs)]
    for i in (seqs // 3, seqs // 2):
        lens[i] = 300 + i
    new = [int(rng.integers(0, n + 1)) for n in lens]
    new[seqs // 3] = lens[seqs // 3]
    for i in (0, seqs // 5, seqs - 1):
        new[i] = 0
    lens[seqs - 1] = 0
    x = Prompts(ctx, dtype, n_q, n_kv, d, page, lens, new, seed=seqs)
    x.call()
    ctx.sync()
    x.check()
    x.free()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("seqs", [33, 1024, 1025])
def test_few_active_of_many_sequences(ctx, dtype, seqs):
    """Most have no new rows: the rows of the others, behind long caches, in parts and not."""
    lens, new = [5] * seqs, [0] * seqs
    for i, rows in ((0, 4), (seqs // 2, 1), (seqs - 1, 3)):
        lens[i], new[i] = 1500 + i, rows
    x = Prompts(ctx, dtype, 8, 2, 128, 16, lens, new)
    x.call()
    ctx.sync()
    x.check()
    x.free()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,seqs", [("bf16", 256), ("bf16", 257), ("bf16", 3000), ("f32", 300)])
def test_decode_of_many_sequences(ctx, dtype, seqs):
    n_q, n_kv, d, page = 4, 2, 64, 16
    rng = np.random.default_rng(seqs)
    lens = [int(x) for x in rng.integers(0, 30, seqs)]
    lens[0] = lens[seqs // 2] = lens[seqs - 1] = 0
    lens[seqs // 3] = 900
    p = Pool(ctx, lens, n_kv, d, page, dtype, seed=seqs)
    q = pm.decode(pm.encode(normal(seqs, seqs, n_q, d), dtype), dtype)
    bq, bo = ctx.array_to_buffer(pm.encode(q, dtype)), ctx.make_buffer(seqs * n_q * d, NP[dtype])
    bo.fill_bytes(0xFF)
    ctx.paged_decode_attention(bq, p.bk, p.bv, bo, p.bt, p.bl, seqs, n_q, 2, n_kv, d, page, p.n_pages, p.width, 0.125, DT[dtype])
    ctx.sync()
    got = pm.decode(bo.download(), dtype).reshape(seqs, n_q, d)
    for b in range(seqs):
        want, tol = pm.attention(q[b:b + 1], p.keys[b], p.values[b], 0.125, False, dtype)
        close(got[b:b + 1], want, tol, f"sequence {b} of {lens[b]}")
    bq.free()
    bo.free()
    p.free()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n_q,n_kv,d,page,lens,new", [
    (14, 2, 128, 16, [200, 37, 19, 18, 0, 1], [200, 37, 19, 2, 0, 1]),         # 18 rows of 7 heads in a tile, two rows of it empty
    (10, 2, 64, 32, [130, 52], [130, 26]),
    (12, 1, 96, 16, [60, 21], [60, 11]),
    (9, 1, 128, 64, [1500, 800], [30, 29]),                                    # keys in parts
    (7, 1, 64, 16, [1200, 2000, 40], [2, 100, 40]),
    (43, 1, 64, 16, [40], [9]),                                                # a group that would leave a third of a tile empty
    (64, 1, 128, 16, [70, 5], [5, 3]),
    (128, 1, 64, 16, [30], [4]),
    (130, 1, 64, 16, [30], [3]),
])
def test_groups_that_share_a_tile(ctx, dtype, n_q, n_kv, d, page, lens, new):
    x = Prompts(ctx, dtype, n_q, n_kv, d, page, lens, new, seed=n_q)
    x.call()
    ctx.sync()
    x.check()
    x.free()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n_q,n_kv,d,page,lens", [
    (8, 2, 256, 16, [1, 15, 16, 17, 0, 63, 64, 65, 300]),
    (16, 1, 256, 64, [1500, 2, 700]),
    (20, 1, 192, 32, [260, 33]),                # more heads in the group than a block serves at once
    (4, 4, 136, 16, [200, 31, 129]),
    (3, 1, 248, 128, [500]),
    (2, 2, 144, 256, [2000, 255, 257]),
])
def test_decode_of_wide_heads(ctx, dtype, n_q, n_kv, d, page, lens):
    p = Pool(ctx, lens, n_kv, d, page, dtype, seed=d)
    step = n_q * d + 8
    full = pm.encode(normal(d, len(lens), step), dtype)
    q = pm.decode(full, dtype)[:, :n_q * d].reshape(len(lens), n_q, d)
    bq, bo = ctx.array_to_buffer(full), ctx.make_buffer((len(lens) + 1) * n_q * d, NP[dtype])
    bo.fill_bytes(0x5A)
    ctx.paged_decode_attention(bq, p.bk, p.bv, bo, p.bt, p.bl, len(lens), n_q, n_q // n_kv, n_kv, d, page, p.n_pages, p.width, d ** -0.5,
                               DT[dtype], ldq=step)
    ctx.sync()
    raw = bo.download().reshape(-1, n_q, d)
    assert (raw[-1].view(np.uint8) == 0x5A).all()
    got = pm.decode(raw[:-1], dtype)
    for b, n in enumerate(lens):
        want, tol = pm.attention(q[b:b + 1], p.keys[b], p.values[b], d ** -0.5, False, dtype)
        close(got[b:b + 1], want, tol, f"sequence {b} of {n}")
    bq.free()
    bo.free()
    p.free()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("n_q,n_kv,d,page,lens,new", [
    (4, 2, 256, 16, [1, 17, 130, 0, 300], [1, 17, 130, 0, 5]),
    (16, 2, 256, 64, [700, 33], [40, 33]),
    (7, 1, 192, 32, [200, 129], [150, 129]),
    (3, 3, 136, 128, [400], [200]),
    (8, 1, 248, 256, [1500, 20], [2, 20]),
    (4, 2, 256, 32, [2500, 1100, 7, 1500], [2, 140, 7, 1]),
    (6, 2, 136, 16, [3000, 0, 1030], [5, 0, 30]),
])
def test_prompts_of_wide_heads(ctx, dtype, n_q, n_kv, d, page, lens, new):
    x = Prompts(ctx, dtype, n_q, n_kv, d, page, lens, new, seed=d)
    x.call()
    ctx.sync()
    x.check()
    x.free()


@pytest.mark.gpu
def test_a_long_prompt_whose_last_rows_are_taken_one_by_one(ctx):
    """An infinity above the diagonal far behind: a block's rows by themselves take longer than any wait in the kernel may, and
    those who wait see that they are at it."""
    n, n_q, d = 80000, 4, 64                                     # (a block: 64 rows of four heads; the last one is full)
    q, k, v = (normal(s, n, h, d) for s, h in ((1, n_q), (2, 1), (3, 1)))
    q, k, v = (pm.from_bf16(pm.to_bf16(x)) for x in (q, k, v))
    v[n - 9, 0, 5] = np.inf
    up = ctx.array_to_buffer
    bq, bk, bv, cu = up(pm.to_bf16(q)), up(pm.to_bf16(k)), up(pm.to_bf16(v)), up(np.array([0, n], np.int32))
    bo = ctx.make_buffer(n * n_q * d, np.uint16)
    ctx.prompt_attention(bq, bk, bv, bo, cu, cu, n, n, 1, n_q, n_q, 1, d, d ** -0.5, True, L.BF16)
    ctx.sync()
    got = pm.from_bf16(bo.download()).reshape(n, n_q, d)
    assert np.isfinite(got[:n - 9]).all() and np.isposinf(got[n - 9:, :, 5]).all()
    v[n - 9, 0, 5] = 0
    keep = [i for i in range(d) if i != 5]
    for r in (0, 63, 64, 70001, n - 64, n - 10, n - 9, n - 1):
        want, tol = pm.attention(q[r:r + 1], k[:r + 1], v[:r + 1], d ** -0.5, False, "bf16")
        close(got[r:r + 1][..., keep], want[..., keep], tol[..., keep], f"row {r}")
    for b in (bq, bk, bv, cu, bo):
        b.free()

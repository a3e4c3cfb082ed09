"""Pages of a cache copied, shared, taken, given back and moved together, against a model that does it one step at a time
(tests/paged_model.py); then all of a serving loop in one run."""
import numpy as np
import pytest

import paged_model as pm
from raster_b200 import _lib as L


class Cache:
    """The state on the device beside its model."""

    def __init__(self, ctx, seqs, n_pages, width, page, layers=2, row=16, seed=0):
        self.ctx, self.m = ctx, pm.Pages(seqs, n_pages, width, page)
        self.seqs, self.n_pages, self.width, self.page, self.layers, self.row = seqs, n_pages, width, page, layers, row
        rng = np.random.default_rng(seed)
        self.k, self.v = (rng.integers(0, 256, (layers, n_pages, page, row)).astype(np.uint8) for _ in range(2))
        up = ctx.array_to_buffer
        self.bk, self.bv, self.bt, self.bl, self.br = up(self.k), up(self.v), up(self.m.table), up(self.m.lens), up(self.m.refs)
        self.bi = ctx.make_buffer(4, np.int32)
        self.sizes = (seqs, n_pages, width, page)

    def ints(self, v):
        return self.ctx.array_to_buffer(np.array(list(v) + [0], np.int32))

    def info(self):
        self.ctx.sync()
        return self.bi.download().tolist()

    def free(self, seqs):
        b = self.ints(seqs)
        self.ctx.pages_free(self.bt, self.bl, self.br, b, self.bi, len(seqs), *self.sizes)
        return self.after(self.m.free(seqs), 0, b)

    def extend(self, seqs, counts):
        a, b = self.ints(seqs), self.ints(counts)
        self.ctx.pages_extend(self.bt, self.bl, self.br, a, b, self.bi, len(seqs), *self.sizes)
        return self.after(self.m.extend(seqs, counts), 0, a, b)

    def fork(self, src, dst):
        a, b = self.ints(src), self.ints(dst)
        self.ctx.pages_fork(self.bk, self.bv, self.bt, self.bl, self.br, a, b, self.bi, len(src), *self.sizes, self.layers, self.row)
        status, pairs = self.m.fork(src, dst)
        self.move(pairs)
        return self.after(status, len(pairs), a, b)

    def move(self, pairs):
        for a, b in pairs:
            self.k[:, b], self.v[:, b] = self.k[:, a], self.v[:, a]

    def compact(self, in_place=True):
        t, r = self.bt, self.br
        if not in_place:
            t, r = self.ints([9] * (self.seqs * self.width - 1)), self.ints([9] * (self.n_pages - 1))
        table, refs = self.m.table.copy(), self.m.refs.copy()
        self.ctx.pages_compact(self.bk, self.bv, self.bt, self.bl, self.br, t, r, self.bi, *self.sizes, self.layers, self.row)
        pairs = self.m.compact()
        self.move(pairs)
        if not in_place:       # the old ones are as they were
            assert self.info()[0] == 0
            assert np.array_equal(self.bt.download().reshape(table.shape), table) and np.array_equal(self.br.download(), refs)
            self.bt.free()
            self.br.free()
            self.bt, self.br = t, r
        return self.after(0, len(pairs))

    def after(self, status, copied, *lists):
        info = self.info()
        for b in lists:
            b.free()
        assert info[:3] == [status, self.m.used(), copied], (info, status, self.m.used(), copied)
        assert np.array_equal(self.bt.download().reshape(self.m.table.shape), self.m.table)
        assert np.array_equal(self.bl.download(), self.m.lens)
        assert np.array_equal(self.br.download(), self.m.refs)
        assert np.array_equal(self.bk.download().reshape(self.k.shape), self.k)
        assert np.array_equal(self.bv.download().reshape(self.v.shape), self.v)
        return info

    def close(self):
        for b in (self.bk, self.bv, self.bt, self.bl, self.br, self.bi):
            b.free()


def test_model_known_answers():
    m = pm.Pages(4, 6, 3, 16)
    assert m.extend([0, 1], [20, 16]) == 0 and m.table[0, :2].tolist() == [0, 1] and m.table[1, 0] == 2
    assert m.fork([0, 1], [2, 3]) == (0, [(1, 3)])
    assert m.table[2].tolist() == [0, 3, -1] and m.table[3].tolist() == [2, -1, -1] and m.refs.tolist() == [2, 1, 2, 1, 0, 0]
    assert m.extend([3], [1]) == 0 and m.table[3, 1] == 4           # behind a full shared page: a page of its own
    assert m.extend([0], [60]) == 3 and m.extend([0], [1, ]) == 0
    assert m.extend([0, 1], [16, 16]) == 1                          # one page is left
    assert m.free([0, 3]) == 0 and m.refs.tolist() == [1, 0, 1, 1, 0, 0]
    assert m.compact() == [(3, 1)] and m.table[2].tolist() == [0, 1, -1] and m.refs.tolist() == [1, 1, 1, 0, 0, 0]


@pytest.mark.gpu
def test_each_call(ctx):
    c = Cache(ctx, 6, 40, 5, 16)
    c.extend([0, 1, 2], [33, 16, 0])
    c.extend([2, 0], [1, 15])                  # 0: to the end of its page
    c.fork([0, 1], [3, 4])
    c.extend([3, 4], [1, 40])
    c.free([1])                                 # its page lives on in 4
    c.free([5])                                 # holds nothing
    c.compact()
    c.fork([4, 4], [1, 5])
    c.free([0, 4, 3])
    c.compact(in_place=False)
    c.compact()                                 # nothing to do
    c.free([])
    c.extend([], [])
    c.fork([], [])
    c.close()


@pytest.mark.gpu
def test_calls_that_cannot_be_done_change_nothing(ctx):
    c = Cache(ctx, 5, 8, 4, 16)
    c.extend([0, 1], [40, 20])
    assert c.extend([2], [64]) [0] == 1 and c.info()[3] == 4       # three pages are free
    c.extend([0, 2], [25, 1])                                       # no room in the table
    c.extend([0, 0], [1, 1])
    c.extend([0, 5], [1, 1])
    c.extend([-1], [1])
    c.extend([2], [-1])
    c.free([1, 1])
    c.free([1 << 30])
    c.fork([0], [1])                                                # not empty
    c.fork([0, 2], [2, 3])                                          # both in src and in dst
    c.fork([0, 1], [2, 2])
    c.fork([0], [7])
    c.fork([0], [0])
    c.fork([0, 1, 0], [2, 3, 4])                                    # takes the three pages that are left
    assert c.info()[0] == 0
    c.free([4])
    c.extend([4], [16])
    c.free([1])
    c.fork([0], [1])
    c.close()
    c = Cache(ctx, 3, 8, 4, 16)
    c.extend([0], [40])
    c.fork([0], [1])
    c.m.lens[1] = 24                                                # cut back into a page that 0 holds too
    c.m.table[1, 2] = -1
    c.m.refs[3] = 0
    for b, a in ((c.bl, c.m.lens), (c.bt, c.m.table), (c.br, c.m.refs)):
        b.upload(a)
    assert c.extend([1], [1])[0] == 4
    assert c.extend([1], [0])[0] == 0
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,n_pages,width,page,layers,row,seed", [
    (9, 50, 7, 16, 1, 16, 1), (40, 3000, 90, 32, 2, 48, 2), (1500, 9001, 12, 16, 1, 32, 3), (3, 5, 3, 256, 3, 256, 4)])
def test_random_calls(ctx, seqs, n_pages, width, page, layers, row, seed):
    rng = np.random.default_rng(seed)
    c = Cache(ctx, seqs, n_pages, width, page, layers, row, seed)
    for step in range(14):
        some = rng.permutation(seqs)[: rng.integers(1, seqs + 1)].tolist()
        what = ("extend", "fork", "free", "compact")[step % 4] if step < 12 else "extend"
        if what == "extend":
            c.extend(some, [int(x) for x in rng.integers(0, page * 3, len(some))])
        elif what == "fork":
            held = [s for s in range(seqs) if c.m.lens[s]] or [0]
            empty = [s for s in range(seqs) if not c.m.lens[s] and s not in held]
            c.fork([held[i % len(held)] for i in range(len(empty))], empty)
        elif what == "free":
            c.free(some[: max(1, len(some) // 2)])
        else:
            c.compact(bool(step % 8 == 3))
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("page_bytes,layers", [(16, 1), (4096, 2), (6160, 3), (65536, 1)])
def test_copy(ctx, page_bytes, layers):
    n_pages = 37
    rng = np.random.default_rng(page_bytes)
    k, v = (rng.integers(0, 256, (layers, n_pages, page_bytes)).astype(np.uint8) for _ in range(2))
    bk, bv, bi = ctx.array_to_buffer(k), ctx.array_to_buffer(v), ctx.make_buffer(4, np.int32)
    for src, dst, status in (([3, 3, 36], [0, 5, 1], 0), ([], [], 0), ([1, 2], [4, 4], 2), ([1, 2], [2, 9], 2), ([7], [7], 2),
                             ([37], [0], 2), ([0], [-1], 2), (list(range(18)), list(range(36, 18, -1)), 0)):
        a, b = ctx.array_to_buffer(np.array(src + [0], np.int32)), ctx.array_to_buffer(np.array(dst + [0], np.int32))
        ctx.pages_copy(bk, bv, a, b, bi, len(src), n_pages, layers, page_bytes)
        ctx.sync()
        info = bi.download().tolist()
        assert info[:3] == [status, 0, 0 if status else len(src)]
        if not status and src:
            k[:, dst], v[:, dst] = k[:, src], v[:, src]
        assert np.array_equal(bk.download().reshape(k.shape), k) and np.array_equal(bv.download().reshape(v.shape), v)
        a.free()
        b.free()
    for b in (bk, bv, bi):
        b.free()


@pytest.mark.gpu
def test_refusals(ctx):
    c = Cache(ctx, 4, 8, 4, 16)
    one = c.ints([0])
    S = c.sizes
    cases = [
        (lambda: ctx.pages_free(c.bt, c.bl, c.br, one, c.bi, 65537, *S), L.E_LIMIT),
        (lambda: ctx.pages_free(c.bt, c.bl, c.br, one, c.bi, 100, *S), L.E_INVALID),
        (lambda: ctx.pages_free(c.bt, c.bl, c.br, one, one, 1, *S), L.E_INVALID),                       # info is too small
        (lambda: ctx.pages_extend(c.bt, c.bl, c.br, one, one, c.bi, 1, 4, 8, 4, 20), L.E_SHAPE),
        (lambda: ctx.pages_extend(c.bt, c.bl, c.br, one, one, c.bi, 1, 4, 9, 4, 16), L.E_INVALID),
        (lambda: ctx.pages_extend(c.bt, c.bl, c.br, one, one, c.bi, -1, *S), L.E_LIMIT),
        (lambda: ctx.pages_fork(c.bk, c.bv, c.bt, c.bl, c.br, one, one, c.bi, 1, *S, 3, 16), L.E_INVALID),  # three layers
        (lambda: ctx.pages_fork(c.bk, c.bv, c.bt, c.bl, c.br, one, one, c.bi, 1, *S, 0, 16), L.E_SHAPE),
        (lambda: ctx.pages_fork(c.bk, c.bv, c.bt, c.bl, c.br, one, one, c.bi, 1, *S, 2, 0), L.E_SHAPE),
        (lambda: ctx.pages_compact(c.bk, c.bv, c.bt, c.bl, c.br, one, c.br, c.bi, *S, 2, 16), L.E_INVALID),
        (lambda: ctx.pages_copy(c.bk, c.bv, one, one, c.bi, 1, 8, 2, 100), L.E_ALIGN),
        (lambda: ctx.pages_copy(c.bk, c.bv, one, one, c.bi, 1, (1 << 20) + 1, 1, 16), L.E_LIMIT)]
    for i, (fn, code) in enumerate(cases):
        with pytest.raises(L.RstqError) as e:
            fn()
        assert e.value.code == code, (i, e.value)
    one.free()
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_serving_loop(ctx, dtype):
    """Prompts in, their rows to the cache, attention over them; then decode steps, forks, ends and a compaction in between, from a
    graph that holds a whole step: every output row against attention over the rows the sequence was made of."""
    n_q, n_kv, d, page, seqs, n_pages, width = 4, 2, 64, 16, 5, 24, 6
    kind, code = {"bf16": (np.uint16, L.BF16), "f32": (np.float32, L.F32)}[dtype]
    scale, theta = d ** -0.5, 1e4
    rng = np.random.default_rng(7)
    m = pm.Pages(seqs, n_pages, width, page)
    up, mk = ctx.array_to_buffer, ctx.make_buffer
    bt, bl, br, bi = up(m.table), up(m.lens), up(m.refs), mk(4, np.int32)
    bk, bv = mk(n_pages * page * n_kv * d, kind), mk(n_pages * page * n_kv * d, kind)
    bk.fill_bytes(0xFF)
    bv.fill_bytes(0xFF)                                       # NaN where nobody has written
    rows = 64
    bq, bkn, bvn = (mk(rows * h * d, np.float32) for h in (n_q, n_kv, n_kv))
    bqt, bo = mk(rows * n_q * d, kind), mk(rows * n_q * d, kind)
    keys, values = [np.zeros((0, n_kv, d)) for _ in range(seqs)], [np.zeros((0, n_kv, d)) for _ in range(seqs)]
    h = pm.HALF[dtype]

    def fresh(n):
        q, k, v = (rng.standard_normal((n, x, d)).astype(np.float32) for x in (n_q, n_kv, n_kv))
        for b, a in ((bq, q), (bkn, k), (bvn, v)):
            b.upload(a)
        return q, k, v

    def grow(b, q, k, v):
        """The sequence's rows grow; returns its new queries, turned and rounded as the device has them."""
        pos = len(keys[b])
        turn = lambda x: np.stack([pm.decode(pm.encode(pm.rope(x[i], pos + i, theta), dtype), dtype) for i in range(len(x))])  # noqa: E731
        keys[b] = np.concatenate([keys[b], turn(k)])
        values[b] = np.concatenate([values[b], pm.decode(pm.encode(v, dtype), dtype)])
        return turn(q)

    def check(got, b, q, what):
        want, tol = pm.attention(q, keys[b], values[b], scale, True, dtype)
        # q and k on the device may be the neighbour of the model's (an angle's last bit): a step each, of scores and so of weights
        close = tol + (4 * h if dtype == "bf16" else 1e-6) * np.abs(q).max() * np.abs(keys[b]).max() * d * scale * np.abs(values[b]).max() * 0.1
        assert np.isfinite(got).all() and (np.abs(got - want) <= close).all(), (what, b, np.abs(got - want).max())

    # prompts of 1, 16 and 37 rows
    counts = [1, 16, 37]
    first, more = up(np.array([0, 1, 2], np.int32)), up(np.array(counts, np.int32))
    ctx.pages_extend(bt, bl, br, first, more, bi, 3, seqs, n_pages, width, page)
    q, k, v = fresh(sum(counts))
    cu = np.concatenate([np.cumsum([0] + counts), [sum(counts)] * 2]).astype(np.int32)
    bcu = up(cu)
    n = sum(counts)
    ctx.paged_rope_append(bq, bkn, bvn, bqt, bk, bv, bt, bl, bcu, n, seqs, n_q, n_kv, d, page, n_pages, width, theta, L.F32, code)
    ctx.paged_prompt_attention(bqt, bk, bv, bo, bt, bcu, bl, n, seqs, n_q, n_q // n_kv, n_kv, d, page, n_pages, width, scale, True, code)
    ctx.sync()
    assert bi.download()[0] == 0
    got = pm.decode(bo.download(n=n * n_q * d), dtype).reshape(n, n_q, d)
    for b in range(3):
        s = slice(cu[b], cu[b + 1])
        check(got[s], b, grow(b, q[s], k[s], v[s]), "prompt")

    # a decode step of all five sequences, recorded once; lists and counts in device memory say who takes part
    everyone, one_each = up(np.arange(seqs, dtype=np.int32)), mk(seqs, np.int32)
    one_each.upload(np.zeros(seqs, np.int32))

    def step():
        ctx.pages_extend(bt, bl, br, everyone, one_each, bi, seqs, seqs, n_pages, width, page)
        ctx.paged_rope_append(bq, bkn, bvn, bqt, bk, bv, bt, bl, None, seqs, seqs, n_q, n_kv, d, page, n_pages, width, theta, L.F32, code)
        ctx.paged_decode_attention(bqt, bk, bv, bo, bt, bl, seqs, n_q, n_q // n_kv, n_kv, d, page, n_pages, width, scale, code)
    ctx.graph_begin()
    step()
    graph = ctx.graph_end()

    def decode_step(live, what):
        one_each.upload(np.array([b in live for b in range(seqs)], np.int32))
        q, k, v = fresh(seqs)
        graph.replay()
        try:
            ctx.sync()
        except L.RstqError as e:        # sequences that hold nothing have no page for their row
            assert e.code == L.E_RANGE and len(live) < seqs
        assert bi.download()[0] == 0
        got = pm.decode(bo.download(n=seqs * n_q * d), dtype).reshape(seqs, n_q, d)
        for b in live:
            check(got[b:b + 1], b, grow(b, q[b:b + 1], k[b:b + 1], v[b:b + 1]), what)

    for _ in range(2):
        decode_step([0, 1, 2], "decode")
    src, dst = up(np.array([2, 1], np.int32)), up(np.array([3, 4], np.int32))
    ctx.pages_fork(bk, bv, bt, bl, br, src, dst, bi, 2, seqs, n_pages, width, page, 1, n_kv * d * kind().itemsize)
    for a, b in ((2, 3), (1, 4)):
        keys[b], values[b] = keys[a].copy(), values[a].copy()
    for _ in range(15):                                       # over the end of a page
        decode_step(range(seqs), "after the fork")
    gone = up(np.array([0, 2], np.int32))
    ctx.pages_free(bt, bl, br, gone, bi, 2, seqs, n_pages, width, page)
    ctx.pages_compact(bk, bv, bt, bl, br, bt, br, bi, seqs, n_pages, width, page, 1, n_kv * d * kind().itemsize)
    ctx.sync()
    info = bi.download().tolist()
    assert info[0] == 0 and info[1] == sum(-(-len(keys[b]) // page) for b in (1, 3, 4)) - 1      # (1 and 4 share a full page)
    assert bt.download().max() == info[1] - 1
    for b in (0, 2):
        keys[b], values[b] = keys[b][:0], values[b][:0]
    for _ in range(3):
        decode_step([1, 3, 4], "after the compaction")
    graph.destroy()
    for b in (bt, bl, br, bi, bk, bv, bq, bkn, bvn, bqt, bo, first, more, bcu, everyone, one_each, src, dst, gone):
        b.free()

"""Which entry of a list a pages call was refused for: the same answer every time, whichever thread looked first."""
import numpy as np
import pytest

from test_pages import Cache


def state(c):
    return [b.download().copy() for b in (c.bt, c.bl, c.br, c.bk, c.bv)]


def same(a, b):
    return all(np.array_equal(x, y) for x, y in zip(a, b))


# ---- fork: sources that may not be there -------------------------------------------------------------
N = 1200           # entries: more than a block has threads, with eight lanes each


@pytest.mark.gpu
@pytest.mark.parametrize("places", [[0], [1], [7], [130], [N - 1], [127, 128], [1100, 3, 600], list(range(5, N))])
def test_fork_refuses_a_source_whose_table_names_no_page(ctx, places):
    c = Cache(ctx, 2 * N, 3 * N, 3, 16, layers=1, row=1)
    c.extend(list(range(N)), [20] * N)
    table = c.m.table.copy()
    for i in places:
        table[i, i % 2] = (-1, c.n_pages, 1 << 30)[i % 3]
    c.bt.upload(table)
    src, dst = c.ints(range(N)), c.ints(range(N, 2 * N))
    before = state(c)
    for _ in range(20):
        ctx.pages_fork(c.bk, c.bv, c.bt, c.bl, c.br, src, dst, c.bi, N, *c.sizes, 1, 1)
        assert c.info() == [2, c.m.used(), 0, min(places)]
    assert same(before, state(c))
    c.bt.upload(c.m.table)
    c.fork(list(range(N)), list(range(N, 2 * N)))
    src.free()
    dst.free()
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("places", [[0], [9], [127], [128], [N - 1], [900, 40, 41], list(range(N))])
def test_fork_refuses_a_source_that_is_a_destination(ctx, places):
    c = Cache(ctx, 2 * N, 3 * N, 3, 16, layers=1, row=1)
    c.extend(list(range(N)), [20] * N)
    sources = np.arange(N)
    sources[places] = 2 * N - 1 - np.array(places)
    src, dst = c.ints(sources.tolist()), c.ints(range(N, 2 * N))
    before = state(c)
    for _ in range(20):
        ctx.pages_fork(c.bk, c.bv, c.bt, c.bl, c.br, src, dst, c.bi, N, *c.sizes, 1, 1)
        assert c.info() == [2, c.m.used(), 0, min(places)]
    assert same(before, state(c))
    src.free()
    dst.free()
    c.close()


# ---- entries that are there twice ----------------------------------------------------------------------
def twice(rng, n, many):
    """A list of n different numbers of which `many` places repeat an earlier one; the first of these places."""
    a = rng.permutation(4 * n)[:n]
    at = np.sort(rng.permutation(np.arange(1, n))[:many])
    for i in at:
        a[i] = a[rng.integers(0, i)]
    seen = set()
    for i, x in enumerate(a.tolist()):
        if x in seen:
            return a.tolist(), i
        seen.add(x)


@pytest.mark.gpu
@pytest.mark.parametrize("n,many", [(2, 1), (33, 1), (700, 1), (700, 60), (3000, 2), (3000, 2900)])
def test_the_place_of_an_entry_that_is_there_twice(ctx, n, many):
    rng = np.random.default_rng(n + many)
    c = Cache(ctx, 8 * n, 16, 1, 16, layers=1, row=1)
    before = state(c)
    for _ in range(25):
        a, place = twice(rng, n, many)
        la, other, ones = c.ints(a), c.ints(range(4 * n, 5 * n)), c.ints([1] * n)
        for call in (lambda: ctx.pages_free(c.bt, c.bl, c.br, la, c.bi, n, *c.sizes),
                     lambda: ctx.pages_extend(c.bt, c.bl, c.br, la, ones, c.bi, n, *c.sizes),
                     lambda: ctx.pages_fork(c.bk, c.bv, c.bt, c.bl, c.br, other, la, c.bi, n, *c.sizes, 1, 1)):
            call()
            assert c.info() == [2, 0, 0, place]
        for b in (la, other, ones):
            b.free()
    assert same(before, state(c))
    c.close()
    k, v, info = (ctx.make_buffer(8 * n * 16, np.uint8) for _ in range(3))
    for _ in range(25):
        a, place = twice(rng, n, many)
        la, other = (ctx.array_to_buffer(np.array(x, np.int32)) for x in (a, range(4 * n, 5 * n)))
        ctx.pages_copy(k, v, other, la, info, n, 8 * n, 1, 16)
        ctx.sync()
        assert info.download().view(np.int32)[:4].tolist() == [2, 0, 0, place]
        la.free()
        other.free()
    for b in (k, v, info):
        b.free()


@pytest.mark.gpu
def test_the_place_of_an_entry_that_is_wrong_by_itself_or_twice(ctx):
    """Whichever comes first."""
    c = Cache(ctx, 40, 16, 1, 16, layers=1, row=1)
    for a, counts, place in (([3, 4, 3, 40], [1] * 4, 2), ([3, 40, 3, 4], [1] * 4, 1), ([3, 4, 5, 3], [1, -1, 1, 1], 1),
                             ([3, 4, 3, 5], [1, 1, 1, -1], 2), ([3, 4, 3, 5], [-1, 1, -1, 1], 0), ([-5, -5], [1, 1], 0)):
        la, lc = c.ints(a), c.ints(counts)
        for _ in range(5):
            ctx.pages_extend(c.bt, c.bl, c.br, la, lc, c.bi, len(a), *c.sizes)
            assert c.info() == [2, 0, 0, place]
        la.free()
        lc.free()
    c.close()


# ---- pages wanted ----------------------------------------------------------------------------------------
@pytest.mark.gpu
def test_pages_wanted_are_said_in_full(ctx):
    """Also where they are more than the pool has, and more than the word holds."""
    c = Cache(ctx, 300, 8, 1 << 17, 256, layers=1, row=1)
    for seqs, each, want in (([0], 9, 9), ([1, 0, 2], 1000, 3000), (list(range(300)), 100000, 30000000), ([5, 6], 0, 0)):
        la, lc = c.ints(seqs), c.ints([each * 256] * len(seqs))
        ctx.pages_extend(c.bt, c.bl, c.br, la, lc, c.bi, len(seqs), *c.sizes)
        assert c.info() == [1 if want else 0, 0, 0, want]
        la.free()
        lc.free()
    assert not c.bl.download().any() and not c.br.download().any()
    c.close()
    c = Cache(ctx, 4096, 2, 1 << 12, 16, layers=1, row=1)      # 2^24 pages
    la, lc = c.ints(range(4096)), c.ints([1 << 16] * 4096)
    ctx.pages_extend(c.bt, c.bl, c.br, la, lc, c.bi, 4096, *c.sizes)
    assert c.info() == [1, 0, 0, 1 << 24]
    la.free()
    lc.free()
    c.close()
    n_pages, seqs, width = 2, 2200, 1 << 20                     # 2200 sequences of 2^20 pages: more than 2^31 - 1
    table, lens, refs = ctx.make_buffer(seqs * width, np.int32), ctx.make_buffer(seqs, np.int32), ctx.make_buffer(n_pages, np.int32)
    info, la = ctx.make_buffer(4, np.int32), ctx.array_to_buffer(np.arange(seqs, dtype=np.int32))
    lc = ctx.array_to_buffer(np.full(seqs, 16 << 20, np.int32))
    for b in (lens, refs):
        b.upload(np.zeros(b.n_elements, np.int32))
    ctx.pages_extend(table, lens, refs, la, lc, info, seqs, seqs, n_pages, width, 16)
    ctx.sync()
    assert info.download().tolist() == [1, 0, 0, (1 << 31) - 1]
    assert not lens.download().any() and not refs.download().any()
    for b in (table, lens, refs, info, la, lc):
        b.free()

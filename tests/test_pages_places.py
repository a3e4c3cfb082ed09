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

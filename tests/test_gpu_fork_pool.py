"""Forks that would take a free page that is none: the call says so and does nothing, as splat_kernel_compact_pages does of the same pool."""
import numpy as np
import pytest

from conftest import report
from test_gpu_pages import BAD_PAGE, POOL_EMPTY, blank, check_fork, dev, host, ptr

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

BAD = [-1, -(2 ** 31), 2 ** 31 - 1, None]   # None: the first number that is no page


def refused(ctx, parents, lens, ps, pages, pool, used, table, in_place, status=BAD_PAGE):
    n, width = table.shape
    d = [dev(x) for x in (parents, lens, pool, [used], table.reshape(-1))]
    lens_out, used_out = (d[1], d[3]) if in_place else (blank(n), blank(1))
    src, dst, rows, got = blank(n), blank(n), blank(n), blank(1)
    torch.cuda.synchronize()
    ctx.kernel_fork_pages(n, ptr(d[0]), 0, ptr(d[1]), ps, pages, ptr(d[2]), len(pool), ptr(d[3]), ptr(d[4]), width, ptr(lens_out), ptr(src),
                          ptr(dst), ptr(rows), ptr(used_out), ptr(got))
    ctx.synchronize()
    assert int(got) == status and int(used_out) == used
    assert np.array_equal(host(d[4]), table.reshape(-1)) and np.array_equal(host(lens_out), lens) and np.array_equal(host(d[2]), pool)
    assert (host(src) == -1).all() and (host(dst) == -1).all() and (host(rows) == 0).all()


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("bad", BAD)
def test_a_free_page_that_is_none(ctx, bad, in_place):
    report("fork.pool", bad=bad, in_place=in_place)
    pages, table, lens = 10, np.array([[4, 5, -1], [3, -1, -1], [7, 7, 7], [8, 8, 8]]), [20, 12, 0, 0]
    bad = pages if bad is None else bad
    for pool, used in (([6, bad], 0), ([bad, 6], 0), ([0, 6, bad, 9], 1)):
        refused(ctx, [-1, -1, 0, 1], lens, 16, pages, pool, used, table, in_place)
    # those that nothing takes are not looked at: before *used, and behind the last one taken
    check_fork(ctx, [-1, -1, 0, 1], None, lens, 16, pages, [bad, 6, 9, bad], 1, table, in_place=in_place)
    check_fork(ctx, [-1, -1, 0, -1], [0, 0, 16, 0], lens, 16, pages, [bad], 0, table, in_place=in_place)
    refused(ctx, [-1, -1, 0, 1], lens, 16, pages, [bad], 0, table, in_place, status=POOL_EMPTY)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("forks,width", [(900, 3), (1500, 40), (5000, 2)])
@pytest.mark.parametrize("at", [0, 511, -1])
def test_one_of_many(ctx, forks, width, at, in_place):
    """More forks than a block has threads, and several blocks."""
    report("fork.pool.many", forks=forks, width=width, at=at, in_place=in_place)
    pages, n = forks + 10, forks + 1
    table = np.full((n, width), -1)
    table[0] = np.arange(width) % 10
    lens, parents = [8 * width - 3] + [0] * forks, [-1] + [0] * forks
    pool = list(range(10, pages))
    check_fork(ctx, parents, None, lens, 8, pages, pool, 0, table, in_place=in_place)
    pool[at] = pages
    refused(ctx, parents, lens, 8, pages, pool, 0, table, in_place)

"""The operators on a cache's pages through the kernel entry points, against their definitions in plain Python: rows that
become forks, pages given back, pages that move, and copies of them. Whole numbers and copied bits: all equal."""
import numpy as np
import pytest

from conftest import report

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TDT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
OK, BAD_LENGTH, POOL_EMPTY, SLOTS_FULL, BAD_ROW, BAD_PAGE = range(6)


def lib():
    import splathip
    return splathip


def ptr(t):
    return 0 if t is None else t.data_ptr()


def dev(v):
    return torch.tensor(np.asarray(v, np.int64).tolist(), dtype=torch.int32, device="cuda")


def blank(m):
    return torch.full((m,), -7, dtype=torch.int32, device="cuda")


def host(t):
    return t.cpu().numpy().astype(np.int64)


# --- the definitions ------------------------------------------------------------------------------

def fork_ref(parents, keep, lens, ps, pages, pool, used, table):
    n, width = table.shape
    status, need = OK, 0
    if not 0 <= used <= len(pool):
        status = BAD_LENGTH
    stray = False
    for i, p in enumerate(parents):
        if p == -1:
            continue
        if not 0 <= p < n or parents[p] != -1 or lens[i] != 0:
            stray = True
            continue
        k = lens[p] if keep is None else keep[i]
        if not 0 <= lens[p] <= width * ps or not 0 <= k <= lens[p]:
            status = BAD_LENGTH
        elif k % ps and 0 <= table[p, k // ps] < pages:
            need += 1
    status = status or (BAD_ROW if stray else POOL_EMPTY if need > len(pool) - used else OK)
    out = dict(table=table.copy(), lens=list(lens), src=[-1] * n, dst=[-1] * n, rows=[0] * n, used=used, status=status)
    if status:
        return out
    for i, p in enumerate(parents):
        if p == -1:
            continue
        k = lens[p] if keep is None else keep[i]
        out["lens"][i] = k
        m = -(-k // ps)
        out["table"][i, :m] = table[p, :m]
        if k % ps and 0 <= table[p, m - 1] < pages:
            out["src"][i], out["dst"][i], out["rows"][i] = table[p, m - 1], pool[out["used"]], k % ps
            out["table"][i, m - 1] = pool[out["used"]]
            out["used"] += 1
    return out


def free_ref(keep, lens, ps, pages, pool, used, table):
    n, width = table.shape
    out = dict(lens=list(lens), pool=list(pool), used=used, status=OK)
    if not 0 <= used <= len(pool) or any(not 0 <= v <= width * ps or not 0 <= k <= v for k, v in zip(keep, lens)):
        return {**out, "status": BAD_LENGTH}
    held, gone = set(pool[used:]), set()
    for row, k in zip(table, keep):
        held.update(row[:-(-k // ps)].tolist())
    for row, k, v in zip(table, keep, lens):
        gone.update(x for x in row[-(-k // ps):-(-v // ps)].tolist() if 0 <= x < pages and x not in held)
    if len(gone) > used:
        return {**out, "status": BAD_PAGE}
    out["pool"][used - len(gone):used] = sorted(gone)
    return dict(lens=list(keep), pool=out["pool"], used=used - len(gone), status=OK)


def compact_ref(lens, ps, pages, pool, used, table, cap):
    n, width = table.shape
    out = dict(table=table.copy(), pool=list(pool), src=[-1] * cap, dst=[-1] * cap, count=0, status=OK)
    if not 0 <= used <= len(pool) or any(not 0 <= v <= width * ps for v in lens):
        return {**out, "status": BAD_LENGTH}
    live = {x for row, v in zip(table, lens) for x in row[:-(-v // ps)].tolist() if 0 <= x < pages}
    free = pool[used:]
    if len(set(free)) < len(free) or live & set(free) or any(not 0 <= x < pages for x in free):
        return {**out, "status": BAD_PAGE}
    both = sorted(live | set(free))
    low, high = both[:len(live)], both[len(live):]
    to = dict(zip((x for x in high if x in live), (x for x in low if x not in live)))
    if len(to) > cap:
        return {**out, "status": SLOTS_FULL}
    for row, v in zip(out["table"], lens):
        m = -(-v // ps)
        row[:m] = [to.get(x, x) for x in row[:m].tolist()]
    out["pool"][used:] = high
    out["src"][:len(to)], out["dst"][:len(to)], out["count"] = list(to), list(to.values()), len(to)
    return out


# --- the calls ------------------------------------------------------------------------------------

def check_fork(ctx, parents, keep, lens, ps, pages, pool, used, table, status=OK, in_place=False):
    ref = fork_ref(parents, keep, lens, ps, pages, pool, used, table)
    assert ref["status"] == status
    n, width = table.shape
    d = {k: dev(v) for k, v in (("parents", parents), ("lens", lens), ("pool", pool), ("used", [used]))}
    d["keep"] = dev(keep) if keep is not None else None
    d["table"] = torch.cat([dev(table).reshape(-1), blank(5)])
    lens_out, used_out = (d["lens"], d["used"]) if in_place else (blank(n), blank(1))
    src, dst, rows, got = blank(n), blank(n), blank(n), blank(1)
    torch.cuda.synchronize()
    ctx.kernel_fork_pages(n, ptr(d["parents"]), ptr(d["keep"]), ptr(d["lens"]), ps, pages, ptr(d["pool"]), len(pool), ptr(d["used"]),
                          ptr(d["table"]), width, ptr(lens_out), ptr(src), ptr(dst), ptr(rows), ptr(used_out), ptr(got))
    ctx.synchronize()
    assert int(got) == status
    assert np.array_equal(host(d["table"])[:n * width].reshape(n, width), ref["table"]) and (host(d["table"])[n * width:] == -7).all()
    for name, t in (("lens", lens_out), ("src", src), ("dst", dst), ("rows", rows)):
        assert np.array_equal(host(t), ref[name]), name
    assert int(used_out) == ref["used"]
    return ref


def run_free(ctx, keep, lens, ps, pages, pool, used, table, lens_out="own"):
    n, width = table.shape
    d = {k: dev(v) for k, v in (("keep", keep), ("lens", lens), ("pool", list(pool) + [-7] * 3), ("used", [used]), ("table", table))}
    out = blank(n) if lens_out == "own" else d[lens_out]
    used_out, got = blank(1) if lens_out == "own" else d["used"], blank(1)
    size = lib().pages_workspace(pages)
    ws = torch.full((size + 64,), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    ctx.kernel_free_pages(n, ptr(d["keep"]), ptr(d["lens"]), ps, pages, ptr(d["pool"]), len(pool), ptr(d["used"]), ptr(d["table"]), width,
                          ptr(out), ptr(used_out), ptr(got), ptr(ws), size)
    ctx.synchronize()
    assert (ws[size:] == 255).all() and np.array_equal(host(d["table"]).reshape(n, width), table)
    p = host(d["pool"])
    assert (p[len(pool):] == -7).all()
    return dict(lens=host(out), pool=p[:len(pool)], used=int(used_out), status=int(got))


def check_free(ctx, keep, lens, ps, pages, pool, used, table, status=OK, **kw):
    ref = free_ref(keep, lens, ps, pages, pool, used, table)
    assert ref["status"] == status
    got = run_free(ctx, keep, lens, ps, pages, pool, used, table, **kw)
    for name in ref:
        assert np.array_equal(got[name], ref[name]), name
    return ref


def check_compact(ctx, lens, ps, pages, pool, used, table, cap, status=OK, in_place=False):
    ref = compact_ref(lens, ps, pages, pool, used, table, cap)
    assert ref["status"] == status
    n, width = table.shape
    d = {k: dev(v) for k, v in (("lens", lens), ("pool", pool), ("used", [used]), ("table", table))}
    table_out, pool_out = (d["table"], d["pool"]) if in_place else (blank(n * width), blank(len(pool)))
    src, dst, count, got = blank(cap + 3), blank(cap + 3), blank(1), blank(1)
    size = lib().pages_workspace(pages)
    ws = torch.full((size + 64,), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    ctx.kernel_compact_pages(n, ptr(d["lens"]), ps, pages, ptr(d["pool"]), len(pool), ptr(d["used"]), ptr(d["table"]), width, ptr(table_out),
                             ptr(pool_out), ptr(src), ptr(dst), cap, ptr(count), ptr(got), ptr(ws), size)
    ctx.synchronize()
    assert int(got) == status and int(count) == ref["count"] and (ws[size:] == 255).all()
    assert np.array_equal(host(table_out).reshape(n, width), ref["table"])
    first = max(0, min(used, len(pool)))
    if status != BAD_LENGTH or 0 <= used <= len(pool):
        assert np.array_equal(host(pool_out)[first:], ref["pool"][first:])
    assert in_place or (host(pool_out)[:first] == -7).all()
    assert np.array_equal(host(src)[:cap], ref["src"]) and np.array_equal(host(dst)[:cap], ref["dst"])
    assert (host(src)[cap:] == -7).all() and (host(dst)[cap:] == -7).all()
    return ref


class World:
    """Rows with pages in random order, some of them forks, and a pool with the free ones."""

    def __init__(self, n, most, ps, *, seed=1, forks=0.5, spare=20, extra=2):
        rng = np.random.default_rng(seed + n + most)
        self.n, self.ps = n, ps
        self.lens = rng.integers(0, most + 1, n)
        if n > 2:
            self.lens[rng.integers(0, n)] = 0
        self.lens[0] = most
        self.width = -(-most // ps) + extra
        parent = [int(rng.integers(0, max(1, i // 2))) if i and rng.random() < forks else -1 for i in range(n)]
        need = sum(-(-int(v) // ps) for v in self.lens)
        self.pages = need + spare
        ids = rng.permutation(self.pages)
        self.table = np.full((n, self.width), -1, np.int64)
        self.table[:] = rng.integers(0, self.pages, self.table.shape)   # what lies behind a row's pages means nothing
        at = 0
        for i, v in enumerate(self.lens):
            m = -(-int(v) // ps)
            common = 0 if parent[i] < 0 else int(rng.integers(0, min(m, int(self.lens[parent[i]]) // ps) + 1))
            self.table[i, :common] = self.table[parent[i], :common]
            self.table[i, common:m] = ids[at:at + m - common]
            at += m - common
        self.pool, self.used = ids.tolist(), at
        self.rng = rng
        self.lens = self.lens.tolist()


SIZES = [(1, 1, 8), (1, 700, 16), (3, 40, 8), (17, 300, 16), (64, 3000, 16), (200, 40, 32), (1025, 60, 8), (130, 5000, 8),
         (7, 70000, 8), (700, 1500, 8)]   # the last three: more pages than one block's map, several chunks


@pytest.mark.parametrize("n,most,ps", SIZES)
@pytest.mark.parametrize("in_place", [False, True])
def test_fork_pages(ctx, n, most, ps, in_place):
    report("fork", n=n, most=most, ps=ps, in_place=in_place)
    w = World(n, most, ps)
    table = np.concatenate([w.table, np.full((n + 3, w.width), -5)])
    lens = w.lens + [0] * (n + 3)
    for whole in (False, True):
        parents = [-1] * n + [int(w.rng.integers(0, n)) if w.rng.random() < 0.8 else -1 for _ in range(n + 3)]
        keep = None if whole else [int(w.rng.integers(0, lens[p] + 1)) if p >= 0 else 99999999 for p in parents]
        if not whole and n > 3:   # a whole page, and nothing
            for i, k in ((n, 0), (n + 1, ps)):
                if parents[i] >= 0 and lens[parents[i]] >= k:
                    keep[i] = k
        check_fork(ctx, parents, keep, lens, ps, w.pages + 2 * n, w.pool + list(range(w.pages, w.pages + 2 * n + 3)), w.used, table, in_place=in_place)


def test_fork_pages_with_nothing_to_do(ctx):
    check_fork(ctx, [], None, [], 16, 4, [1, 2], 1, np.zeros((0, 3), np.int64))
    check_fork(ctx, [-1, -1], None, [5, 0], 16, 4, [], 0, np.array([[1, 2], [3, 4]]))


@pytest.mark.parametrize("in_place", [False, True])
def test_fork_pages_take_all_or_nothing(ctx, in_place):
    table, lens, pool = np.array([[4, 5, -1], [3, -1, -1], [7, 7, 7], [8, 8, 8]]), [20, 16, 0, 0], [6, 9]
    def fork(parents, keep=None, lens=lens, used=0, status=OK, table=table, pool=pool):
        check_fork(ctx, parents, keep, lens, 16, 10, pool, used, table, status=status, in_place=in_place)
    fork([-1, -1, 0, 0])
    fork([-1, -1, 0, 1], used=1)
    fork([-1, -1, 0, 0], used=1, status=POOL_EMPTY)
    fork([-1, -1, 0, 0], used=3, status=BAD_LENGTH)
    fork([-1, -1, 0, 0], used=-1, status=BAD_LENGTH)
    fork([-1, -1, 0, 0], keep=[0, 0, 21, 1], status=BAD_LENGTH)
    fork([-1, -1, 0, 0], keep=[0, 0, 1, -1], status=BAD_LENGTH)
    fork([-1, -1, 0, -1], lens=[49, 16, 0, 0], status=BAD_LENGTH)
    fork([-1, -1, 0, -1], lens=[-1, 16, 0, 0], status=BAD_LENGTH)
    fork([-1, -1, 4, -1], status=BAD_ROW)
    fork([-1, -1, -2, -1], status=BAD_ROW)
    fork([-1, -1, 2 ** 31 - 1, -1], status=BAD_ROW)
    fork([-1, -1, 0, 2], status=BAD_ROW)     # a fork of a fork
    fork([-1, -1, 2, -1], status=BAD_ROW)    # of itself
    fork([-1, 0, -1, -1], status=BAD_ROW)    # over a row in use
    fork([-1, -1, -1, -1], lens=[2 ** 31 - 1, -9, 0, 0])   # rows that no fork asks for are not looked at
    # a begun page that is none stays one, and takes none
    for bad in (-1, -(2 ** 31), 10, 2 ** 31 - 1):
        t = table.copy()
        t[0, 1] = bad
        fork([-1, -1, 0, 0], table=t, pool=[], keep=[0, 0, 20, 17])


@pytest.mark.parametrize("n,most,ps", SIZES)
@pytest.mark.parametrize("lens_out", ["own", "lens", "keep"])
def test_free_pages(ctx, n, most, ps, lens_out):
    report("free", n=n, most=most, ps=ps, lens_out=lens_out)
    w = World(n, most, ps)
    for share in (0.0, 0.3, 1.0):
        keep = [int(w.rng.integers(0, v + 1)) if w.rng.random() < share / 2 else 0 if w.rng.random() < share else v for v in w.lens]
        check_free(ctx, keep, w.lens, ps, w.pages, w.pool, w.used, w.table, lens_out=lens_out)
    ref = check_free(ctx, [0] * n, w.lens, ps, w.pages, w.pool, w.used, w.table, lens_out=lens_out)
    assert ref["used"] == 0 and sorted(ref["pool"]) == list(range(w.pages))


@pytest.mark.parametrize("pages", [10, 40000, 100000])   # one block, one chunk more, several
def test_free_pages_takes_all_or_nothing(ctx, pages):
    table = np.array([[4, 5, -1], [4, 3, 5], [7, -2, pages]])
    def free(keep, lens, used=6, pool=(0, 1, 2, 6, 8, 9, 9), status=OK):
        return check_free(ctx, keep, lens, 16, pages, list(pool), used, table, status=status)
    assert free([0, 48, 48], [32, 48, 48])["used"] == 6        # both pages are in the other row
    assert free([0, 0, 48], [32, 48, 48])["pool"][3:6] == [3, 4, 5]
    assert free([16, 0, 0], [32, 48, 48])["pool"][3:6] == [3, 5, 7]
    free([0, 0, 0], [32, 48, 48], used=4, pool=[0, 1, 2, 6])
    free([0, 0, 0], [32, 48, 48], used=3, pool=[0, 1, 2, 6], status=BAD_PAGE)   # four pages, three taken
    free([0, 0, 0], [32, 48, 48], used=0, pool=[4, 5, 3, 7])   # all free already
    free([0, 0, 0], [32, 48, 48], used=2, pool=[4, 5, 3, -7, 2 ** 31 - 1], status=BAD_PAGE)   # three of them are not free
    free([0, 0, 0], [32, 48, 48], used=3, pool=[4, 5, 8, 3, -7, 2 ** 31 - 1])
    free([33, 0, 0], [32, 48, 48], status=BAD_LENGTH)
    free([-1, 0, 0], [32, 48, 48], status=BAD_LENGTH)
    free([0, 0, 0], [32, 49, 48], status=BAD_LENGTH)
    free([0, 0, 0], [32, -1, 48], status=BAD_LENGTH)
    free([0, 0, 0], [32, 48, 48], used=8, status=BAD_LENGTH)
    free([0, 0, 0], [32, 48, 48], used=-1, status=BAD_LENGTH)
    check_free(ctx, [], [], 16, pages, [1, 2], 1, np.zeros((0, 3), np.int64))


@pytest.mark.parametrize("n,most,ps", SIZES)
@pytest.mark.parametrize("in_place", [False, True])
def test_compact_pages(ctx, n, most, ps, in_place):
    for spare in (0, 1, 30, 3000, 120000):
        report("compact", n=n, most=most, ps=ps, spare=spare, in_place=in_place)
        w = World(n, most, ps, spare=spare)
        ref = check_compact(ctx, w.lens, ps, w.pages, w.pool, w.used, w.table, w.pages // 2 + 1, in_place=in_place)
        live = {x for row, v in zip(ref["table"], w.lens) for x in row[:-(-v // ps)].tolist()}
        assert live == set(range(len(live))) and ref["pool"][w.used:] == list(range(len(live), w.pages))
    # the pool does not hold every page: those it does not know stay out of it
    some = w.pool[:w.used] + w.pool[w.used + 2::3]
    check_compact(ctx, w.lens, ps, w.pages, some, w.used, w.table, w.pages // 2, in_place=in_place)
    # rows have lost pages: holes that the pool does not know
    lens = [v // 2 for v in w.lens]
    check_compact(ctx, lens, ps, w.pages, w.pool, w.used, w.table, w.pages // 2, in_place=in_place)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("pages", [10, 40000, 100000])
def test_compact_pages_does_all_or_nothing(ctx, pages, in_place):
    table = np.array([[4, 9, -1, 6], [4, 3, 9, 6], [7, -2, pages, 6]])
    def compact(lens=(32, 48, 48), used=2, pool=(9, 9, 0, 1, 5), cap=4, status=OK):
        return check_compact(ctx, list(lens), 16, pages, list(pool), used, table, cap, status=status, in_place=in_place)
    assert compact()["src"] == [7, 9, -1, -1]
    compact(cap=2)
    compact(cap=1, status=SLOTS_FULL)
    compact(cap=0, status=SLOTS_FULL)
    compact(pool=(9, 9), cap=0)
    compact(lens=(0, 0, 0), cap=0)
    compact(pool=(0, 0, 0, 1, 0), status=BAD_PAGE)
    compact(pool=(0, 0, 0, 1, 3), status=BAD_PAGE)       # free and in use
    compact(pool=(0, 0, 0, 1, -1), status=BAD_PAGE)
    compact(pool=(0, 0, 0, 1, pages), status=BAD_PAGE)
    compact(lens=(32, 65, 48), status=BAD_LENGTH)
    compact(lens=(32, -1, 48), status=BAD_LENGTH)
    compact(used=6, status=BAD_LENGTH)
    compact(used=-1, status=BAD_LENGTH)
    check_compact(ctx, [], 16, pages, [1, 2], 1, np.zeros((0, 3), np.int64), 3, in_place=in_place)


# --- copies -----------------------------------------------------------------------------------------

def test_millions_of_pages(ctx):
    """More chunks of the maps than a block has threads, with the rows' pages in the first, the last and ones between."""
    pages, ps, rng = 4096 * 1024 + 50000, 8, np.random.default_rng(5)
    report("pages.millions", pages=pages)
    ids = rng.permutation(pages)
    ids[:4] = [0, pages - 1, 4096 * 1024 - 1, 4096 * 1024]
    ids = np.concatenate([ids[:4], rng.permutation(np.setdiff1d(np.arange(pages), ids[:4]))])
    table = np.full((3, 2000), -1, np.int64)
    table[0], table[1, :1500], table[2, :700] = ids[:2000], ids[1000:2500], ids[:700]
    lens = [16000, 12000 - 3, 5600]
    used, pool = 2500, [0] * 2500 + ids[2500:].tolist()
    check_free(ctx, [4000, 0, 5600], lens, ps, pages, pool, used, table)
    check_compact(ctx, lens, ps, pages, pool, used, table, 2500)
    half = 2110000   # nearly all pages in use: the last of them lies in a chunk past the 1024th
    check_compact(ctx, [half * ps - 3, half * ps], ps, pages, [0] * 7 + ids[2 * half:].tolist(), 7, ids[:2 * half].reshape(2, half), pages - 2 * half, in_place=True)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("kv,ps,layers,gap,bounds", [(1, 8, 1, 0, False), (3, 16, 2, 64, True), (12, 32, 5, 0, True), (8, 64, 64, 8, False), (2, 256, 3, 0, True)])
def test_copy_pages(ctx, dtype, kv, ps, layers, gap, bounds):
    L, td, pages = lib(), TDT[dtype], 23
    g = torch.Generator().manual_seed(kv * ps)
    stride = kv * ps * 64 + gap
    pools = [[torch.randn(pages, stride, generator=g).to(td).cuda() for _ in range(2)] for _ in range(layers)]
    for k, _ in pools:
        k[3, :70] = float("nan")   # bits go along as they are
    low = [torch.randn(pages, kv, 2, 64, generator=g).to(td).cuda() for _ in range(layers)] if bounds else None
    caches = L.layers(L.KvCache(L.DTYPES[dtype], ptr(k), ptr(v), pages, ps, kv, stride) for k, v in pools)
    order = torch.randperm(pages, generator=g).tolist()
    src, dst = order[:10] + [-1, 5, pages, 2 ** 31 - 1, 4, 4], order[10:20] + [order[20], -1, order[21], order[22], pages, 4]
    rows = [0, 1, ps - 1, ps, ps + 5, 7, -3, 2, 8, 5] + [ps] * 6
    for r, count in ((None, None), (rows, None), (rows, 7), (None, 0), (None, -4), (None, 2 ** 31 - 1)):
        report("copy", dtype=dtype, kv=kv, ps=ps, layers=layers, rows=r is not None, count=count)
        want = [[p.cpu().clone() for p in pair] for pair in pools]
        wlow = [b.cpu().clone() for b in low] if bounds else []
        n = len(src) if count is None else max(0, min(count, len(src)))
        for s, t, m in list(zip(src, dst, r or [ps] * len(src)))[:n]:
            if not (0 <= s < pages and 0 <= t < pages) or s == t:
                continue
            for x in (p for pair in want for p in pair):
                x = x[:, :kv * ps * 64].view(pages, kv, ps, 64)
                x[t, :, :max(m, 0)] = x[s, :, :max(m, 0)]
            for b in wlow:
                b[t] = b[s]
        d = [dev(src), dev(dst), dev(r) if r else None, dev([count]) if count is not None else None]
        torch.cuda.synchronize()
        ctx.kernel_copy_pages(caches, L.pointers(ptr(b) for b in low) if bounds else None, len(src), *[ptr(x) for x in d])
        ctx.synchronize()
        same = lambda a, b: torch.equal(a.cpu().view(torch.int32 if dtype == "f32" else torch.int16), b.view(torch.int32 if dtype == "f32" else torch.int16))  # noqa: E731
        assert all(same(p, x) for pair, xs in zip(pools, want) for p, x in zip(pair, xs))
        assert all(same(b, x) for b, x in zip(low or [], wlow))


def test_copy_pages_of_many_pairs(ctx):
    """More pieces than a launch has blocks."""
    L, pages, kv, ps = lib(), 9001, 3, 32
    k, v = (torch.randint(-2 ** 15, 2 ** 15, (pages, kv, ps, 64), dtype=torch.int16, device="cuda") for _ in range(2))
    want = [x.clone() for x in (k, v)]
    order = torch.randperm(pages, device="cuda")
    src, dst = order[:4400], order[4400:8800]
    for x in want:
        x[dst] = x[src]
    a, b = src.int(), dst.int()
    torch.cuda.synchronize()
    ctx.kernel_copy_pages(L.KvCache(L.BF16, ptr(k), ptr(v), pages, ps, kv), None, 4400, ptr(a), ptr(b))
    ctx.synchronize()
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


def test_copy_pages_with_offsets_past_32_bits(ctx):
    """Pages 4 GiB apart."""
    L, pages, stride = lib(), 3, 2 ** 31
    k, v = (torch.zeros((pages - 1) * stride + 2 * 8 * 64, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for x, a in ((k, 1.0), (v, 5.0)):
        x[2 * stride:] = a
    d = [dev([2]), dev([1])]
    torch.cuda.synchronize()
    ctx.kernel_copy_pages(L.KvCache(L.BF16, ptr(k), ptr(v), pages, 8, 2, stride), None, 1, *[ptr(x) for x in d])
    ctx.synchronize()
    for x, a in ((k, 1.0), (v, 5.0)):
        assert (x[stride:stride + 1024] == a).all() and (x[:1024] == 0).all() and float(x[stride + 1024:stride + 4096].abs().max()) == 0


def test_calls_without_layers_or_pairs(ctx):
    L = lib()
    ctx.kernel_copy_pages(L.layers([]), None, 5, 0, 0)
    ctx.kernel_copy_pages(L.KvCache(L.BF16, 1 << 20, 1 << 30, 4, 16, 2), None, 0, 0, 0)

"""Scenes of a few layers whose rows fork, grow side by side, attend over what they share, end, and whose pages move:
block tables, forks, copies of pages, norms with rotation into the cache, page bounds, attention over the shared prefix,
pages given back and compacted, as a serving program calls them; against plain restatements of what every row was fed. Tolerances
of rotated keys and of attention as in test_gpu_cache.py. What the calls refuse stands at the end."""
import numpy as np
import pytest

from conftest import report

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_gpu_cache import TDT, Cache, bounds_ref, check_paged, ints, lib, ptr, rope_ref, rope_tol  # noqa: E402

SCENES, EACH = 2, 4            # rows: a scene, then its forks
N = SCENES * EACH


class Branches:
    """What a serving program keeps on the device, and beside it the rows that every sequence was fed."""

    def __init__(self, dtype, heads=6, kv=2, ps=16, layers=2, cap=400, width=30, pages=150):
        self.__dict__.update(dtype=dtype, heads=heads, kv=kv, ps=ps, layers=layers, cap=cap, width=width, pages=pages)
        td, L = TDT[dtype], lib()
        cuda = lambda *s, v=0, t=torch.int32: torch.full(s, v, dtype=t, device="cuda")  # noqa: E731
        self.k, self.v = (cuda(layers, pages, kv, ps, 64, v=float("nan"), t=td) for _ in range(2))
        self.bounds = cuda(layers, pages, kv, 2, 64, v=float("nan"), t=td)
        self.caches = [L.KvCache(L.DTYPES[dtype], ptr(self.k[l]), ptr(self.v[l]), pages, ps, kv) for l in range(layers)]
        self.lens, self.add, self.parents, self.fork_keep, self.keep = (cuda(N) for _ in range(5))
        self.src, self.dst, self.rows_of, self.moved, self.moved_to = (cuda(N), cuda(N), cuda(N), cuda(pages // 2), cuda(pages // 2))
        self.used, self.count, self.status = cuda(1), cuda(1), cuda(4, v=-7)
        self.table, self.shared = cuda(N, width, v=-1), cuda(SCENES)
        self.starts, self.slots, self.pos, self.groups = cuda(N + 1), cuda(cap), cuda(cap), ints([g * EACH for g in range(SCENES + 1)]).cuda()
        self.pool = torch.randperm(pages, generator=torch.Generator().manual_seed(2)).to(torch.int32).cuda()
        self.qkv = cuda(layers, cap, (heads + 2 * kv) * 64, v=0.0, t=td)
        self.q, self.last, self.out = cuda(cap, heads * 64, v=0.0, t=td), cuda(layers, N, heads * 64, v=0.0, t=td), cuda(layers, N, heads * 64, v=0.0, t=td)
        self.max_len = width * ps
        self.size = L.prefix_attention_workspace(self.caches[0], N, heads, SCENES, self.max_len, self.max_len)
        self.ws, self.map = cuda(self.size, t=torch.uint8, v=255), cuda(L.pages_workspace(pages), t=torch.uint8, v=255)
        self.fed = [torch.zeros(0, layers, heads + 2 * kv, 64) for _ in range(N)]
        self.common = [0] * SCENES

    def calls(self, ctx):
        L, h, kv, d, bounds = lib(), self.heads, self.kv, self.heads * 64, lib().pointers([ptr(b) for b in self.bounds])
        caches, pages = L.layers(self.caches), (self.ps, self.pages, ptr(self.pool), self.pages, ptr(self.used))
        at = lambda i: ptr(self.status) + 4 * i  # noqa: E731
        ctx.kernel_fork_pages(N, ptr(self.parents), ptr(self.fork_keep), ptr(self.lens), *pages, ptr(self.table), self.width, ptr(self.lens), ptr(self.src),
                              ptr(self.dst), ptr(self.rows_of), ptr(self.used), at(0))
        ctx.kernel_copy_pages(caches, bounds, N, ptr(self.src), ptr(self.dst), ptr(self.rows_of))
        ctx.kernel_block_tables(N, ptr(self.lens), ptr(self.add), self.ps, ptr(self.pool), self.pages, ptr(self.used), ptr(self.table), self.width,
                                ptr(self.lens), ptr(self.starts), ptr(self.slots), ptr(self.pos), self.cap, ptr(self.used), at(1))
        for l, cache in enumerate(self.caches):
            ctx.kernel_qk_norm_rope(L.DTYPES[self.dtype], ptr(self.qkv[l]), (h + 2 * kv) * 64, self.cap, h, kv, L.NORM_RMS, 0, 0, 0, 0, 1e-6,
                                    L.ROPE_LINE, 100.0, ptr(self.pos), ptr(self.q), d, 0, 0, cache, ptr(self.slots))
            ctx.kernel_page_bounds(cache, N, ptr(self.table), self.width, ptr(self.lens), ptr(self.add), 64, ptr(self.bounds[l]))
            # a scene's row is every EACH-th of the table
            ctx.kernel_prefix_attention(cache, ptr(self.last[l]), d, N, h, ptr(self.groups), SCENES, ptr(self.table), EACH * self.width, ptr(self.shared),
                                        self.max_len, ptr(self.table), self.width, ptr(self.lens), self.max_len, 0.125, ptr(self.out[l]), d, ptr(self.ws),
                                        self.size)
        ctx.kernel_free_pages(N, ptr(self.keep), ptr(self.lens), *pages, ptr(self.table), self.width, ptr(self.lens), ptr(self.used), at(2), ptr(self.map),
                              self.map.numel())
        ctx.kernel_compact_pages(N, ptr(self.lens), *pages, ptr(self.table), self.width, ptr(self.table), ptr(self.pool), ptr(self.moved), ptr(self.moved_to),
                                 self.pages // 2, ptr(self.count), at(3), ptr(self.map), self.map.numel())
        ctx.kernel_copy_pages(caches, bounds, self.pages // 2, ptr(self.moved), ptr(self.moved_to), 0, ptr(self.count))

    def feed(self, forks=(), add=(0,) * N, end=(), cut=(), seed=0):
        """forks: (row, parent, positions); add: new tokens of each row; end: rows that end after the step; cut: (row, by so many)."""
        g, td = torch.Generator().manual_seed(seed), TDT[self.dtype]
        parents, fork_keep = [-1] * N, [-3] * N
        before = list(self.fed)
        for row, parent, positions in forks:
            parents[row], fork_keep[row] = parent, positions
            self.fed[row] = before[parent][:positions]
            lived = any(len(before[i]) for i in range(parent + 1, parent + EACH))
            self.common[parent // EACH] = min(positions, self.common[parent // EACH]) if lived else positions
        x = torch.full((self.layers, self.cap, self.heads + 2 * self.kv, 64), float("nan"))   # garbage behind the rows
        x[:, :sum(add)] = torch.randn(self.layers, sum(add), self.heads + 2 * self.kv, 64, generator=g)
        x = x.to(td)
        t = 0
        for i, a in enumerate(add):
            self.fed[i] = torch.cat([self.fed[i], x[:, t:t + a].float().transpose(0, 1)])
            t += a
        for s in range(SCENES):
            if not any(len(self.fed[i]) for i in range(s * EACH + 1, s * EACH + EACH)):
                self.common[s] = len(self.fed[s * EACH])
        self.shared_now = [min(c, len(self.fed[s * EACH])) for s, c in enumerate(self.common)]
        self.whole = [i not in end and i not in dict(cut) for i in range(N)]
        self.seen = [len(r) for r in self.fed]
        for i in range(N):
            self.fed[i] = self.fed[i][:0 if i in end else len(self.fed[i]) - dict(cut).get(i, 0)]
        self.qkv.copy_(x.reshape(self.layers, self.cap, -1).cuda())
        self.last.copy_(torch.randn(self.last.shape, generator=g).to(td).cuda())
        self.out.fill_(float("nan"))
        for t, v in ((self.add, add), (self.parents, parents), (self.fork_keep, fork_keep), (self.keep, [len(r) for r in self.fed]), (self.shared, self.shared_now)):
            t.copy_(ints(list(v)).cuda())
        torch.cuda.synchronize()

    def check(self):
        assert self.status.tolist() == [0] * 4
        lens, table = [len(r) for r in self.fed], self.table.cpu()
        assert self.lens.tolist() == lens
        held = {int(p) for row, v in zip(table, lens) for p in row[:-(-v // self.ps)]}
        used, pool = int(self.used), self.pool.tolist()
        assert held == set(range(len(held))) and used == len(held) and pool[used:] == list(range(used, self.pages))   # compact, nothing lost
        for s in range(SCENES):   # the whole pages of what they have in common are one page each
            for i in range(s * EACH + 1, s * EACH + EACH):
                if lens[i]:
                    m = min(self.shared_now[s], lens[i], lens[s * EACH]) // self.ps
                    assert torch.equal(table[i, :m], table[s * EACH, :m])
        h, kv = self.heads, self.kv
        for l in range(self.layers):
            c = Cache.__new__(Cache)
            c.__dict__.update(dtype=self.dtype, lens=lens, kv=kv, ps=self.ps, n=N, pages=self.pages, width=self.width, table=table,
                              k=self.k[l].cpu().reshape(self.pages, -1), v=self.v[l].cpu().reshape(self.pages, -1))
            for i, r in enumerate(self.fed):
                if not len(r):
                    continue
                x, at = r[:, l, h:h + kv].double(), range(len(r))
                want = rope_ref(x, None, None, "rms", "line", 100.0, torch.arange(len(r)), 1e-6)
                tol = rope_tol(x, want, self.dtype)
                for j in range(kv):
                    assert ((c.head(c.k, i, j, at) - want[:, j]).abs() <= tol[:, j]).all()
                    assert torch.equal(c.head(c.v, i, j, at), r[:, l, h + kv + j].to(TDT[self.dtype]).double())
            b = self.bounds[l].cpu().double()
            for p, v in bounds_ref(c, table, lens, None).items():   # of a page that was cut they may be wider
                assert (b[p][:, 0] <= v[:, 0]).all() and (b[p][:, 1] >= v[:, 1]).all()
            out, rows = self.out[l].cpu(), [i for i in range(N) if self.whole[i]]
            assert torch.isfinite(out).all()
            c.lens = [lens[i] for i in rows]
            c.table = table[rows]
            check_paged(None, c, h, self.last[l].cpu()[rows], out[rows])


STEPS = [
    dict(add=[160, 0, 0, 0, 37, 0, 0, 0]),
    dict(forks=[(1, 0, 160), (2, 0, 160), (5, 4, 37), (6, 4, 33), (7, 4, 32)], add=[0, 1, 1, 0, 0, 1, 1, 1]),
    dict(add=[0, 20, 1, 0, 1, 1, 40, 1]),
    dict(forks=[(3, 0, 100)], add=[3, 1, 1, 0, 1, 0, 0, 0], end=[1, 5], cut=[(6, 9)]),
    dict(add=[1, 0, 16, 17, 0, 0, 1, 1]),
    dict(),
    dict(forks=[(1, 0, 164), (5, 4, 1)], add=[0, 0, 1, 1, 0, 30, 1, 1], cut=[(2, 1), (3, 1)]),
    dict(add=[1, 100, 1, 1, 1, 1, 100, 1], end=[1, 2, 3, 5, 6, 7]),
    dict(forks=[(7, 4, 40)], add=[1, 0, 0, 0, 1, 0, 0, 1], end=[0]),
    dict(add=[50, 0, 0, 0, 1, 0, 0, 1]),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_scenes_that_fork(ctx, dtype):
    s = Branches(dtype)
    for step, what in enumerate(STEPS):
        report("forks", dtype=dtype, step=step, **what)
        s.feed(**what, seed=100 + step)
        s.calls(ctx)
        ctx.synchronize()
        s.check()


def test_scenes_that_fork_in_a_captured_graph(ctx):
    """All calls captured once on the context's stream and replayed every step, with eager work of the same context and of
    torch between the replays; nothing is allocated by them."""
    s, other = Branches("bf16"), Branches("bf16", heads=16, kv=2, ps=8, layers=1, width=40)
    other.feed(add=[30, 0, 0, 0, 5, 0, 0, 0], seed=1)
    other.calls(ctx)          # the code objects are loaded
    ctx.synchronize()
    other.check()
    stream = torch.cuda.ExternalStream(ctx.stream)
    graph = torch.cuda.CUDAGraph()
    s.feed()
    with torch.cuda.graph(graph, stream=stream):
        s.calls(ctx)
    for step, what in enumerate(STEPS):
        report("forks.graph", step=step, **what)
        s.feed(**what, seed=100 + step)
        with torch.cuda.stream(stream):
            graph.replay()
        ctx.synchronize()
        s.check()
        other.feed(forks=[(1 + step % 3, 0, 30)], add=[0, 1, 1, 1, 1, 0, 0, 0], end=[1, 2, 3], seed=50 + step)
        other.calls(ctx)
        ctx.synchronize()
        other.check()


def test_two_contexts_at_once(ctx):
    """Two streams with tables and workspaces of their own, both under way before either is waited for."""
    L = lib()
    second = L.Context(0)
    both = [(Branches("f16"), ctx), (Branches("bf16", heads=8, kv=1, ps=32, layers=3, width=20, pages=90), second)]
    try:
        for step, what in enumerate(STEPS):
            report("forks.two", step=step)
            for s, _ in both:
                s.feed(**what, seed=7 * step)
            for s, c in both:
                s.calls(c)
            for s, c in both:
                c.synchronize()
                s.check()
    finally:
        second.close()


@pytest.mark.parametrize("dtype,members,shared,heads,kv", [("bf16", 700, 2000, 12, 12), ("f16", 40, 3000, 32, 8), ("f32", 100, 900, 8, 2), ("bf16", 3, 9000, 6, 6)])
def test_prefix_attention_in_a_captured_graph(ctx, dtype, members, shared, heads, kv):
    """Each form, captured with its parts and their join, replayed over other lengths, starts, queries and pages."""
    from test_gpu_prefix import Shared
    L = lib()
    full = Shared(dtype, [members], [shared], None, heads, kv, 16)
    cache_k, cache_v = full.k.cuda(), full.v.cuda()
    cache = L.KvCache(L.DTYPES[dtype], ptr(cache_k), ptr(cache_v), full.pages, 16, kv, full.stride)
    q, out, starts, prefix, own, lens = (t.cuda() for t in (full.q, torch.zeros_like(full.q), ints([0, members, members]), torch.cat([full.prefix] * 2),
                                                            ints([shared, 0]), ints([shared] * members)))
    size = L.prefix_attention_workspace(cache, members, heads, 2, shared, 0)
    ws = torch.full((size + 16,), 255, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()

    def call():
        ctx.kernel_prefix_attention(cache, ptr(q), heads * 64, members, heads, ptr(starts), 2, ptr(prefix), full.prefix_width, ptr(own), shared, 0, 0, ptr(lens), 0,
                                    0.125, ptr(out), heads * 64, ptr(ws), size)
    call()
    ctx.synchronize()
    stream, graph = torch.cuda.ExternalStream(ctx.stream), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        call()
    g = torch.Generator().manual_seed(3)
    for step, (middle, a, b) in enumerate([(members, shared, 0), (1, 17, shared), (members // 2, shared // 2, shared), (0, 0, shared - 1), (members - 1, 0, 5)]):
        report("prefix.graph", dtype=dtype, step=step)
        full.q = torch.randn(members, heads * 64, generator=g).to(TDT[dtype])
        see = torch.randint(0, shared + 1, (members,), generator=g).tolist()
        for t, v in ((q, full.q), (starts, ints([0, middle, members])), (own, ints([a, b])), (lens, ints(see))):
            t.copy_(v.cuda())
        out.fill_(float("nan"))
        ws.fill_(255)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        ctx.synchronize()
        once = out.cpu()
        call()
        ctx.synchronize()
        assert torch.equal(out.cpu(), once)     # the same sums in the same order
        full.lens = [min(v, a if i < middle else b) for i, v in enumerate(see)]
        full.check(once, rows=sorted({0, 1, middle % members, members // 2, members - 1}))


def test_profiling_names_the_operators(ctx):
    s = Branches("bf16")
    s.feed(**STEPS[0])
    ctx.profile_begin()
    s.calls(ctx)
    names = {r["name"] for r in ctx.profile_end()}
    assert {"fork_pages", "free_pages", "compact_pages", "copy_pages", "prefix_attention"} <= names


def test_refused_calls_say_why_and_launch_nothing(ctx):
    L = lib()
    s = Branches("bf16")
    for step in (0, 1):
        s.feed(**STEPS[step], seed=step)
        s.calls(ctx)
    s.feed(**STEPS[2], seed=2)
    ctx.synchronize()
    keys = ("k", "v", "bounds", "lens", "table", "pool", "used", "src", "dst", "rows_of", "moved", "moved_to", "count", "out")
    before = {k: getattr(s, k).clone().view(torch.uint8) for k in keys}
    d, caches, bounds = s.heads * 64, L.layers(s.caches), L.pointers([ptr(b) for b in s.bounds])
    stat, map_bytes = ptr(s.status), s.map.numel()
    calls = {
        "kernel_fork_pages": (dict(n=N, parents=ptr(s.parents), keep=0, lens=ptr(s.lens), page_size=16, pages=s.pages, pool=ptr(s.pool), pool_size=s.pages,
                                   used=ptr(s.used), table=ptr(s.table), width=s.width, lens_out=ptr(s.lens), src=ptr(s.src), dst=ptr(s.dst),
                                   rows=ptr(s.rows_of), used_out=ptr(s.used), status=stat),
                              [dict(n=-1), dict(n=65537), dict(page_size=12), dict(pages=0), dict(parents=0), dict(src=ptr(s.dst)), dict(table=ptr(s.pool)),
                               dict(lens_out=ptr(s.lens) + 4), dict(width=0), dict(pool_size=-1), dict(status=stat + 2)]),
        "kernel_free_pages": (dict(n=N, keep=ptr(s.keep), lens=ptr(s.lens), page_size=16, pages=s.pages, pool=ptr(s.pool), pool_size=s.pages, used=ptr(s.used),
                                   table=ptr(s.table), width=s.width, lens_out=ptr(s.lens), used_out=ptr(s.used), status=stat, workspace=ptr(s.map),
                                   workspace_bytes=map_bytes),
                              [dict(keep=0), dict(workspace=0), dict(workspace_bytes=map_bytes - 1), dict(pool=ptr(s.table)), dict(used_out=ptr(s.lens)),
                               dict(workspace=ptr(s.table)), dict(pages=s.pages * 1000)]),
        "kernel_compact_pages": (dict(n=N, lens=ptr(s.lens), page_size=16, pages=s.pages, pool=ptr(s.pool), pool_size=s.pages, used=ptr(s.used), table=ptr(s.table),
                                      width=s.width, table_out=ptr(s.table), pool_out=ptr(s.pool), src=ptr(s.moved), dst=ptr(s.moved_to), cap=s.pages // 2,
                                      count=ptr(s.count), status=stat, workspace=ptr(s.map), workspace_bytes=map_bytes),
                                 [dict(cap=-1), dict(count=0), dict(table_out=ptr(s.table) + 4), dict(pool_out=ptr(s.lens)), dict(src=ptr(s.moved_to)),
                                  dict(workspace=ptr(s.map) + 4), dict(cap=1 << 30)]),
        "kernel_copy_pages": (dict(caches=caches, bounds=bounds, n=N, src=ptr(s.src), dst=ptr(s.dst), rows=0, count=0),
                              [dict(n=-1), dict(src=0), dict(dst=ptr(s.dst) + 1), dict(caches=L.layers([s.caches[0]] * 2)), dict(bounds=L.pointers([ptr(s.bounds)])),
                               dict(bounds=L.pointers([0, ptr(s.bounds[1])])), dict(caches=L.layers(s.caches * 33), bounds=None), dict(src=ptr(s.k))]),
        "kernel_prefix_attention": (dict(cache=s.caches[0], q=ptr(s.last[0]), ldq=d, n=N, heads=s.heads, starts=ptr(s.groups), groups=SCENES, prefix=ptr(s.table),
                                         prefix_width=EACH * s.width, shared=ptr(s.shared), max_shared=s.max_len, table=ptr(s.table), width=s.width,
                                         lens=ptr(s.lens), max_own=s.max_len, scale=0.125, out=ptr(s.out[0]), ldo=d, workspace=ptr(s.ws), workspace_bytes=s.size),
                                    [dict(heads=5), dict(cache=None), dict(ldq=d - 4), dict(ldo=d - 8), dict(q=0), dict(lens=0), dict(groups=65537), dict(max_own=-1),
                                     dict(scale=float("inf")), dict(out=ptr(s.last[0])), dict(workspace_bytes=0), dict(out=ptr(s.k)), dict(prefix_width=0)]),
    }
    for name, (args, bad) in calls.items():
        for change in bad:
            with pytest.raises(L.SplatError) as e:
                getattr(ctx, name)(**{**args, **change})
            assert e.value.code == L.BAD_ARGUMENT and len(str(e.value)) > 10, (name, change)
    for bad in ((s.caches[0], N, 5, SCENES, 10, 0), (s.caches[0], N, 6, -1, 10, 0), (s.caches[0], N, 6, 2, -1, 0), (None, N, 6, 2, 1, 0)):
        with pytest.raises(L.SplatError):
            L.prefix_attention_workspace(*bad)
    for bad in (0, -1, (1 << 28) + 1):
        with pytest.raises(L.SplatError):
            L.pages_workspace(bad)
    ctx.synchronize()
    for k in keys:
        assert torch.equal(getattr(s, k).view(torch.uint8), before[k]), k
    s.calls(ctx)
    ctx.synchronize()
    s.check()

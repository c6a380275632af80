"""Attention over a prefix that tokens share, through the kernel entry points, against the definition in 64 bits on the CPU: each
token's positions gathered from the prefix's row and its own.

Tolerance (u = 2^-24, h = half a rounding step of the storage type, as in test_gpu_cache.py): |out - ref| <= h |ref| +
(h_w + 2 e + (L + 8) u) A with A = sum w |v| / sum w, h_w = h for 16-bit types, whose weights may be rounded to the type, and e = 70 u
scale sum |q_c k_c| the error of a score; joins of parts are a few u more, of the 8. In f16 weights lose bits 2^-37 below the
largest, L 2^-37 max |v|, and the output 2^-25."""
import numpy as np
import pytest

from conftest import report

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = 2.0 ** -24
TDT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
DTYPES = ["bf16", "f16", "f32"]


def lib():
    import splathip
    return splathip


def ptr(t):
    return 0 if t is None else t.data_ptr()


def ints(v):
    return torch.as_tensor(v, dtype=torch.int32)


class Shared:
    """Groups of tokens (members [groups]), shared [groups] positions of each, `own` more of each token (None: no table); `sees`:
    the tokens' lengths (None: everything). Garbage (NaN, infinities) wherever no position of anybody lies."""

    def __init__(self, dtype, members, shared, own, heads, kv, ps, *, sees=None, seed=1, gap=0, behind=2):
        g = torch.Generator().manual_seed(seed)
        self.__dict__.update(dtype=dtype, members=list(members), shared=list(shared), heads=heads, kv=kv, ps=ps)
        self.n, td = sum(members), TDT[dtype]
        self.group = [i for i, m in enumerate(members) for _ in range(m)]
        held = [-(-v // ps) for v in shared]
        self.prefix_width = max(held + [0]) + behind
        self.lens = sees if sees is not None else [shared[k] + (own[i] if own else 0) for i, k in enumerate(self.group)]
        self.has_table, self.has_lens = own is not None, own is not None or sees is not None
        mine = [max(0, -(-v // ps) - shared[k] // ps) if own and v > shared[k] else 0 for v, k in zip(self.lens, self.group)]
        self.width = (max([-(-v // ps) for v in self.lens] + [0]) + behind) if own is not None else 0
        self.pages = sum(held) + sum(mine) + 3
        ids = torch.randperm(self.pages, generator=g).tolist()
        self.prefix = torch.full((len(members), self.prefix_width), -1, dtype=torch.int32)
        self.table = torch.full((self.n, max(self.width, 1)), -1, dtype=torch.int32)
        self.stride = kv * ps * 64 + gap
        bad = torch.tensor([float("nan"), float("inf"), -float("inf")])
        self.k, self.v = (bad[torch.randint(0, 3, (self.pages, self.stride), generator=g)].to(td) for _ in range(2))
        at = 0
        for x, v in enumerate(shared):
            for j in range(held[x]):
                self.fill(ids[at], 0, min(ps, v - j * ps), g)
                self.prefix[x, j] = ids[at]
                at += 1
        for i, k in enumerate(self.group):
            for j in range(mine[i]):
                place = shared[k] // ps + j
                self.fill(ids[at], max(0, shared[k] - place * ps), min(ps, self.lens[i] - place * ps), g)
                self.table[i, place] = ids[at]
                at += 1
        self.q = torch.randn(self.n, heads * 64, generator=g).to(td)
        self.starts = [0] + np.cumsum(members).tolist()

    def fill(self, page, first, end, g):
        for p in (self.k, self.v):
            x = p[page, :self.kv * self.ps * 64].view(self.kv, self.ps, 64)
            x[:, first:end] = (0.5 * torch.randn(self.kv, 1, 64, generator=g) + torch.randn(self.kv, end - first, 64, generator=g)).to(p.dtype)

    def seen(self, i):
        """(page, row) of the positions that token i sees."""
        k, v = self.group[i], self.lens[i]
        out = [(int(self.prefix[k, p // self.ps]), p % self.ps) for p in range(min(v, self.shared[k]))]
        if self.has_table:
            out += [(int(self.table[i, p // self.ps]), p % self.ps) for p in range(self.shared[k], v)]
        return [x for x in out if 0 <= x[0] < self.pages]

    def run(self, ctx, *, scale=0.125, ldq=None, ldo=None, max_shared=None, max_own=None, n=None, starts=None, shared=None, lens=None, graph=None):
        L, td, w = lib(), TDT[self.dtype], self.heads * 64
        n = n or self.n
        ldq, ldo = ldq or w, ldo or w
        q = torch.full((n, ldq), float("nan"), dtype=td)
        q[:self.n, :w] = self.q
        d = dict(q=q, k=self.k, v=self.v, prefix=self.prefix, starts=ints(self.starts if starts is None else starts),
                 shared=ints(self.shared if shared is None else shared), lens=ints(self.lens if lens is None else lens),
                 table=torch.cat([self.table, self.table.new_full((n - self.n, self.table.shape[1]), -1)]))
        if lens is None:
            d["lens"] = torch.cat([d["lens"], d["lens"].new_zeros(n - self.n)])
        d = {k: t.cuda() for k, t in d.items()}
        out = torch.full((n + 1, ldo), float("nan"), dtype=td, device="cuda")
        cache = L.KvCache(L.DTYPES[self.dtype], ptr(d["k"]), ptr(d["v"]), self.pages, self.ps, self.kv, self.stride)
        max_shared = max(self.shared + [0]) if max_shared is None else max_shared
        if max_own is None:
            max_own = max([v - self.shared[k] for v, k in zip(self.lens, self.group)] + [0]) if self.has_table else 0
        size = L.prefix_attention_workspace(cache, n, self.heads, len(self.members), max_shared, max_own)
        ws = torch.full((size + 64,), 255, dtype=torch.uint8, device="cuda")   # NaN wherever it is read unwritten
        torch.cuda.synchronize()
        ctx.kernel_prefix_attention(cache, ptr(d["q"]), ldq, n, self.heads, ptr(d["starts"]), len(self.members), ptr(d["prefix"]), self.prefix_width,
                                    ptr(d["shared"]), max_shared, ptr(d["table"]) if self.has_table else 0, self.width,
                                    ptr(d["lens"]) if self.has_lens else 0, max_own, scale, ptr(out), ldo, ptr(ws), size)
        ctx.synchronize()
        out = out.cpu()
        assert torch.isnan(out[n]).all() and torch.isnan(out[:, w:]).all() and (ws[size:] == 255).all()
        return out[:n, :w]

    def ref(self, i, scale=0.125, at=None):
        """(out [kv, G, 64], tolerance) of token i."""
        G = self.heads // self.kv
        at = self.seen(i) if at is None else at
        if not at:
            return torch.zeros(self.kv, G, 64, dtype=torch.float64), torch.zeros(self.kv, G, 64, dtype=torch.float64)
        page, row = (torch.tensor(x) for x in zip(*at))
        body = [p[:, :self.kv * self.ps * 64].view(self.pages, self.kv, self.ps, 64)[page, :, row].double().transpose(0, 1) for p in (self.k, self.v)]
        q = self.q[i].double().view(self.kv, G, 64)
        w = torch.softmax(q @ body[0].transpose(1, 2) * scale, -1)
        ref, A = w @ body[1], w @ body[1].abs()
        e = 70 * U * abs(scale) * (q.abs() @ body[0].abs().transpose(1, 2)).amax(-1, keepdim=True)
        h = torch.finfo(TDT[self.dtype]).eps / 2
        tol = h * ref.abs() + ((0 if self.dtype == "f32" else h) + 2 * e + (len(at) + 8) * U) * A
        if self.dtype == "f16":
            tol = tol + len(at) * 2.0 ** -37 * body[1].abs().max() + 2.0 ** -25
        return ref, tol

    def check(self, out, scale=0.125, rows=None):
        worst = 0.0
        for i in range(self.n) if rows is None else rows:
            ref, tol = self.ref(i, scale)
            d = (out[i].double().view(ref.shape) - ref).abs()
            assert (d <= tol).all(), (i, float((d / tol.clamp(min=1e-300)).max()))
            worst = max(worst, float((d / tol.clamp(min=1e-300)).max()))
        report("prefix.err", of_tolerance=f"{worst:.3f}")


# (tokens of the groups, shared positions, own positions as a function of the token, heads, key heads, page size)
FORKS = [
    ([1], [1], lambda i: 0, 1, 1, 8), ([1], [0], lambda i: 1, 1, 1, 8), ([2, 1], [0, 5], lambda i: i, 2, 1, 8), ([3, 3], [188, 40], lambda i: 7 * i % 20, 6, 6, 8),
    ([5, 0, 4], [31, 100, 33], lambda i: i % 3, 4, 2, 16), ([16], [64], lambda i: 0, 12, 12, 16), ([17, 1], [65, 63], lambda i: 33 * i % 70, 8, 1, 32),
    ([7, 9, 40], [1037, 0, 300], lambda i: 19 * i % 400, 8, 2, 64), ([33], [2000], lambda i: i, 20, 4, 256), ([3], [6223], lambda i: 1000 * i, 6, 3, 16),
    ([64], [1037], lambda i: 5 * i, 12, 12, 16), ([2, 60, 1, 1], [5000, 700, 0, 1], lambda i: i % 2 * 40, 32, 8, 64), ([1] * 40, [50 + 3 * i for i in range(40)], lambda i: i, 6, 2, 8),
    ([3] * 300, [8 * (i % 5) for i in range(300)], lambda i: i % 4, 2, 1, 8), ([2], [13000], lambda i: 9000 * i, 17, 1, 128), ([130], [520], lambda i: 0, 3, 1, 32),
    ([200], [777], lambda i: i % 9, 2, 2, 8),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("members,shared,own,heads,kv,ps", FORKS)
def test_forks(ctx, dtype, members, shared, own, heads, kv, ps):
    report("prefix", dtype=dtype, members=members[:4], shared=shared[:4], heads=heads, kv=kv, ps=ps)
    s = Shared(dtype, members, shared, [own(i) for i in range(sum(members))], heads, kv, ps, gap=64)
    s.check(s.run(ctx))


TOKENS = [([1], [1], 1, 1, 8), ([37], [500], 6, 6, 16), ([300, 1, 70], [1037, 0, 90], 12, 12, 16), ([129], [2074], 8, 2, 64), ([257], [400], 4, 1, 8), ([513], [640], 2, 2, 256),
          ([64], [9000], 20, 4, 32), ([1037], [2075], 6, 6, 16)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("members,shared,own,heads,kv", [
    ([90, 0, 91] * 35 + [0], [40 + 7 * i % 300 for i in range(106)], lambda i: i % 5 * 9, 1, 1), ([1, 70, 450], [0, 1500, 2000], lambda i: i % 40, 12, 2),
    ([300] * 3, [3000, 700, 5], lambda i: 0, 7, 1),
])
def test_many_tokens_and_heads(ctx, dtype, members, shared, own, heads, kv):
    """Parts of several groups' columns in a wave of the join."""
    n = sum(members)
    report("prefix.many", dtype=dtype, members=members[:4], heads=heads, kv=kv)
    s = Shared(dtype, members, shared, [own(i) for i in range(n)], heads, kv, 16)
    out = s.run(ctx)
    ends = np.cumsum(members)
    s.check(out, rows=sorted({i for e in [0, *ends.tolist()] for i in (e - 1, e, e + 1) if 0 <= i < n} | set(range(0, n, 97))))
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("members,shared,heads,kv,ps", TOKENS)
def test_tokens_of_requests(ctx, dtype, causal, members, shared, heads, kv, ps):
    report("prefix.tokens", dtype=dtype, causal=causal, members=members, shared=shared, heads=heads, kv=kv, ps=ps)
    sees = [max(0, shared[k] - m + 1 + t) for k, m in enumerate(members) for t in range(m)] if causal else None
    s = Shared(dtype, members, shared, None, heads, kv, ps, sees=sees, gap=64)
    rows = list(range(s.n)) if s.n < 200 else sorted({0, 1, s.n - 1, *range(0, s.n, 17), *range(120, 140)})
    out = s.run(ctx)
    s.check(out, rows=rows)
    assert not torch.isnan(out.float()).any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_lengths_in_no_order(ctx, dtype):
    """Tokens of a group that see any part of the prefix, nothing among them."""
    sees = [0, 500, 3, 1, 64, 65, 0, 31, 32, 33, 400, 499, 8, 7] * 20
    s = Shared(dtype, [280], [500], None, 2, 1, 16, sees=sees)
    s.check(s.run(ctx))
    s = Shared(dtype, [280], [500], [max(0, v - 500) for v in [2 * x for x in sees]], 2, 1, 16, sees=[2 * x for x in sees])
    s.check(s.run(ctx))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_scale_and_rows_behind_the_last_group(ctx, dtype):
    s = Shared(dtype, [5, 6], [300, 45], [i for i in range(11)], 6, 2, 16, behind=90)
    s.check(s.run(ctx, scale=-0.3, ldq=400, ldo=448, max_shared=1500, max_own=1000), scale=-0.3)
    s.check(s.run(ctx, scale=0.0, max_shared=2 ** 31 - 1, max_own=2 ** 31 - 1), scale=0.0)
    out = s.run(ctx, n=20)
    s.check(out[:11])
    assert torch.isnan(out[11:].float()).all()
    out = s.run(ctx, starts=[3, 5, 9])     # tokens before the first group and behind the last stay
    assert torch.isnan(out[:3].float()).all() and torch.isnan(out[9:].float()).all() and not torch.isnan(out[3:5].float()).any()
    for starts in ([5, 3, 11], [0, 2 ** 31 - 1, 0], [11, 0, 11]):
        s.run(ctx, starts=starts)          # descending: no fault
    out = s.run(ctx, starts=[-5, 5, 2 ** 31 - 1])   # cut to the tokens there are
    s.check(out)


@pytest.mark.parametrize("dtype", DTYPES)
def test_lengths_past_the_rows_or_the_bounds_are_cut(ctx, dtype):
    s = Shared(dtype, [4], [100], [30, 0, 7, 20], 4, 2, 16)
    cut = Shared(dtype, [4], [100], [30, 0, 7, 20], 4, 2, 16)
    out = s.run(ctx, max_own=5)
    cut.lens = [105, 100, 105, 105]
    cut.check(out)
    out = s.run(ctx, lens=[-3, 50, 107, -2 ** 31])
    cut.lens = [0, 50, 107, 0]
    cut.check(out)
    t = Shared(dtype, [4], [100], None, 4, 2, 16)
    out = t.run(ctx, max_shared=64)
    t.lens = [64] * 4
    t.check(out)
    assert (t.run(ctx, max_shared=0) == 0).all() and (t.run(ctx, shared=[-5]) == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ps", [8, 16, 32, 64, 128])
@pytest.mark.parametrize("members", [3, 150])
def test_pages_that_are_not_there(ctx, dtype, ps, members):
    s = Shared(dtype, [members], [10 * ps - 3], [i % 40 for i in range(members)], 2, 1, ps)
    for j, bad in ((0, -1), (3, s.pages), (7, -(2 ** 31)), (9, 2 ** 31 - 1)):
        s.prefix[0, j] = bad
    s.table[::2, 10] = -1
    s.table[1, 9] = s.pages + 5
    s.check(s.run(ctx))
    s.prefix[:], s.table[:] = -1, s.pages
    assert (s.run(ctx) == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("members", [4, 200])
def test_large_scores(ctx, dtype, members):
    """Scores of hundreds to thousands, of both signs: only differences count."""
    s = Shared(dtype, [members], [700], [i % 50 for i in range(members)], 2, 1, 16)
    s.q *= 60
    rows = list(range(0, members, max(1, members // 40)))
    s.check(s.run(ctx), rows=rows)
    s.check(s.run(ctx, scale=16.0), scale=16.0, rows=rows)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("members", [5, 150])
def test_infinities_and_nan_count_where_they_are_seen(ctx, dtype, members):
    """Values of positions that some tokens see and others do not; a NaN query. What they do not reach stays within the bound of
    the file's head, whose sum A is over values that nearly cancel: two results within it differ by up to twice the bound, which
    a step of the output's type can be far below."""
    sees = [(53 * i) % 301 for i in range(members)]
    s = Shared(dtype, [members], [300], None, 4, 2, 16, sees=sees)
    clean, refs = s.run(ctx), [s.ref(i) for i in range(members)]
    marks = {17: float("inf"), 100: float("nan"), 160: -float("inf"), 161: float("inf"), 299: float("nan")}
    for p, x in marks.items():
        s.v[int(s.prefix[0, p // 16])].view(s.kv, 16, 64)[1, p % 16, 3 * (p % 5)] = x
    out = s.run(ctx).view(members, 4, 64)
    clean = clean.view(members, 4, 64)
    assert torch.equal(out[:, :2], clean[:, :2])   # the other key head
    for i, v in enumerate(sees):
        for c in range(64):
            x = [m for p, m in marks.items() if p < v and 3 * (p % 5) == c]
            got = out[i, 2:, c].float()
            if not x:
                ref, tol = (r[1, :, c] for r in refs[i])
                assert ((got.double() - ref).abs() <= tol).all(), (i, c)
            elif any(m != m for m in x) or (float("inf") in x and -float("inf") in x):
                assert torch.isnan(got).all(), (i, c)
            else:
                assert (got == x[0]).all(), (i, c)
    # keys: NaN where a token sees one, nobody else
    t = Shared(dtype, [members], [300], None, 4, 2, 16, sees=sees)
    refs = [t.ref(i) for i in range(members)]
    t.k[int(t.prefix[0, 200 // 16])].view(t.kv, 16, 64)[0, 200 % 16, 5] = float("nan")
    t.q[2, 2 * 64 + 7] = float("nan")
    out = t.run(ctx).view(members, 4, 64)
    for i, v in enumerate(sees):
        for h in range(4):
            if v and (h < 2 and v > 200 or (i, h) == (2, 2)):
                assert torch.isnan(out[i, h]).all(), (i, h)
            else:
                ref, tol = (r.view(4, 64)[h] for r in refs[i])
                assert ((out[i, h].double() - ref).abs() <= tol).all(), (i, h)


def test_offsets_past_32_bits(ctx):
    """Pages 4 GiB apart, of the prefix and of the token's own."""
    L, stride, ps = lib(), 2 ** 31, 8
    k, v = (torch.zeros(2 * stride + 512, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    g = torch.Generator().manual_seed(4)
    rows = torch.randn(2, 3, 8, 64, generator=g).to(torch.bfloat16)
    for x, r in ((k, rows[0]), (v, rows[1])):
        for p in range(3):
            x[p * stride:p * stride + 512] = r[p].reshape(-1).cuda()
    q = torch.randn(2, 64, generator=g).to(torch.bfloat16)
    d = [t.cuda() for t in (q, ints([0, 2]), ints([[2, 1]]), ints([16]), ints([[0, 0, 0], [0, 0, 0]]), ints([24, 20]))]
    out = torch.empty(2, 64, dtype=torch.bfloat16, device="cuda")
    cache = L.KvCache(L.BF16, ptr(k), ptr(v), 3, ps, 1, stride)
    size = L.prefix_attention_workspace(cache, 2, 1, 1, 16, 8)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    ctx.kernel_prefix_attention(cache, ptr(d[0]), 64, 2, 1, ptr(d[1]), 1, ptr(d[2]), 2, ptr(d[3]), 16, ptr(d[4]), 3, ptr(d[5]), 8, 0.125, ptr(out), 64,
                                ptr(ws), size)
    ctx.synchronize()
    for i, m in enumerate((24, 20)):
        K, V = (r[[2, 1, 0]].reshape(24, 64)[:m].double() for r in rows)
        ref = torch.softmax(q[i].double() @ K.T / 8, -1) @ V
        assert ((out[i].cpu().double() - ref).abs() <= 2 ** -8 * (ref.abs() + V.abs().max())).all()


@pytest.mark.parametrize("starts", [[0, 5, 3, 4], [0, 5, 3, 8], [8, 0, 0, 0], [0, 8, 7, 7], [3, 2, 5, 8]])
@pytest.mark.parametrize("shared,own", [(40, None), (40, 9), (6000, 9)])
def test_starts_that_descend_write_nothing(ctx, starts, shared, own):
    """Also where the groups' tokens are no more than there are: one of them would be in two groups."""
    s = Shared("bf16", [3, 3, 2], [shared] * 3, own and [own] * 8, 6, 2, 16)
    report("prefix.descends", starts=starts, shared=shared, own=own)
    assert torch.isnan(s.run(ctx, starts=starts)).all()
    s.check(s.run(ctx))


def test_calls_without_tokens_or_groups(ctx):
    L = lib()
    cache = L.KvCache(L.BF16, 1 << 20, 1 << 30, 4, 16, 2)
    ctx.kernel_prefix_attention(cache, 0, 256, 0, 4, 0, 1, 0, 5, 0, 80, 0, 0, 0, 0, 0.125, 0, 256, 0, 0)
    ctx.kernel_prefix_attention(cache, 0, 256, 7, 4, 0, 0, 0, 5, 0, 80, 0, 0, 0, 0, 0.125, 0, 256, 0, 0)

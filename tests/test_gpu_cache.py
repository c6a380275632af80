"""The paged cache's operators through the kernel entry points, against plain restatements in 64 bits on the CPU
of the same rounded operands.

Tolerances (u = 2^-24, h = half a rounding step of the storage type relative to the value: bf16 2^-8, f16 2^-11,
fp32 2^-24) come from counting roundings:
  norms with rotation: a value ends at h |value| from its rounding. Before it, in fp32: at most 11 roundings of the
    sums over 64 channels (8 in a lane, 3 across), the same again for the variance, and less than 20 for difference,
    root, scale, shift, and the two products and the sum of the rotation with its factors' own: 64 u of the largest
    magnitude in the head's row before and after the norm.
  attention: |out - ref| <= h |ref| + (h_w + 2 e + (L + 8) u) A, with A = sum w |v| / sum w: h_w = h for the 16-bit
    types, whose weights are rounded to the type (0 for fp32), e the error of a score, 70 u scale sum |q_c k_c| at most
    (a weight 2^s moves by a factor of e^(2 e) when its score and the largest one move by e), L u for sums of L terms. In f16
    a weight below the smallest normal value is off by half a step of the subnormals, 2^-25; the weights are kept up to
    2^12, so that this is 2^-37 of the largest weight: L 2^-37 max |v| more.
"""
import ctypes

import numpy as np
import pytest

from conftest import report

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

U = 2.0 ** -24
TDT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
DTYPES = ["bf16", "f16", "f32"]


def half(dtype):
    return torch.finfo(TDT[dtype]).eps / 2


def lib():
    import splathip
    return splathip


def ptr(t):
    return 0 if t is None else t.data_ptr()


def ints(v):
    return torch.tensor(v, dtype=torch.int32)


# --- block tables ---------------------------------------------------------------------------------

def tables_ref(past, add, ps, pool, used, table, cap):
    """The operator in plain Python, one request at a time: all or nothing."""
    n, width = table.shape
    need = sum(-(-(p + a) // ps) - -(-p // ps) for p, a in zip(past, add))
    status = 0
    if any(p < 0 or a < 0 or p + a > width * ps for p, a in zip(past, add)) or not 0 <= used <= len(pool):
        status = 1
    elif need > len(pool) - used:
        status = 2
    elif sum(add) > cap:
        status = 3
    table = table.copy()
    slots, pos = np.full(cap, -1, np.int64), np.zeros(cap, np.int64)
    if status:
        return dict(table=table, lens=past, starts=[0] * (n + 1), slots=slots, positions=pos, used=used, status=status)
    t, starts = 0, [0]
    for i, (p, a) in enumerate(zip(past, add)):
        for j in range(-(-p // ps), -(-(p + a) // ps)):
            table[i, j] = pool[used]
            used += 1
        for x in range(p, p + a):
            page = int(table[i, x // ps])
            slots[t] = page * ps + x % ps if page >= 0 else -1
            pos[t] = x
            t += 1
        starts.append(t)
    return dict(table=table, lens=[p + a for p, a in zip(past, add)], starts=starts, slots=slots, positions=pos, used=used,
                status=0)


def run_tables(ctx, past, add, ps, pool, used, table, cap, in_place=False, positions=True):
    d = {k: ints(v).cuda() for k, v in (("past", past), ("add", add), ("pool", pool), ("used", [used]))}
    n, width = table.shape
    d["table"] = torch.from_numpy(table.astype(np.int32)).cuda()
    d["lens"] = d["past"] if in_place else torch.full((n,), -7, dtype=torch.int32, device="cuda")
    d["used_out"] = d["used"] if in_place else torch.full((1,), -7, dtype=torch.int32, device="cuda")
    for k, m in (("starts", n + 1), ("slots", cap), ("positions", cap), ("status", 1)):
        d[k] = torch.full((m,), -7, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    ctx.kernel_block_tables(n, ptr(d["past"]), ptr(d["add"]), ps, ptr(d["pool"]), len(pool), ptr(d["used"]), ptr(d["table"]),
                            width, ptr(d["lens"]), ptr(d["starts"]), ptr(d["slots"]), ptr(d["positions"]) if positions else 0,
                            cap, ptr(d["used_out"]), ptr(d["status"]))
    ctx.synchronize()
    return {k: v.cpu().numpy() for k, v in d.items()}


def check_tables(ctx, past, add, ps, pool, used, table, cap, status=0, **kw):
    ref = tables_ref(past, add, ps, pool, used, table, cap)
    assert ref["status"] == status
    got = run_tables(ctx, past, add, ps, pool, used, table, cap, **kw)
    assert got["status"][0] == status
    assert np.array_equal(got["table"], ref["table"])
    assert np.array_equal(got["lens"], ref["lens"])
    assert np.array_equal(got["starts"], ref["starts"])
    assert np.array_equal(got["slots"], ref["slots"])
    if kw.get("positions", True):
        assert np.array_equal(got["positions"], ref["positions"])
    else:
        assert (got["positions"] == -7).all()
    assert got["used_out"][0] == ref["used"]


def requests(rng, n, most_past, most_add, ps, spare=4):
    past = rng.integers(0, most_past + 1, n).tolist()
    add = rng.integers(0, most_add + 1, n).tolist()
    width = max(1, max(-(-(p + a) // ps) for p, a in zip(past, add))) + 2
    have = sum(-(-p // ps) for p in past)
    ids = rng.permutation(have + sum(-(-a // ps) + 1 for a in add) + spare)
    table = np.full((n, width), -1, np.int64)
    at = 0
    for i, p in enumerate(past):
        m = -(-p // ps)
        table[i, :m] = ids[at:at + m]
        at += m
    return past, add, table, ids[at:].tolist()


@pytest.mark.parametrize("n,most_past,most_add,ps", [
    (1, 0, 1, 8), (1, 40, 1, 16), (3, 100, 40, 8), (64, 3000, 1, 16), (257, 50, 3, 32), (40, 500, 900, 64),
    (1023, 30, 2, 8), (1024, 30, 2, 8), (1025, 30, 5, 8), (5000, 100, 4, 16), (7, 5, 20000, 256),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_block_tables(ctx, n, most_past, most_add, ps, in_place):
    report("tables", n=n, past=most_past, add=most_add, ps=ps, in_place=in_place)
    rng = np.random.default_rng(n * 7 + ps)
    past, add, table, pool = requests(rng, n, most_past, most_add, ps)
    used = int(rng.integers(0, 4))
    pool = [0] * used + pool
    for cap in {sum(add), sum(add) + 100}:
        check_tables(ctx, past, add, ps, pool, used, table, cap, in_place=in_place)


def test_block_tables_without_requests_tokens_or_positions(ctx):
    check_tables(ctx, [], [], 16, [1, 2], 1, np.zeros((0, 3), np.int64), 5)
    check_tables(ctx, [5, 0], [0, 0], 16, [1, 2], 1, np.array([[4, -1], [-1, -1]]), 0)
    check_tables(ctx, [5, 0], [20, 3], 16, [1, 2, 9], 1, np.array([[4, -1], [-1, -1]]), 23, positions=False)


@pytest.mark.parametrize("cap", [40, 5000])   # one launch and two
def test_block_tables_take_all_or_nothing(ctx, cap):
    past, add, table = [5, 16, 0], [20, 1, 3], np.array([[4, -1, 5], [3, -1, -1], [-1, -1, -1]])
    check_tables(ctx, past, add, 16, [9, 8, 7], 0, table, cap)
    check_tables(ctx, past, add, 16, [9, 8, 7], 1, table, cap, status=2)
    check_tables(ctx, past, add, 16, [9, 8, 7], 4, table, cap, status=1)
    check_tables(ctx, past, add, 16, [9, 8, 7], -1, table, cap, status=1)
    check_tables(ctx, [5, -1, 0], add, 16, [9, 8, 7], 0, table, cap, status=1)
    check_tables(ctx, past, [20, -1, 3], 16, [9, 8, 7], 0, table, cap, status=1)
    check_tables(ctx, past, [44, 1, 3], 16, [9, 8, 7], 0, table, cap, status=1)
    check_tables(ctx, [2 ** 31 - 1, 16, 0], [2 ** 31 - 1, 1, 3], 16, [9, 8, 7], 0, table, cap, status=1)
    check_tables(ctx, past, [20, 1, 3], 16, [9, 8, 7], 0, table, 23, status=3)
    check_tables(ctx, past, [20, 1, 3], 16, [9, 8, 7], 0, table, 23, status=3, in_place=True)


def test_block_tables_bad_entries_give_no_slots(ctx):
    """A page below 0 in the table or the pool: its tokens get slot -1."""
    check_tables(ctx, [5, 16], [20, 1], 16, [-3, 8, 7], 0, np.array([[-1, -1], [3, -1]]), 21)


# --- norms with rotation --------------------------------------------------------------------------

def rope_ref(x, w, b, norm, rope, base, pos, eps):
    """x [T, H, 64] in 64 bits; the largest magnitude of each row before and after."""
    y = x
    if norm == "layer":
        y = (y - y.mean(-1, keepdim=True)) / torch.sqrt(y.var(-1, unbiased=False, keepdim=True) + eps)
    elif norm == "rms":
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
    if norm != "none":
        y = y * (w.double() if w is not None else 1) + (b.double() if b is not None else 0)
    if rope == "none":
        return y
    out = y.clone()
    spans = [(0, 32, pos if pos.ndim == 1 else None)] if rope == "line" else [(0, 16, pos[:, 0]), (32, 16, pos[:, 1])]
    for c0, h, p in spans:
        for c in range(h):
            a = p.double() * base ** (-c / h)
            cs, sn = torch.cos(a)[:, None], torch.sin(a)[:, None]
            lo, hi = y[:, :, c0 + c], y[:, :, c0 + c + h]
            out[:, :, c0 + c], out[:, :, c0 + c + h] = lo * cs - hi * sn, hi * cs + lo * sn
    return out


def rope_tol(x, ref, dtype):
    """See the top of the file; a row's scale is what the norm divides by times what comes out."""
    big = ref.abs().amax(-1, keepdim=True) * (1 + x.abs().amax(-1, keepdim=True) / x.std(-1, unbiased=False, keepdim=True).clamp(min=1e-3))
    big = torch.maximum(big, x.abs().amax(-1, keepdim=True))
    return half(dtype) * ref.abs() + 64 * U * big + (2.0 ** -25 if dtype == "f16" else 0.0)   # half a step of f16's subnormals


class Rope:
    def __init__(self, dtype, T, heads, kv, norm, rope, *, seed=1, base=100.0, ps=16, cache=True, pad=0, weights=True, bias=True,
                 far=False, eps=1e-5):
        g = torch.Generator().manual_seed(seed + T)
        self.__dict__.update(dtype=dtype, T=T, heads=heads, kv=kv, norm=norm, rope=rope, base=base, ps=ps, eps=eps, pad=pad, cache=cache)
        self.ld = (heads + 2 * kv) * 64 + pad
        self.qkv = (torch.randn(T, self.ld, generator=g) + 0.3 * torch.randn(self.ld, generator=g)).to(TDT[dtype])
        self.w = [1 + 0.2 * torch.randn(64, generator=g) if weights else None for _ in range(2)]
        self.b = [0.2 * torch.randn(64, generator=g) if bias else None for _ in range(2)]
        most = 2 ** 31 - 1 if far else 500
        shape = (T, 2) if rope == "grid" else (T,)
        self.pos = torch.randint(0, most, shape, generator=g, dtype=torch.int64).to(torch.int32)
        self.pages = -(-T // ps) + 2
        self.slots = torch.randperm(self.pages * ps, generator=g)[:T].to(torch.int32)

    def call(self, ctx, q, ldq, k, ldk, kc, vc, qkv=None, slots=None, stride=0):
        L = lib()
        d = {n: t.cuda() if t is not None else None for n, t in
             (("qw", self.w[0]), ("kw", self.w[1]), ("qb", self.b[0]), ("kb", self.b[1]), ("pos", self.pos),
              ("slots", self.slots if slots is None else slots))}
        qkv = self.qkv.cuda() if qkv is None else qkv
        code = L.DTYPES[self.dtype]
        cache = L.KvCache(code, ptr(kc), ptr(vc), self.pages, self.ps, self.kv, stride) if kc is not None else None
        torch.cuda.synchronize()
        ctx.kernel_qk_norm_rope(code, ptr(qkv), self.ld, self.T, self.heads, self.kv,
                                {"none": 0, "layer": 1, "rms": 2}[self.norm], ptr(d["qw"]), ptr(d["qb"]), ptr(d["kw"]), ptr(d["kb"]),
                                self.eps, {"none": 0, "line": 1, "grid": 2}[self.rope], self.base,
                                0 if self.rope == "none" else ptr(d["pos"]), ptr(q), ldq, ptr(k), ldk, cache,
                                ptr(d["slots"]) if cache is not None else 0)
        ctx.synchronize()

    def refs(self):
        x = self.qkv[:, :self.ld - self.pad].double().reshape(self.T, -1, 64)
        h, kv = self.heads, self.kv
        q = rope_ref(x[:, :h], self.w[0], self.b[0], self.norm, self.rope, self.base, self.pos, self.eps)
        k = rope_ref(x[:, h:h + kv], self.w[1], self.b[1], self.norm, self.rope, self.base, self.pos, self.eps)
        return (x[:, :h], q), (x[:, h:h + kv], k), x[:, h + kv:]

    def check(self, ctx):
        td, T, kv, ps = TDT[self.dtype], self.T, self.kv, self.ps
        q = torch.full((T, self.heads * 64 + 8), float("nan"), dtype=td, device="cuda")
        k = torch.full((T, kv * 64 + 16), float("nan"), dtype=td, device="cuda")
        stride = kv * ps * 64 + 64
        kc = torch.full((self.pages, stride), 7.0, dtype=td, device="cuda") if self.cache else None
        vc = torch.full((self.pages, stride), 7.0, dtype=td, device="cuda") if self.cache else None
        self.call(ctx, q, self.heads * 64 + 8, k, kv * 64 + 16, kc, vc, stride=stride)
        (xq, rq), (xk, rk), rv = self.refs()
        q, k = q.cpu(), k.cpu()
        assert torch.isnan(q[:, self.heads * 64:]).all() and torch.isnan(k[:, kv * 64:]).all()
        err = []
        for got, x, ref in ((q[:, :self.heads * 64], xq, rq), (k[:, :kv * 64], xk, rk)):
            d = (got.double().reshape(ref.shape) - ref).abs()
            tol = rope_tol(x, ref, self.dtype)
            err.append(float((d / tol).max()))
            assert (d <= tol).all(), float((d / tol).max())
        report("rope.err", of_tolerance=f"{max(err):.2f}")
        if not self.cache:
            return
        want = torch.full((self.pages, stride), 7.0, dtype=td)
        body = want[:, :kv * ps * 64].reshape(self.pages, kv, ps, 64)
        s = self.slots.long()
        for pool, rows in ((kc, k[:, :kv * 64].reshape(T, kv, 64)), (vc, rv.to(td))):
            w = body.clone()
            w[s // ps, :, s % ps] = rows
            pool = pool.cpu()
            assert torch.equal(pool[:, :kv * ps * 64].reshape(w.shape), w)
            assert (pool[:, kv * ps * 64:] == 7).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norm", ["none", "layer", "rms"])
@pytest.mark.parametrize("rope", ["none", "line", "grid"])
def test_qk_norm_rope(ctx, dtype, norm, rope):
    for T, heads, kv, kw in ((1, 1, 1, {}), (3, 6, 6, {"ps": 8}), (67, 12, 12, {"bias": False, "pad": 64}),
                             (130, 20, 4, {"base": 10000.0, "ps": 64}), (9, 3, 1, {"weights": False, "cache": False})):
        report("rope", dtype=dtype, norm=norm, rope=rope, T=T, heads=heads, kv=kv, **kw)
        Rope(dtype, T, heads, kv, norm, rope, **kw).check(ctx)


@pytest.mark.parametrize("dtype", DTYPES)
def test_qk_norm_rope_of_a_scene(ctx, dtype):
    """Many tokens: as many waves as fill the chip several times over."""
    Rope(dtype, 6221, 12, 12, "layer", "grid", ps=32).check(ctx)


@pytest.mark.parametrize("rope", ["line", "grid"])
def test_qk_norm_rope_far_positions(ctx, rope):
    """Positions up to 2^31 - 1: the angle's error is half an ulp of the position's turns in 64 bits, below 2^-24."""
    Rope("f32", 40, 2, 2, "layer", rope, far=True, base=10000.0).check(ctx)


@pytest.mark.parametrize("dtype", DTYPES)
def test_qk_norm_rope_in_place(ctx, dtype):
    """q and k over qkv's own blocks give the same bits; the values and what lies behind them stay."""
    r = Rope(dtype, 41, 6, 2, "rms", "line", pad=64, cache=False)
    q = torch.empty(41, 384, dtype=TDT[dtype], device="cuda")
    k = torch.empty(41, 128, dtype=TDT[dtype], device="cuda")
    r.call(ctx, q, 384, k, 128, None, None)
    x = r.qkv.cuda()
    r.call(ctx, x, r.ld, x[:, 384:], r.ld, None, None, qkv=x)
    assert torch.equal(x[:, :384].cpu(), q.cpu()) and torch.equal(x[:, 384:512].cpu(), k.cpu())
    assert torch.equal(x[:, 512:].cpu(), r.qkv[:, 512:])


def test_qk_norm_rope_slots_outside_the_pool_store_nothing(ctx):
    r = Rope("bf16", 30, 4, 2, "layer", "grid", ps=8)
    slots = r.slots.clone()
    bad = [-1, -(2 ** 31), r.pages * 8, 2 ** 31 - 1]
    slots[[2, 11, 12, 29]] = ints(bad)
    td = torch.bfloat16
    pools = {}
    for name, s in (("all", r.slots), ("some", slots)):
        q = torch.empty(30, 256, dtype=td, device="cuda")
        pools[name] = [torch.full((r.pages, 2, 8, 64), 7.0, dtype=td, device="cuda") for _ in range(2)]
        r.call(ctx, q, 256, None, 0, *pools[name], slots=s)
    for a, b in zip(pools["all"], pools["some"]):
        a = a.cpu()
        s = r.slots.long()[[2, 11, 12, 29]]
        a[s // 8, :, s % 8] = 7
        assert torch.equal(a, b.cpu())


def test_qk_norm_rope_without_tokens(ctx):
    L = lib()
    ctx.kernel_qk_norm_rope(L.BF16, 0, 384, 0, 2, 2, L.NORM_LAYER, 0, 0, 0, 0, 1e-5, L.ROPE_GRID, 100.0, 0, 0, 128)


# --- caches ---------------------------------------------------------------------------------------

class Cache:
    """Pools with pages in random order, a table, and garbage (NaN, infinities) wherever no position lies."""

    def __init__(self, dtype, lens, kv, ps, *, seed=1, extra_width=2, gap=0, garbage=True, scale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.lens, self.kv, self.ps, self.n = dtype, list(lens), kv, ps, len(lens)
        td = TDT[dtype]
        used = [-(-v // ps) for v in lens]
        self.pages = sum(used) + 3
        self.width = max(used) + extra_width
        ids = torch.randperm(self.pages, generator=g)
        self.table = torch.full((self.n, self.width), -1, dtype=torch.int32)
        self.stride = kv * ps * 64 + gap
        self.k = torch.empty(self.pages, self.stride)
        self.v = torch.empty(self.pages, self.stride)
        bad = torch.tensor([float("nan"), float("inf"), -float("inf")])
        for p in (self.k, self.v):
            p[:] = bad[torch.randint(0, 3, p.shape, generator=g)] if garbage else 0.0
        at = 0
        for i, v in enumerate(lens):
            m = used[i]
            self.table[i, :m] = ids[at:at + m].to(torch.int32)
            at += m
            for j in range(m):
                rows = min(ps, v - j * ps)
                for p in (self.k, self.v):
                    x = p[self.table[i, j], :kv * ps * 64].view(kv, ps, 64)
                    x[:, :rows] = scale * torch.randn(kv, 1, 64, generator=g) * 0.5 + scale * torch.randn(kv, rows, 64, generator=g)
        self.k, self.v = self.k.to(td), self.v.to(td)

    def head(self, pool, i, h, positions):
        t = self.table[i].long()
        p = torch.as_tensor(positions).long()
        body = pool[:, :self.kv * self.ps * 64].view(self.pages, self.kv, self.ps, 64)
        return body[t[p // self.ps], h, p % self.ps].double()

    def device(self):
        self.dk, self.dv, self.dtable, self.dlens = self.k.cuda(), self.v.cuda(), self.table.cuda(), ints(self.lens).cuda()
        L = lib()
        torch.cuda.synchronize()
        return L.KvCache(L.DTYPES[self.dtype], ptr(self.dk), ptr(self.dv), self.pages, self.ps, self.kv, self.stride)


def attention_ref(q, k, v, scale):
    """q [G, 64], k, v [L, 64] in 64 bits: out [G, 64], and its tolerance without h |out| (see the top)."""
    s = (q @ k.T) * scale
    w = torch.softmax(s, -1)
    return w @ v, w @ v.abs(), 70 * U * abs(scale) * (q.abs() @ k.abs().T).amax(-1, keepdim=True)


def attention_check(got, q, ks, vs, scale, dtype):
    ref, A, e = attention_ref(q, ks, vs, scale)
    h = half(dtype)
    tol = h * ref.abs() + ((0 if dtype == "f32" else h) + 2 * e + (len(ks) + 8) * U) * A
    if dtype == "f16":   # the output's own subnormals too
        tol = tol + len(ks) * 2.0 ** -37 * vs.abs().max() + 2.0 ** -25
    d = (got - ref).abs()
    assert (d <= tol).all(), float((d / tol).max())
    return float((d / tol).max())


def run_paged(ctx, c, q, heads, *, max_len=None, scale=0.125, ldq=None, ldo=None, table=None, lens=None, fill=float("nan")):
    L = lib()
    cache = c.device()
    td = TDT[c.dtype]
    ldq, ldo = ldq or heads * 64, ldo or heads * 64
    dq = torch.full((c.n, ldq), float("nan"), dtype=td)
    dq[:, :heads * 64] = q
    dq = dq.cuda()
    out = torch.full((c.n + 1, ldo), fill, dtype=td, device="cuda")
    max_len = max(max(c.lens), 1) if max_len is None else max_len
    size = L.paged_attention_workspace(cache, c.n, heads, max_len)
    ws = torch.full((size + 64,), 255, dtype=torch.uint8, device="cuda")   # NaN wherever it is read unwritten
    dt, dl = (c.dtable if table is None else table.cuda()), (c.dlens if lens is None else lens.cuda())
    torch.cuda.synchronize()
    ctx.kernel_paged_attention(cache, ptr(dq), ldq, c.n, heads, ptr(dt), c.width, ptr(dl), max_len, scale, ptr(out), ldo,
                               ptr(ws), size)
    ctx.synchronize()
    out = out.cpu()
    assert torch.isnan(out[c.n]).all() and torch.isnan(out[:, heads * 64:]).all()
    assert (ws[size:] == 255).all()
    return out[:c.n, :heads * 64]


def queries(c, heads, seed=3, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (scale * torch.randn(c.n, heads * 64, generator=g)).to(TDT[c.dtype])


def check_paged(ctx, c, heads, q, out, scale=0.125, positions=None):
    worst, G = 0.0, heads // c.kv
    for i, v in enumerate(c.lens):
        at = list(range(v)) if positions is None else positions[i]
        for h in range(c.kv):
            got = out[i].view(c.kv, G, 64)[h].double()
            if not len(at):
                assert (got == 0).all()
                continue
            worst = max(worst, attention_check(got, q[i].view(c.kv, G, 64)[h].double(), c.head(c.k, i, h, at),
                                               c.head(c.v, i, h, at), scale, c.dtype))
    report("paged.err", of_tolerance=f"{worst:.3f}")


PAGED = [
    # (lens, heads, kv_heads, page_size)
    ([1], 1, 1, 8), ([1, 0, 2], 2, 1, 8), ([7, 8, 9], 6, 6, 8), ([31, 32, 33], 4, 2, 16), ([63, 64, 65, 0], 12, 12, 16),
    ([127, 128, 129], 8, 1, 32), ([255, 256, 257], 16, 1, 64), ([500, 1, 300], 17, 1, 256), ([600, 0, 1037], 40, 2, 64),
    ([973], 6, 6, 128), ([2000, 3, 1111], 20, 4, 16), ([6223], 12, 12, 16), ([4096, 4097], 8, 2, 8), ([10000, 17], 6, 3, 64),
    ([24889], 1, 1, 16), ([5] * 40, 3, 3, 8), ([700] * 9, 33, 1, 32), ([13000, 5000], 24, 8, 256),
    # parts of a block joined, sequences that end inside one, and more sequences than a block sums up
    ([9000, 1, 0, 7000, 40], 16, 1, 16), ([3000, 3001, 2999, 64, 0, 1], 2, 1, 8), ([1500] + [3, 0, 40] * 400, 2, 1, 8),
    ([3, 0, 40] * 400 + [9000, 0], 2, 1, 8), ([5, 0, 4500] + [0, 1] * 520, 18, 1, 32),   # the same, cut into parts
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,heads,kv,ps", PAGED)
def test_paged_attention(ctx, dtype, lens, heads, kv, ps):
    report("paged", dtype=dtype, lens=lens[:4], n=len(lens), heads=heads, kv=kv, ps=ps)
    c = Cache(dtype, lens, kv, ps, gap=64)
    q = queries(c, heads)
    check_paged(ctx, c, heads, q, run_paged(ctx, c, q, heads))


@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_attention_strides_scale_and_generous_max_len(ctx, dtype):
    c = Cache(dtype, [300, 0, 45], 2, 16, extra_width=90)
    q = queries(c, 6)
    a = run_paged(ctx, c, q, 6, scale=-0.3, ldq=400, ldo=448, max_len=1500)
    check_paged(ctx, c, 6, q, a, scale=-0.3)
    check_paged(ctx, c, 6, q, run_paged(ctx, c, q, 6, scale=0.0, max_len=2 ** 31 - 1), scale=0.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_attention_lengths_past_the_row_or_max_len_are_cut(ctx, dtype):
    c = Cache(dtype, [200, 90, 64], 2, 16, extra_width=0)
    q = queries(c, 4)
    lens = ints([2 ** 31 - 1, -4, 64])
    out = run_paged(ctx, c, q, 4, max_len=1000, lens=lens)   # the row holds 13 pages: 208 positions, 8 of them garbage
    assert torch.isnan(out[0].float()).any() and (out[1] == 0).all()
    out = run_paged(ctx, c, q, 4, max_len=77, lens=lens)
    check_paged(ctx, c, 4, q, out, positions=[list(range(77)), [], list(range(64))])
    assert (run_paged(ctx, c, q, 4, max_len=0) == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ps", [8, 16, 32, 64, 128])
def test_paged_attention_leaves_out_pages_that_are_not_there(ctx, dtype, ps):
    """Entries outside the pool hold no keys; a row of nothing else gives zeros."""
    lens = [10 * ps - 3, 3 * ps, 2 * ps + 1, 40 * ps]
    c = Cache(dtype, lens, 2, ps)
    table = c.table.clone()
    gone = {0: [0, 4, 9], 1: [0, 1, 2], 2: [2], 3: list(range(3, 30))}
    for i, js in gone.items():
        for x, j in enumerate(js):
            table[i, j] = [-1, c.pages, 2 ** 31 - 1, -(2 ** 31)][x % 4]
    q = queries(c, 6)
    out = run_paged(ctx, c, q, 6, table=table)
    check_paged(ctx, c, 6, q, out, positions=[[p for p in range(v) if p // ps not in gone[i]] for i, v in enumerate(lens)])


@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_attention_large_scores(ctx, dtype):
    """Scores of some thousands, one key far above the others, and all keys alike."""
    c = Cache(dtype, [700, 1500, 64], 2, 16, scale=20.0)
    q = queries(c, 4, scale=20.0)
    check_paged(ctx, c, 4, q, run_paged(ctx, c, q, 4))


@pytest.mark.parametrize("dtype", DTYPES)
def test_paged_attention_infinities_and_nan(ctx, dtype):
    """In a key or value that is there they go where the formula takes them, and nowhere else: heads of their
    own, the other heads keep their bits."""
    c = Cache(dtype, [400, 700], 4, 16)
    q = queries(c, 4)
    clean = run_paged(ctx, c, q, 4)
    inf, nan = float("inf"), float("nan")
    body = lambda p: p[:, :4 * 16 * 64].view(c.pages, 4, 16, 64)  # noqa: E731
    page = int(c.table[0, 3])
    q[0, 5] = 0.75                       # channel 5 of head 0: a key of -inf there has weight 0
    body(c.k)[page, 0, 2, 5] = -inf
    body(c.k)[page, 1, 2, 5] = nan       # head 1: a score of NaN
    body(c.v)[page, 2, 2, 5] = inf       # head 2: an infinite value
    out = run_paged(ctx, c, q, 4).float()
    assert torch.equal(out[1], clean[1].float()) and torch.equal(out[0, 192:], clean[0, 192:].float())
    keep = [p for p in range(400) if p != 50]
    attention_check(out[0, :64].double()[None], q[0, :64].double()[None], c.head(c.k, 0, 0, keep), c.head(c.v, 0, 0, keep), 0.125, dtype)
    assert torch.isnan(out[0, 64:128]).all()
    assert out[0, 128 + 5] == inf and torch.isfinite(out[0, 128:192]).sum() == 63
    body(c.k)[int(c.table[0, 0]), 3] = -inf   # every key of a page and more: all scores NaN or -inf
    q[0, 192:] = q[0, 192:].abs() + 0.5
    for j in range(25):
        body(c.k)[int(c.table[0, j]), 3] = -inf
    out = run_paged(ctx, c, q, 4).float()
    assert torch.isnan(out[0, 192:]).all() and torch.equal(out[1], clean[1].float())


def test_paged_attention_offsets_past_32_bits(ctx):
    """Pages 2^27 elements apart: 34 of them reach past 2^32 elements (8.6 GB a pool)."""
    L = lib()
    ps, kv, heads, stride, pages = 16, 2, 4, 1 << 27, 34
    pool = torch.empty(pages * stride, dtype=torch.bfloat16, device="cuda")
    c = Cache("bf16", [16 * 28, 16 * 2 + 3], kv, ps, seed=4)
    assert c.pages == pages
    far = [torch.as_strided(pool, (pages, kv * ps * 64), (stride, 1), off) for off in (0, 2048)]
    for dst, src in zip(far, (c.k, c.v)):
        dst.copy_(src.cuda())
    table = c.table.cuda()
    q = queries(c, heads)
    dq, out, lens = q.cuda(), torch.empty(2, heads * 64, dtype=torch.bfloat16, device="cuda"), ints(c.lens).cuda()
    cache = L.KvCache(L.BF16, ptr(far[0]), ptr(far[1]), pages, ps, kv, stride)
    size = L.paged_attention_workspace(cache, 2, heads, 480)
    ws = torch.empty(size + 16, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    ctx.kernel_paged_attention(cache, ptr(dq), 256, 2, heads, ptr(table), c.width, ptr(lens), 480, 0.125, ptr(out), 256, ptr(ws), size)
    ctx.synchronize()
    check_paged(ctx, c, heads, q, out.cpu())


# --- bounds ---------------------------------------------------------------------------------------

def bounds_ref(c, table, lens, add):
    """{page: [kv, 2, 64]} of the pages that are written."""
    out = {}
    for i, v in enumerate(lens):
        v = max(0, min(v, c.width * c.ps))
        a = v if add is None else min(max(add[i], 0), v)
        for j in range((v - a) // c.ps, -(-v // c.ps)) if a else ():
            p = int(table[i, j])
            if 0 <= p < c.pages:
                k = c.k[p, :c.kv * c.ps * 64].view(c.kv, c.ps, 64)[:, :min(c.ps, v - j * c.ps)].double()
                out[p] = torch.stack([k.amin(1), k.amax(1)], 1)   # NaN where a row has it
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,kv,ps,add,max_add", [
    ([1], 1, 8, None, 0), ([40, 0, 7], 3, 8, None, 0), ([1037, 16, 17], 12, 16, [1, 1, 1], 1), ([300, 64, 0], 2, 64, [100, 64, 5], 64),
    ([900, 33], 6, 32, [700, 0], 1), ([1000], 5, 256, [2 ** 31 - 1], 0), ([500] * 30, 1, 128, [3] * 30, 2 ** 31 - 1),
    ([2 ** 31 - 1, -5], 2, 16, [20, 20], 20),
])
def test_page_bounds(ctx, dtype, lens, kv, ps, add, max_add):
    report("bounds", dtype=dtype, lens=lens[:4], kv=kv, ps=ps, add=None if add is None else add[:3], max_add=max_add)
    L = lib()
    c = Cache(dtype, [max(0, min(v, 5000)) for v in lens], kv, ps, gap=8, extra_width=0 if max(lens) > 5000 else 2)
    body = c.k[:, :kv * ps * 64].view(c.pages, kv, ps, 64)
    body[int(c.table[0, 0]), 0, 0, 3] = float("nan")
    cache = c.device()
    dl = ints(lens).cuda()
    bounds = torch.full((c.pages, kv, 2, 64), 7.0, dtype=TDT[dtype], device="cuda")
    da = ints(add).cuda() if add is not None else None
    torch.cuda.synchronize()
    ctx.kernel_page_bounds(cache, c.n, ptr(c.dtable), c.width, ptr(dl), ptr(da), max_add, ptr(bounds))
    ctx.synchronize()
    got = bounds.cpu().double()
    want = torch.full_like(got, 7.0)
    for p, b in bounds_ref(c, c.table, lens, add).items():
        want[p] = b
    assert torch.equal(torch.nan_to_num(got, nan=1e9), torch.nan_to_num(want, nan=1e9))


def test_page_bounds_bad_pages_are_left_out(ctx):
    c = Cache("bf16", [100], 2, 16)
    cache = c.device()
    t = c.table.clone()
    t[0, 1], t[0, 3], t[0, 5] = -1, c.pages, 2 ** 31 - 1
    dt = t.cuda()
    bounds = torch.full((c.pages, 2, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    ctx.kernel_page_bounds(cache, 1, ptr(dt), c.width, ptr(c.dlens), 0, 0, ptr(bounds))
    ctx.synchronize()
    want = torch.full((c.pages, 2, 2, 64), 7.0, dtype=torch.float64)
    for p, b in bounds_ref(c, t, [100], None).items():
        want[p] = b
    assert torch.equal(bounds.cpu().double(), want)


# --- sparse attention -----------------------------------------------------------------------------

def choose(c, table, bounds, q, heads, topk, lens):
    """selected [n, kv, topk] in 64 bits, from the definition."""
    G = heads // c.kv
    out = torch.full((c.n, c.kv, topk), -1, dtype=torch.int64)
    b = bounds.double()
    for i, v in enumerate(lens):
        held = -(-v // c.ps)
        there = [j for j in range(held) if 0 <= int(table[i, j]) < c.pages]
        for h in range(c.kv):
            x = q[i].view(c.kv, G, 64)[h].double()
            up, down = x.clamp(min=0).sum(0), x.clamp(max=0).sum(0)
            keyed = []
            for j in there:
                lo, hi = b[int(table[i, j]), h]
                s = float((lo * down + hi * up).sum())
                keyed.append((0 if j == held - 1 else 1 if s != s else 2, -s if s == s else 0.0, j))
            take = sorted(j for _, _, j in sorted(keyed)[:topk])
            out[i, h, :len(take)] = torch.tensor(take, dtype=torch.int64)
    return out


def run_sparse(ctx, c, q, heads, bounds, topk, *, table=None, lens=None, max_len=None, scale=0.125, workspace=None):
    L = lib()
    cache = c.device()
    dq, db = q.cuda(), bounds.cuda()
    out = torch.full((c.n, heads * 64), float("nan"), dtype=TDT[c.dtype], device="cuda")
    sel = torch.full((c.n * c.kv * topk + 8,), -7, dtype=torch.int32, device="cuda")
    max_len = max(max(c.lens), 1) if max_len is None else max_len
    size = L.sparse_attention_workspace(cache, c.n, heads, max_len, topk)
    ws = torch.full((size + 64,), 255, dtype=torch.uint8, device="cuda")
    dt, dl = (c.dtable if table is None else table.cuda()), (c.dlens if lens is None else lens.cuda())
    torch.cuda.synchronize()
    ctx.kernel_sparse_attention(cache, ptr(db), ptr(dq), heads * 64, c.n, heads, ptr(dt), c.width, ptr(dl), max_len, topk, scale,
                                ptr(out), heads * 64, ptr(sel), ptr(ws), size)
    ctx.synchronize()
    assert (sel[c.n * c.kv * topk:] == -7).all() and (ws[size:] == 255).all()
    return out.cpu(), sel[:c.n * c.kv * topk].cpu().view(c.n, c.kv, topk).long()


def page_bounds_of(c):
    b = torch.full((c.pages, c.kv, 2, 64), float("nan"), dtype=TDT[c.dtype])
    for p, v in bounds_ref(c, c.table, c.lens, None).items():
        b[p] = v.to(b.dtype)
    return b


def check_sparse(c, table, bounds, q, heads, topk, out, sel, lens=None, scale=0.125):
    lens = c.lens if lens is None else lens
    want = choose(c, table, bounds, q, heads, topk, lens)
    assert torch.equal(sel, want)
    G, worst = heads // c.kv, 0.0
    real, c.table = c.table, table
    for i, v in enumerate(lens):
        for h in range(c.kv):
            at = [p for j in want[i, h].tolist() if j >= 0 for p in range(j * c.ps, min((j + 1) * c.ps, v))]
            got = out[i].view(c.kv, G, 64)[h].double()
            if not at:
                assert (got == 0).all()
                continue
            worst = max(worst, attention_check(got, q[i].view(c.kv, G, 64)[h].double(), c.head(c.k, i, h, at), c.head(c.v, i, h, at),
                                               scale, c.dtype))
    c.table = real
    report("sparse.err", of_tolerance=f"{worst:.3f}")


SPARSE = [
    # (lens, heads, kv_heads, page_size, topk)
    ([1], 1, 1, 8, 1), ([100, 0, 9], 4, 2, 8, 1), ([100, 0, 8], 4, 4, 8, 3), ([300, 31], 12, 12, 16, 7), ([1037, 16], 8, 1, 16, 64),
    ([1037, 500, 700], 17, 1, 16, 20), ([2000], 6, 6, 8, 100), ([5000, 4999], 16, 4, 32, 33), ([9000], 3, 3, 8, 1024), ([640] * 6, 20, 4, 64, 200),
    ([6223], 2, 2, 16, 16), ([20000, 300], 2, 1, 8, 300), ([3000], 33, 3, 256, 2),
    ([1500] + [3, 0, 40] * 400, 2, 1, 8, 150),   # more sequences than a block sums up
    ([3, 0, 40] * 400 + [9000, 0], 2, 1, 8, 700),   # the same, cut into parts
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,heads,kv,ps,topk", SPARSE)
def test_sparse_attention(ctx, dtype, lens, heads, kv, ps, topk):
    report("sparse", dtype=dtype, lens=lens[:4], n=len(lens), heads=heads, kv=kv, ps=ps, topk=topk)
    c = Cache(dtype, lens, kv, ps)
    q, b = queries(c, heads), page_bounds_of(c)
    out, sel = run_sparse(ctx, c, q, heads, b, topk)
    check_sparse(c, c.table, b, q, heads, topk, out, sel)


@pytest.mark.parametrize("longest", [50, 100, 128, 129, 291, 1025, 4200])   # pages: every way that a page is scored and taken
@pytest.mark.parametrize("topk", [1, 2, 5, 63, 64, 65, 300])
def test_sparse_attention_equal_scores_go_to_the_lower_page(ctx, topk, longest):
    """Bounds from three values only, in all pages of two sequences: many pages score alike."""
    ps = 8 if longest > 1000 else 16
    c = Cache("bf16", [ps * (longest - 1) + 3, ps * 40], 2, ps)
    g = torch.Generator().manual_seed(topk)
    kinds = torch.randn(3, 2, 2, 64, generator=g).sort(2).values.to(torch.bfloat16)
    b = kinds[torch.randint(0, 3, (c.pages,), generator=g)]
    q = queries(c, 4)
    out, sel = run_sparse(ctx, c, q, 4, b, topk)
    check_sparse(c, c.table, b, q, 4, topk, out, sel)


def test_sparse_attention_over_more_pages_than_registers_hold(ctx):
    c = Cache("bf16", [8 * 16500 - 5], 1, 8, garbage=False)
    q, b = queries(c, 2), page_bounds_of(c)
    for topk in (1, 300, 20000):
        out, sel = run_sparse(ctx, c, q, 2, b, topk)
        check_sparse(c, c.table, b, q, 2, topk, out, sel)


@pytest.mark.parametrize("dtype", DTYPES)
def test_sparse_attention_nan_infinite_bounds_and_missing_pages(ctx, dtype):
    """A page with NaN in its bounds comes before every number, infinities in their order, missing pages never."""
    c = Cache(dtype, [16 * 60, 16 * 3, 16 * 2], 2, 16)
    q, b = queries(c, 4), page_bounds_of(c)
    t = c.table.clone()
    inf = float("inf")
    b[int(t[0, 7]), 0, 0, 3] = float("nan")
    q[0, 2], q[0, 66] = 1.5, 0.5
    b[int(t[0, 9]), :, 1, 2] = inf
    b[int(t[0, 11]), :, 1, 2] = -inf
    t[0, 5], t[0, 59], t[0, 20], t[1, 0], t[1, 1], t[1, 2] = -1, c.pages, 2 ** 31 - 1, -5, -1, c.pages + 3
    for topk in (1, 2, 3, 50, 57, 58, 80):
        out, sel = run_sparse(ctx, c, q, 4, b, topk, table=t)
        assert 59 not in sel[0] and (sel[1] == -1).all()
        check_sparse(c, t, b, q, 4, topk, out, sel)


def test_sparse_attention_lengths_past_the_row_or_max_len_are_cut(ctx):
    c = Cache("f16", [200, 90, 64], 2, 16, extra_width=0, garbage=False)
    q, b = queries(c, 4), page_bounds_of(c)
    out, sel = run_sparse(ctx, c, q, 4, b, 3, lens=ints([2 ** 31 - 1, -4, 64]), max_len=77)
    check_sparse(c, c.table, b, q, 4, 3, out, sel, lens=[77, 0, 64])
    out, sel = run_sparse(ctx, c, q, 4, b, 3, max_len=0)
    assert (out == 0).all() and (sel == -1).all()


# --- refusals -------------------------------------------------------------------------------------

def test_refused_calls_say_why_and_launch_nothing(ctx):
    L = lib()
    c = Cache("bf16", [40], 2, 16)
    cache = c.device()
    q, out = torch.zeros(1, 256, dtype=torch.bfloat16, device="cuda"), torch.full((1, 256), 7.0, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    call = lambda **k: ctx.kernel_paged_attention(**{**dict(  # noqa: E731
        cache=cache, q=ptr(q), ldq=256, n=1, heads=4, table=ptr(c.dtable), width=c.width, lens=ptr(c.dlens), max_len=40, scale=0.1,
        out=ptr(out), ldo=256, workspace=0, workspace_bytes=0), **k})
    for bad in ({"heads": 3}, {"cache": None}, {"ldq": 252}, {"q": 0}, {"max_len": -1}, {"scale": float("nan")}, {"out": ptr(q)}):
        with pytest.raises(L.SplatError) as e:
            call(**bad)
        assert e.value.code == L.BAD_ARGUMENT and len(str(e.value)) > 10
    with pytest.raises(L.SplatError):
        L.paged_attention_workspace(cache, 1, 3, 40)
    with pytest.raises(L.SplatError):
        L.sparse_attention_workspace(cache, 1, 4, 40, 0)
    ctx.synchronize()
    assert (out == 7).all()
    call()
    ctx.synchronize()
    assert not (out == 7).any()


# --- together -------------------------------------------------------------------------------------

class Scene:
    """A few scenes that grow: what a serving program keeps, and the plain restatement beside it."""

    def __init__(self, dtype, n=3, heads=6, kv=2, ps=16, cap=400, width=40, topk=4):
        self.__dict__.update(dtype=dtype, n=n, heads=heads, kv=kv, ps=ps, cap=cap, width=width, topk=topk)
        td, L = TDT[dtype], lib()
        cuda = lambda *s, v=0, t=torch.int32: torch.full(s, v, dtype=t, device="cuda")  # noqa: E731
        self.pages = n * width
        self.k, self.v = cuda(self.pages, kv, ps, 64, v=float("nan"), t=td), cuda(self.pages, kv, ps, 64, v=float("nan"), t=td)
        self.bounds = cuda(self.pages, kv, 2, 64, v=float("nan"), t=td)
        self.cache = L.KvCache(L.DTYPES[dtype], ptr(self.k), ptr(self.v), self.pages, ps, kv)
        self.lens, self.add, self.used, self.status = cuda(n), cuda(n), cuda(1), cuda(1)
        self.table, self.starts, self.slots, self.pos = cuda(n, width, v=-1), cuda(n + 1), cuda(cap), cuda(cap)
        self.pool = torch.randperm(self.pages, generator=torch.Generator().manual_seed(2)).to(torch.int32).cuda()
        self.qkv, self.q = cuda(cap, (heads + 2 * kv) * 64, v=0.0, t=td), cuda(cap, heads * 64, v=0.0, t=td)
        self.last, self.dense, self.sparse = (cuda(n, heads * 64, v=0.0, t=td) for _ in range(3))
        self.selected = cuda(n, kv, topk)
        self.max_len = width * ps
        self.sizes = (L.paged_attention_workspace(self.cache, n, heads, self.max_len),
                      L.sparse_attention_workspace(self.cache, n, heads, self.max_len, topk))
        self.ws = [cuda(s + 16, t=torch.uint8, v=255) for s in self.sizes]
        self.rows = [torch.zeros(0, heads + 2 * kv, 64) for _ in range(n)]

    def calls(self, ctx):
        L = lib()
        h, kv, d = self.heads, self.kv, self.heads * 64
        ctx.kernel_block_tables(self.n, ptr(self.lens), ptr(self.add), self.ps, ptr(self.pool), self.pages, ptr(self.used),
                                ptr(self.table), self.width, ptr(self.lens), ptr(self.starts), ptr(self.slots), ptr(self.pos), self.cap,
                                ptr(self.used), ptr(self.status))
        ctx.kernel_qk_norm_rope(L.DTYPES[self.dtype], ptr(self.qkv), (h + 2 * kv) * 64, self.cap, h, kv, L.NORM_RMS, 0, 0, 0, 0, 1e-6,
                                L.ROPE_LINE, 100.0, ptr(self.pos), ptr(self.q), d, 0, 0, self.cache, ptr(self.slots))
        ctx.kernel_page_bounds(self.cache, self.n, ptr(self.table), self.width, ptr(self.lens), ptr(self.add), 64, ptr(self.bounds))
        ctx.kernel_paged_attention(self.cache, ptr(self.last), d, self.n, h, ptr(self.table), self.width, ptr(self.lens), self.max_len,
                                   0.125, ptr(self.dense), d, ptr(self.ws[0]), self.sizes[0])
        ctx.kernel_sparse_attention(self.cache, ptr(self.bounds), ptr(self.last), d, self.n, h, ptr(self.table), self.width,
                                    ptr(self.lens), self.max_len, self.topk, 0.125, ptr(self.sparse), d, ptr(self.selected),
                                    ptr(self.ws[1]), self.sizes[1])

    def feed(self, add, seed):
        """New tokens' rows (garbage behind them) and the queries of this step, on torch's stream."""
        g = torch.Generator().manual_seed(seed)
        td = TDT[self.dtype]
        x = torch.full((self.cap, self.heads + 2 * self.kv, 64), float("nan"))
        x[:sum(add)] = torch.randn(sum(add), self.heads + 2 * self.kv, 64, generator=g)
        x = x.to(td)
        self.qkv.copy_(x.reshape(self.cap, -1).cuda())
        self.last.copy_(torch.randn(self.n, self.heads * 64, generator=g).to(td).cuda())
        self.add.copy_(ints(add).cuda())
        t = 0
        for i, a in enumerate(add):
            self.rows[i] = torch.cat([self.rows[i], x[t:t + a].float()])
            t += a
        torch.cuda.synchronize()

    def check(self, add):
        assert int(self.status) == 0
        td = TDT[self.dtype]
        c = Cache.__new__(Cache)
        c.__dict__.update(dtype=self.dtype, lens=[len(r) for r in self.rows], kv=self.kv, ps=self.ps, n=self.n, pages=self.pages,
                          width=self.width, table=self.table.cpu(), k=self.k.cpu().reshape(self.pages, -1), v=self.v.cpu().reshape(self.pages, -1))
        assert self.lens.cpu().tolist() == c.lens
        h = self.heads
        for i, r in enumerate(self.rows):   # what the cache holds is what was fed, normed and turned
            if not len(r):
                continue
            want = rope_ref(r[:, h:h + self.kv].double(), None, None, "rms", "line", 100.0, torch.arange(len(r)), 1e-6)
            tol = rope_tol(r[:, h:h + self.kv].double(), want, self.dtype)
            for j in range(self.kv):
                at = range(len(r))
                assert ((c.head(c.k, i, j, at) - want[:, j]).abs() <= tol[:, j]).all()
                assert torch.equal(c.head(c.v, i, j, at), r[:, h + self.kv + j].to(td).double())
        q = self.last.cpu()
        check_paged(None, c, h, q, self.dense.cpu())
        b = self.bounds.cpu()
        for p, v in bounds_ref(c, c.table, c.lens, None).items():
            assert torch.equal(b[p].double(), v)
        check_sparse(c, c.table, b, q, h, self.topk, self.sparse.cpu(), self.selected.cpu().long())


STEPS = [[37, 0, 160], [1, 1, 1], [1, 1, 1], [200, 16, 1], [0, 0, 0], [1, 300, 47], [15, 1, 64]]


@pytest.mark.parametrize("dtype", DTYPES)
def test_scenes_that_grow(ctx, dtype):
    s = Scene(dtype)
    for step, add in enumerate(STEPS):
        report("scene", dtype=dtype, step=step, add=add)
        s.feed(add, 100 + step)
        s.calls(ctx)
        ctx.synchronize()
        s.check(add)


def test_scenes_that_grow_in_a_captured_graph(ctx):
    """The five calls captured once on the context's stream and replayed every step, with eager work of the same
    context and of torch between the replays; nothing is allocated by them."""
    s, other = Scene("bf16"), Scene("bf16", n=2, cap=100)
    other.feed([30, 5], 1)
    other.calls(ctx)          # the code objects are loaded
    ctx.synchronize()
    stream = torch.cuda.ExternalStream(ctx.stream)
    graph = torch.cuda.CUDAGraph()
    s.feed([0, 0, 0], 0)
    with torch.cuda.graph(graph, stream=stream):
        s.calls(ctx)
    for step, add in enumerate(STEPS):
        report("scene.graph", step=step, add=add)
        s.feed(add, 100 + step)
        with torch.cuda.stream(stream):
            graph.replay()
        ctx.synchronize()
        s.check(add)
        other.feed([1, 2], 50 + step)
        other.calls(ctx)
        ctx.synchronize()
        other.check([1, 2])


@pytest.mark.parametrize("n,most,ps,topk", [(2, 6000, 16, 130), (1030, 4400, 8, 530)])
def test_long_scenes_in_a_captured_graph(ctx, n, most, ps, topk):
    """Attention cut into parts and joined, scores and selection in launches of their own, captured once and replayed
    over other lengths, queries and bounds in the same memory."""
    L = lib()
    full = Cache("bf16", [most] + [9] * (n - 1), 1, ps)
    heads, cache = 2, full.device()
    q, b = torch.zeros(n, heads * 64, dtype=torch.bfloat16, device="cuda"), page_bounds_of(full).cuda()
    lens = full.dlens
    dense, sparse = torch.zeros_like(q), torch.zeros_like(q)
    sel = torch.zeros(n, 1, topk, dtype=torch.int32, device="cuda")
    sizes = L.paged_attention_workspace(cache, n, heads, most), L.sparse_attention_workspace(cache, n, heads, most, topk)
    assert min(sizes) > 0
    ws = [torch.full((s,), 255, dtype=torch.uint8, device="cuda") for s in sizes]

    def calls():
        at = (ptr(q), heads * 64, n, heads, ptr(full.dtable), full.width, ptr(lens), most)
        ctx.kernel_paged_attention(cache, *at, 0.125, ptr(dense), heads * 64, ptr(ws[0]), sizes[0])
        ctx.kernel_sparse_attention(cache, ptr(b), *at, topk, 0.125, ptr(sparse), heads * 64, ptr(sel), ptr(ws[1]), sizes[1])

    torch.cuda.synchronize()
    calls()   # the code objects are loaded
    ctx.synchronize()
    stream = torch.cuda.ExternalStream(ctx.stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        calls()
    for step, first in enumerate((most, 0, 77, most - 1, most // 2)):
        report("long.graph", n=n, step=step, first=first)
        now = [first] + [(5 * i + step) % 10 for i in range(n - 1)]
        q.copy_(queries(full, heads, seed=step).cuda())
        lens.copy_(ints(now).cuda())
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            graph.replay()
        ctx.synchronize()
        got = dense.clone(), sparse.clone(), sel.clone()
        for w in ws:
            w.fill_(255)   # eager work between the replays; nothing of a call stays in its workspace
        torch.cuda.synchronize()
        calls()
        ctx.synchronize()
        assert torch.equal(got[0], dense) and torch.equal(got[1], sparse) and torch.equal(got[2], sel)
        check_sparse(full, full.table, b.cpu(), q.cpu(), heads, topk, sparse.cpu(), sel.cpu().long(), lens=now)
        real, full.lens = full.lens, now
        check_paged(None, full, heads, q.cpu(), dense.cpu())
        full.lens = real


def test_scenes_of_two_contexts_at_once(ctx):
    """Two contexts, two streams, calls enqueued in turn without a wait between them: the same bits as one after
    the other."""
    L = lib()
    ctx2 = L.Context(0)
    try:
        pairs = [(ctx, Scene("bf16")), (ctx2, Scene("bf16"))]
        alone = Scene("bf16")
        for step, add in enumerate(STEPS[:4]):
            for k, (_, s) in enumerate(pairs):
                s.feed(add, 100 + step)
            for c, s in pairs:
                s.calls(c)
            alone.feed(add, 100 + step)
            ctx.synchronize()
            ctx2.synchronize()
            alone.calls(ctx)
            ctx.synchronize()
            for _, s in pairs:
                assert torch.equal(s.dense, alone.dense) and torch.equal(s.sparse, alone.sparse)
                assert torch.equal(s.selected, alone.selected) and torch.equal(s.table, alone.table)
    finally:
        ctx2.close()


def test_profiling_names_the_operators(ctx):
    s = Scene("bf16")
    s.feed([30, 20, 10], 5)
    ctx.profile_begin()
    s.calls(ctx)
    names = {r["name"] for r in ctx.profile_end()}
    assert {"block_tables", "qk_norm_rope", "page_bounds", "paged_attention", "sparse_attention"} <= names

"""What the paged cache's operators keep of their operands, against restatements in 64 bits on the CPU that share no
formula with the kernels. u = 2^-24, h = half a rounding step of the storage type relative to the value: bf16 2^-8, f16
2^-11, fp32 2^-24."""
import math

import pytest

from conftest import report
from test_gpu_cache import DTYPES, TDT, U, Cache, Rope, attention_ref, half, lib, page_bounds_of, ptr, queries, run_paged, run_sparse

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


# --- weights of 16-bit types ----------------------------------------------------------------------

def weights_tol(ref, A, e, keys, top, dtype):
    """|out - ref| <= h |ref| + (h_w + 2 e + (L + 8) u) A as for any softmax over L keys. A weight of a 16-bit type is the sum of
    two of its numbers: the rest that the first leaves is at most h of the weight, and h of that is lost: h_w = h^2. Terms of
    f16 below its smallest normal value are off by 2^-25, which is 2^-37 of the largest weight, 2^12."""
    h = half(dtype)
    tol = h * ref.abs() + ((0 if dtype == "f32" else h * h) + 2 * e + (keys + 8) * U) * A
    return tol + (keys * 2.0 ** -37 * top + 2.0 ** -25 if dtype == "f16" else 0.0)


def even_cache(dtype, lens, kv, ps):
    """Keys whose scores differ little, and values of 1 and -1 in equal numbers: the sums nearly cancel, so that the result's own
    rounding hides nothing of the weights'."""
    c = Cache(dtype, lens, kv, ps, scale=0.1)
    g = torch.Generator().manual_seed(len(lens))
    v = c.v[:, :kv * ps * 64].view(c.pages, kv, ps, 64)
    for i, n in enumerate(lens):
        signs = torch.stack([torch.randperm(n, generator=g) % 2 for _ in range(kv * 64)]).T.reshape(n, kv, 64) * 2.0 - 1
        for j in range(-(-n // ps)):
            x = signs[j * ps:(j + 1) * ps].transpose(0, 1)
            v[int(c.table[i, j]), :, :x.shape[1]] = x.to(TDT[dtype])
    return c


def check_weights(c, q, heads, out, places=None):
    G, worst = heads // c.kv, 0.0
    for i, n in enumerate(c.lens):
        for h in range(c.kv):
            at = range(n) if places is None else [p for j in places[i, h].tolist() if j >= 0 for p in range(j * c.ps, min(n, (j + 1) * c.ps))]
            k, v = c.head(c.k, i, h, at), c.head(c.v, i, h, at)
            ref, A, e = attention_ref(q[i].view(c.kv, G, 64)[h].double(), k, v, 0.125)
            d = (out[i].view(c.kv, G, 64)[h].double() - ref).abs() / weights_tol(ref, A, e, len(k), 1.0, c.dtype)
            worst = max(worst, float(d.max()))
    report("weights.err", of_tolerance=f"{worst:.3f}")
    assert worst <= 1, worst


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,heads,kv,ps", [([2, 16, 17, 40], 4, 2, 8), ([64, 200, 31], 12, 12, 16), ([2500, 90], 16, 1, 32),
                                              ([4001], 6, 6, 16)])
def test_weights_keep_more_than_their_type_holds(ctx, dtype, lens, heads, kv, ps):
    report("weights", dtype=dtype, lens=lens, heads=heads, kv=kv, ps=ps)
    c = even_cache(dtype, lens, kv, ps)
    q = queries(c, heads)
    check_weights(c, q, heads, run_paged(ctx, c, q, heads))
    out, sel = run_sparse(ctx, c, q, heads, page_bounds_of(c), 3)
    check_weights(c, q, heads, out, sel)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,heads,kv,ps", [([17, 40], 2, 2, 8), ([300, 31], 6, 2, 16), ([2500, 90], 16, 1, 32)])
def test_a_key_of_infinity_costs_the_others_no_bits(ctx, dtype, lens, heads, kv, ps):
    """Keys whose score is -inf have weight 0; the other keys' weights keep all their bits."""
    report("infinite.key", dtype=dtype, lens=lens, heads=heads, kv=kv)
    c = even_cache(dtype, lens, kv, ps)
    q = queries(c, heads)
    x = q.view(c.n, heads, 64)
    x[:, :, 5] = x[:, :, 5].abs() + 0.25
    gone = {}
    for i, n in enumerate(lens):
        gone[i] = [n // 2, n - 1]
        for at in gone[i]:
            c.k[int(c.table[i, at // ps]), :kv * ps * 64].view(kv, ps, 64)[:, at % ps, 5] = -float("inf")
    out = run_paged(ctx, c, q, heads)
    G, worst = heads // kv, 0.0
    for i, n in enumerate(lens):
        at = [p for p in range(n) if p not in gone[i]]
        for h in range(kv):
            k, v = c.head(c.k, i, h, at), c.head(c.v, i, h, at)
            ref, A, e = attention_ref(q[i].view(kv, G, 64)[h].double(), k, v, 0.125)
            d = (out[i].view(kv, G, 64)[h].double() - ref).abs() / weights_tol(ref, A, e, n, 1.0, dtype)
            worst = max(worst, float(d.max()))
    report("infinite.key.err", of_tolerance=f"{worst:.3f}")
    assert worst <= 1, worst


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,heads,kv", [([1, 2, 33, 300], 6, 2), ([3000], 6, 2), ([2000, 5, 1999], 32, 2)])
def test_infinite_values(ctx, dtype, lens, heads, kv):
    """An infinite value has a weight above 0: the channel is infinite, of no number where both signs meet or a value is
    NaN, and the other channels are what they are without it."""
    report("infinite", dtype=dtype, lens=lens, heads=heads, kv=kv)
    c = Cache(dtype, lens, kv, 16, scale=0.3)   # scores of a few units: no weight is too small for f16
    q = queries(c, heads)
    v = c.v[:, :kv * 16 * 64].view(c.pages, kv, 16, 64)
    clean = c.v.clone()
    inf, want = float("inf"), {}
    for i, n in enumerate(lens):
        for at, channel, value in ((0, 3, inf), (n - 1, 17, -inf), (n // 2, 40, inf), (n // 3, 40, -inf), (n // 2, 63, float("nan"))):
            if n == 1 and channel == 40 and value < 0:
                continue   # one key holds one value
            v[int(c.table[i, at // 16]), kv - 1, at % 16, channel] = value
        want[i] = {3: inf, 17: -inf, 40: inf if n == 1 else math.nan, 63: math.nan}
    out = run_paged(ctx, c, q, heads).float()
    c.v = clean
    G = heads // kv
    for i, n in enumerate(lens):
        x = out[i].view(kv, G, 64)[kv - 1]
        for channel, value in want[i].items():
            y = x[:, channel]
            assert torch.isnan(y).all() if value != value else (y == value).all(), (i, channel, y)
        rest = [ch for ch in range(64) if ch not in want[i]]
        k, vals = c.head(c.k, i, kv - 1, range(n)), c.head(c.v, i, kv - 1, range(n))
        ref, A, e = attention_ref(q[i].view(kv, G, 64)[kv - 1].double(), k, vals, 0.125)
        # beside such a channel a weight is one number of its type: h_w = h
        h = half(dtype)
        tol = h * ref.abs() + ((0 if dtype == "f32" else h) + 2 * e + (n + 8) * U) * A
        if dtype == "f16":
            tol = tol + n * 2.0 ** -37 * vals.abs().max() + 2.0 ** -25
        assert ((x.double() - ref).abs() <= tol)[:, rest].all()
        assert torch.isfinite(out[i].view(kv, G, 64)[:kv - 1]).all()


# --- large scores ---------------------------------------------------------------------------------

def exact_scores(dtype, lens, heads, kv, ps):
    """Whole numbers whose products and sums hold no rounding: scores of 8192 and some units more or less, in eighths."""
    c = Cache(dtype, lens, kv, ps, garbage=False)
    g = torch.Generator().manual_seed(len(lens) + heads)
    k = torch.randint(-2, 3, (c.pages, kv, ps, 64), generator=g).float()
    v = torch.randint(0, 2, (c.pages, kv, ps, 64), generator=g) * 2.0 - 1
    q = torch.randint(-2, 3, (c.n, heads, 64), generator=g).float()
    k[..., 0] = q[..., 0] = 256.0
    c.k[:, :kv * ps * 64], c.v[:, :kv * ps * 64] = k.view(c.pages, -1).to(TDT[dtype]), v.view(c.pages, -1).to(TDT[dtype])
    return c, q.view(c.n, -1).to(TDT[dtype])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,heads,kv,ps", [([2, 9, 40], 4, 2, 8), ([33, 100], 16, 1, 16), ([3000, 7], 6, 6, 16)])
def test_large_scores_lose_nothing(ctx, dtype, lens, heads, kv, ps):
    """A score s that holds no rounding gives the weight e^d, d = s - max, which is off by 2 u |d| (log2(e) and its product) and 3 u
    (exp2 and a product); each later tile or part that moves the largest score adds 3 u, L u in all; and the sums L u, the
    weights of 16-bit types h^2: |out - ref| <= h |ref| + sum w (|v| + |ref|) (2 |d| + 3 + 2 L + 8) u / sum w + h_w A."""
    report("large", dtype=dtype, lens=lens, heads=heads, kv=kv)
    c, q = exact_scores(dtype, lens, heads, kv, ps)
    out = run_paged(ctx, c, q, heads)
    G, worst, h = heads // kv, 0.0, half(dtype)
    for i, n in enumerate(lens):
        for hk in range(kv):
            k, v = c.head(c.k, i, hk, range(n)), c.head(c.v, i, hk, range(n))
            s = q[i].view(kv, G, 64)[hk].double() @ k.T * 0.125
            assert s.min() > 8000
            d = s - s.amax(-1, keepdim=True)
            w = torch.softmax(s, -1)
            ref = w @ v
            of = 2 * d.abs() + 3 + 2 * n + 8
            tol = h * ref.abs() + U * ((w * of) @ v.abs() + (w * of).sum(-1, keepdim=True) * ref.abs())
            if dtype != "f32":
                tol = tol + h * h * (w @ v.abs())
            if dtype == "f16":
                tol = tol + n * 2.0 ** -37 + 2.0 ** -25
            worst = max(worst, float(((out[i].view(kv, G, 64)[hk].double() - ref).abs() / tol).max()))
    report("large.err", of_tolerance=f"{worst:.3f}")
    assert worst <= 1, worst


def test_fp32_scores_are_summed_in_quarters(ctx):
    """Products of 2^16 and -2^16 in the first and last channel, and 32 small ones between, whose sum is 3.6 steps of fp32 at 2^16.
    A chain through all channels rounds each of them off there; sums of a quarter's 16 channels hold them, and their three
    additions round by half a step, 2^-8, each: the score is off by 3 2^-8, tanh(score / 2) by half of that."""
    c = Cache("f32", [2], 1, 16, garbage=False)
    t = 0.1125 * 2.0 ** -7   # four of them, a step's products, are less than half of the step at 2^16, 2^-7
    k, q = torch.zeros(64), torch.ones(64)
    k[0], q[0], k[63], q[63] = 256.0, 256.0, 256.0, -256.0
    k[16:48] = t
    page = c.k[int(c.table[0, 0])].view(16, 64)
    page[0], page[1] = 0.0, k
    c.v[int(c.table[0, 0])].view(16, 64)[0], c.v[int(c.table[0, 0])].view(16, 64)[1] = -1.0, 1.0
    out = run_paged(ctx, c, q[None], 1, scale=1.0).double()
    ref = math.tanh(float((q.double() * k.double()).sum()) / 2)
    worst = float((out - ref).abs().max())
    report("quarters", ref=f"{ref:.5f}", off=f"{worst:.5f}")
    assert worst <= 1.5 * 2.0 ** -8 + 8 * U


# --- angles ---------------------------------------------------------------------------------------

def run_turns(ctx, rope, pos, base):
    """Cosines and sines as the rotation has them: [tokens, 32] each, the pairs (1, 0) turned."""
    L = lib()
    T = len(pos)
    x = torch.zeros(T, 3, 2, 2, 16)   # q, k, v of one head; halves of two spans of 16 (grid), or of one of 32 (line)
    x[:, 0, :, 0] = 1.0 if rope == "grid" else 0.0
    if rope == "line":
        x[:, 0, 0] = 1.0
    qkv, d_pos = x.reshape(T, 192).cuda(), pos.to(torch.int32).cuda()
    out = torch.full((T, 64), float("nan"), device="cuda")
    torch.cuda.synchronize()
    ctx.kernel_qk_norm_rope(L.F32, ptr(qkv), 192, T, 1, 1, L.NORM_NONE, 0, 0, 0, 0, 0.0,
                            L.ROPE_GRID if rope == "grid" else L.ROPE_LINE, base, ptr(d_pos), ptr(out), 64)
    ctx.synchronize()
    out = out.cpu().double()
    if rope == "line":
        return out[:, :32], out[:, 32:]
    out = out.view(T, 2, 2, 16)
    return out[:, :, 0].reshape(T, 32), out[:, :, 1].reshape(T, 32)


@pytest.mark.parametrize("rope", ["line", "grid"])
@pytest.mark.parametrize("base", [100.0, 10000.0, 1.0])
def test_angles(ctx, rope, base):
    """At positions up to 4096 the turns in 64 bits are off by less than 2^-40. What 32 bits take of them is below an eighth of a
    turn, 2^-27 of a half turn off at most (pi 2^-27 in the angle), and cosine and sine of it by one ulp of numbers below
    1, 2^-24."""
    n = 4097
    if rope == "line":
        pos = torch.arange(n)
        turns = pos.double()[:, None] * base ** (-torch.arange(32, dtype=torch.float64) / 32)
    else:
        pos = torch.stack([torch.arange(n), torch.arange(n).flip(0)], 1)
        turns = (pos.double()[:, :, None] * base ** (-torch.arange(16, dtype=torch.float64) / 16)).reshape(n, 32)
    cs, sn = run_turns(ctx, rope, pos, base)
    worst = max(float((cs - torch.cos(turns)).abs().max()), float((sn - torch.sin(turns)).abs().max()))
    report("angles.err", rope=rope, base=base, units=f"{worst / 2.0 ** -24:.3f}")
    assert worst <= 2.0 ** -24 + math.pi * 2.0 ** -27


# --- norms, each within its own bound -------------------------------------------------------------

def norm_tol(x, w, b, norm, rope, eps, ref, dtype):
    """Rows x [.., 64] in 64 bits. In units of u, before the rounding to the type (h |ref|):
      sums of 64 terms of one sign: 8 additions in a lane, 3 across, a rounding of each term: 12.
      rms: the root halves those, and it, eps, the division, x r, w and b add one each: 12 S at most, S = |x| r |w| + |b|.
      layer: the mean is off by 12 M (M = max |x|), so a difference by that and 1 of itself, and the variance, relative to itself, by
        2 * 12 M / sd + 12 + 2: y = d r by 12 M / sd (1 + |y|) + 12 |y|, and w and b add one each of S.
      rotation: cosines and sines are off by 1.4 and two products and their sum round: the parts' errors add up, and
        2 * 2.4 + 1 of the largest S.
    """
    top = lambda t: t.abs().amax(-1, keepdim=True)  # noqa: E731
    W = top(w) if w is not None else 1.0
    B = top(b) if b is not None else 0.0
    if norm == "none":
        S, E = top(x), 0.0
    elif norm == "rms":
        S = top(x) / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * W + B
        E = 12 * S
    else:
        sd = torch.sqrt(x.var(-1, unbiased=False, keepdim=True) + eps)
        Y = top(x - x.mean(-1, keepdim=True)) / sd
        S = Y * W + B
        E = W * (12 * top(x) / sd * (1 + Y) + 12 * Y) + 2 * S
    tol = half(dtype) * ref.abs() + U * (E if rope == "none" else 2 * E + 6 * S)
    return tol + (2.0 ** -25 if dtype == "f16" else 0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norm", ["none", "layer", "rms"])
@pytest.mark.parametrize("rope", ["none", "line", "grid"])
def test_norms_within_their_own_bound(ctx, dtype, norm, rope):
    for T, heads, kv, kw in ((33, 6, 6, {}), (70, 8, 2, {"bias": False}), (5, 3, 1, {"weights": False, "bias": False})):
        report("norms", dtype=dtype, norm=norm, rope=rope, T=T, heads=heads, kv=kv, **kw)
        r = Rope(dtype, T, heads, kv, norm, rope, cache=False, **kw)
        x = r.qkv.float()
        x[::3] = x[::3] * 0.05 + 4.0      # a mean far from 0
        x[1::3] *= 30.0
        r.qkv = x.to(TDT[dtype])
        q = torch.empty(T, heads * 64, dtype=TDT[dtype], device="cuda")
        k = torch.empty(T, kv * 64, dtype=TDT[dtype], device="cuda")
        r.call(ctx, q, heads * 64, k, kv * 64, None, None)
        (xq, rq), (xk, rk), _ = r.refs()
        worst = 0.0
        for got, xs, ref, w, b in ((q, xq, rq, r.w[0], r.b[0]), (k, xk, rk, r.w[1], r.b[1])):
            w, b = (None if t is None else t.double() for t in (w, b))
            d = (got.cpu().double().reshape(ref.shape) - ref).abs()
            worst = max(worst, float((d / norm_tol(xs, w, b, norm, rope, r.eps, ref, dtype).clamp(min=1e-300)).max()))
        report("norms.err", of_tolerance=f"{worst:.3f}")
        assert worst <= 1, worst


# --- the choice of pages --------------------------------------------------------------------------

def most_between(lo, hi, q):
    """The most that q k can be for k between lo and hi, head by head and summed over them: q [G, 64], lo and hi [64]. A maximum
    over both ends of every channel, as IEEE products have it (0 inf and NaN give NaN)."""
    at_lo, at_hi = q * lo, q * hi
    return float(torch.where(torch.isnan(at_lo) | torch.isnan(at_hi), math.nan, torch.maximum(at_lo, at_hi)).sum())


def pages_from_the_maximum(c, bounds, q, heads, topk):
    G = heads // c.kv
    out = torch.full((c.n, c.kv, topk), -1, dtype=torch.int64)
    b = bounds.double()
    for i, n in enumerate(c.lens):
        held = -(-n // c.ps)
        for h in range(c.kv):
            x = q[i].view(c.kv, G, 64)[h].double()
            s = [most_between(*b[int(c.table[i, j]), h], x) for j in range(held)]
            # the newest, then NaN, then the largest; the lower page where they are equal
            order = sorted(range(held), key=lambda j: (j != held - 1, s[j] == s[j], -s[j] if s[j] == s[j] else 0.0, j))
            take = sorted(order[:topk])
            out[i, h, :len(take)] = torch.tensor(take, dtype=torch.int64)
    return out


def check_choice(ctx, c, bounds, q, heads, topks, scale=0.125):
    for topk in topks:
        want = pages_from_the_maximum(c, bounds, q, heads, topk)
        _, got = run_sparse(ctx, c, q, heads, bounds, topk, scale=scale)
        assert torch.equal(got, want), (topk, (got != want).nonzero()[:4])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pages", [40, 400])   # scored by the selection, and before it
@pytest.mark.parametrize("heads,kv", [(2, 2), (6, 2), (17, 1)])
def test_infinite_bounds_take_part_where_the_query_does(ctx, dtype, pages, heads, kv):
    """Bounds of one infinite side in random channels, beside queries of one sign, of both and of 0 in the group."""
    report("infinite.bounds", dtype=dtype, pages=pages, heads=heads, kv=kv)
    c = Cache(dtype, [16 * pages, 16 * 7 + 3], kv, 16, garbage=False)
    b = page_bounds_of(c)
    g = torch.Generator().manual_seed(pages + heads)
    inf = float("inf")
    for p in range(0, c.pages, 2):
        for h in range(kv):
            low, high = torch.randint(0, 16, (2,), generator=g).tolist()   # lowest bounds in channels 0-15, highest in 16-31
            b[p, h, 0, low] = -inf
            if p % 4:
                b[p, h, 1, 16 + high] = inf
            if p % 16 == 6:   # both sides of one channel
                b[p, h, 0, 32 + high], b[p, h, 1, 32 + high] = -inf, inf
            if p % 32 == 12:   # every key of the page
                b[p, h, :, 48] = -inf if h else inf
    q = queries(c, heads)
    x = q.view(c.n, kv, heads // kv, 64)
    x[:, :, :, :14] = x[:, :, :, :14].abs() + 0.01    # -inf is the least there, whatever the head
    x[:, :, :, 16:30] = -x[:, :, :, 16:30].abs() - 0.01
    x[1, :, 0, 5], x[1, :, -1, 20], x[1, :, 0, 33] = 0.0, 0.0, 0.0   # no number in the second sequence
    check_choice(ctx, c, b, q, heads, (1, 2, 5, 17, pages // 2, pages + 3))


@pytest.mark.parametrize("dtype", DTYPES)
def test_one_harmless_infinity_displaces_no_page(ctx, dtype):
    """Queries above 0 and a key of -inf, or below 0 and +inf: the page's score is that of its other end."""
    for sign, side in ((1.0, 0), (-1.0, 1)):
        c = Cache(dtype, [16 * 4], 1, 16, garbage=False)
        b = page_bounds_of(c)
        q = queries(c, 1)
        q[0, 2] = sign
        scores = [most_between(*b[int(c.table[0, j]), 0].double(), q[0].view(1, 64).double()) for j in range(3)]
        least = scores.index(min(scores))
        b[int(c.table[0, least]), 0, side, 2] = -sign * float("inf")
        _, got = run_sparse(ctx, c, q, 1, b, 3)
        assert got.flatten().tolist() == [j for j in range(4) if j != least]
        check_choice(ctx, c, b, q, 1, (1, 2, 3, 4))


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_score_is_the_sum_of_each_heads_most(ctx, dtype):
    """Two heads of opposite signs: the page with the wide channel comes first, though one key there gives their sum nothing."""
    c = Cache(dtype, [16 * 5], 1, 16, garbage=False)
    b = torch.zeros(c.pages, 1, 2, 64, dtype=TDT[dtype])
    at = c.table[0].long()
    b[at[1], 0, 0, 7], b[at[1], 0, 1, 7] = -4.0, 4.0   # 8 by two heads of 1 and -1
    b[at[2], 0, :, 9] = 3.0                            # 6 by two heads of 1
    q = torch.zeros(1, 128, dtype=TDT[dtype])
    q[0, 7], q[0, 64 + 7], q[0, 9], q[0, 64 + 9] = 1.0, -1.0, 1.0, 1.0
    _, got = run_sparse(ctx, c, q, 2, b, 2)
    assert got.flatten().tolist() == [1, 4]
    check_choice(ctx, c, b, q, 2, (1, 2, 3, 4, 5))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pages,heads,kv", [(30, 12, 4), (300, 16, 2), (1500, 3, 3)])
def test_the_choice_is_the_definitions(ctx, dtype, pages, heads, kv):
    c = Cache(dtype, [16 * pages - 5, 16 * 9], kv, 16, garbage=False)
    check_choice(ctx, c, page_bounds_of(c), queries(c, heads), heads, (2, 9, pages // 3, pages))


# --- workspaces -----------------------------------------------------------------------------------

@pytest.mark.parametrize("sparse", [False, True])
def test_a_workspace_for_the_largest_batch_serves_smaller_ones(ctx, sparse):
    """A serving loop: one workspace, sized for 100 sequences (one launch, no parts), and batches that shrink (parts)."""
    L = lib()
    heads, ps, topk, most = 12, 16, 100, 2000
    full = Cache("bf16", [most] + [(37 * i) % 60 for i in range(99)], heads, ps, garbage=False)
    cache, bounds = full.device(), page_bounds_of(full).cuda()
    size = L.sparse_attention_workspace(cache, 100, heads, most, topk) if sparse else L.paged_attention_workspace(cache, 100, heads, most)
    ws = torch.empty(size + 16, dtype=torch.uint8, device="cuda")
    q = queries(full, heads)
    dq, sel = q.cuda(), torch.empty(100, heads, topk, dtype=torch.int32, device="cuda")
    outs = []
    for n in (100, 86, 85, 3, 1):
        out = torch.full((100, heads * 64), float("nan"), dtype=torch.bfloat16, device="cuda")
        at = (ptr(dq), heads * 64, n, heads, ptr(full.dtable), full.width, ptr(full.dlens), most)
        ws.fill_(255)
        torch.cuda.synchronize()
        if sparse:
            ctx.kernel_sparse_attention(cache, ptr(bounds), *at, topk, 0.125, ptr(out), heads * 64, ptr(sel), ptr(ws), size)
        else:
            ctx.kernel_paged_attention(cache, *at, 0.125, ptr(out), heads * 64, ptr(ws), size)
        ctx.synchronize()
        outs.append(out.cpu().float())
        assert torch.isnan(outs[-1][n:]).all() and torch.isfinite(outs[-1][:n]).all()
        # other cuts of the same sums: each result is off by one rounding to the type, h |ref|, and before it by (L + 8) u + h_w of
        # the largest value (e is the same for both), so two of them differ by twice that
        d, h = (outs[-1][:n] - outs[0][:n]).abs(), half("bf16")
        assert (d <= 2 * (1 + h) * h * outs[0][:n].abs() + 2 * ((most + 8) * U + h * h) * float(full.v.float().abs().max())).all()

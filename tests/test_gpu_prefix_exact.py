"""What attention over a shared prefix keeps of its operands, in each of its forms, against the definition in 64 bits of test_gpu_prefix.py. u = 2^-24,
h = half a rounding step of the storage type relative to the value: bf16 2^-8, f16 2^-11, fp32 2^-24."""
import pytest

from conftest import report
from test_gpu_prefix import DTYPES, TDT, U, Shared

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


class Even(Shared):
    """Keys whose scores differ little, and values of 1 and -1 in equal numbers: the sums nearly cancel, so that the result's own
    rounding hides nothing of the weights'."""

    def fill(self, page, first, end, g):
        at = [p[page, :self.kv * self.ps * 64].view(self.kv, self.ps, 64) for p in (self.k, self.v)]
        at[0][:, first:end] = (0.1 * torch.randn(self.kv, end - first, 64, generator=g)).to(self.k.dtype)
        signs = torch.rand(self.kv, end - first, 64, generator=g).argsort(1) % 2 * 2.0 - 1
        at[1][:, first:end] = (signs * (1 - 2 * (page % 2))).to(self.v.dtype)

    def tolerance(self, i, scale=0.125):
        """|out - ref| <= h |ref| + (h_w + 2 e + (L + 8) u) A as in test_gpu_prefix.py, but a weight of a 16-bit type is the sum of two of its
        numbers: the rest that the first leaves is at most h of the weight, and h of that is lost: h_w = h^2. Terms of f16
        below its smallest normal value are off by 2^-25, which is at most 2^-29 of the largest weight: that is 2^4 or more. A is at most 1
        here, all values being 1 or -1."""
        L = len(self.seen(i))
        ref, tol = self.ref(i, scale)
        if self.dtype == "f32" or not L:
            return ref, tol
        h = torch.finfo(TDT[self.dtype]).eps / 2
        page, row = (torch.tensor(x) for x in zip(*self.seen(i)))
        k = self.k[:, :self.kv * self.ps * 64].view(self.pages, self.kv, self.ps, 64)[page, :, row].double().transpose(0, 1)
        q = self.q[i].double().view(self.kv, -1, 64)
        e = 70 * U * abs(scale) * (q.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True)
        tol = h * ref.abs() + h * h + 2 * e + (L + 8) * U
        return ref, tol + (L * 2.0 ** -29 + 2.0 ** -25 if self.dtype == "f16" else 0.0)


# few rows of a group and key head (16 and 32 in one item), and more than 64
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("members,shared,own,heads,kv", [
    ([1], [900], None, 4, 2), ([5], [1037], lambda i: 0, 2, 1), ([7, 9], [500, 2000], lambda i: 40 * i % 300, 6, 2), ([130], [200], None, 2, 2),
    ([300, 20], [1500, 64], None, 1, 1), ([90], [1037], lambda i: 3 * i % 200, 4, 2), ([40], [5000], lambda i: 600, 12, 4), ([60, 70], [2000, 3000], None, 6, 1),
])
def test_weights_keep_more_than_their_type_holds(ctx, dtype, members, shared, own, heads, kv):
    report("prefix.weights", dtype=dtype, members=members, shared=shared, heads=heads, kv=kv)
    n = sum(members)
    s = Even(dtype, members, shared, own and [own(i) for i in range(n)], heads, kv, 16)
    out, worst = s.run(ctx), 0.0
    for i in sorted({0, n - 1, *range(0, n, 5)}):
        ref, tol = s.tolerance(i)
        worst = max(worst, float(((out[i].double().view(ref.shape) - ref).abs() / tol).max()))
    report("prefix.weights.err", of_tolerance=f"{worst:.3f}")
    assert worst <= 1, worst


class Whole(Shared):
    """Whole numbers whose products and sums hold no rounding: scores of 8196 and some units more or less, in eighths; values of 1 and -1."""

    def __init__(self, *args, **named):
        super().__init__(*args, **named)
        g = torch.Generator().manual_seed(self.n)
        q = torch.randint(-2, 3, (self.n, self.heads, 64), generator=g).float()
        q[..., 0], q[..., 1] = 256.0, 8.0
        self.q = q.view(self.n, -1).to(self.q.dtype)

    def fill(self, page, first, end, g):
        at = [p[page, :self.kv * self.ps * 64].view(self.kv, self.ps, 64) for p in (self.k, self.v)]
        k = torch.randint(-2, 3, (self.kv, end - first, 64), generator=g).float()
        k[..., 0], k[..., 1] = 256.0, 4.0
        at[0][:, first:end] = k.to(self.k.dtype)
        at[1][:, first:end] = (torch.randint(0, 2, (self.kv, end - first, 64), generator=g) * 2.0 - 1).to(self.v.dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.125, -0.125])
@pytest.mark.parametrize("members,shared,own,heads,kv", [
    ([3], [300], lambda i: 20 * i, 2, 2), ([7], [1037], None, 2, 1), ([20, 9], [600, 90], lambda i: 13 * i % 60, 6, 3), ([90], [1200], None, 4, 2),
    ([150, 5], [520, 700], lambda i: i % 70, 2, 1), ([200], [64], lambda i: 64, 1, 1),
])
def test_large_scores_lose_nothing_where_parts_join(ctx, dtype, scale, members, shared, own, heads, kv):
    """A score s that holds no rounding gives the weight e^d, d = s - max, which is off by 2 u |d| (log2(e) and its product) and 3 u
    (exp2 and a product); each later tile or part that moves the largest score adds 3 u, L u in all; and the sums L u, the
    weights of 16-bit types h^2: |out - ref| <= h |ref| + sum w (|v| + |ref|) (2 |d| + 3 + 2 L + 8) u / sum w + h^2 A."""
    report("prefix.large", dtype=dtype, scale=scale, members=members, shared=shared, heads=heads, kv=kv)
    n = sum(members)
    s = Whole(dtype, members, shared, own and [own(i) for i in range(n)], heads, kv, 16)
    out, worst, h = s.run(ctx, scale=scale), 0.0, torch.finfo(TDT[dtype]).eps / 2
    for i in sorted({0, n - 1, *range(0, n, 3)}):
        at = s.seen(i)
        page, row = (torch.tensor(x) for x in zip(*at))
        k, v = (p[:, :kv * 16 * 64].view(s.pages, kv, 16, 64)[page, :, row].double().transpose(0, 1) for p in (s.k, s.v))
        x = s.q[i].double().view(kv, -1, 64) @ k.transpose(1, 2) * scale
        assert x.abs().min() > 8000
        d = x - x.amax(-1, keepdim=True)
        w = torch.softmax(x, -1)
        ref, of = w @ v, 2 * d.abs() + 3 + 2 * len(at) + 8
        tol = h * ref.abs() + U * ((w * of) @ v.abs() + (w * of).sum(-1, keepdim=True) * ref.abs())
        if dtype != "f32":
            tol = tol + h * h * (w @ v.abs())
        if dtype == "f16":
            tol = tol + len(at) * 2.0 ** -29 + 2.0 ** -25
        worst = max(worst, float(((out[i].double().view(ref.shape) - ref).abs() / tol).max()))
    report("prefix.large.err", of_tolerance=f"{worst:.3f}")
    assert worst <= 1, worst

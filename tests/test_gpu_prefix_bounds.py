"""Attention over a shared prefix at the ends of what it is given: its workspace. Scenes, the definition in 64 bits and the tolerance are those of
test_gpu_prefix.py."""
import pytest

from conftest import report
from test_gpu_prefix import DTYPES, Shared

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,G,shared,max_own", [(16, 24, 128, 16384), (32, 17, 128, 8192), (10, 24, 32, 24889), (64, 24, 64, 8192), (64, 31, 100, 8192), (300, 17, 0, 64)])
def test_parts_of_heads_that_fill_no_group_of_16(ctx, dtype, n, G, shared, max_own):
    """A short prefix and long own positions, whose parts take nearly all of the workspace: run() has the bytes behind it stay."""
    report("prefix.workspace", dtype=dtype, n=n, G=G, shared=shared, max_own=max_own)
    own = [max_own // 8 if i % 13 == 1 else 37 * i % (1 + max_own // 60) for i in range(n)]
    s = Shared(dtype, [n - n // 3, n // 3], [shared, shared // 2], own, G, 1, 16)
    s.check(s.run(ctx, max_own=max_own), rows=sorted({0, 1, n - 1, *range(0, n, 7)}))


class Cut(Shared):
    """Of a group's shared positions the first `most` are seen; own ones begin behind all of them."""

    def seen(self, i):
        k, v = self.group[i], self.lens[i]
        out = [(int(self.prefix[k, p // self.ps]), p % self.ps) for p in range(min(v, self.shared[k], self.most))]
        out += [(int(self.table[i, p // self.ps]), p % self.ps) for p in range(self.shared[k], min(v, self.shared[k] + self.most_own))]
        return [x for x in out if 0 <= x[0] < self.pages]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("members,shared,most,most_own", [([4], [100], 64, 1000), ([3, 150], [1037, 90], 70, 20), ([150, 2], [300, 5000], 0, 33), ([1] * 70, [40] * 70, 33, 50)])
def test_own_positions_begin_behind_a_prefix_that_is_cut(ctx, dtype, members, shared, most, most_own):
    """By max_shared, then by the width of the prefix's rows."""
    report("prefix.cut", dtype=dtype, members=members[:4], shared=shared[:4], most=most, most_own=most_own)
    s = Cut(dtype, members, shared, [(23 * i + 30) % 61 for i in range(sum(members))], 4, 2, 16)
    s.most, s.most_own = most, most_own
    rows = sorted({*range(0, s.n, 5), s.n - 1})
    s.check(s.run(ctx, max_shared=most, max_own=most_own), rows=rows)
    s.prefix_width = max(1, most // 16)
    s.prefix = s.prefix[:, :s.prefix_width].contiguous()
    s.most = s.prefix_width * 16
    s.check(s.run(ctx, max_own=most_own), rows=rows)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("members", [4, 150])
def test_a_shared_length_past_every_token(ctx, dtype, members):
    """No position of a token's own lies behind it, up to the largest number there is."""
    s = Cut(dtype, [members], [100], [(23 * i + 30) % 61 for i in range(members)], 4, 2, 16)
    s.most, s.most_own = 64, 0
    for shared in (161, 2 ** 30, 2 ** 31 - 1):
        s.check(s.run(ctx, shared=[shared], max_shared=64, max_own=2 ** 31 - 1), rows=range(0, members, 3))

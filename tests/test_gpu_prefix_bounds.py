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

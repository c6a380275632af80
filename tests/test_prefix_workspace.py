"""Attention over a shared prefix stays within the workspace that its size query asks for (splatting-rs_amd/csrc/cache_checks.cpp), for
every number of query heads a key head: by the kernels' own indexes, on the CPU under AddressSanitizer and
UndefinedBehaviorSanitizer."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lines(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ is not installed")
    out = str(tmp_path_factory.mktemp("checks") / "prefix_workspace_main")
    subprocess.run([gxx, "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined,float-cast-overflow",
                    "-fno-sanitize-recover=all", os.path.join(ROOT, "tests", "host", "prefix_workspace_main.cpp"),
                    os.path.join(ROOT, "splatting-rs_amd", "csrc", "cache_checks.cpp"), "-o", out],
                   check=True, capture_output=True, timeout=300)
    r = subprocess.run([out], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0 and "runtime error" not in r.stderr, r.stderr[-3000:]
    return r.stdout.splitlines()


@pytest.mark.parametrize("dtype", [0, 1, 2])
@pytest.mark.parametrize("kv", [1, 3])
def test_parts_lie_in_the_workspace(lines, dtype, kv):
    found = [l for l in lines if l.startswith(f"extent ok {dtype} {kv} ")]
    assert len(found) == 40
    assert all(l.endswith(" OK") for l in found), [l for l in found if not l.endswith(" OK")][:4]

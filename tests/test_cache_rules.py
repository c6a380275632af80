"""Rules of the paged cache's calls (splatting-rs_amd/csrc/cache_checks.cpp), on the CPU: which arguments may share
memory, and how workspaces and launches follow the sizes."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "splatting-rs_amd", "csrc")


@pytest.fixture(scope="module")
def lines(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ is not installed")
    out = str(tmp_path_factory.mktemp("rules") / "cache_rules_main")
    subprocess.run([gxx, "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined,float-cast-overflow",
                    "-fno-sanitize-recover=all", os.path.join(ROOT, "tests", "host", "cache_rules_main.cpp"),
                    os.path.join(CSRC, "cache_checks.cpp"), "-o", out], check=True, capture_output=True, timeout=300)
    r = subprocess.run([out], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "runtime error" not in r.stderr, r.stderr[-3000:]
    return r.stdout.splitlines()


def check(lines, first, least):
    """Lines of one kind: calls with " ok" in their name pass, the others are refused."""
    found = [l for l in lines if l.split(" ")[0] == first]
    assert len(found) >= least
    for line in found:
        assert line.endswith(" OK") if " ok" in line else " ERR 1 " in line, line


def test_bounds_lie_over_no_other_argument(lines):
    check(lines, "bounds", 8)


def test_rows_and_pools_lie_over_no_other_argument(lines):
    check(lines, "qk", 24)


def test_a_workspace_for_the_largest_call_serves_every_smaller_one(lines):
    check(lines, "workspace", 3 * 4 * 3 * 5 + 13)

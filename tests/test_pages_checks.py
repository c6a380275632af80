"""Argument checks, launch rules and workspaces of the calls on a cache's pages and of attention over a shared prefix
(splatting-rs_amd/csrc/cache_checks.cpp), under AddressSanitizer and UndefinedBehaviorSanitizer on the CPU; registers and scratch
of their kernels and the waits before their loads into LDS, read from the built library."""
import os
import shutil
import subprocess

import pytest

from test_kernel_resources import kernels  # noqa: F401  (the fixture)
from test_lds_load_waits import functions, missing  # noqa: F401

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "splatting-rs_amd", "csrc")


@pytest.fixture(scope="module")
def lines(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ is not installed")
    out = str(tmp_path_factory.mktemp("checks") / "pages_checks_main")
    subprocess.run([gxx, "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined,float-cast-overflow",
                    "-fno-sanitize-recover=all", os.path.join(ROOT, "tests", "host", "pages_checks_main.cpp"),
                    os.path.join(CSRC, "cache_checks.cpp"), "-o", out], check=True, capture_output=True, timeout=300)
    r = subprocess.run([out], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "runtime error" not in r.stderr, r.stderr[-3000:]
    return r.stdout.splitlines()


@pytest.mark.parametrize("call,least", [("fork", 38), ("free", 35), ("compact", 37), ("copy", 26), ("prefix", 42), ("workspace", 35)])
def test_allowed_calls_pass_and_every_other_one_is_refused(lines, call, least):
    found = [l for l in lines if l.split(" ")[0] == call]
    assert len(found) >= least
    for line in found:
        if " ok" in line:
            assert line.endswith(" OK"), line
        else:
            assert " ERR 1 " in line and len(line.split(" ERR 1 ")[1]) > 10, line


def test_bounds_past_the_rows_size_no_launch(lines):
    assert "cuts 320 480" in lines


def test_kernels_keep_their_values_in_registers(kernels):  # noqa: F811
    """The wide form alone has scratch, for the sums that are taken again with care, whose registers three blocks a CU do not leave; and
    the fp32 form of 64 columns three values of its set-up."""
    for want, count in (("prefix_parts_kernel", 3 + 2 + 2), ("prefix_wide_kernel", 2), ("prefix_own_kernel", 2), ("prefix_join_kernel", 6), ("fork_pages_kernel", 3),
                        ("pages_mark_kernel", 2), ("pages_free_kernel", 1), ("pages_free_small_kernel", 1), ("pages_move_kernel", 1), ("pages_rewrite_kernel", 1),
                        ("pages_compact_small_kernel", 1), ("copy_pages_kernel", 1)):
        found = {k: v for k, v in kernels.items() if want in k}
        assert len(found) == count, (want, len(found))
        for name, (registers, scratch) in found.items():
            assert registers <= (168 if "wide" in want else 256), (name, registers)
            assert scratch <= (128 if "wide" in want else 16 if "parts_kernelIfLi4" in name else 0), (name, scratch)


@pytest.mark.parametrize("kernel", ["prefix_parts_kernel", "prefix_wide_kernel", "prefix_own_kernel"])
def test_loads_into_lds_wait_for_their_registers(functions, kernel):  # noqa: F811
    found = {k: v for k, v in functions.items() if kernel in k}
    assert found
    for name, lines_of in found.items():
        loads, bad = missing(lines_of)
        assert loads and not bad, (name, loads, len(bad), bad[:3])

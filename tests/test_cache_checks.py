"""The paged cache's argument checks (splatting-rs_amd/csrc/cache_checks.cpp), under AddressSanitizer and
UndefinedBehaviorSanitizer on the CPU: calls that are allowed pass, everything else is refused with
SPLAT_BAD_ARGUMENT before a kernel could see it; and the index checks that the kernels make themselves."""
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
    out = str(tmp_path_factory.mktemp("checks") / "cache_checks_main")
    subprocess.run([gxx, "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined,float-cast-overflow",
                    "-fno-sanitize-recover=all", os.path.join(ROOT, "tests", "host", "cache_checks_main.cpp"),
                    os.path.join(CSRC, "cache_checks.cpp"), "-o", out], check=True, capture_output=True, timeout=300)
    r = subprocess.run([out], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "runtime error" not in r.stderr, r.stderr[-3000:]
    return r.stdout.splitlines()


def test_calls_that_are_allowed_pass(lines):
    for line in lines:
        if " ok" in line:
            assert line.endswith(" OK"), line


def test_every_other_call_is_refused(lines):
    calls = [l for l in lines if l.split(" ")[0] in ("tables", "qk", "bounds", "cache", "paged", "sparse", "workspace") and " ok" not in l]
    assert len(calls) > 80
    for line in calls:
        assert " ERR 1 " in line and len(line.split(" ERR 1 ")[1]) > 10, line


def test_the_kernels_index_checks(lines):
    got = {l.split(" ")[0]: l.split(" ")[1:] for l in lines if " OK" not in l and " ERR" not in l}
    assert got["pages"] == ["0", "1", "1", "0"]
    assert got["slots"] == ["0", "1", "1", "0", "0"]
    assert got["lengths"] == ["0", "0", "299", "310", str(2 ** 30)]
    assert got["offsets"] == [str(99 * 2 ** 31 + 3 * 1024), str(99 * 2 ** 31 + 3 * 1024 + 15 * 64)]
    assert got["turns"] == ["1"]

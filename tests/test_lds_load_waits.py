"""Wait states before the loads from memory straight into LDS, read from the disassembly of the built library's own
code objects. The compiler does not look into the inline assembly that issues them, so nothing else inserts these: such a
load needs one after a scalar instruction wrote m0 (its place in LDS), and five after a vector instruction wrote a
scalar register of its descriptor or offset."""
import os
import re
import shutil
import subprocess

import pytest

import splathip
from test_kernel_resources import _code_objects

OBJDUMP = shutil.which("llvm-objdump") or "/opt/rocm/llvm/bin/llvm-objdump"


def scalars(arg):
    """The scalar registers that an operand names."""
    m = re.match(r"s\[(\d+):(\d+)\]$", arg)
    if m:
        return set(range(int(m[1]), int(m[2]) + 1))
    m = re.match(r"s(\d+)$", arg)
    return {int(m[1])} if m else set()


def missing(lines):
    """(loads, those with too few wait states) of one function's instructions."""
    seen, loads, bad = [], 0, []
    for line in lines:
        op, _, rest = line.partition(" ")
        args = [a.strip().split(" ")[0] for a in rest.split(",")]
        if op.startswith("buffer_load") and re.search(r"\blds\b", rest):
            loads += 1
            need, m0, states = set().union(*(scalars(a) for a in args)), True, 0
            for o, a, n in reversed(seen[-12:]):
                if o.startswith("s_") and a[0] == "m0":
                    if m0 and states < 1:
                        bad.append(f"{o} m0, then {states} before {line}")
                    m0 = False
                wrote = scalars(a[0]) & need
                if wrote and o.startswith("v_") and states < 5:
                    bad.append(f"{o} {a[0]}, then {states} before {line}")
                need -= wrote
                states += n
        seen.append((op, args, int(args[0], 0) + 1 if op == "s_nop" else 1))
    return loads, bad


def test_the_count_itself():
    load = "buffer_load_dwordx4 v1, s[4:7], 0 offen lds"
    assert missing(["s_mov_b32 m0, s9", load])[1] and missing(["s_add_i32 m0, s9, 16", load])[1]
    assert missing(["s_mov_b32 m0, s9", "s_nop 0", load]) == (1, [])
    assert missing(["v_readfirstlane_b32 s6, v2", "s_nop 3", load])[1]
    assert missing(["v_readfirstlane_b32 s6, v2", "s_nop 4", load]) == (1, [])
    assert missing(["v_readfirstlane_b32 s8, v2", load]) == (1, [])
    assert missing(["v_readfirstlane_b32 s6, v2", "s_lshl_b32 s6, s6, 8", load]) == (1, [])


@pytest.fixture(scope="module")
def functions(tmp_path_factory):
    """Kernel name -> its instructions, of the kernels that load into LDS."""
    if not os.path.exists(splathip.LIB_PATH) or not os.path.exists(OBJDUMP):
        pytest.skip("no built library or no llvm-objdump")
    out, tmp = {}, tmp_path_factory.mktemp("objects")
    for k, image in enumerate(_code_objects(splathip.LIB_PATH)):
        path = tmp / f"{k}.elf"
        path.write_bytes(image)
        name = None
        p = subprocess.Popen([OBJDUMP, "-d", "--no-show-raw-insn", "--no-leading-addr", str(path)], stdout=subprocess.PIPE, text=True)
        for line in p.stdout:
            m = re.match(r"(?:[0-9a-f]+ )?<(\S+)>:$", line.strip())
            if m:
                name = m[1]
                out[name] = []
            elif name and line.strip():
                out[name].append(re.sub(r"\s+", " ", line.split("//")[0]).strip())
        assert p.wait() == 0
    return {k: v for k, v in out.items() if any("lds" in i and i.startswith("buffer_load") for i in v)}


@pytest.mark.parametrize("kernel", ["paged_whole_kernel", "paged_parts_kernel", "gemm_mfma_kernel", "conv3x3_halo_kernel", "attn_bf16_kernel",
                                    "attn_f32_kernel"])
def test_loads_into_lds_wait_for_their_registers(functions, kernel):
    found = {k: v for k, v in functions.items() if kernel in k}
    assert found
    for name, lines in found.items():
        loads, bad = missing(lines)
        assert loads and not bad, (name, loads, len(bad), bad[:3])

"""The built key-value cache kernels' matrix instructions: no operands in partly
overlapping registers. A build of the 16-row kernel once held its weights and
a fragment of V so, where its loop stood under a condition that the compiler
could not see to be the same in every lane."""
import os
import re
import subprocess

import pytest

from eos_amd import build

LLVM = os.path.join(build.ROCM, "llvm", "bin")
KERNELS = os.path.join(build.BUILD_DIR, "kv.hsaco")


def _operands(line):
    """Register file, first and last register of each operand of a listing's line."""
    return [(f, int(a), int(b)) for f, a, b in re.findall(r"\b([va])\[(\d+):(\d+)\]", line.split("//")[0])]


def _overlap(x, y):
    return x != y and x[0] == y[0] and x[1] <= y[2] and y[1] <= x[2]


def test_the_rule_itself():
    a, b, c = (_operands(s) for s in (
        "v_mfma_f32_16x16x32_f16 a[4:7], v[18:21], v[20:23], a[4:7]",
        "v_mfma_f32_16x16x32_f16 v[4:7], v[18:21], v[22:25], v[6:9]",
        "v_mfma_f32_32x32x16_f16 a[16:31], v[16:19], v[20:23], a[16:31] // v[1:2]"))
    assert _overlap(*a[1:3]) and not _overlap(a[0], a[3])
    assert _overlap(b[0], b[3]) and not _overlap(*b[1:3])
    assert len(c) == 4 and not _overlap(c[0], c[1]) and not _overlap(c[1], c[2])


def test_matrix_operands_do_not_overlap(tmp_path):
    if not os.path.exists(KERNELS) or not os.path.exists(os.path.join(LLVM, "llvm-objdump")):
        pytest.skip("no built kernels, or no disassembler")
    out = str(tmp_path / "kv.o")
    subprocess.run([os.path.join(LLVM, "clang-offload-bundler"), "--unbundle", "--type=o",
                    f"--targets=hipv4-amdgcn-amd-amdhsa--{build.ARCH}", f"--input={KERNELS}",
                    f"--output={out}"], check=True)
    listing = subprocess.run([os.path.join(LLVM, "llvm-objdump"), "-d", "--no-show-raw-insn", out],
                             check=True, capture_output=True, text=True).stdout
    kernel, seen, bad = "", 0, []
    for line in listing.splitlines():
        m = re.search(r"<(eos_kv_\w+)>:", line)
        kernel = m.group(1) if m else kernel
        if "v_mfma" not in line:
            continue
        r = _operands(line)
        seen += 1
        # result, two factors and, where it is no constant, the summand (which the
        # result of four registers may overlap: it is written after the last read)
        if _overlap(r[1], r[2]) or (len(r) == 4 and r[0][2] - r[0][1] > 3 and _overlap(r[0], r[3])):
            bad.append((kernel, line.strip()))
    assert seen > 1000
    assert not bad, bad[:5]

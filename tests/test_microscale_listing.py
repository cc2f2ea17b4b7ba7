"""The built MXFP4 kernels' matrix instructions: no operands in partly
overlapping registers, no spilled registers in the kernels' inner loops."""
import os
import re
import subprocess

import pytest

from eos_amd import build
from test_kv_cache_listing import LLVM, _operands, _overlap

KERNELS = os.path.join(build.BUILD_DIR, "mx.hsaco")


def test_matrix_operands_do_not_overlap(tmp_path):
    if not os.path.exists(KERNELS) or not os.path.exists(os.path.join(LLVM, "llvm-objdump")):
        pytest.skip("no built kernels, or no disassembler")
    out = str(tmp_path / "mx.o")
    subprocess.run([os.path.join(LLVM, "clang-offload-bundler"), "--unbundle", "--type=o",
                    f"--targets=hipv4-amdgcn-amd-amdhsa--{build.ARCH}", f"--input={KERNELS}",
                    f"--output={out}"], check=True)
    listing = subprocess.run([os.path.join(LLVM, "llvm-objdump"), "-d", "--no-show-raw-insn", out],
                             check=True, capture_output=True, text=True).stdout
    kernel, seen, bad, spills = "", {}, [], []
    after_mfma = 0
    for line in listing.splitlines():
        m = re.search(r"<(eos_mx_\w+)>:", line)
        if m:
            kernel, after_mfma = m.group(1), 0
        if "v_mfma" in line:
            after_mfma = 40
            r = _operands(line)
            seen[kernel] = seen.get(kernel, 0) + 1
            # result, two factors and, where it is no constant, the summand
            if _overlap(r[1], r[2]) or any(_overlap(r[0], f) and r[0][0] == f[0] for f in r[1:3]):
                bad.append((kernel, line.strip()))
            if len(r) == 4 and r[0][2] - r[0][1] > 3 and _overlap(r[0], r[3]):
                bad.append((kernel, line.strip()))
        elif after_mfma:
            after_mfma -= 1
            if "scratch_" in line:
                spills.append((kernel, line.strip()))
    assert len([k for k in seen if "product" in k]) == 9 and len(seen) > 25
    assert not bad, bad[:5]
    assert not spills, spills[:5]

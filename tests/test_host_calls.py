"""What the host side of the device entry points refuses and asks for, on a
stand-in for devices (no GPU call)."""
import os
import subprocess
import sys

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
ROCM = os.environ.get("ROCM_PATH", "/opt/rocm")

CASES = ["linear_overlap", "rows_overlap", "rotary_overlap", "pager_overlap",
         "rotary_alignment", "another_current_device",
         "largest_calls"]


@pytest.fixture(scope="module")
def stub(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("stub") / "hip_stub.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-Wall", "-Wextra", "-Werror",
                    "-D__HIP_PLATFORM_AMD__", "-isystem", os.path.join(ROCM, "include"), "-o", out,
                    os.path.join(HERE, "hip_stub.cpp")], check=True)
    return out


@pytest.mark.parametrize("case", CASES)
def test_host_side(stub, case):
    r = subprocess.run([sys.executable, os.path.join(HERE, "hip_stub_cases.py"), stub, case],
                       capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "OK", r.stdout + r.stderr


def test_rows_that_meet(tmp_path):
    exe = str(tmp_path / "row_ranges_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror",
                    "-fsanitize=address,undefined", "-fno-sanitize-recover=undefined",
                    "-I", os.path.join(ROOT, "eos_amd", "csrc"), "-o", exe,
                    os.path.join(HERE, "row_ranges_check.cpp")], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "OK", r.stdout + r.stderr

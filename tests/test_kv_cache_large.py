"""The paged key-value cache's index arithmetic at its largest, on the host."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_steps_of_the_longest_sequences_pass_32_bits(tmp_path):
    exe = str(tmp_path / "kv_large_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror",
                    "-fsanitize=address,undefined", "-fno-sanitize-recover=undefined",
                    "-I", os.path.join(ROOT, "eos_amd", "csrc", "kernels"), "-o", exe,
                    os.path.join(ROOT, "tests", "kv_large_check.cpp")], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "OK", r.stdout + r.stderr

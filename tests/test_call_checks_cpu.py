"""More refusals and bounds of the paged-cache calls, without a GPU (tests/call_checks.cu)."""
import os
import shutil
import subprocess

import pytest

from yuuka_b200 import build

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


def test_refusals_and_bounds(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    exe = str(tmp_path / "call_checks")
    cmd = [nvcc, "-O0", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "--expt-relaxed-constexpr", "-Xptxas", "-O0",
           "-I", os.path.join(ROOT, "include"), "-I", build.CSRC, os.path.join(HERE, "call_checks.cu"), "-o", exe]
    done = subprocess.run(cmd, capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    done = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0 and "all checks passed" in done.stdout, done.stdout + done.stderr

"""Views that begin between words, refused by the calls that read words, without a GPU (tests/view_checks.cpp)."""
import os
import shutil
import subprocess

import pytest

from yuuka_b200 import build

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


def test_misaligned_views_are_refused(tmp_path):
    cxx, nvcc = shutil.which("g++"), shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if cxx is None or not os.path.exists(nvcc):
        pytest.skip("no host C++ compiler, or no CUDA headers")
    build.build_all(force=False, verbose=False)
    exe, libdir = str(tmp_path / "view_checks"), os.path.dirname(build.CUDA_LIB)
    toolkit = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(nvcc))), "include")
    cmd = [cxx, "-std=c++17", "-O1", "-I", os.path.join(ROOT, "include"), "-I", build.CSRC, "-isystem", toolkit, os.path.join(HERE, "view_checks.cpp"), "-o", exe,
           "-L", libdir, "-lyuuka_cuda", f"-Wl,-rpath,{libdir}"]
    done = subprocess.run(cmd, capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    done = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0 and "all checks passed" in done.stdout, done.stdout + done.stderr

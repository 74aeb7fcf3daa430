"""Refusals and lookups of the paged-cache calls, without a GPU (tests/cache_checks.cu)."""
import os
import shutil
import subprocess

import pytest

from yuuka_b200 import build, cuda

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)


def test_refusals_and_lookups(tmp_path):
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    if not os.path.exists(nvcc):
        pytest.skip("no nvcc")
    exe = str(tmp_path / "cache_checks")
    # (-O0 and no device code for what is not run: a few seconds)
    cmd = [nvcc, "-O0", "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "--expt-relaxed-constexpr", "-Xptxas", "-O0",
           "-I", os.path.join(ROOT, "include"), "-I", build.CSRC, os.path.join(HERE, "cache_checks.cu"), "-o", exe]
    done = subprocess.run(cmd, capture_output=True, text=True)
    assert done.returncode == 0, done.stderr
    done = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert done.returncode == 0 and "all checks passed" in done.stdout, done.stdout + done.stderr


@pytest.mark.parametrize("heads,dim", [(1, 64), (3, 64), (4, 128), (7, 256), (1024, 256)])
def test_row_bytes(heads, dim):
    n = heads * dim
    assert cuda.kv_row_bytes(cuda.KV_F32, heads, dim) == 4 * n
    assert cuda.kv_row_bytes(cuda.KV_F16, heads, dim) == 2 * n
    assert cuda.kv_row_bytes(cuda.KV_Q8_0, heads, dim) == n // 32 * 34
    f8 = cuda.kv_row_bytes(cuda.KV_F8, heads, dim)
    assert f8 % 16 == 0 and n + 4 * heads <= f8 < n + 4 * heads + 16
    assert cuda.kv_row_bytes(cuda.KV_F8 + 1, heads, dim) == 0


@pytest.mark.parametrize("heads,dim", [(0, 64), (-1, 64), (1025, 64), (1, 0), (1, 32), (1, 96), (1, 512)])
def test_shapes_without_a_form(heads, dim):
    assert all(cuda.kv_row_bytes(f, heads, dim) == 0 for f in range(4))


def test_null_handles_are_refused():
    lib = cuda.lib()
    assert lib.yuuka_kv_write(None, None, None, None) == cuda.ERR_INVALID_ARGUMENT
    assert lib.yuuka_kv_read(None, None, None, None) == cuda.ERR_INVALID_ARGUMENT
    assert lib.yuuka_attention_decode(None, None, None, None, None) == cuda.ERR_INVALID_ARGUMENT
    assert lib.yuuka_attention_scratch_create(None, None) == cuda.ERR_INVALID_ARGUMENT
    assert lib.yuuka_buffer_view(None, None, 0, None) == cuda.ERR_INVALID_ARGUMENT
    assert lib.yuuka_stream_view(None, None, None) == cuda.ERR_INVALID_ARGUMENT
    lib.yuuka_attention_scratch_destroy(None)

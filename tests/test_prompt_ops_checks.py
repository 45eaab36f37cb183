"""Refusals of the packed-prompt and cache entry points and the range checks
their kernels use, on the CPU (no device is touched)."""
import os
import shutil
import subprocess

import pytest

from conftest import PKG, ROOT


def test_refusals_and_range_checks(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("no g++")
    exe = str(tmp_path / "prompt_ops_checks")
    cmd = [gxx, "-std=c++17", "-O1", "-Wall", "-I/usr/local/cuda/include",
           os.path.join(ROOT, "tests", "prompt_ops_checks.cpp"), "-L" + PKG, "-lsam3cuda",
           "-L/usr/local/cuda/lib64", "-lcudart", "-Wl,-rpath," + PKG,
           "-Wl,-rpath,/usr/local/cuda/lib64", "-o", exe]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "all checks passed" in r.stdout


def test_cache_struct_layout(sam3):
    import ctypes as C
    assert C.sizeof(sam3.KVCache) == 4 * 8 + 4 * 4
    c = sam3.kv_cache(16, 32, 48, 64, 5, 16, 2, 64)
    assert (c.k, c.v, c.k_scale, c.v_scale) == (16, 32, 48, 64)
    assert (c.num_pages, c.page_size, c.kv_heads, c.head_dim) == (5, 16, 2, 64)


def test_dtype_and_limit_constants_match_the_header(sam3):
    src = open(os.path.join(ROOT, "include", "sam3cuda.h")).read()
    assert f"SAM3_F16 = {sam3.F16}, SAM3_BF16 = {sam3.BF16}" in src
    assert f"#define SAM3_CACHED_MAX_SEQS {sam3.CACHED_MAX_SEQS}" in src


def test_a_device_buffer_is_not_asked_for_data_ptr(sam3):
    class Buffer(sam3.DeviceBuffer):
        def __init__(self):  # no device
            self.ptr = 4096

        def data_ptr(self):
            raise AssertionError("asked")

    assert sam3.ptr(Buffer()) == 4096
    assert [sam3.ptr(x) for x in (None, 0, 1 << 40)] == [None, 0, 1 << 40]

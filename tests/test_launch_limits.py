"""Launches of 2^32 threads are refused by name, before anything is launched, and those just below are not; nothing is launched
here. The kernels take a wave of 64 threads for a row's 512 columns, four waves a workgroup, in whole workgroups."""

import os

import pytest

from forgeserve_amd import _lib
from forgeserve_amd.build import LIB

MOST = (1 << 26) - 4   # waves: (2^26 - 4) / 4 workgroups of 256 threads


@pytest.fixture
def lib():
    if not os.path.exists(LIB):
        pytest.skip("library not built")
    return _lib.load()


@pytest.mark.parametrize("m,k", [(MOST + 1, 128), (MOST + 3, 512), (MOST + 4, 128), (MOST // 2 + 1, 640)])
def test_rows_encoded_within_a_product(lib, m, k):
    call = _lib.Linear(x=256, w=256, w_scales=256, out=256, ldx=k, ldw=k, ldo=1, m=m, n=1, k=k, x_dtype=_lib.BF16, dtype=_lib.BF16)
    assert lib.fs_linear_e4m3(call, 256, 1 << 62, None) == -1 and b"linear_e4m3: M" in lib.fs_last_error()
    assert lib.fs_linear_e4m3_workspace_size(call) == 0
    call.m = MOST if k <= 512 else MOST // 2
    assert lib.fs_linear_e4m3_workspace_size(call) > call.m * k
    call.m, call.x_scales = m, 256   # (rows in codes are encoded by nobody)
    assert lib.fs_linear_e4m3_workspace_size(call) == 0 and lib.fs_linear_e4m3_plan(call, (_lib.c_i32 * 4)()) == 0


@pytest.mark.parametrize("m,n", [(MOST + 1, 128), (MOST + 3, 1024), (1 << 22, 1152)])
def test_norm(lib, m, n):
    assert lib.fs_add_rmsnorm_e4m3(256, n, None, 0, None, 0, 256, 256, n, 256, m, n, 1e-5, _lib.BF16, None) == -1
    assert b"add_rmsnorm_e4m3: M" in lib.fs_last_error()


@pytest.mark.parametrize("rows,k", [(MOST + 1, 128), (MOST + 3, 512), (MOST // 2 + 1, 640)])
def test_values(lib, rows, k):
    assert lib.fs_dequantize_e4m3(256, k, 256, rows, k, _lib.BF16, 256, k, None) == -1
    assert b"dequantize_e4m3: rows" in lib.fs_last_error()


@pytest.mark.parametrize("rows,k", [(MOST + 1, 128), (MOST + 3, 512), (MOST // 2 + 1, 640), (1 << 29, 128)])
def test_encoding(lib, rows, k):
    assert lib.fs_quantize_e4m3(256, k, rows, k, _lib.BF16, 256, k, 256, None) == -1
    assert b"quantize_e4m3: rows" in lib.fs_last_error()


@pytest.mark.parametrize("m,n,k", [(MOST + 1, 1, 128), (MOST + 3, 1, 512), (MOST // 2 + 1, 1, 640), (1 << 28, 1, 128), (1 << 25, 1 << 20, 128),
                                   (1, (1 << 29) - 1, 128)])
def test_product(lib, m, n, k):
    """Its rows' encoding, and its tiles."""
    assert lib.fs_gemm_e4m3(256, k, 256, k, 256, 256, n, None, 0, m, n, k, _lib.BF16, 256, 1 << 62, None) == -1
    assert b"gemm_e4m3: M" in lib.fs_last_error()

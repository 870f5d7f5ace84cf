"""A workspace for a number of rows serves any fewer, so that a program may
allocate it once for its largest batch."""
import ctypes

import pytest

import relpos_mhsa as M


def rows_up_to(most):
    return sorted(set(list(range(1, 400)) + [int(1.013 ** i) for i in range(400, 1000) if 1.013 ** i <= most]))


@pytest.mark.parametrize("e,d,f", [(1, 128, 256), (8, 1024, 4096), (16, 64, 64), (64, 1024, 4096), (256, 512, 2048), (1024, 64, 192)])
@pytest.mark.parametrize("top_k", [1, 2, 5, 32])
def test_experts_workspace_grows_with_the_rows(e, d, f, top_k):
    lib, h = M.library(), ctypes.c_void_p()
    assert lib.mhsa_experts_create(e, d, f, 0, ctypes.byref(h)) == 0
    rows = set(rows_up_to(300000))
    for pairs in (256, 1024, 24 * e, 192 * e, 1 << 18):  # about every change of kernels
        rows |= {r for r in range(pairs // top_k - 3, pairs // top_k + 4) if r > 0}
    need = [lib.mhsa_experts_workspace(h, r, top_k) for r in sorted(rows)]
    lib.mhsa_experts_destroy(h)
    assert need[0] > 0
    assert all(a <= b for a, b in zip(need, need[1:]))


@pytest.mark.parametrize("i,o", [(64, 64), (256, 384), (1024, 4096), (4096, 1024), (2048, 2048), (32768, 8192)])
def test_linear_workspace_grows_with_the_rows(i, o):
    lib, h = M.library(), ctypes.c_void_p()
    assert lib.mhsa_fp8_linear_create(i, o, 0, ctypes.byref(h)) == 0
    need = [lib.mhsa_fp8_linear_workspace(h, r) for r in rows_up_to(300000)]
    lib.mhsa_fp8_linear_destroy(h)
    assert all(a <= b for a, b in zip(need, need[1:]))

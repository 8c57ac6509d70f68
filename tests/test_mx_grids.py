"""Sizes past what a grid counts (2^32 threads along x) are refused before a launch.  CPU only."""

from __future__ import annotations

import ctypes

import pytest

from int8_linear import _lib

P = ctypes.c_void_p(0x1000)   # never read: every call below is refused before a launch
MANY = 1 << 26                # waves of 64 lanes


@pytest.mark.parametrize("m", [MANY, MANY - 3])
@pytest.mark.parametrize("ldx", [40, 41])
def test_rows_of_a_slice(m, ldx):
    """A row of 32 of a wider matrix is a wave."""
    L = _lib.lib()
    assert L.i8l_mxfp4_quant(P, ldx, P, P, m, 32, _lib.BF16, 0, None) == _lib.UNSUPPORTED
    assert L.i8l_mxfp4_dequant(P, ldx, P, 1, P, m, 32, _lib.BF16, None) == _lib.UNSUPPORTED
    assert _lib.last_error()


@pytest.mark.parametrize("m", [MANY, MANY - 3])
def test_rows_of_the_fused_quantizers(m):
    L = _lib.lib()
    assert L.i8l_add_rmsnorm_mxfp4_quant(P, None, P, 1e-6, P, P, None, m, 32, _lib.BF16, _lib.BF16, 0,
                                         None) == _lib.UNSUPPORTED
    assert L.i8l_silu_mul_mxfp4_quant(P, P, P, m, 32, _lib.BF16, 0, None) == _lib.UNSUPPORTED
    assert _lib.last_error()


def test_elements_of_an_unaligned_matrix():
    """Rows that touch are one long row; off 16 bytes a wave takes 512 elements."""
    odd = ctypes.c_void_p(0x1002)
    assert _lib.lib().i8l_mxfp4_quant(odd, 1 << 13, P, P, 1 << 22, 1 << 13, _lib.BF16, 0,
                                      None) == _lib.UNSUPPORTED


@pytest.mark.parametrize("n,k", [(1 << 30, 32), ((1 << 30) - 63, 128), ((1 << 31) - 1, 160)])
def test_columns_of_a_product(n, k):
    st = _lib.lib().i8l_mxfp4_mm(P, k // 2, P, k // 2, P, k // 32, P, k // 32, None, 0, P, n, _lib.BF16,
                                 1, n, k, None)
    assert st == _lib.UNSUPPORTED and _lib.last_error()

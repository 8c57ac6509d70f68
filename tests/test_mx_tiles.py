"""The macro tiles of the MXFP4 product, without a GPU: which sizes launch which, as the tests that run
them (test_mx_tiles_gpu.py) take it, so that a change of the rule cannot empty those."""

from __future__ import annotations

import ctypes

import pytest

from int8_linear import _lib

# (tile, parts of K, M, N, K): each tile with more tiles than the card has CUs (256), so that a
# workgroup takes several, then with K in parts; ragged in M and N.  1536: an odd number of
# pairs of K steps, so that a workgroup's next tile starts in the other buffer of scales.
MANY = [((128, 128), 1, 1035, 14440, 1024), ((128, 192), 1, 521, 26736, 1024),
        ((128, 192), 1, 521, 26736, 1536), ((128, 256), 1, 535, 33056, 1024),
        ((256, 128), 1, 16789, 792, 1024), ((256, 192), 1, 1037, 26520, 1024),
        ((256, 256), 1, 771, 38296, 1024), ((256, 256), 1, 771, 38296, 1536)]
PARTS = [((128, 128), 4, 300, 520, 4096), ((128, 192), 2, 33, 20680, 8192),
         ((128, 256), 3, 33, 21040, 6144), ((256, 128), 4, 132, 6224, 14336),
         ((256, 192), 2, 131, 16456, 14336)]


def tile_of(m: int, n: int, k: int):
    """((tokens, columns) of the macro tile that is launched, parts of K)."""
    bm, bn, parts = ctypes.c_int32(-1), ctypes.c_int32(-1), ctypes.c_int32(-1)
    assert _lib.lib().i8l_mxfp4_mm_tile(m, n, k, bm, bn, parts) == _lib.OK
    return (bm.value, bn.value), parts.value


@pytest.mark.parametrize("tile,parts,m,n,k", MANY + PARTS)
def test_the_sizes_launch_their_tiles(tile, parts, m, n, k):
    assert tile_of(m, n, k) == (tile, parts)
    bm, bn = tile
    work = -(-m // bm) * -(-n // bn) * parts
    assert work > 256 if parts == 1 else work <= 256
    assert m % bm and n % bn
    need = _lib.lib().i8l_mxfp4_mm_workspace_bytes(m, n, k)
    assert need == (parts * m * n * 4 if parts > 1 else 0)


@pytest.mark.parametrize("m,n,k", [(1, 4096, 2048), (4096, 4096, 1792), (4096, 4097, 2048),
                                   (4096, 120, 2048), (4096, 4096, 512), (0, 4096, 2048),
                                   (128, 4096, 2048)])
def test_no_tile_where_another_kernel_runs(m, n, k):
    assert tile_of(m, n, k) == ((0, 0), 1)


def test_an_output_that_is_not_there_is_refused():
    i = ctypes.c_int32()
    assert _lib.lib().i8l_mxfp4_mm_tile(4096, 4096, 2048, i, None, i) == _lib.INVALID_ARG

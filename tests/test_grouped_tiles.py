"""The schedules of the grouped product, without a GPU: which sizes launch which, as the tests that run
them (test_grouped_tiles_gpu.py) take it, so that a change of the rule cannot empty those."""

from __future__ import annotations

import ctypes

import pytest

from int8_linear import _lib

CUS = 256

# Rows of experts: last tiles of every kind (up to half of a tile's rows, one past it, whole, one row),
# experts without rows, and with several tiles.
ROWS = {(64, True): ([1, 32, 33, 0, 40, 5, 0, 17] * 7 + [1, 32, 33, 0, 70, 5, 0, 17]),
        (64, False): ([1, 32, 33, 0, 40, 5, 0, 17] * 7 + [1, 32, 33, 0, 70, 5, 0, 17]),
        (128, True): [64, 65, 0, 128, 129, 1, 20, 200] * 2,
        (128, False): [300, 65, 0, 128, 129, 257, 20, 400] * 2,
        (256, False): [1000, 129, 128, 700, 0, 257, 384, 900]}

# (rows of a tile, weights past the caches): (rows of the experts, N, K).  MANY: three tiles a workgroup
# and more, so that each of its three tables of rows is used again, at a K of more steps than are held
# ahead; LONG: more than the 32 tiles that a workgroup's table holds, at a short K.
MANY = {(64, True): (ROWS[64, True], 5104, 640), (64, False): (ROWS[64, False], 5104, 656),
        (128, True): (ROWS[128, True], 13040, 640), (128, False): (ROWS[128, False], 8176, 1008),
        (256, False): (ROWS[256, False], 14320, 1168)}
LONG = {(64, True): (ROWS[64, True], 44272, 128), (64, False): (ROWS[64, False], 44272, 48),
        (128, True): (ROWS[128, True] * 4, 30192, 128), (128, False): (ROWS[128, False] * 4, 18160, 64),
        (256, False): (ROWS[256, False] * 4, 31984, 64)}

# (rows an expert on average where the schedule changes, experts, N, K; the schedule below and from there on)
BORDERS = [(6, 6, 64, 256, (16, 64, 1), (32, 64, 1)), (14, 6, 64, 256, (32, 64, 1), (64, 64, 1)),
           (10, 64, 5104, 144, (32, 64, 1), (64, 256, 0)), (10, 64, 5104, 128, (32, 64, 1), (64, 256, 1)),
           (18, 60, 1000, 256, (64, 64, 1), (64, 256, 1)), (34, 60, 1000, 4112, (64, 64, 1), (128, 256, 0)),
           (44, 6, 64, 256, (64, 64, 1), (128, 256, 1)), (24, 64, 5104, 128, (64, 256, 1), (128, 256, 1)),
           (112, 6, 264, 128, (128, 256, 1), (128, 256, 0)), (208, 6, 264, 1040, (128, 256, 0), (256, 256, 0)),
           (400, 6, 264, 1024, (128, 256, 0), (256, 256, 0))]


def schedule_of(r: int, e: int, n: int, k: int, lines: bool | None = None):
    """(rows, columns of a tile, whether the weights go past the caches)."""
    m, cols, streamed = ctypes.c_int32(-1), ctypes.c_int32(-1), ctypes.c_int32(-1)
    lines = k % 128 == 0 if lines is None else lines      # (of a contiguous weight)
    assert _lib.lib().i8l_w8a8_grouped_mm_tile(r, e, n, k, lines, m, cols, streamed) == _lib.OK
    return m.value, cols.value, streamed.value


def tiles_of(rows, n: int, bm: int) -> int:
    return sum(-(-r // bm) for r in rows) * -(-n // 256)


@pytest.mark.parametrize("gone", [0, 9])
@pytest.mark.parametrize("bm,stream", list(MANY))
def test_the_sizes_launch_their_tiles(bm, stream, gone):
    for sizes, least in ((MANY, 3), (LONG, 33)):
        rows, n, k = sizes[bm, stream]
        assert schedule_of(sum(rows) + gone, len(rows), n, k) == (bm, 256, int(stream))
        assert tiles_of(rows, n, bm) > least * CUS
        assert n % 16 == 0 and n % 256 and k % 16 == 0        # both products, a ragged last column block
        last = {(r - 1) % bm + 1 for r in rows if r}
        assert any(x <= bm // 2 for x in last) and any(x > bm // 2 for x in last)


@pytest.mark.parametrize("border,e,n,k,below,above", BORDERS)
def test_the_borders(border, e, n, k, below, above):
    assert schedule_of(border * e - 1, e, n, k) == below
    assert schedule_of(border * e, e, n, k) == above


def test_every_schedule_stands_at_a_border():
    at = {s for *_, below, above in BORDERS for s in (below, above)}
    assert at == {(16, 64, 1), (32, 64, 1), (64, 64, 1)} | {(bm, 256, int(s)) for bm, s in MANY}


def test_a_grid_too_large_for_the_ring_is_tiled():
    """A workgroup of the ring for each of its tiles: more than a grid counts go to macro tiles."""
    assert schedule_of(2 ** 20, 512, 2 ** 24, 64)[1] == 256 and schedule_of(1, 1, 2 ** 17, 64)[1] == 64


def test_the_query_refuses():
    L, i = _lib.lib(), ctypes.c_int32()
    good = (100, 4, 64, 64, 1)
    assert L.i8l_w8a8_grouped_mm_tile(*good, i, i, i) == _lib.OK
    for outs in ((None, i, i), (i, None, i), (i, i, None)):
        assert L.i8l_w8a8_grouped_mm_tile(*good, *outs) == _lib.INVALID_ARG
    for at, bad in ((0, -1), (0, 2 ** 25 + 1), (1, 0), (1, 513), (2, -1), (2, 2 ** 24 + 1), (3, 0), (3, 2 ** 17)):
        sizes = list(good)
        sizes[at] = bad
        assert L.i8l_w8a8_grouped_mm_tile(*sizes, i, i, i) == _lib.INVALID_ARG

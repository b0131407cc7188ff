"""How the product with an epilogue is split over two launches (CPU): the library's own rule, and its refusal of empty launches."""
import ctypes

import pytest

from _blocks import plan
from h3_tp2_amd import _lib


def first_rows(M, N, cus):
    """The rows of a call's first launch (csrc/gemm_blocks_act.hip)."""
    f = _lib.load()["_ZN6h3host20gemm_blocks_act_rowsElli"]
    f.restype = ctypes.c_int64
    return f(ctypes.c_int64(M), ctypes.c_int64(N), cus)


@pytest.mark.parametrize("N", [272, 1536, 2048, 4096, 4608, 5376, 6144, 7168, 8192, 8208, 14336, 16384, 21504])
@pytest.mark.parametrize("cus", [64, 80, 256, 304])
def test_both_parts_are_rows_of_the_call(N, cus):
    """Every number of rows: the first launch has some and no more than there are, and only whole tiles where a second follows."""
    f = _lib.load()["_ZN6h3host20gemm_blocks_act_rowsElli"]
    f.restype, f.argtypes = ctypes.c_int64, (ctypes.c_int64, ctypes.c_int64, ctypes.c_int)
    cols = -(-N // 256)
    for M in range(1, 70001):
        head = f(M, N, cus)
        if head == M:
            continue
        assert 0 < head < M and head % 256 == 0, (M, head)
        # whole rounds of the tiles, and up to half a round of them left
        tiles = -(-M // 256) * cols
        assert 0 < tiles - head // 256 * cols <= cus // 2, (M, head)


def test_rounds_that_are_full_with_a_ragged_last_tile_are_one_launch():
    """Tiles that fill whole rounds leave nothing for a second launch, whether the last row tile is full or not; where rows are left
    over there is one."""
    for M, N in ((4000, 4096), (4096, 4096), (8000, 4096), (8000, 6144), (8000, 14336), (2000, 8192), (1000, 16384), (16200, 7168),
                 (32600, 4608), (65400, 5376)):
        assert plan(M, N)[:2] == (256, 256) and first_rows(M, N, 256) == M, (M, N)
    for M, N, head in ((6200, 5376, 6144), (18880, 5376, 18688), (18880, 14336, 18688), (12500, 5376, 12288)):
        assert first_rows(M, N, 256) == head, (M, N)
    # 16 columns of tiles: 8 row tiles left are half a round, 9 are more
    assert first_rows(4096 + 8 * 256, 4096, 256) == 4096 and first_rows(4096 + 8 * 256 + 1, 4096, 256) == 4096 + 8 * 256 + 1

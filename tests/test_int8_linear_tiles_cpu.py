"""The tile order of the int8 product's many-row kernel: every tile once, in range, up to the largest products."""
import ctypes

import pytest

from axonml_b200 import _native as N


def _tile(M, Nn, K, bn, t):
    out = (ctypes.c_int * 2)(-7, -7)
    return N.cuda()._lib.ax_int8_gemm_tile(M, Nn, K, bn, t, ctypes.addressof(out)), out[0], out[1]


@pytest.mark.parametrize("bn", [128, 256])
@pytest.mark.parametrize("M,Nn,K", [(1, 1, 1), (300, 1000, 77), (8192, 28672, 4096), (5000, 700, 131071), (100_000, 130, 16), (1, 50_000, 16)])
def test_every_tile_once(M, Nn, K, bn):
    tiles = _tile(M, Nn, K, bn, -1)[0]
    rows, cols = -(-M // 256), -(-Nn // bn)
    assert tiles == rows * cols
    assert {_tile(M, Nn, K, bn, t)[1:] for t in range(tiles)} == {(m, n) for m in range(rows) for n in range(cols)}


@pytest.mark.parametrize("bn", [128, 256])
@pytest.mark.parametrize("M,Nn", [(m, n) for m in (1, 300) for n in (2 ** 28, 2 ** 29 - 128, 2 ** 29, 2 ** 29 + 128, 2 ** 29 + 70_000, 2 ** 30)]
                         + [(2 ** 30, 16), (2 ** 29 + 1, 300)])
@pytest.mark.parametrize("K", [16, 136, 4096])
def test_tiles_of_very_many_channels_and_rows(M, Nn, K, bn):
    """Near 2^29 channels a group's tiles times its columns once wrapped to zero: sampled tiles are in range and distinct, and
    the column goes up by one after each group's rows."""
    tiles = _tile(M, Nn, K, bn, -1)[0]
    rows, cols = -(-M // 256), -(-Nn // bn)
    assert tiles == rows * cols
    step = max(1, tiles // 5000)
    seen = [_tile(M, Nn, K, bn, t)[1:] for t in [*range(0, tiles, step), *range(max(0, tiles - 3000), tiles)]]
    assert all(0 <= m < rows and 0 <= n < cols for m, n in seen)
    assert len(set(seen)) == len(set([*range(0, tiles, step), *range(max(0, tiles - 3000), tiles)]))
    if rows <= 2:                                          # one group: all its rows, then the next column
        for t in (0, 1, tiles // 2, tiles - 1):
            assert _tile(M, Nn, K, bn, t)[1:] == (t % rows, t // rows)

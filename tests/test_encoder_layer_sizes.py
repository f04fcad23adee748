"""Sizes of the entry points of a text encoder's layer whose products leave the range that they are counted in: refused before a device is touched (no GPU needed)."""
from __future__ import annotations

import ctypes as C

import pytest


@pytest.mark.parametrize("N,K", [(2 ** 40, 2 ** 24), (2 ** 40, 2 ** 23), (2 ** 36, 2 ** 28 + 16), (2 ** 34, 2 ** 30), (2 ** 62, 2 ** 31 - 16), (2 ** 63 - 1, 16), (2 ** 38 + 128, 16)])
def test_weights_of_more_than_all_codes(pkg, N, K):
    """N K past 64 bits comes back as a small number, 0 among them."""
    assert pkg.lib.gpu_f8_dequant(0, 16, 16, 128, 16, N, K, 0) == -1
    assert pkg.lib.gpu_f8_requant(0, 16, K, 16, 16, N, K, 0) == -1


@pytest.mark.parametrize("rows,H,scale,D", [(140000000, 16, -1.0, 8), (2 ** 27, 16, -1.0, 8), (2 ** 31 - 600, 2, 0.0, 8), (2 ** 30, 2, 1.0, 136)])
def test_rows_times_heads_of_a_tile(pkg, rows, H, scale, D):
    """The form on mma.sync, which heads above 128 values and scales that are not positive take, counts a sequence's rows as token times heads that share a tile."""
    strides = (C.c_int64 * 8)(*[H * D, D] * 4)
    assert pkg.lib.gpu_packed_attention(2, 16, 16, 16, 16, strides, 16, 1, 1, rows, H, 1, D, scale, 0) == -1

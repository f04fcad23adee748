"""Sizes of the entry points of a text encoder's layer whose products leave the range that they are counted in: refused before a device is touched (no GPU needed)."""
from __future__ import annotations

import pytest


@pytest.mark.parametrize("N,K", [(2 ** 40, 2 ** 24), (2 ** 40, 2 ** 23), (2 ** 36, 2 ** 28 + 16), (2 ** 34, 2 ** 30), (2 ** 62, 2 ** 31 - 16), (2 ** 63 - 1, 16), (2 ** 38 + 128, 16)])
def test_weights_of_more_than_all_codes(pkg, N, K):
    """N K past 64 bits comes back as a small number, 0 among them."""
    assert pkg.lib.gpu_f8_dequant(0, 16, 16, 128, 16, N, K, 0) == -1
    assert pkg.lib.gpu_f8_requant(0, 16, K, 16, 16, N, K, 0) == -1

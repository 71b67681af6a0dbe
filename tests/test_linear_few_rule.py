"""Products of few rows with long sums go to the tiles, whose parts many blocks take (no device needed)."""
import ctypes

import pytest

from naiwa_moe import _lib
from test_linear_rules import FEW16, FEW32, MID, SHORT, THIN, BIG


def kind(rows, experts, n, k, pair=False, odd=False):
    return ctypes.CDLL(_lib.LIB_PATH).naiwa_linear_kind(ctypes.c_int64(rows), experts, n, k, int(pair) + 2 * int(odd))


@pytest.mark.parametrize("rows,experts,n,k,pair,want", [
    (1, 0, 32, 262144, False, THIN), (1, 0, 1, 1 << 21, False, THIN), (64, 0, 32, 100000, False, MID), (200, 0, 16, 8192, True, MID),
    (16, 8, 16, 20000, True, THIN), (1, 0, 16, 4096, False, FEW16), (1, 0, 16, 4104, False, THIN), (200, 0, 1003, 4096, False, FEW32),
    (200, 0, 1003, 4104, False, MID), (64, 0, 16, 131072, True, MID), (64, 0, 16, 262144, True, BIG),
    (1, 0, 8192, 16384, False, FEW16), (64, 64, 1000, 8192, False, FEW16),            # a block a CU and more
])
def test_long_sums(rows, experts, n, k, pair, want):
    assert kind(rows, experts, n, k, pair) == want


@pytest.mark.parametrize("rows,experts,n,k,pair,few", [
    (5, 0, 1003, 1001, False, True), (1, 0, 16, 1536, False, True), (1, 0, 16, 1537, False, False), (64, 0, 200, 2501, True, False),
    (1, 0, 8192, 1001, True, True), (1, 0, 14336, 1001, True, False), (64, 64, 1000, 1001, False, False), (1, 0, 14336, 4097, False, False),
])
def test_odd_rows(rows, experts, n, k, pair, few):
    assert (kind(rows, experts, n, k, pair, odd=True) >= FEW16) == few
    assert kind(rows, experts, n, k, pair) >= FEW16          # the same at multiples of 4 bytes

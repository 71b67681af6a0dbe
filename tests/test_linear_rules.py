"""Which kernel a product and its gradients take (no device needed)."""
import ctypes

import pytest

from naiwa_moe import _lib

THIN, SHORT, MID, BIG, FEW16, FEW32, FEW64 = range(7)


def forward(rows, experts, n, k, pair):
    return ctypes.CDLL(_lib.LIB_PATH).naiwa_linear_kind(ctypes.c_int64(rows), experts, n, k, int(pair))


def input_grad(rows, experts, n, k, dual):
    return ctypes.CDLL(_lib.LIB_PATH).naiwa_linear_input_grad_kind(ctypes.c_int64(rows), experts, n, k, int(dual))


def weight_grad(rows, experts, n, k):
    return ctypes.CDLL(_lib.LIB_PATH).naiwa_linear_weight_grad_kind(ctypes.c_int64(rows), experts, n, k)


@pytest.mark.parametrize("rows,experts,n,k,pair,kind", [
    (1, 0, 2048, 2048, False, FEW16), (64, 0, 2048, 2048, False, FEW16), (65, 0, 2048, 2048, False, FEW32),   # a block a CU
    (129, 0, 2048, 2048, False, FEW64), (256, 0, 2048, 2048, False, FEW64), (257, 0, 2048, 2048, False, MID),   # 16 MB at most
    (1, 0, 14336, 4096, False, FEW16), (3, 0, 14336, 4096, False, THIN), (32, 0, 14336, 4096, False, THIN),     # rows a segment
    (33, 0, 14336, 4096, False, BIG), (128, 8, 14336, 4096, True, THIN), (1, 0, 4096, 14336, False, THIN),      # (128 strips)
    (64, 64, 1408, 2048, True, FEW16), (1024, 64, 1408, 2048, True, THIN), (6144, 64, 1408, 2048, True, BIG),
    (4096, 0, 4096, 14336, False, BIG), (4096, 0, 2048, 2048, False, BIG), (1024, 0, 2048, 2048, False, MID),
    (16384, 0, 4096, 64, False, SHORT), (16384, 0, 4096, 576, False, SHORT), (16384, 0, 4096, 584, False, BIG),
    (1024, 0, 4096, 584, False, MID), (1024, 128, 576, 64, True, SHORT), (32, 8, 14336, 200, True, SHORT), (32, 8, 14336, 256, True, THIN),
])
def test_forward(rows, experts, n, k, pair, kind):
    assert forward(rows, experts, n, k, pair) == kind


@pytest.mark.parametrize("rows,experts,n,k,dual,kind", [
    (1, 0, 2048, 2048, False, THIN), (32, 0, 14336, 4096, True, THIN), (33, 0, 1024, 4096, True, MID),
    (32, 0, 255, 4096, False, SHORT), (32, 0, 128, 4096, True, THIN), (16384, 0, 576, 5120, False, SHORT),
    (16384, 0, 584, 5120, False, BIG), (16384, 0, 288, 5120, True, SHORT), (16384, 0, 296, 5120, True, BIG),
    (16384, 64, 1408, 2048, True, BIG), (2048, 0, 1408, 2048, True, BIG), (2048, 0, 1408, 2048, False, MID),
    (58752, 64, 1240, 88, True, MID), (58752, 64, 1240, 264, True, BIG),                                       # half a tile empty
])
def test_input_grad(rows, experts, n, k, dual, kind):
    assert input_grad(rows, experts, n, k, dual) == kind


@pytest.mark.parametrize("rows,experts,n,k,kind", [
    (0, 1, 2048, 2048, SHORT), (384, 1, 2048, 2048, SHORT), (385, 1, 2048, 2048, MID), (2048, 1, 2048, 2048, MID),
    (4096, 1, 2048, 2048, BIG), (4096, 64, 1408, 2048, SHORT), (24576, 64, 1408, 2048, BIG),
    (9335, 1, 208, 6952, MID), (10085, 1, 3200, 2288, BIG), (46080, 64, 56, 2384, MID),                         # few tiles, empty ones
])
def test_weight_grad(rows, experts, n, k, kind):
    assert weight_grad(rows, experts, n, k) == kind

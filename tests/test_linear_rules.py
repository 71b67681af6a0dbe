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
    (33, 0, 14336, 4096, False, MID), (128, 8, 14336, 4096, True, THIN), (1, 0, 4096, 14336, False, THIN),      # (128 strips)
    (64, 64, 1408, 2048, True, FEW16), (1024, 64, 1408, 2048, True, THIN), (6144, 64, 1408, 2048, True, BIG),
    (4096, 0, 4096, 14336, False, BIG), (4096, 0, 2048, 2048, False, BIG), (1024, 0, 2048, 2048, False, MID),
    (16384, 0, 4096, 64, False, SHORT), (16384, 0, 4096, 72, False, MID), (1024, 128, 576, 64, True, SHORT),
    (32, 8, 14336, 200, True, MID), (32, 8, 14336, 256, True, THIN),                                          # rings to fill
])
def test_forward(rows, experts, n, k, pair, kind):
    assert forward(rows, experts, n, k, pair) == kind


@pytest.mark.parametrize("rows,experts,n,k,dual,kind", [
    (1, 0, 2048, 2048, False, THIN), (32, 0, 14336, 4096, True, THIN), (33, 0, 14336, 4096, True, MID),
    (32, 0, 255, 4096, False, MID), (32, 0, 64, 4096, False, SHORT), (16384, 0, 64, 5120, False, SHORT),
    (16384, 0, 72, 5120, False, MID), (16384, 64, 1408, 2048, True, BIG), (2048, 0, 1408, 2048, True, MID),
    (4096, 0, 1408, 2048, True, BIG), (4096, 0, 1408, 2048, False, MID),
])
def test_input_grad(rows, experts, n, k, dual, kind):
    assert input_grad(rows, experts, n, k, dual) == kind


@pytest.mark.parametrize("rows,experts,n,k,kind", [
    (0, 1, 2048, 2048, SHORT), (64, 1, 2048, 2048, SHORT), (65, 1, 2048, 2048, MID), (2048, 1, 2048, 2048, MID),
    (4096, 1, 2048, 2048, BIG), (4096, 64, 1408, 2048, SHORT), (4097, 64, 1408, 2048, BIG),
])
def test_weight_grad(rows, experts, n, k, kind):
    assert weight_grad(rows, experts, n, k) == kind

"""The products at the documented limits: the longest sums and rows, most experts, millions of rows; one kept value or one bias of two.
Tolerances as in test_gpu_linear."""
import numpy as np
import pytest

import test_gpu_linear as base
from test_gpu_linear import ULP, Stack, off
from test_gpu_tokens import Rows, close, raw_of, values

pytestmark = pytest.mark.gpu

MOST = 1 << 21


@pytest.mark.parametrize("rows,n,k", [(3, 2, MOST), (3, 2, MOST - 1), (1, 1, MOST), (2, MOST, 8), (2, MOST - 1, 3), (40, 24, MOST)])
def test_linear(gpu, rows, n, k):
    # (the residual's rows are one value longer there, which is past the limit of the longest)
    base.test_linear(gpu, rows, n, k, 1, "dense", "bf16", "none", False, True, n < MOST, True, False, True)


@pytest.mark.parametrize("rows,n,k", [(3, 2, MOST), (2, 3, MOST - 1), (2, MOST, 8), (3, MOST - 1, 3)])
def test_gradients(gpu, rows, n, k):
    base.test_input_grad(gpu, rows, n, k, 1, "dense", "bf16", False, "plain", "none", True, True)
    base.test_weight_grad(gpu, rows, n, k, 1, "dense", "bf16", True, True, True, True)


@pytest.mark.parametrize("rows", [1, 5000])
def test_most_experts(gpu, rows):
    for how in (("bf16", "silu", True, True, False, False, True, True), ("f16", "none", False, False, True, True, False, False)):
        base.test_linear(gpu, rows, 24, 16, 4096, "all", *how)
    base.test_input_grad(gpu, rows, 24, 16, 4096, "all", "bf16", False, "pair", "silu", False, True)
    base.test_weight_grad(gpu, rows, 24, 16, 4096, "some", "bf16", True, False, True, True)


def test_millions_of_rows(gpu):
    """Two experts' 20,000,003 rows of 8, some before, between and behind their segments; the gradients of whole numbers are exact."""
    nm = gpu
    rng = np.random.default_rng(1)
    rows, n, k = 20_000_003, 8, 8
    o = np.array([5, 9_000_001, 19_999_000], np.uint32)
    W = Stack(nm, rng, 2, n, k, "bf16", bias=False)
    W.v = rng.integers(-4, 5, (2, n, k)).astype(np.float64)
    W.buf.upload(raw_of(W.v, "bf16")[0])
    xv = rng.integers(-2, 3, (rows, k)).astype(np.float32)
    raw = raw_of(xv, "bf16")[0]
    x, od = nm.DeviceBuffer.from_array(raw), off(nm, o)
    out = nm.DeviceBuffer.from_array(np.full((rows, n), 9.0, np.float32))
    nm.linear(W.w, x, rows, out, offsets=od, out_dtype=nm.F32)
    want = np.full((rows, n), 9.0, np.float32)
    for e in range(2):
        want[o[e]:o[e + 1]] = xv[o[e]:o[e + 1]] @ W.v[e].T.astype(np.float32)
    assert np.array_equal(out.download(np.float32).reshape(rows, n), want)
    # whole numbers below 2^24: sums over 11 million rows of 0 and 1
    g, y = (rng.integers(0, 2, (rows, 8)).astype(np.float32) for _ in range(2))
    gd, yd = (nm.DeviceBuffer.from_array(raw_of(t, "bf16")[0]) for t in (g, y))
    dw, db = nm.DeviceBuffer(2 * n * k * 4), nm.DeviceBuffer(2 * n * 4)
    nm.linear_weight_grad(gd, yd, nm.BF16, rows, n, k, dw, experts=2, offsets=od, dbias=db)
    nm.linear_input_grad(W.w, gd, rows, out, offsets=od, dx_dtype=nm.F32)
    for e in range(2):
        s = slice(o[e], o[e + 1])
        assert np.array_equal(dw.download(np.float32).reshape(2, n, k)[e], g[s].T.astype(np.float64) @ y[s])
        assert np.array_equal(db.download(np.float32).reshape(2, n)[e], g[s].sum(0, dtype=np.float64))
        want[s] = g[s] @ W.v[e].astype(np.float32)
    want[:5], want[19_999_000:] = 9.0, 9.0
    assert np.array_equal(out.download(np.float32).reshape(rows, n), want)


@pytest.mark.parametrize("rows,n,k", [(4, 40, 24), (300, 264, 136), (90, 2056, 4104), (130, 71, 33)])
def test_one_of_two(gpu, rows, n, k):
    """Of a gated product the gate's or the up's values kept alone, and a bias for one of them."""
    nm = gpu
    rng = np.random.default_rng(rows)
    W, U = Stack(nm, rng, 1, n, k, "bf16", bias=False), Stack(nm, rng, 1, n, k, "bf16")
    x = Rows(nm, rng.standard_normal((rows, k)).astype(np.float32), "bf16")
    xv = values(x.start[:-1, :k], "bf16")
    bounds = [(k + 4) * ULP * (np.abs(xv) @ np.abs(t.v[0].T) + (0 if t.b is None else np.abs(t.b[0]))) for t in (W, U)]
    for first, second in ((W, U), (U, W)):
        for keep in ("pre", "pre_up"):
            out, kept = (Rows(nm, np.zeros((rows, n), np.float32), "bf16") for _ in range(2))
            nm.linear(first.w, x.ptr, rows, out.ptr, up=second.w, act=nm.ACT_SILU, **{keep: kept.ptr})
            t = first if keep == "pre" else second
            close(kept.get(), xv @ t.v[0].T + (0 if t.b is None else t.b[0]), bounds[0 if t is W else 1], "bf16")
            both = [Rows(nm, np.zeros((rows, n), np.float32), "bf16") for _ in range(3)]
            nm.linear(first.w, x.ptr, rows, both[0].ptr, up=second.w, act=nm.ACT_SILU, pre=both[1].ptr, pre_up=both[2].ptr)
            assert np.array_equal(out.raw(), both[0].raw())

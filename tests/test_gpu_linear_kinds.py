"""Every kernel of the products and their gradients, at sizes that end inside its tiles and steps: few rows, thin, short, split and
whole-LDS tiles; and rows, weights and results more than 2^32 bytes apart.  Tolerances as in test_gpu_linear."""
import numpy as np
import pytest

import test_gpu_linear as base
import test_linear_rules as rules
from test_gpu_linear import ULP, Stack, off, segments, spans
from test_gpu_tokens import close, dtype_of, np_of, raw_of, values

pytestmark = pytest.mark.gpu

# dt, act, gated, bias, residual, f32, keep, tight
PLAIN = ("bf16", "none", False, True, False, True, False, True)
GATED = ("f16", "silu", True, False, False, False, True, False)
WHOLE = ("bf16", "gelu", True, True, True, False, True, False)
ADDED = ("f16", "gelu", False, True, True, False, True, True)


@pytest.mark.parametrize("rows,n,k,experts,kind,how,takes", [
    (900, 2600, 5128, 1, "dense", ADDED, rules.BIG), (300, 520, 50008, 1, "dense", PLAIN, rules.BIG),
    (700, 1288, 8000, 3, "all", WHOLE, rules.BIG), (1000, 1032, 8400, 3, "some", GATED, rules.BIG),
    (2100, 3600, 2104, 2, "past", PLAIN, rules.BIG), (1800, 3600, 1048, 1, "dense", GATED, rules.BIG),
    (29, 8200, 1064, 1, "dense", ADDED, rules.THIN), (32, 8200, 1064, 1, "dense", GATED, rules.THIN),
    (100, 1000, 1000, 10, "all", WHOLE, rules.THIN), (170, 1384, 520, 12, "one", PLAIN, rules.THIN),
    (600, 1000, 264, 60, "some", GATED, rules.THIN),
    (4500, 1032, 64, 1, "dense", WHOLE, rules.SHORT), (5000, 520, 40, 1, "dense", ADDED, rules.SHORT),
    (700, 1000, 16, 9, "all", GATED, rules.SHORT), (33, 700, 56, 200, "all", PLAIN, rules.SHORT),
    (600, 2056, 1048, 1, "dense", ADDED, rules.MID), (700, 1000, 264, 7, "all", WHOLE, rules.SHORT), (700, 1000, 584, 7, "all", WHOLE, rules.MID),
    (100, 264, 33000, 1, "dense", GATED, rules.MID), (70, 2056, 4104, 1, "dense", PLAIN, rules.MID),     # parts of sums
    (100, 2056, 4104, 2, "all", WHOLE, rules.MID),
    (90, 136, 80, 1, "dense", WHOLE, rules.FEW16), (100, 2040, 1048, 1, "dense", PLAIN, rules.FEW32),
    (240, 2040, 1048, 1, "dense", ADDED, rules.FEW64), (115, 1016, 1000, 1, "dense", GATED, rules.FEW32),
    (240, 1016, 1000, 2, "all", GATED, rules.FEW64),
])
def test_linear(gpu, rows, n, k, experts, kind, how, takes):
    assert rules.forward(rows, 0 if kind == "dense" else experts, n, k, how[2]) == takes
    base.test_linear(gpu, rows, n, k, experts, kind, *how)


@pytest.mark.parametrize("rows,n,k,experts,kind,how", [
    (100, 2051, 4099, 1, "dense", PLAIN), (700, 1003, 263, 7, "all", WHOLE), (60, 1003, 4099, 2, "some", GATED),
    (1000, 999, 63, 1, "dense", ADDED),
])
def test_linear_of_odd_rows(gpu, rows, n, k, experts, kind, how):
    base.test_linear(gpu, rows, n, k, experts, kind, *how)


# dt, dual, mode, act, f32, tight
@pytest.mark.parametrize("rows,n,k,experts,kind,how,takes", [
    (900, 5128, 2600, 1, "dense", ("bf16", False, "plain", "none", True, True), rules.BIG),
    (700, 6504, 1288, 3, "all", ("f16", True, "pair", "silu", False, False), rules.BIG),
    (700, 6504, 1288, 3, "all", ("bf16", True, "add", "none", True, False), rules.BIG),
    (1000, 8400, 2056, 3, "some", ("bf16", False, "pair", "gelu", False, True), rules.BIG),
    (2100, 2104, 3600, 2, "past", ("f16", False, "pre", "silu", False, True), rules.BIG),
    (29, 1064, 2056, 1, "dense", ("bf16", False, "pair", "silu", False, True), rules.THIN),
    (100, 1000, 1000, 10, "all", ("f16", True, "add", "none", False, False), rules.THIN),
    (170, 520, 1384, 12, "one", ("bf16", True, "plain", "none", True, True), rules.THIN),
    (7, 20008, 136, 1, "dense", ("bf16", True, "pre", "gelu", False, True), rules.THIN),                  # parts
    (4500, 64, 1032, 1, "dense", ("bf16", True, "pair", "gelu", False, True), rules.SHORT),
    (700, 16, 1000, 9, "all", ("f16", False, "add", "none", True, False), rules.SHORT),
    (600, 1048, 2056, 1, "dense", ("f16", True, "pair", "silu", False, True), rules.MID),
    (100, 33000, 264, 1, "dense", ("bf16", False, "pair", "silu", False, True), rules.MID),
])
def test_input_grad(gpu, rows, n, k, experts, kind, how, takes):
    assert rules.input_grad(rows, 0 if kind == "dense" else experts, n, k, how[1]) == takes
    base.test_input_grad(gpu, rows, n, k, experts, kind, *how)


# dt, f32, accumulate, bias, tight
@pytest.mark.parametrize("rows,n,k,experts,kind,how,takes", [
    (5003, 1544, 2056, 1, "dense", ("bf16", True, False, True, True), rules.BIG),
    (3000, 2056, 2600, 3, "all", ("f16", True, True, True, False), rules.BIG),
    (3000, 2056, 2600, 3, "some", ("bf16", False, True, True, True), rules.BIG),
    (30000, 520, 264, 2, "one", ("f16", False, False, True, False), rules.MID),
    (60, 1032, 1000, 1, "dense", ("bf16", True, True, True, False), rules.SHORT),
    (500, 520, 264, 9, "all", ("f16", False, False, True, True), rules.SHORT),
    (0, 520, 264, 3, "all", ("bf16", True, False, True, True), rules.SHORT),
    (4000, 520, 264, 9, "past", ("bf16", True, True, False, False), rules.MID),
])
def test_weight_grad(gpu, rows, n, k, experts, kind, how, takes):
    assert rules.weight_grad(rows, experts, n, k) == takes
    base.test_weight_grad(gpu, rows, n, k, experts, kind, *how)


# ---- far apart

LD = 1 << 21                                                  # values, the longest rows that calls take


class Far:
    """Rows LD values apart: 1100 of 16 bits are 4.6 GB."""

    def __init__(self, nm, v, dt):
        raw, self.v = raw_of(v.astype(np.float32), dt)
        self.dt, self.shape, self.step = dt, v.shape, LD * np.dtype(np_of(dt)).itemsize
        self.buf = nm.DeviceBuffer(v.shape[0] * self.step)
        self.ptr = self.buf.ptr
        for i in range(v.shape[0]):
            self.buf.upload(raw[i], offset=i * self.step)

    def get(self):
        return values(np.stack([self.buf.download(np_of(self.dt), self.shape[1], offset=i * self.step)
                                for i in range(self.shape[0])]), self.dt)


@pytest.mark.parametrize("n,k,takes", [(72, 136, rules.FEW16), (2000, 1032, rules.MID), (2000, 5640, rules.BIG), (2000, 64, rules.SHORT),
                                       (1003, 263, None)])
def test_rows_far_apart(gpu, n, k, takes):
    nm = gpu
    rng = np.random.default_rng(n + k)
    rows = 1100
    if takes is not None:
        assert rules.forward(rows, 0, n, k, False) == takes
    normal = lambda w: rng.standard_normal((rows, w))  # noqa: E731
    W = Stack(nm, rng, 1, n, k, "bf16", bias=False)
    x, out, res = Far(nm, normal(k), "bf16"), Far(nm, normal(n), "f32"), Far(nm, normal(n), "f32")
    nm.linear(W.w, x.ptr, rows, out.ptr, residual=res.ptr, out_dtype=nm.F32, x_ld=LD, residual_ld=LD, out_ld=LD)
    want, size = x.v @ W.v[0].T, np.abs(x.v) @ np.abs(W.v[0].T)
    close(out.get(), want + res.v, (k + 4) * ULP * size + ULP * (np.abs(want) + np.abs(res.v)), "f32")
    del out, res
    dy, dx = Far(nm, normal(n), "bf16"), Far(nm, normal(k), "f32")
    nm.linear_input_grad(W.w, dy.ptr, rows, dx.ptr, dx_dtype=nm.F32, dy_ld=LD, dx_ld=LD)
    close(dx.get(), dy.v @ W.v[0], (n + 4) * ULP * (np.abs(dy.v) @ np.abs(W.v[0])), "f32")
    del dx
    dw = nm.DeviceBuffer(n * k * 4)
    nm.linear_weight_grad(dy.ptr, x.ptr, nm.BF16, rows, n, k, dw, dy_ld=LD, x_ld=LD)
    close(dw.download(np.float32).reshape(n, k), dy.v.T @ x.v, (rows + 4) * ULP * (np.abs(dy.v).T @ np.abs(x.v)), "f32")


@pytest.mark.parametrize("rows,n,k", [(6, 40, 72), (90, 136, 264), (3000, 1032, 1304), (90, 135, 263)])
def test_experts_far_apart(gpu, rows, n, k):
    """Three experts 2^31 values apart, their rows 2^20: few rows, and the larger tiles."""
    nm = gpu
    rng = np.random.default_rng(rows)
    stride, ld, experts = 1 << 31, 1 << 20, 3
    raw, wv = raw_of(rng.standard_normal((experts, n, k)).astype(np.float32), "bf16")
    w = nm.DeviceBuffer(2 * (2 * stride + n * ld))
    for e in range(experts):
        for i in range(n):
            w.upload(raw[e, i], offset=2 * (e * stride + i * ld))
    W = nm.Weights(w, nm.BF16, experts, n, k, ld=ld, stride=stride)
    o = segments(rng, rows, experts, "all")
    od = off(nm, o)
    (xr, xv), (gr, gv) = (raw_of(rng.standard_normal((rows, m)).astype(np.float32), "bf16") for m in (k, n))
    x, g = nm.DeviceBuffer.from_array(xr), nm.DeviceBuffer.from_array(gr)
    out, dx = nm.DeviceBuffer(rows * n * 4), nm.DeviceBuffer(rows * k * 4)
    nm.linear(W, x, rows, out, offsets=od, out_dtype=nm.F32)
    nm.linear_input_grad(W, g, rows, dx, offsets=od, dx_dtype=nm.F32)
    got, gdx = out.download(np.float32).reshape(rows, n), dx.download(np.float32).reshape(rows, k)
    for e, s in spans(o, rows, experts):
        close(got[s], xv[s] @ wv[e].T, (k + 4) * ULP * (np.abs(xv[s]) @ np.abs(wv[e].T)), "f32")
        close(gdx[s], gv[s] @ wv[e], (n + 4) * ULP * (np.abs(gv[s]) @ np.abs(wv[e])), "f32")
    nm.linear_weight_grad(g, x, nm.BF16, rows, n, k, w, experts=experts, offsets=od, dw_dtype=nm.BF16, ld=ld, stride=stride)
    for e, s in spans(o, rows, experts):
        d = values(np.stack([w.download(np.uint16, k, offset=2 * (e * stride + i * ld)) for i in range(n)]), "bf16")
        close(d, gv[s].T @ xv[s], (max(s.stop - s.start, 0) + 4) * ULP * (np.abs(gv[s]).T @ np.abs(xv[s])), "bf16")


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_token_rows_far_apart(gpu, dt):
    """Tokens moved between rows more than 2^32 bytes apart from first to last."""
    nm = gpu
    rng = np.random.default_rng(4)
    T, k, E, H = 550, 2, 16, 200
    x, y, out, dy = (Far(nm, rng.standard_normal((m, H)), dt) for m in (T, T * k, T, T * k))
    wv = rng.random((T, k)).astype(np.float32)
    w, dw = nm.DeviceBuffer.from_array(wv), nm.DeviceBuffer(T * k * 4)
    iv = rng.permutation(T * k).astype(np.uint32).reshape(T, k)
    inv = nm.DeviceBuffer.from_array(iv)
    d = dtype_of(nm, dt)
    nm.tokens_to_experts(x.ptr, d, inv, T, k, H, y.ptr, ld=LD, rows_ld=LD)
    rows = np.zeros((T * k, H))
    for j in range(k):
        rows[iv[:, j]] = x.v
    assert np.array_equal(y.get(), rows)
    nm.tokens_from_experts(y.ptr, d, inv, T, k, H, out.ptr, w=w, ld=LD, out_ld=LD)
    want = wv.sum(1, dtype=np.float64)[:, None] * x.v
    close(out.get(), want, 4 * ULP * np.abs(x.v) * wv.sum(1)[:, None], dt)
    o = out.get()
    nm.tokens_from_experts_backward(out.ptr, d, y.ptr, d, inv, T, k, H, dy=dy.ptr, dw=dw, w=w, dout_ld=LD, ld=LD, dy_ld=LD)
    for j in range(k):
        rows[iv[:, j]] = wv[:, j, None].astype(np.float64) * o
    close(dy.get(), rows, 2.0 ** -24 * np.abs(rows), dt)
    want = np.repeat((o * x.v).sum(1)[:, None], k, 1)
    close(dw.download(np.float32).reshape(T, k), want, H * 2.0 ** -24 * np.repeat(np.abs(o * x.v).sum(1)[:, None], k, 1), "f32")


# ---- results too large for the caches

def some(rng, n):
    """The first and last 200 of n, and 600 between."""
    return np.unique(np.concatenate([np.arange(200), np.arange(n - 200, n), rng.integers(0, n, 600)]))


@pytest.mark.parametrize("rows,n,k,dt", [(70000, 1000, 24, "f32"), (70001, 2003, 17, "bf16"), (40000, 3600, 1096, "bf16")])
def test_large_results(gpu, rows, n, k, dt):
    """Forward and input gradient of 256 MB and more, where stores go past the caches; rows behind them stay."""
    nm = gpu
    rng = np.random.default_rng(rows)
    W = Stack(nm, rng, 1, n, k, "bf16")
    (xr, xv), d = raw_of(rng.standard_normal((rows, k)).astype(np.float32), "bf16"), dtype_of(nm, dt)
    x, size = nm.DeviceBuffer.from_array(xr), np.dtype(np_of(dt)).itemsize
    assert rows * n * size >= 1 << 28
    out = nm.DeviceBuffer((rows + 1) * n * size)
    mark = raw_of(np.full(n, 1.25, np.float32), dt)[0]
    out.upload(mark, offset=rows * n * size)
    nm.linear(W.w, x, rows, out, out_dtype=d)
    for m in some(rng, rows):
        got = values(out.download(np_of(dt), n, offset=int(m) * n * size), dt)
        close(got, xv[m] @ W.v[0].T + W.b[0], (k + 4) * ULP * (np.abs(xv[m]) @ np.abs(W.v[0].T) + np.abs(W.b[0])), dt)
    assert np.array_equal(out.download(np_of(dt), n, offset=rows * n * size), mark)
    # as an input gradient: the weights' transposes, [k, n] here
    T = nm.DeviceBuffer.from_array(np.ascontiguousarray(raw_of(W.v[0], "bf16")[0].T))
    nm.linear_input_grad(nm.Weights(T, nm.BF16, 1, k, n), x, rows, out, dx_dtype=d)
    for m in some(rng, rows):
        got = values(out.download(np_of(dt), n, offset=int(m) * n * size), dt)
        close(got, xv[m] @ W.v[0].T, (k + 4) * ULP * (np.abs(xv[m]) @ np.abs(W.v[0].T)), dt)
    assert np.array_equal(out.download(np_of(dt), n, offset=rows * n * size), mark)


@pytest.mark.parametrize("rows,n,k,dt", [(600, 1408, 2048, "f32"), (5000, 1408, 1504, "f32"), (90, 2003, 2051, "bf16")])
def test_large_weight_gradients(gpu, rows, n, k, dt):
    nm = gpu
    rng = np.random.default_rng(rows)
    experts, size = 34, np.dtype(np_of(dt)).itemsize
    assert experts * n * k * size >= 1 << 28
    o = segments(rng, rows, experts, "all")
    (gr, gv), (xr, xv) = (raw_of(rng.standard_normal((rows, m)).astype(np.float32), "bf16") for m in (n, k))
    g, x, dw = nm.DeviceBuffer.from_array(gr), nm.DeviceBuffer.from_array(xr), nm.DeviceBuffer(experts * n * k * size)
    nm.linear_weight_grad(g, x, nm.BF16, rows, n, k, dw, experts=experts, offsets=off(nm, o), dw_dtype=dtype_of(nm, dt))
    for e, s in spans(o, rows, experts):
        got = values(dw.download(np_of(dt), n * k, offset=e * n * k * size).reshape(n, k), dt)
        m = max(s.stop - s.start, 0)
        close(got, gv[s].T @ xv[s], (m + 4) * ULP * (np.abs(gv[s]).T @ np.abs(xv[s])), dt)

"""Products over 16-bit weights with everything behind them, and their gradients, against 64 bits.

Tolerances, value by value.  Products of 16-bit values are exact in f32.  A sum of K of them added up in any order in f32,
by additions that round or cut, errs by at most K 2^-23 sum |a b|; with bias, gate and residual a few 2^-24 more, which the
same bound holds for K >= 4 (4 are added for shorter ones).  SiLU and GELU have slopes of at most 1.13 and their
slopes' own of at most 1.2; their values in f32 are good to 16 2^-24 of |v| + 2^-20 (the exponential of v by |v| 2^-24,
tanh by a few 2^-24; GELU's 1 + tanh loses up to 2^-24 of v).  Then one rounding by half a step of the type.
"""
import numpy as np
import pytest

from test_gpu_mxfp4 import Graph
from test_gpu_tokens import Rows, close, dtype_of, np_of, raw_of, values

pytestmark = pytest.mark.gpu

ULP = 2.0 ** -23
ACTS = {"none": -1, "silu": 0, "gelu": 1}


def act(name, v):
    """(act(v), act'(v)) in f64."""
    if name == "none":
        return v, np.ones_like(v)
    if name == "silu":
        with np.errstate(over="ignore"):
            s = 1 / (1 + np.exp(-v))
        return v * s, s * (1 + v * (1 - s))
    a = np.sqrt(2 / np.pi)
    t = np.tanh(a * (v + 0.044715 * v ** 3))
    return 0.5 * v * (1 + t), 0.5 * (1 + t) + 0.5 * v * (1 - t * t) * a * (1 + 3 * 0.044715 * v * v)


def act_error(name, v, dv):
    """How far act(v + dv) in f32 may be from act(v), and its slope."""
    if name == "none":
        return dv, np.zeros_like(v)
    own = 16 * 2.0 ** -24 * (np.abs(v) + 2.0 ** -4)
    return 1.13 * dv + own, 1.2 * dv + 16 * 2.0 ** -24 * (1 + np.abs(v))


def segments(rng, rows, experts, kind):
    """offsets [experts + 1], or None."""
    if kind == "dense":
        return None
    if kind == "one":                  # all rows one expert's, the others empty
        o = np.zeros(experts + 1, np.uint32)
        o[experts // 2 + 1:] = rows
        return o
    if kind == "past":                 # entries past the rows count as the last
        o = segments(rng, rows, experts, "some")
        o[o == o[-1]] = rows + 1000
        return o
    cuts = np.sort(rng.integers(0, rows + 1, experts + 1)).astype(np.uint32)
    cuts[0] = 0
    if kind == "all":
        cuts[-1] = rows
    return cuts


def spans(o, rows, experts):
    o = np.array([0, rows]) if o is None else np.minimum(o, rows).astype(int)
    return [(e, slice(o[e], o[e + 1])) for e in range(experts)]


class Stack:
    """Weights [experts, n, k] with rows `ld` and experts `stride` values apart, NaN between."""

    def __init__(self, nm, rng, experts, n, k, dt, ld=0, gap=0, shift=0, bias=True):
        self.ld, self.v = ld or k, rng.standard_normal((experts, n, k)).astype(np.float32) * 0.5
        self.stride = n * self.ld + gap
        raw = raw_of(np.full((experts, self.stride), np.nan, np.float32), dt)[0]
        body, self.v = raw_of(self.v, dt)
        for e in range(experts):
            raw[e, :n * self.ld].reshape(n, self.ld)[:, :k] = body[e]
        self.buf = nm.DeviceBuffer(raw.nbytes + 64)
        self.buf.upload(raw, offset=2 * shift)
        self.b = rng.standard_normal((experts, n)).astype(np.float32) if bias else None
        self.bd = nm.DeviceBuffer.from_array(self.b) if bias else None
        self.w = nm.Weights(self.buf.ptr + 2 * shift, dtype_of(nm, dt), experts, n, k, bias=self.bd, ld=ld,
                            stride=self.stride if gap or ld else 0)


def off(nm, o):
    return None if o is None else nm.DeviceBuffer.from_array(o)


# rows, n, k, experts, segments: one and few rows, tiles' edges, odd sizes, empty experts, more experts than lanes
SHAPES = [
    (1, 1, 1, 1, "dense"), (1, 16, 8, 1, "dense"), (5, 1003, 1001, 1, "dense"), (16, 64, 64, 1, "dense"), (17, 72, 40, 1, "dense"),
    (128, 128, 128, 1, "dense"), (129, 136, 200, 1, "dense"), (300, 257, 520, 1, "dense"), (40, 2048, 256, 1, "dense"),
    (513, 320, 1048, 1, "dense"), (700, 512, 64, 1, "dense"), (33, 48, 4096, 1, "dense"), (256, 256, 384, 1, "dense"),
    (1, 64, 64, 4, "one"), (9, 65, 33, 3, "some"), (200, 136, 72, 5, "some"), (64, 40, 24, 130, "all"), (600, 264, 136, 3, "all"),
    (300, 128, 64, 8, "one"), (300, 96, 128, 8, "past"), (50, 24, 16, 1000, "all"), (1500, 384, 192, 2, "all"), (32, 512, 512, 8, "all"),
]


@pytest.mark.parametrize("rows,n,k,experts,kind", SHAPES)
@pytest.mark.parametrize("dt,a,gated,bias,residual,f32,keep,tight", [
    ("bf16", "none", False, False, False, True, False, True), ("bf16", "silu", True, True, False, False, True, True),
    ("f16", "gelu", False, True, True, False, True, False), ("f16", "silu", True, False, True, True, False, False),
    ("bf16", "gelu", True, True, True, False, True, False),
])
def test_linear(gpu, rows, n, k, experts, kind, dt, a, gated, bias, residual, f32, keep, tight):
    nm = gpu
    rng = np.random.default_rng(rows + 7 * n + k)
    o = segments(rng, rows, experts, kind)
    pad = 0 if tight else 8 if k % 8 == 0 else 3      # rows that stay multiples of 16 bytes, and others
    W = Stack(nm, rng, experts, n, k, dt, ld=k + pad if pad else 0, gap=8 if pad else 0, bias=bias)
    U = Stack(nm, rng, experts, n, k, dt, ld=k + 2 * pad if pad else 0, gap=16 if pad else 0, bias=bias) if gated else None
    x = Rows(nm, rng.standard_normal((rows, k)).astype(np.float32), dt, k + pad)
    xv = values(x.start[:-1, :k], dt)
    od = "f32" if f32 else dt
    r = Rows(nm, rng.standard_normal((rows, n)).astype(np.float32), od, n + 1) if residual else None
    out = Rows(nm, np.full((rows, n), 9.0, np.float32), od, 0 if tight else n + 5)
    pre, pre_up = ([Rows(nm, np.full((rows, n), 9.0, np.float32), dt, 0 if tight else n + 3) for _ in range(2)] if keep
                   else (None, None))
    live = spans(o, rows, experts)
    if o is not None:   # what rows that are no expert's hold does not matter
        raw = x.start[:-1].copy()
        raw[live[-1][1].stop:] = raw_of(np.full(1, np.nan), dt)[0]
        x.buf.upload(raw)
    print(f"[linear {rows} {n} {k} {experts} {kind} {dt} {a}]", flush=True)
    nm.linear(W.w, x.ptr, rows, out.ptr, up=U.w if gated else None, offsets=off(nm, o), act=ACTS[a],
              residual=r.ptr if residual else None, out_dtype=dtype_of(nm, od), pre=pre.ptr if keep else None,
              pre_up=pre_up.ptr if keep and gated else None, x_ld=x.ld, residual_ld=r.ld if residual else 0, out_ld=out.ld,
              pre_ld=pre.ld if keep else 0)
    want, bound = np.full((rows, n), 9.0), np.zeros((rows, n))
    p9, q9, pb, qb = (np.full((rows, n), v) for v in (9.0, 9.0, 0.0, 0.0))
    for e, s in live:
        p, dp = xv[s] @ W.v[e].T, np.abs(xv[s]) @ np.abs(W.v[e].T)
        if bias:
            p, dp = p + W.b[e], dp + np.abs(W.b[e])
        dp = (k + 4) * ULP * dp
        v = act(a, p)[0]
        dv = act_error(a, p, dp)[0]
        p9[s], pb[s] = p, dp
        if gated:
            q, dq = xv[s] @ U.v[e].T, np.abs(xv[s]) @ np.abs(U.v[e].T)
            if bias:
                q, dq = q + U.b[e], dq + np.abs(U.b[e])
            dq = (k + 4) * ULP * dq
            q9[s], qb[s] = q, dq
            v, dv = v * q, dv * (np.abs(q) + dq) + np.abs(v) * dq + ULP * np.abs(v * q)
        if residual:
            rv = values(r.start[:-1, :n], od)[s]
            v, dv = v + rv, dv + ULP * (np.abs(v) + np.abs(rv))
        want[s], bound[s] = v, dv
    close(out.get(), want, bound, od)
    if keep:
        close(pre.get(), p9, pb, dt)
        close(pre_up.get(), q9 if gated else np.full((rows, n), 9.0), qb, dt)


@pytest.mark.parametrize("shift", [1, 4])
def test_linear_off_alignment(gpu, shift):
    """Rows and weights of lengths that are multiples of 16 bytes, at addresses that are not."""
    nm = gpu
    rng = np.random.default_rng(shift)
    rows, n, k = 70, 72, 96
    W = Stack(nm, rng, 1, n, k, "bf16", shift=shift, bias=False)
    x = Rows(nm, rng.standard_normal((rows, k)).astype(np.float32), "bf16", 0, shift)
    out = Rows(nm, np.zeros((rows, n), np.float32), "f32")
    nm.linear(W.w, x.ptr, rows, out.ptr, out_dtype=nm.F32)
    xv = values(x.start[:-1, :k], "bf16")
    close(out.get(), xv @ W.v[0].T, (k + 4) * ULP * (np.abs(xv) @ np.abs(W.v[0].T)), "f32")


def test_linear_residual_in_place(gpu):
    nm = gpu
    rng = np.random.default_rng(5)
    rows, n, k = 150, 200, 64
    W = Stack(nm, rng, 1, n, k, "bf16")
    x = Rows(nm, rng.standard_normal((rows, k)).astype(np.float32), "bf16")
    a, b = (Rows(nm, rng.standard_normal((rows, n)).astype(np.float32), "bf16", n + 8) for _ in range(2))
    b.buf.upload(a.start)
    nm.linear(W.w, x.ptr, rows, a.ptr, residual=a.ptr, residual_ld=a.ld, out_ld=a.ld)
    c = Rows(nm, np.zeros((rows, n), np.float32), "bf16")
    nm.linear(W.w, x.ptr, rows, c.ptr, residual=b.ptr, residual_ld=b.ld)
    assert np.array_equal(a.raw(), c.raw())


@pytest.mark.parametrize("rows", [3, 40, 300])
def test_not_a_number_stays_in_its_row_and_expert(gpu, rows):
    nm = gpu
    rng = np.random.default_rng(rows)
    experts, n, k = 3, 136, 72
    o = np.array([0, rows // 3, 2 * rows // 3, rows], np.uint32)
    W = Stack(nm, rng, experts, n, k, "bf16", bias=False)
    W.v[1, 5, 3], W.v[1, 9, 0] = np.nan, np.inf
    W.buf.upload(raw_of(W.v, "bf16")[0])
    xv = rng.standard_normal((rows, k)).astype(np.float32)
    xv[0, 70], xv[rows - 1, 1] = np.inf, np.nan
    x, out = Rows(nm, xv, "bf16"), Rows(nm, np.zeros((rows, n), np.float32), "f32")
    nm.linear(W.w, x.ptr, rows, out.ptr, offsets=off(nm, o), out_dtype=nm.F32)
    got, xf = out.get(), values(x.start[:-1], "bf16")
    with np.errstate(invalid="ignore"):
        want = np.concatenate([xf[s] @ W.v[e].T for e, s in spans(o, rows, experts)])
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(want))
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])


@pytest.mark.parametrize("rows,n,k,experts,kind", SHAPES)
@pytest.mark.parametrize("dt,dual,mode,a,f32,tight", [
    ("bf16", False, "plain", "none", True, True), ("f16", True, "add", "none", False, False), ("bf16", False, "pre", "gelu", False, True),
    ("f16", False, "pair", "silu", False, False), ("bf16", True, "pair", "gelu", True, True), ("bf16", True, "add", "none", True, False),
])
def test_input_grad(gpu, rows, n, k, experts, kind, dt, dual, mode, a, f32, tight):
    nm = gpu
    rng = np.random.default_rng(rows + 7 * n + k)
    o = segments(rng, rows, experts, kind)
    pad = 0 if tight else 8 if n % 8 == 0 and k % 8 == 0 else 3
    W = Stack(nm, rng, experts, n, k, dt, ld=k + pad if pad else 0, gap=8 if pad else 0)
    U = Stack(nm, rng, experts, n, k, dt, ld=k + 2 * pad if pad else 0, gap=16 if pad else 0)
    normal = lambda width, t, ld=0: Rows(nm, rng.standard_normal((rows, width)).astype(np.float32), t, ld)  # noqa: E731
    dy, dy_up = (normal(n, dt, n + pad) for _ in range(2))
    live = spans(o, rows, experts)
    for d in (dy, dy_up):
        if o is not None:
            raw = d.start[:-1].copy()
            raw[live[-1][1].stop:] = raw_of(np.full(1, np.nan), dt)[0]
            d.buf.upload(raw)
    xd = "f32" if f32 else dt
    dx, dx_up = (normal(k, xd, 0 if tight else k + 5) for _ in range(2))
    pre, pre_up = (normal(k, dt, 0 if tight else k + 3) for _ in range(2))
    has, pair = mode in ("pre", "pair"), mode == "pair"
    print(f"[input grad {rows} {n} {k} {experts} {kind} {dt} {mode}]", flush=True)
    nm.linear_input_grad(W.w, dy.ptr, rows, dx.ptr, up=U.w if dual else None, dy_up=dy_up.ptr if dual else None,
                         offsets=off(nm, o), act=ACTS[a], pre=pre.ptr if has else None, pre_up=pre_up.ptr if pair else None,
                         dx_up=dx_up.ptr if pair else None, dx_dtype=dtype_of(nm, xd), accumulate=mode == "add", dy_ld=dy.ld,
                         pre_ld=pre.ld, dx_ld=dx.ld)
    start, start_up = (values(d.start[:-1, :k], xd) for d in (dx, dx_up))
    want, want_up, bound, bound_up = start.copy(), start_up.copy(), np.zeros((rows, k)), np.zeros((rows, k))
    dv, du = values(dy.start[:-1, :n], dt), values(dy_up.start[:-1, :n], dt)
    for e, s in live:
        g, eg = dv[s] @ W.v[e], np.abs(dv[s]) @ np.abs(W.v[e])
        if dual:
            g, eg = g + du[s] @ U.v[e], eg + np.abs(du[s]) @ np.abs(U.v[e])
        eg = ((2 if dual else 1) * n + 4) * ULP * eg
        if mode == "add":
            want[s], bound[s] = start[s] + g, eg + ULP * np.abs(start[s])
        elif not has:
            want[s], bound[s] = g, eg
        else:
            p, q = values(pre.start[:-1, :k], dt)[s], values(pre_up.start[:-1, :k], dt)[s] if pair else 1.0
            v, slope = act(a, p)
            ev, es = act_error(a, p, np.zeros_like(p))
            want[s] = g * slope * q
            bound[s] = (eg * (np.abs(slope) + es) + np.abs(g) * es) * np.abs(q) + 4 * ULP * np.abs(want[s])
            if pair:
                want_up[s] = g * v
                bound_up[s] = eg * (np.abs(v) + ev) + np.abs(g) * ev + 4 * ULP * np.abs(want_up[s])
    close(dx.get(), want, bound, xd)
    close(dx_up.get(), want_up, bound_up, xd)


@pytest.mark.parametrize("rows,n,k,experts,kind", SHAPES + [(0, 24, 40, 1, "dense"), (0, 24, 40, 3, "all"), (5000, 40, 24, 1, "dense"),
                                                            (9001, 130, 70, 2, "all")])
@pytest.mark.parametrize("dt,f32,acc,bias,tight", [("bf16", True, False, True, True), ("f16", False, True, True, False),
                                                   ("f16", True, True, False, False), ("bf16", False, False, True, True)])
def test_weight_grad(gpu, rows, n, k, experts, kind, dt, f32, acc, bias, tight):
    nm = gpu
    rng = np.random.default_rng(rows + 7 * n + k)
    o = segments(rng, rows, experts, kind)
    pad = 0 if tight else 8 if n % 8 == 0 and k % 8 == 0 else 3
    dy = Rows(nm, rng.standard_normal((rows, n)).astype(np.float32), dt, n + pad)
    x = Rows(nm, rng.standard_normal((rows, k)).astype(np.float32), dt, k + pad)
    live = spans(o, rows, experts)
    for d in (dy, x):
        if o is not None:
            raw = d.start[:-1].copy()
            raw[live[-1][1].stop:] = raw_of(np.full(1, np.nan), dt)[0]
            d.buf.upload(raw)
    wd = "f32" if f32 else dt
    ld, gap = (0, 0) if tight else (k + 3, 1)
    stride = n * (ld or k) + gap
    dw = Rows(nm, rng.standard_normal((experts, stride)).astype(np.float32), wd)
    db = Rows(nm, rng.standard_normal((experts, n)).astype(np.float32), "f32")
    print(f"[weight grad {rows} {n} {k} {experts} {kind} {dt}]", flush=True)
    nm.linear_weight_grad(dy.ptr, x.ptr, dtype_of(nm, dt), rows, n, k, dw.ptr, experts=experts, offsets=off(nm, o),
                          dw_dtype=dtype_of(nm, wd), dbias=db.ptr if bias else None, accumulate=acc, dy_ld=dy.ld, x_ld=x.ld, ld=ld,
                          stride=stride if gap else 0)
    start = values(dw.start[:-1], wd)[:, :n * (ld or k)].reshape(experts, n, -1)
    whole = dw.get()
    got = whole[:, :n * (ld or k)].reshape(experts, n, -1)
    if ld:                                     # between rows and experts nothing is written
        assert np.array_equal(got[:, :, k:], start[:, :, k:])
        assert np.array_equal(whole[:, n * ld:], values(dw.start[:-1], wd)[:, n * ld:])
    gotb, startb = db.get(), values(db.start[:-1], "f32")
    dv, xv = values(dy.start[:-1, :n], dt), values(x.start[:-1, :k], dt)
    for e, s in live:
        m = max(s.stop - s.start, 0)
        w0, b0 = (start[e, :, :k], startb[e]) if acc else (0.0, 0.0)
        close(got[e, :, :k], w0 + dv[s].T @ xv[s], (m + 4) * ULP * (np.abs(dv[s]).T @ np.abs(xv[s]) + np.abs(w0)), wd)
        if bias:
            close(gotb[e], b0 + dv[s].sum(0), (m + 4) * ULP * (np.abs(dv[s]).sum(0) + np.abs(b0)), "f32")
        else:
            assert np.array_equal(gotb, startb)


@pytest.mark.parametrize("rows,n", [(1, 1), (3, 7), (5, 8), (17, 129), (300, 1408), (2, 4001)])
@pytest.mark.parametrize("dt,a,pair,place", [("f32", "silu", True, True), ("bf16", "gelu", False, False), ("f16", "silu", True, False),
                                             ("f32", "gelu", False, True), ("bf16", "none", True, False)])
def test_act_backward(gpu, rows, n, dt, a, pair, place):
    nm = gpu
    rng = np.random.default_rng(rows + n)
    ld = n + 3
    d, p, q = (Rows(nm, 3 * rng.standard_normal((rows, n)).astype(np.float32), dt, ld) for _ in range(3))
    dp, dq = (p, q) if place else (Rows(nm, np.zeros((rows, n), np.float32), dt, ld) for _ in range(2))
    nm.act_backward(d.ptr, p.ptr, dtype_of(nm, dt), rows, n, ACTS[a], dp.ptr, pre_up=q.ptr if pair else None,
                    dpre_up=dq.ptr if pair else None, ld=ld)
    dv, pv, qv = (values(t.start[:-1, :n], dt) for t in (d, p, q))
    v, slope = act(a, pv)
    ev, es = act_error(a, pv, np.zeros_like(pv))
    f = qv if pair else 1.0
    close(dp.get(), dv * slope * f, np.abs(dv * f) * es + 4 * ULP * np.abs(dv * slope * f), dt)
    if pair:
        close(dq.get(), dv * v, np.abs(dv) * ev + 4 * ULP * np.abs(dv * v), dt)


@pytest.mark.parametrize("v", [-1e4, -200.0, -90.0, -20.0, -0.0, 0.0, 20.0, 90.0, 200.0, 1e4])
def test_activations_far_out(gpu, v):
    """No infinity or NaN from large finite values, and the limits of both activations and their slopes."""
    nm = gpu
    for a in ("silu", "gelu"):
        d, p = Rows(nm, np.ones((1, 8), np.float32), "f32"), Rows(nm, np.full((1, 8), v, np.float32), "f32")
        q = Rows(nm, np.ones((1, 8), np.float32), "f32")
        dp, dq = (Rows(nm, np.zeros((1, 8), np.float32), "f32") for _ in range(2))
        nm.act_backward(d.ptr, p.ptr, nm.F32, 1, 8, ACTS[a], dp.ptr, pre_up=q.ptr, dpre_up=dq.ptr)
        w, slope = act(a, np.full((1, 8), v))
        assert np.abs(dp.get() - slope).max() < 1e-4 and np.abs(dq.get() - w).max() <= 1e-4 * max(1, abs(v))


def test_gradients_against_differences(gpu):
    """<g, out(x + h d) - out(x - h d)> / 2h of the gated product in f32 against the gradients from the calls, for the rows, a
    weight and the biases; x, the weights and the steps are multiples of 2^-6 that bf16 holds."""
    nm = gpu
    rng = np.random.default_rng(8)
    rows, n, k = 24, 40, 32
    grid = lambda *s: (rng.integers(-40, 41, s) / 64).astype(np.float32)  # noqa: E731
    xs, ws, us, b, c, g = grid(rows, k), grid(1, n, k), grid(1, n, k), grid(1, n), grid(1, n), grid(rows, n)

    def run(xs, ws, b):
        x = Rows(nm, xs, "bf16")
        assert np.array_equal(x.get(), xs)
        keep = [nm.DeviceBuffer.from_array(t) for t in (raw_of(ws, "bf16")[0], raw_of(us, "bf16")[0], b, c)]
        W = nm.Weights(keep[0], nm.BF16, 1, n, k, bias=keep[2])
        U = nm.Weights(keep[1], nm.BF16, 1, n, k, bias=keep[3])
        out, pre, pre_up = Rows(nm, np.zeros((rows, n), np.float32), "f32"), *(Rows(nm, np.zeros((rows, n), np.float32), "bf16")
                                                                            for _ in range(2))
        nm.linear(W, x.ptr, rows, out.ptr, up=U, act=nm.ACT_SILU, out_dtype=nm.F32, pre=pre.ptr, pre_up=pre_up.ptr)
        return out.get(), x, W, U, pre, pre_up, keep

    out, x, W, U, pre, pre_up, keep = run(xs, ws, b)
    gd = Rows(nm, g, "bf16")
    dp, dq, dx = (Rows(nm, np.zeros((rows, m), np.float32), t) for m, t in ((n, "bf16"), (n, "bf16"), (k, "f32")))
    nm.act_backward(gd.ptr, pre.ptr, nm.BF16, rows, n, nm.ACT_SILU, dp.ptr, pre_up=pre_up.ptr, dpre_up=dq.ptr)
    nm.linear_input_grad(W, dp.ptr, rows, dx.ptr, up=U, dy_up=dq.ptr, dx_dtype=nm.F32)
    dw, db = Rows(nm, np.zeros((n, k), np.float32), "f32"), Rows(nm, np.zeros((1, n), np.float32), "f32")
    nm.linear_weight_grad(dp.ptr, x.ptr, nm.BF16, rows, n, k, dw.ptr, dbias=db.ptr)
    h = 1 / 64
    for what in ("x", "w", "b"):
        d = rng.choice([-1.0, 1.0], {"x": (rows, k), "w": (1, n, k), "b": (1, n)}[what]).astype(np.float32)
        at = lambda s: run(xs + s * h * d if what == "x" else xs, ws + s * h * d if what == "w" else ws,  # noqa: E731
                           b + s * h * d if what == "b" else b)[0]
        per = g * (at(1) - at(-1)) / (2 * h)
        got = {"x": dx, "w": dw, "b": db}[what].get()
        # Third derivatives of sums of a few units leave h^2 of a value's size; the gradients entered in bf16, 2^-8 of a
        # value each: 2 % of the terms' sizes covers both, added up as squares over the terms.
        assert abs((got * d.reshape(got.shape)).sum() - per.sum()) < 0.02 * np.sqrt((per ** 2).sum()) + 0.02 * abs(per.sum())


def test_captured_and_replayed(gpu):
    """Forward and both gradients of grouped and dense calls in one graph, replayed on new values between eager calls of other
    sizes, on a stream of its own."""
    nm = gpu
    rng = np.random.default_rng(9)
    st = nm.Stream()

    class Calls:
        def __init__(self, rows, n, k, experts):
            self.sizes = rows, n, k, experts
            self.W, self.U = (Stack(nm, rng, experts, n, k, "bf16") for _ in range(2))
            self.x, self.dy = (nm.DeviceBuffer(rows * w * 2) for w in (k, n))
            self.o = nm.DeviceBuffer((experts + 1) * 4)
            zeros = lambda b: nm.DeviceBuffer.from_array(np.zeros(b // 4 + 1, np.uint32))  # noqa: E731
            self.out = [zeros(rows * n * 2) for _ in range(3)] + [zeros(rows * k * 2), zeros(experts * n * k * 4), zeros(experts * n * 4)]

        def fill(self):
            rows, n, k, experts = self.sizes
            for b, w in ((self.x, k), (self.dy, n)):
                b.upload(raw_of(rng.standard_normal((rows, w)), "bf16")[0])
            self.o.upload(segments(rng, rows, experts, "some"))
            nm.synchronize()

        def __call__(self, s):
            rows, n, k, experts = self.sizes
            o, offsets = self.out, self.o if experts > 1 else None
            nm.linear(self.W.w, self.x, rows, o[0], up=self.U.w, offsets=offsets, act=nm.ACT_SILU, pre=o[1], pre_up=o[2], stream=s)
            nm.linear_input_grad(self.W.w, self.dy, rows, o[3], offsets=offsets, stream=s)
            nm.linear_weight_grad(self.dy, self.x, nm.BF16, rows, n, k, o[4], experts=experts, offsets=offsets, dbias=o[5], stream=s)

        def results(self):
            nm.synchronize()
            r = [b.download(np.uint32) for b in self.out]
            for b in self.out:
                b.upload(np.zeros(b.nbytes // 4, np.uint32))
            nm.synchronize()
            return r

    mine = [Calls(3, 96, 64, 1), Calls(200, 136, 72, 4), Calls(20, 64, 2048, 1), Calls(2000, 64, 128, 1)]
    other = Calls(4000, 200, 264, 1)
    for c in mine:
        c.fill()
        c(st.handle)
    st.sync()
    g = Graph(nm, st, lambda: [c(st.handle) for c in mine])
    for _ in range(3):
        for c in mine + [other]:
            c.fill()
            c.results()
        other(0)
        nm.synchronize()
        g.launch()
        st.sync()
        got = [c.results() for c in mine]
        for c, r in zip(mine, got):
            c(0)
            assert all(np.array_equal(a, b) for a, b in zip(r, c.results()))
    g.close()

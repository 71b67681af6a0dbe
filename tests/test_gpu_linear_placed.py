"""Every kernel of the products and their gradients: arguments at addresses that are no multiples of 16 bytes though their rows' lengths
are, residuals in the results' place, segments that begin behind the first row, and NaN and infinity in one row or weight.
Tolerances as in test_gpu_linear; which kernel aligned calls take is asserted."""
import numpy as np
import pytest

import test_linear_rules as rules
from test_gpu_linear import ULP, Stack, off, spans
from test_gpu_tokens import Rows, close, dtype_of, raw_of, values

pytestmark = pytest.mark.gpu

# rows, n, k, experts, the kernel that takes them if aligned (None: rows of odd lengths)
FORWARD = [
    (90, 136, 80, 1, rules.FEW16), (100, 2040, 1048, 1, rules.FEW32), (240, 2040, 1048, 1, rules.FEW64), (29, 8200, 1064, 1, rules.THIN),
    (100, 1000, 1000, 10, rules.THIN), (4500, 1032, 64, 1, rules.SHORT), (700, 1000, 264, 7, rules.SHORT), (600, 2056, 1048, 1, rules.MID),
    (700, 1000, 584, 7, rules.MID), (70, 2056, 4104, 1, rules.MID), (520, 264, 40008, 1, rules.BIG), (520, 16648, 1288, 1, rules.BIG), (780, 2056, 5960, 3, rules.BIG),
    (40, 1003, 1701, 1, None), (300, 1003, 1701, 1, None), (300, 1003, 263, 7, None), (900, 1003, 263, 7, None),
]
INPUT = [
    (29, 1064, 2056, 1, rules.THIN), (100, 1000, 1000, 10, rules.THIN), (4500, 64, 1032, 1, rules.SHORT), (700, 16, 1000, 9, rules.SHORT),
    (600, 1048, 2056, 1, rules.MID), (100, 33000, 264, 1, rules.MID), (900, 5128, 2600, 1, rules.BIG), (1000, 8400, 2056, 3, rules.BIG),
    (40, 1003, 263, 1, None), (300, 1003, 263, 1, None), (900, 263, 1003, 7, None),
]
WEIGHT = [
    (60, 1032, 1000, 1, rules.SHORT), (500, 520, 264, 9, rules.SHORT), (9001, 520, 264, 1, rules.MID), (4000, 520, 264, 9, rules.MID),
    (5003, 1544, 2056, 1, rules.BIG), (3000, 2056, 2600, 3, rules.BIG), (60, 1003, 263, 1, None), (9001, 131, 71, 2, None),
]


def offsets(rows, experts, late=0):
    """Segments of unequal lengths, one of them empty, all from row `late` on and to rows - late."""
    if experts == 1 and not late:
        return None
    w = np.arange(1, experts + 1) * (np.arange(experts) != 2)
    cuts = np.concatenate([[0], np.cumsum(w)]) * (rows - 2 * late) // max(w.sum(), 1)
    return (cuts + late).astype(np.uint32)


def normal(nm, rng, rows, width, dt, ld=0, shift=0):
    return Rows(nm, rng.standard_normal((rows, width)).astype(np.float32), dt, ld, shift)


def of(r, dt):
    return values(r.start[:-1, :r.shape[1]], dt)


def padded(width):
    return (width + 7) // 8 * 8 if width % 8 else width + 8


# ---- addresses: every argument alone, and all, by 2 and by 8 bytes

@pytest.mark.parametrize("rows,n,k,experts,takes", [f for f in FORWARD if f[4] is not None])
@pytest.mark.parametrize("gated,shift,which", [(False, 1, "x"), (False, 4, "w"), (True, 4, "x"), (True, 1, "u"), (True, 1, "out"),
                                               (False, 4, "all"), (True, 4, "all")])
def test_linear_addresses(gpu, rows, n, k, experts, takes, gated, shift, which):
    nm, dt = gpu, "bf16"
    assert gated or rules.forward(rows, 0 if experts == 1 else experts, n, k, False) == takes
    at = lambda name: shift if which in (name, "all") else 0  # noqa: E731
    rng = np.random.default_rng(rows + n)
    o = offsets(rows, experts)
    W, U = Stack(nm, rng, experts, n, k, dt, shift=at("w")), Stack(nm, rng, experts, n, k, dt, shift=at("u"))
    x = normal(nm, rng, rows, k, dt, 0, at("x"))
    r, out, pre, pre_up = (normal(nm, rng, rows, n, dt, n + 8, at("out")) for _ in range(4))
    print(f"[addresses {rows} {n} {k} {experts} {which} {shift}]", flush=True)
    nm.linear(W.w, x.ptr, rows, out.ptr, up=U.w if gated else None, offsets=off(nm, o), residual=r.ptr, pre=pre.ptr,
              pre_up=pre_up.ptr if gated else None, residual_ld=r.ld, out_ld=out.ld, pre_ld=pre.ld)
    xv = of(x, dt)
    want, wp, wq = of(out, dt), of(pre, dt), of(pre_up, dt)
    bound, bp, bq = (np.zeros_like(want) for _ in range(3))
    for e, s in spans(o, rows, experts):
        a = np.abs(xv[s])
        wp[s], bp[s] = xv[s] @ W.v[e].T + W.b[e], (k + 4) * ULP * (a @ np.abs(W.v[e].T) + np.abs(W.b[e]))
        v, dv = wp[s], bp[s]
        if gated:
            wq[s], bq[s] = xv[s] @ U.v[e].T + U.b[e], (k + 4) * ULP * (a @ np.abs(U.v[e].T) + np.abs(U.b[e]))
            v, dv = v * wq[s], dv * (np.abs(wq[s]) + bq[s]) + np.abs(v) * bq[s] + ULP * np.abs(v * wq[s])
        rv = of(r, dt)[s]
        want[s], bound[s] = v + rv, dv + ULP * (np.abs(v) + np.abs(rv))
    close(pre.get(), wp, bp, dt)
    close(pre_up.get(), wq, bq, dt)
    close(out.get(), want, bound, dt)


@pytest.mark.parametrize("rows,n,k,experts,takes", [f for f in INPUT if f[4] is not None])
@pytest.mark.parametrize("dual,shift,which", [(False, 1, "dy"), (False, 4, "w"), (True, 4, "dy_up"), (True, 1, "u"), (True, 1, "dx"),
                                              (False, 4, "all"), (True, 4, "all")])
def test_input_grad_addresses(gpu, rows, n, k, experts, takes, dual, shift, which):
    nm, dt = gpu, "f16"
    assert dual or rules.input_grad(rows, 0 if experts == 1 else experts, n, k, False) == takes
    at = lambda name: shift if which in (name, "all") else 0  # noqa: E731
    rng = np.random.default_rng(rows + n)
    o = offsets(rows, experts)
    W, U = Stack(nm, rng, experts, n, k, dt, shift=at("w")), Stack(nm, rng, experts, n, k, dt, shift=at("u"))
    dy, dy_up = normal(nm, rng, rows, n, dt, 0, at("dy")), normal(nm, rng, rows, n, dt, 0, at("dy_up"))
    dx = normal(nm, rng, rows, k, "f32", k + 8, at("dx"))
    print(f"[addresses {rows} {n} {k} {experts} {which} {shift}]", flush=True)
    nm.linear_input_grad(W.w, dy.ptr, rows, dx.ptr, up=U.w if dual else None, dy_up=dy_up.ptr if dual else None, offsets=off(nm, o),
                         dx_dtype=nm.F32, dx_ld=dx.ld)
    want, dv, du = of(dx, "f32"), of(dy, dt), of(dy_up, dt)
    bound = np.zeros_like(want)
    for e, s in spans(o, rows, experts):
        want[s], size = dv[s] @ W.v[e], np.abs(dv[s]) @ np.abs(W.v[e])
        if dual:
            want[s], size = want[s] + du[s] @ U.v[e], size + np.abs(du[s]) @ np.abs(U.v[e])
        bound[s] = ((2 if dual else 1) * n + 4) * ULP * size
    close(dx.get(), want, bound, "f32")


@pytest.mark.parametrize("rows,n,k,experts,takes", [f for f in WEIGHT if f[4] is not None])
@pytest.mark.parametrize("wd", ["f32", "bf16"])
@pytest.mark.parametrize("shift,which", [(1, "dy"), (4, "x"), (1, "dw"), (4, "all")])
def test_weight_grad_addresses(gpu, rows, n, k, experts, takes, wd, shift, which):
    nm, dt = gpu, "bf16"
    assert rules.weight_grad(rows, experts, n, k) == takes
    at = lambda name: shift if which in (name, "all") else 0  # noqa: E731
    rng = np.random.default_rng(rows + n)
    o = offsets(rows, experts)
    dy, x = normal(nm, rng, rows, n, dt, 0, at("dy")), normal(nm, rng, rows, k, dt, 0, at("x"))
    dw, db = normal(nm, rng, experts, n * k, wd, 0, at("dw")), normal(nm, rng, experts, n, "f32", 0, at("dw"))
    print(f"[addresses {rows} {n} {k} {experts} {which} {shift}]", flush=True)
    nm.linear_weight_grad(dy.ptr, x.ptr, nm.BF16, rows, n, k, dw.ptr, experts=experts, offsets=off(nm, o), dw_dtype=dtype_of(nm, wd),
                          dbias=db.ptr)
    got, gotb, dv, xv = dw.get().reshape(experts, n, k), db.get(), of(dy, dt), of(x, dt)
    for e, s in spans(o, rows, experts):
        m = s.stop - s.start
        close(got[e], dv[s].T @ xv[s], (m + 4) * ULP * (np.abs(dv[s]).T @ np.abs(xv[s])), wd)
        close(gotb[e], dv[s].sum(0), (m + 4) * ULP * np.abs(dv[s]).sum(0), "f32")


# ---- the residual in the result's place: the bits of a call with a copy of it

@pytest.mark.parametrize("rows,n,k,experts,takes", FORWARD)
@pytest.mark.parametrize("gated,od,ld", [(False, "bf16", 0), (True, "f32", 0), (True, "bf16", 5), (False, "f32", 8)])
def test_residual_in_place(gpu, rows, n, k, experts, takes, od, ld, gated):
    nm, dt = gpu, "bf16"
    assert gated or takes is None or rules.forward(rows, 0 if experts == 1 else experts, n, k, False) == takes
    rng = np.random.default_rng(rows + n)
    o = offsets(rows, experts, 3 if experts > 1 else 0)
    W, U = Stack(nm, rng, experts, n, k, dt), Stack(nm, rng, experts, n, k, dt) if gated else None
    x, a = normal(nm, rng, rows, k, dt), normal(nm, rng, rows, n, od, n + ld)
    copy, out = Rows(nm, np.zeros((rows, n), np.float32), od, n + ld), Rows(nm, np.zeros((rows, n), np.float32), od, n + ld)
    copy.buf.upload(a.start), out.buf.upload(a.start)
    copy.start = out.start = a.start
    more = dict(up=U.w if gated else None, offsets=off(nm, o), act=nm.ACT_SILU, out_dtype=dtype_of(nm, od), out_ld=a.ld, residual_ld=a.ld)
    print(f"[in place {rows} {n} {k} {experts} {od}]", flush=True)
    nm.linear(W.w, x.ptr, rows, a.ptr, residual=a.ptr, **more)
    nm.linear(W.w, x.ptr, rows, out.ptr, residual=copy.ptr, **more)
    got, want = a.raw(), out.raw()
    assert np.array_equal(got, want)
    live = np.zeros(rows, bool)
    for _, s in spans(o, rows, experts):
        live[s] = True
    assert np.array_equal(got[~live], a.start[:-1, :n][~live])
    # (half of p is positive or nearly so, and SiLU(p) then moves a residual: the gate's product with it too)
    assert (got[live] != a.start[:-1, :n][live]).mean() > 0.4


# ---- NaN and infinity stay in the results that they have a part in; rows before the first segment and behind the last are not read

def poison(v, *at):
    """v's copy with infinity, NaN, minus infinity, ... at the places that exist."""
    v = v.copy()
    for i, place in enumerate(at):
        v[place] = (np.inf, np.nan, -np.inf)[i % 3]
    return v


def kinds_alike(got, want):
    assert np.array_equal(np.isnan(got), np.isnan(want))
    inf = np.isinf(want)
    assert np.array_equal(np.isinf(got), inf) and np.array_equal(got[inf], want[inf])
    assert 0 < np.isfinite(want).sum() < want.size


def values_of(rng, *shape):
    """Values that bf16 holds, none of them 0."""
    return ((rng.integers(1, 128, shape) * rng.choice([-1, 1], shape)) / 64).astype(np.float32)


def placed(rows, experts):
    o = offsets(rows, experts, 3)
    e = int(np.argmax(np.diff(o.astype(int))))
    return o, e, int(o[e]), int(o[e + 1]) - 1      # the longest segment, its first and last row


@pytest.mark.parametrize("rows,n,k,experts,takes", FORWARD)
def test_not_a_number_in_a_product(gpu, rows, n, k, experts, takes):
    nm = gpu
    rng = np.random.default_rng(rows + n)
    assert takes is None or rules.forward(rows, experts, n, k, False) == takes
    o, e, first, last = placed(rows, experts)
    w = values_of(rng, experts, n, k)
    w[e] = poison(w[e], (0, k - 1), (n - 1, 0), (n // 2, k // 2))
    xv = poison(values_of(rng, rows, k), (last, 0), (first, k - 1), ((first + last) // 2, k // 2))
    xv[:3], xv[rows - 3:] = np.nan, np.inf
    W = nm.Weights(nm.DeviceBuffer.from_array(raw_of(w, "bf16")[0]), nm.BF16, experts, n, k)
    x, out = Rows(nm, xv, "bf16"), Rows(nm, np.full((rows, n), 5.0, np.float32), "f32")
    print(f"[nan {rows} {n} {k} {experts}]", flush=True)
    nm.linear(W, x.ptr, rows, out.ptr, offsets=off(nm, o), out_dtype=nm.F32)
    want = np.full((rows, n), 5.0)
    with np.errstate(invalid="ignore"):
        for i, s in spans(o, rows, experts):
            want[s] = xv[s].astype(np.float64) @ w[i].T.astype(np.float64)
    kinds_alike(out.get(), want)
    assert (out.get()[:3] == 5.0).all() and (out.get()[rows - 3:] == 5.0).all()


@pytest.mark.parametrize("rows,n,k,experts,takes", INPUT)
@pytest.mark.parametrize("dual", [False, True])
def test_not_a_number_in_an_input_gradient(gpu, rows, n, k, experts, takes, dual):
    nm = gpu
    assert takes is None or dual or rules.input_grad(rows, experts, n, k, False) == takes
    rng = np.random.default_rng(rows + n)
    o, e, first, last = placed(rows, experts)
    w, u = values_of(rng, experts, n, k), values_of(rng, experts, n, k)
    w[e] = poison(w[e], (n - 1, 0), (0, k - 1))
    u[e] = poison(u[e], (0, k // 2))
    dy = poison(values_of(rng, rows, n), (last, n - 1), (first, 0))
    dy_up = poison(values_of(rng, rows, n), ((first + last) // 2, n // 2))
    for d in (dy, dy_up):
        d[:3], d[rows - 3:] = np.nan, np.inf
    W, U = (nm.Weights(nm.DeviceBuffer.from_array(raw_of(v, "bf16")[0]), nm.BF16, experts, n, k) for v in (w, u))
    d, d_up, dx = Rows(nm, dy, "bf16"), Rows(nm, dy_up, "bf16"), Rows(nm, np.full((rows, k), 5.0, np.float32), "f32")
    print(f"[nan {rows} {n} {k} {experts} {dual}]", flush=True)
    nm.linear_input_grad(W, d.ptr, rows, dx.ptr, up=U if dual else None, dy_up=d_up.ptr if dual else None, offsets=off(nm, o),
                         dx_dtype=nm.F32)
    want = np.full((rows, k), 5.0)
    with np.errstate(invalid="ignore"):
        for i, s in spans(o, rows, experts):
            want[s] = dy[s].astype(np.float64) @ w[i].astype(np.float64)
            if dual:
                want[s] += dy_up[s].astype(np.float64) @ u[i].astype(np.float64)
    kinds_alike(dx.get(), want)
    assert (dx.get()[:3] == 5.0).all() and (dx.get()[rows - 3:] == 5.0).all()


@pytest.mark.parametrize("rows,n,k,experts,takes", WEIGHT)
@pytest.mark.parametrize("acc", [False, True])
def test_not_a_number_in_a_weight_gradient(gpu, rows, n, k, experts, takes, acc):
    nm = gpu
    assert takes is None or rules.weight_grad(rows, experts, n, k) == takes
    rng = np.random.default_rng(rows + n)
    o, e, first, last = placed(rows, experts)
    dy = poison(values_of(rng, rows, n), (first, 0), (last, n - 1))
    xv = poison(values_of(rng, rows, k), (last, k - 1), (first, 0), ((first + last) // 2, k // 2))
    for d in (dy, xv):
        d[:3], d[rows - 3:] = np.nan, np.inf
    start = values_of(rng, experts, n * k)
    d, x, dw = Rows(nm, dy, "bf16"), Rows(nm, xv, "bf16"), Rows(nm, start, "f32")
    db = Rows(nm, np.zeros((experts, n), np.float32), "f32")
    print(f"[nan {rows} {n} {k} {experts} {acc}]", flush=True)
    nm.linear_weight_grad(d.ptr, x.ptr, nm.BF16, rows, n, k, dw.ptr, experts=experts, offsets=off(nm, o), dbias=db.ptr, accumulate=acc)
    want, wantb = start.reshape(experts, n, k).astype(np.float64) * acc, np.zeros((experts, n))
    with np.errstate(invalid="ignore"):
        for i, s in spans(o, rows, experts):
            want[i] += dy[s].astype(np.float64).T @ xv[s].astype(np.float64)
            wantb[i] = dy[s].astype(np.float64).sum(0)
    kinds_alike(dw.get().reshape(want.shape), want)
    kinds_alike(db.get(), wantb)

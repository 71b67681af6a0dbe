"""The activations and their slopes out to their tails, relative to the value itself, against 64 bits.

With u = v (SiLU) or 1.5957691 (v + 0.044715 v^3) (GELU), s = 1 / (1 + exp(-u)), the activation is v s and its slope s + v u' s (1 - s).
In units of 2^-24, relative: SiLU's u is exact, GELU's errs by 7 (five roundings, two constants, all terms of one sign).  exp(-u) is 2
to the power u log2(e): the product and the constant move the exponent by 1.22 |u|, the power itself by 2; 1 + errs by 1, the
reciprocal by 2, the product with v by 1.  So the activation errs by (1.22 |u| + 6) or (8.22 |u| + 6), call it a: an error in v of a few
half steps does as much.  Where s < 2^-126 the reciprocal may be 0: an absolute 2^-126 |v|, under 2^-119.

The slope, v < 0: s errs by a, 1 - s by a s / (1 - s) + 1 <= a + 1, their product with v u' by 2 a + 1 + 4 (GELU's u' has four
roundings): (s + |v u'| s (1 - s)) (2 a + 6) in all.  v >= 0: s errs by exp(-u) a + 4 and so does 1 - s, now absolutely:
(1 + |v u'|) (exp(-u) a + 5) + 6 |slope|."""
import numpy as np
import pytest

import test_linear_rules as rules
from test_gpu_tokens import Rows, raw_of, values

pytestmark = pytest.mark.gpu

UNIT = 2.0 ** -24
C, D = 1.5957691216057308, 0.044715


def exact(name, v):
    """Activation, slope and their bounds, in f64."""
    u = v if name == "silu" else C * (v + D * v ** 3)
    du = np.ones_like(v) if name == "silu" else C * (1 + 3 * D * v * v)
    with np.errstate(over="ignore", under="ignore"):
        e = np.exp(np.minimum(-u, 700.0))
    s = 1 / (1 + e)
    t = e * s                                   # 1 - s, with nothing lost
    a = ((1.22 if name == "silu" else 8.22) * np.abs(u) + 6) * UNIT
    act, slope = v * s, s + v * du * s * t
    tiny = 2.0 ** -126 * np.abs(v)
    left = (s + np.abs(v * du) * s * t) * (2 * a + 6 * UNIT) + tiny * (1 + du)
    right = (1 + np.abs(v * du)) * (np.minimum(e, 1.0) * a + 5 * UNIT) + 6 * UNIT * np.abs(slope)
    return act, slope, a * np.abs(act) + tiny + 2.0 ** -149, np.where(v < 0, left, right) + 2.0 ** -149


def points():
    near = np.linspace(-12, 12, 4001)
    far = np.linspace(-104, 104, 4001)
    small = np.concatenate([s * np.logspace(-30, 0, 500) for s in (-1, 1)])
    v = np.concatenate([near, far, small, [0.0, -0.0]]).astype(np.float32)
    return v[:v.size // 8 * 8]


@pytest.mark.parametrize("name", ["silu", "gelu"])
def test_gradient_of_the_activation(gpu, name):
    nm = gpu
    v = points()
    rows, n = v.size // 8, 8
    p = Rows(nm, v.reshape(rows, n), "f32")
    one = Rows(nm, np.ones((rows, n), np.float32), "f32")
    slope, act = (Rows(nm, np.zeros((rows, n), np.float32), "f32") for _ in range(2))
    code = {"silu": nm.ACT_SILU, "gelu": nm.ACT_GELU_PYTORCH_TANH}[name]
    nm.act_backward(one.ptr, p.ptr, nm.F32, rows, n, code, slope.ptr, pre_up=one.ptr, dpre_up=act.ptr)
    a, s, ea, es = exact(name, v.astype(np.float64))
    for got, want, bound in ((act, a, ea), (slope, s, es)):
        off = np.abs(got.get().reshape(-1) - want) / bound
        print(f"[{name}: {off.max():.2f} of the bound, at {v[off.argmax()]}]", flush=True)
        assert off.max() <= 1


# rows of one value each times ones: p is the value itself
@pytest.mark.parametrize("name", ["silu", "gelu"])
@pytest.mark.parametrize("copies,n,k,odd,takes", [
    (1, 16, 8, 0, rules.FEW16), (1, 2056, 40, 0, rules.SHORT), (3, 264, 648, 0, rules.MID), (1, 2600, 1600, 0, rules.BIG), (1, 2200, 45, 1, None)])
def test_product(gpu, name, copies, n, k, odd, takes):
    nm = gpu
    v = np.unique(values(raw_of(points(), "bf16")[0], "bf16"))
    v = np.tile(v, copies)
    assert takes in (None, rules.forward(v.size, 0, n, k, False))
    x, w = np.zeros((v.size, k), np.float32), np.zeros((1, n, k), np.float32)
    x[:, k // 2], w[0, :, k // 2] = v, 1.0
    xd, out = Rows(nm, x, "bf16", k + odd, odd), Rows(nm, np.zeros((v.size, n), np.float32), "f32")
    wd = nm.DeviceBuffer.from_array(raw_of(w, "bf16")[0])
    code = {"silu": nm.ACT_SILU, "gelu": nm.ACT_GELU_PYTORCH_TANH}[name]
    nm.linear(nm.Weights(wd, nm.BF16, 1, n, k), xd.ptr, v.size, out.ptr, act=code, out_dtype=nm.F32, x_ld=xd.ld)
    a, _, ea, _ = exact(name, v)
    off = np.abs(out.get() - a[:, None]) / ea[:, None]
    print(f"[{name} {n} {k}: {off.max():.2f} of the bound, at {v[off.argmax() // n]}]", flush=True)
    assert off.max() <= 1

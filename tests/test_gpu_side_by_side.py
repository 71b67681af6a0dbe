"""Arguments that lie side by side in wider rows: a gate's and its up's values as halves of one buffer, inputs and outputs as columns
of another.  They share no memory, so calls take them, and give the bits that they give in buffers of their own."""
import numpy as np
import pytest

from test_gpu_linear import Stack, off, segments
from test_gpu_tokens import dtype_of, np_of, raw_of, routing, sort_ref

pytestmark = pytest.mark.gpu


class Wide:
    """One buffer of rows of several fields' values side by side, or a buffer of such rows for each field (apart)."""

    def __init__(self, nm, rng, rows, widths, dt, apart):
        self.nm, self.rows, self.widths, self.dt, self.ld = nm, rows, widths, dt, sum(widths)
        self.start = raw_of(rng.standard_normal((rows, self.ld)).astype(np.float32), dt)[0]
        self.bufs = [nm.DeviceBuffer.from_array(self.start) for _ in (widths if apart else widths[:1])]
        self.at = np.concatenate([[0], np.cumsum(widths)])

    def __getitem__(self, i):
        return self.bufs[i if len(self.bufs) > 1 else 0].ptr + int(self.at[i]) * self.start.itemsize

    def get(self, i):
        b = self.bufs[i if len(self.bufs) > 1 else 0].download(np_of(self.dt)).reshape(self.start.shape)
        return b[:, self.at[i]:self.at[i + 1]]


def both(run, *changed):
    """run(apart) -> Wide: the fields that the call changed, and those it did not, alike in one buffer and in several."""
    one, several = run(False), run(True)
    for i in range(len(one.widths)):
        assert np.array_equal(one.get(i), several.get(i)), i
        assert np.array_equal(one.get(i), one.start[:, one.at[i]:one.at[i + 1]]) == (i not in changed), i


# rows, n, k, experts: few rows, 128 x 128, 256 x 256, odd rows
SIZES = [(5, 40, 24, 1), (300, 264, 136, 3), (2100, 1544, 1048, 2), (130, 71, 33, 2)]


@pytest.mark.parametrize("rows,n,k,experts", SIZES)
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_linear(gpu, rows, n, k, experts, dt):
    nm = gpu

    def run(apart):
        rng = np.random.default_rng(rows + n)
        o = off(nm, segments(rng, rows, experts, "all" if experts > 1 else "dense"))
        W, U = (Stack(nm, rng, experts, n, k, dt) for _ in range(2))
        f = Wide(nm, rng, rows, [k, n, n, n, n], dt, apart)
        nm.linear(W.w, f[0], rows, f[1], up=U.w, offsets=o, act=nm.ACT_SILU, residual=f[2], pre=f[3], pre_up=f[4], x_ld=f.ld,
                  out_ld=f.ld, residual_ld=f.ld, pre_ld=f.ld)
        return f

    both(run, 1, 3, 4)


@pytest.mark.parametrize("rows,n,k,experts", SIZES)
@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_input_grad(gpu, rows, n, k, experts, dt):
    nm = gpu

    def run(apart):
        rng = np.random.default_rng(rows + n)
        o = off(nm, segments(rng, rows, experts, "all" if experts > 1 else "dense"))
        W, U = (Stack(nm, rng, experts, n, k, dt) for _ in range(2))
        f = Wide(nm, rng, rows, [n, n, k, k, k, k], dt, apart)
        nm.linear_input_grad(W.w, f[0], rows, f[4], up=U.w, dy_up=f[1], offsets=o, act=nm.ACT_SILU, pre=f[2], pre_up=f[3],
                             dx_up=f[5], dy_ld=f.ld, pre_ld=f.ld, dx_ld=f.ld)
        return f

    both(run, 4, 5)


@pytest.mark.parametrize("rows,n", [(3, 9), (40, 128)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_act_backward(gpu, rows, n, dt):
    nm = gpu

    def run(apart):
        f = Wide(nm, np.random.default_rng(n), rows, [n] * 5, dt, apart)
        nm.act_backward(f[0], f[1], dtype_of(nm, dt), rows, n, nm.ACT_SILU, f[3], pre_up=f[2], dpre_up=f[4], ld=f.ld)
        return f

    both(run, 3, 4)


@pytest.mark.parametrize("T,H", [(7, 33), (100, 640)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_tokens(gpu, T, H, dt):
    """With one expert a token, tokens' rows and sorted rows are as many: x, the experts' rows, the sum and the gradient in one."""
    nm = gpu
    d = dtype_of(nm, dt)

    def run(apart):
        rng = np.random.default_rng(T)
        inv = nm.DeviceBuffer.from_array(sort_ref(*routing(rng, T, 1, 4), 4)[1])
        f = Wide(nm, rng, T, [H] * 4, dt, apart)
        nm.tokens_to_experts(f[0], d, inv, T, 1, H, f[1], ld=f.ld, rows_ld=f.ld)
        nm.tokens_from_experts(f[1], d, inv, T, 1, H, f[2], w=None, ld=f.ld, out_ld=f.ld)
        nm.tokens_from_experts_backward(f[0], d, f[1], d, inv, T, 1, H, dy=f[3], dw=nm.DeviceBuffer(T * 4), dout_ld=f.ld, ld=f.ld,
                                        dy_ld=f.ld)
        return f

    both(run, 1, 2, 3)

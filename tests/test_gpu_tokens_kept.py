"""Sums added to what is there: tokens without rows keep their bits, of zeros with a sign and the smallest numbers too."""
import numpy as np
import pytest

from test_gpu_tokens import NO, Rows, dtype_of, np_of

pytestmark = pytest.mark.gpu

SPECIAL = [-0.0, 0.0, np.inf, -np.inf, 2.0 ** -24, -(2.0 ** -24), 2.0 ** -133, -(2.0 ** -133), 1.0, -65504.0]


@pytest.mark.parametrize("H", [5, 8, 64, 1031])
@pytest.mark.parametrize("k", [1, 8, 9])
@pytest.mark.parametrize("dt,od", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("weighted", [False, True])
def test_tokens_without_rows(gpu, H, k, dt, od, weighted):
    nm, T = gpu, 6
    with np.errstate(over="ignore"):
        out = Rows(nm, np.resize(np.array(SPECIAL, np.float32), (T, H)), od)
    inv = np.full((T, k), NO, np.uint32)
    inv[2], inv[4, 0] = T * k, T * k + 7                   # outside the rows: none, either
    y, w = Rows(nm, np.full((T * k, H), np.nan, np.float32), dt), np.full((T, k), -1.0, np.float32)
    invd, wd = nm.DeviceBuffer.from_array(inv), nm.DeviceBuffer.from_array(w)
    nm.tokens_from_experts(y.ptr, dtype_of(nm, dt), invd, T, k, H, out.ptr, w=wd if weighted else None,
                           out_dtype=dtype_of(nm, od), accumulate=True)
    bits = lambda a: np.ascontiguousarray(a).view(np.uint32 if od == "f32" else np.uint16)  # noqa: E731
    assert np.array_equal(bits(out.raw()), bits(out.start[:-1]))


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_tokens_with_fewer_rows_than_pairs(gpu, dt):
    """The pairs without rows add nothing: -0 from a row stays -0 where the sum began with it."""
    nm, T, k, H = gpu, 4, 3, 16
    out, y = (Rows(nm, np.full((n, H), -0.0, np.float32), dt) for n in (T, T * k))
    inv = np.full((T, k), NO, np.uint32)
    inv[:, 1] = np.arange(T)
    invd = nm.DeviceBuffer.from_array(inv)
    nm.tokens_from_experts(y.ptr, dtype_of(nm, dt), invd, T, k, H, out.ptr, accumulate=True)
    assert np.array_equal(np.signbit(raw_f32(out.raw(), dt)), np.ones((T, H), bool))


def raw_f32(raw, dt):
    return raw if np_of(dt) is np.float32 else (raw.astype(np.uint32) << 16).view(np.float32)

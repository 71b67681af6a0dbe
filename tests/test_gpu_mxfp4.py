"""MXFP4 on the device: quantisation bit for bit, and the expert products against 64 bits.

Tolerance of the products.  An activation enters in planes of E2M3 whose last rounding has
steps of at most 2^-2 2^(-5 (P - 1)) where the block's largest magnitude M is at least 2
(csrc/mxfp4_experts.hip): an error of rms at most 2^-3 2^(-5 (P - 1)) / sqrt(12) M, that is
3.4e-8 M for 5 planes (f32 x, h); bf16 x in 4 planes is exact but for values under 2^-12 M.
In a block of normal values M is about 2.5 times the rms, for h up to 5 times: 2e-7 of a
value.  f32 sums of K products add about sqrt(K) 2^-24, 4e-6 at K 4096 and 1.1e-5 at 33024 if
the additions' errors were all of the size of the whole sum; partial sums grow as they are
added, which halves that: 6e-6.  Gate and up enter as a product, down on top: as squares at
most sqrt(2 * 6^2 + 4^2) 1e-6 = 9.4e-6; 1e-5 holds every case.
"""
import numpy as np
import pytest

import mxfp4_ref as M

pytestmark = pytest.mark.gpu

REL = 1e-5


def bf16(a):
    """f32 values rounded to bf16, as bits."""
    b = np.ascontiguousarray(a, np.float32).view(np.uint32).astype(np.uint64)
    nan = (b & 0x7FFFFFFF) > 0x7F800000
    return np.where(nan, (b >> 16) | 0x40, (b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def f32_of(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


def rel(got, want):
    return np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-300)


# ---- quantisation ---------------------------------------------------------------------------


def awkward(rng, n, k):
    """Rows with ties, saturation, zeros, subnormals, the largest finite values and signs of zero."""
    x = rng.standard_normal((n, k)).astype(np.float32)
    x[0, :32] = np.arange(32) * 0.25                      # ties of the codes (largest 7.75: above 6)
    x[1, :32] = -np.arange(32) * 0.125
    x[2, :32] = 0
    x[2, 1::2][:16] = -0.0
    x[3, :32] = rng.standard_normal(32) * 1e-39           # subnormal
    x[4, :32] = rng.standard_normal(32) * 1e38
    x[4, 5] = 3.4028235e38
    x[5, :32] = 2.0 ** np.arange(-20, 12)
    return x


@pytest.mark.parametrize("batch,n,k", [(1, 16, 32), (1, 32, 96), (2, 16, 128), (1, 48, 672), (3, 16, 512), (1, 16, 8192),
                                       (2, 2048, 1408)])
@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
def test_quantize_bit_for_bit(gpu, batch, n, k, dt):
    nm = gpu
    rng = np.random.default_rng(n + k)
    x = np.stack([awkward(rng, n, k) for _ in range(batch)])
    if dt == "bf16":
        raw = bf16(x)
        x = f32_of(raw)
    elif dt == "f16":
        with np.errstate(over="ignore"):
            raw = np.clip(x, -65504, 65504).astype(np.float16)
        x = raw.astype(np.float32)
    else:
        raw = x
    size = nm.projection_bytes(nm.MXFP4_T, n, k)
    src = nm.DeviceBuffer.from_array(raw)
    packed = nm.DeviceBuffer.from_array(np.full(batch * size, 0xA5, np.uint8))
    ids = {"f32": nm.F32, "bf16": nm.BF16, "f16": nm.F16}
    print(f"[quantize {batch} {n} {k} {dt}]", flush=True)
    nm.mxfp4_quantize(src, ids[dt], n, k, packed, batch=batch)
    got = packed.download(np.uint8).reshape(batch, size)
    for b in range(batch):
        code, s = M.quantize(x[b])
        assert np.array_equal(got[b], M.tiled(code, s))
        want = M.values(code, s)
    back = nm.DeviceBuffer(batch * n * k * 4)
    nm.mxfp4_dequantize(packed, n, k, back, nm.F32, batch=batch)
    v = back.download(np.float32).reshape(batch, n, k)
    assert np.array_equal(v[-1].view(np.uint32), want.astype(np.float32).view(np.uint32))
    nm.mxfp4_dequantize(packed, n, k, back, nm.BF16, batch=batch)
    v = back.download(np.uint16, batch * n * k).reshape(batch, n, k)
    assert np.array_equal(v[-1], bf16(want.astype(np.float32)))


def test_quantize_strides_and_bad_values(gpu):
    """Rows and projections apart, bytes between them left alone; NaN and infinities make their block NaN."""
    nm = gpu
    batch, n, k, ld, gap = 2, 16, 160, 176, 16 * 176 + 8
    rng = np.random.default_rng(3)
    x = rng.standard_normal(batch * gap).astype(np.float32)
    at = lambda b, r, c: b * gap + r * ld + c  # noqa: E731
    x[at(0, 3, 40)], x[at(0, 5, 100)], x[at(1, 0, 0)], x[at(1, 15, 159)] = np.nan, np.inf, -np.inf, np.nan
    rows = [np.stack([x[at(b, r, 0):at(b, r, k)] for r in range(n)]) for b in range(batch)]
    size = nm.projection_bytes(nm.MXFP4_T, n, k)
    dst = np.full(batch * (size + 64), 0xEE, np.uint8)
    src, out = nm.DeviceBuffer.from_array(x), nm.DeviceBuffer.from_array(dst)
    nm.mxfp4_quantize(src, nm.F32, n, k, out, batch=batch, ld=ld, src_stride=gap, dst_stride=size + 64)
    got = out.download(np.uint8).reshape(batch, size + 64)
    assert (got[:, size:] == 0xEE).all()
    for b in range(batch):
        code, s = M.quantize(rows[b])
        assert np.array_equal(got[b, :size], M.tiled(code, s))
    y = np.full(batch * gap, 7.0, np.float32)
    back = nm.DeviceBuffer.from_array(y)
    nm.mxfp4_dequantize(out, n, k, back, nm.F32, batch=batch, ld=ld, src_stride=size + 64, dst_stride=gap)
    v = back.download(np.float32)
    seen = np.zeros(v.size, bool)
    for b in range(batch):
        want = M.values(*M.quantize(rows[b]))
        for r in range(n):
            np.testing.assert_array_equal(v[at(b, r, 0):at(b, r, k)], want[r].astype(np.float32))
            seen[at(b, r, 0):at(b, r, k)] = True
    assert (v[~seen] == 7.0).all() and np.isnan(v).sum() == 4 * 32


# ---- the expert products --------------------------------------------------------------------


class Experts:
    """E random experts in tile-order banks and in f64."""

    def __init__(self, nm, seed, E, H, I, std=0.05, contiguous=False):
        rng = np.random.default_rng(seed)
        self.banks = nm.LayerBanks(E, H, I, (nm.MXFP4_T,) * 3, contiguous=contiguous)
        self.w = [[], [], []]
        for e in range(E):
            tiles = []
            for p, (n, k) in enumerate(((I, H), (I, H), (H, I))):
                code, s = M.quantize((rng.standard_normal((n, k)) * std).astype(np.float32))
                self.w[p].append(M.values(code, s))
                tiles.append(M.tiled(code, s))
            self.banks.load(e, *tiles)


def route(rng, T, E, k, drop=0.0, past=None):
    ids = np.stack([rng.permutation(E)[:k] for _ in range(T)]).astype(np.uint32) if k <= E else \
        rng.integers(0, E, (T, k)).astype(np.uint32)
    w = rng.random((T, k)).astype(np.float32) + 0.1
    out = rng.random((T, k)) < drop
    if past is None:
        ids[out], w[out] = 0, 0
    else:
        ids[out] = past
    return ids, w


def decode(nm, ex, x, ids, w, act="silu", out0=None, f32=False, noalloc=False):
    T, k = ids.shape
    H = x.shape[1]
    xd = nm.DeviceBuffer.from_array(x.astype(np.float32) if f32 else bf16(x))
    out = nm.DeviceBuffer.from_array(np.full((T, H), np.nan, np.float32) if out0 is None else out0)
    a = nm.ACT_SILU if act == "silu" else nm.ACT_GELU_PYTORCH_TANH
    idd, wd = nm.DeviceBuffer.from_array(ids), nm.DeviceBuffer.from_array(w)
    if noalloc:
        import ctypes as C
        g, u, d = ex.banks.gate.desc(), ex.banks.up.desc(), ex.banks.down.desc()
        nm._lib.check(nm.lib().naiwa_moe_decode_noalloc(C.byref(g), C.byref(u), C.byref(d), xd.ptr,
                                                        nm.F32 if f32 else nm.BF16, idd.ptr, wd.ptr, T, k, a, out.ptr,
                                                        0 if out0 is None else 1, 0), "noalloc")
    else:
        nm.indexed_moe_fused_decode(ex.banks, xd, nm.F32 if f32 else nm.BF16, idd, wd, T, k, out, act=a,
                                    accumulate=out0 is not None)
    return out.download(np.float32).reshape(T, H)


@pytest.mark.parametrize("T,E,H,I,k", [
    (1, 1, 32, 32, 1), (1, 8, 1024, 2048, 2), (1, 16, 2048, 768, 8), (2, 4, 160, 96, 3), (3, 8, 672, 1408, 6),
    (5, 8, 2048, 1408, 6), (16, 4, 512, 512, 2), (17, 2, 416, 224, 1), (33, 3, 288, 160, 2), (64, 4, 2880, 736, 2),
    (130, 4, 256, 128, 3), (96, 16, 544, 96, 8), (7, 2, 64, 4096, 2),
    (9, 2, 4256, 1056, 2),     # 33.25 steps of x: a last group of two
    (5, 3, 96, 2080, 2),       # h in two unequal K parts
    (300, 8, 128, 96, 4),      # more pairs than are sorted beside the planes
    (1, 8, 128, 4096, 8),      # one token whose h fills more than LDS
    (1, 1, 33024, 32, 1),      # and whose x does
    (1, 3, 64, 10496, 3), (1, 1, 32256, 32, 1),   # one token whose h and whose x just fit
    (1, 2, 64, 12288, 2), (1, 1, 24576, 32, 1),
    (1, 2, 11008, 64, 2), (2, 64, 64, 32, 64),
    (8, 8, 96, 64, 2), (4, 16, 288, 160, 6), (3, 8, 544, 736, 5),   # few tokens by pair
    (2, 1, 96, 64, 2), (4, 4, 288, 160, 3),    # as few in tiles
    (2, 8, 64, 4096, 8), (2, 2, 33024, 32, 2),  # by pair but for h and x that fill more than LDS
])
@pytest.mark.parametrize("f32", [False, True])
def test_decode_against_64_bits(gpu, T, E, H, I, k, f32):
    rng = np.random.default_rng(T * H + I)
    print(f"[decode {T} {E} {H} {I} {k} {f32}]", flush=True)
    ex = Experts(gpu, 11, E, H, I)
    x = rng.standard_normal((T, H)).astype(np.float32)
    if not f32:
        x = f32_of(bf16(x))
    ids, w = route(rng, T, E, k, drop=0.2 if T > 4 else 0.0)
    want = M.experts(x, ids, w, *ex.w)
    got = decode(gpu, ex, x, ids, w, f32=f32)
    assert rel(got, want) < REL


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_decode_accumulates_and_noalloc_agrees(gpu, act):
    rng = np.random.default_rng(4)
    T, E, H, I, k = 6, 4, 384, 160, 3
    ex = Experts(gpu, 12, E, H, I, contiguous=True)
    x = f32_of(bf16(rng.standard_normal((T, H))))
    ids, w = route(rng, T, E, k)
    out0 = rng.standard_normal((T, H)).astype(np.float32)
    want = M.experts(x, ids, w, *ex.w, name=act, out0=out0)
    got = decode(gpu, ex, x, ids, w, act=act, out0=out0)
    assert rel(got, want) < REL
    assert np.array_equal(decode(gpu, ex, x, ids, w, act=act, out0=out0, noalloc=True), got)


@pytest.mark.parametrize("T", [1, 3, 40])
def test_decode_split_by_slot_gives_the_same_bits(gpu, T):
    """A call over the pairs of low slots and an accumulating one over the rest add the same terms in the
    same order as one call."""
    rng = np.random.default_rng(T)
    E, H, I, k = 8, 256, 128, 4
    ex = Experts(gpu, 13, E, H, I)
    x = f32_of(bf16(rng.standard_normal((T, H))))
    ids, w = route(rng, T, E, k)
    whole = decode(gpu, ex, x, ids, w)
    low = decode(gpu, ex, x, np.where(ids < 4, ids, 0), np.where(ids < 4, w, 0).astype(np.float32))
    both = decode(gpu, ex, x, np.where(ids < 4, 0, ids).astype(np.uint32), np.where(ids < 4, 0, w).astype(np.float32),
                  out0=low)
    assert np.array_equal(both, whole)


def test_decode_edges(gpu):
    """No pairs, no valid pair, the same slot twice, ids past the bank, width 0, a row of zeros."""
    rng = np.random.default_rng(6)
    T, E, H, I, k = 5, 4, 192, 64, 3
    ex = Experts(gpu, 14, E, H, I)
    x = f32_of(bf16(rng.standard_normal((T, H))))
    x[4] = 0
    ids, w = route(rng, T, E, k)
    w[0] = 0                              # a token without experts
    ids[1] = 2                            # one expert three times
    ids[2, 1] = E                         # past the bank: nothing
    ids[3, 0] = 0xFFFFFFFF
    want = M.experts(x, np.where(ids >= E, E, ids), w, *ex.w)
    got = decode(gpu, ex, x, ids, w)
    assert rel(got, want) < REL and (got[0] == 0).all() and (got[4] == 0).all()
    none = decode(gpu, ex, x, ids, np.zeros_like(w))
    assert (none == 0).all()
    # width 0: zeros, or out as it is
    nm = gpu
    xd, out = nm.DeviceBuffer.from_array(bf16(x)), nm.DeviceBuffer.from_array(np.ones((T, H), np.float32))
    nm.indexed_moe_fused_decode(ex.banks, xd, nm.BF16, 0, 0, T, 0, out, accumulate=True)
    assert (out.download(np.float32) == 1).all()
    nm.indexed_moe_fused_decode(ex.banks, xd, nm.BF16, 0, 0, T, 0, out)
    assert (out.download(np.float32) == 0).all()


def test_nan_and_infinity_stay_in_their_row(gpu):
    rng = np.random.default_rng(7)
    T, E, H, I, k = 20, 2, 256, 64, 2
    ex = Experts(gpu, 15, E, H, I)
    x = f32_of(bf16(rng.standard_normal((T, H))))
    ids, w = route(rng, T, E, k)
    clean = decode(gpu, ex, x, ids, w)
    x[3, 100], x[11, 255] = np.nan, np.inf
    got = decode(gpu, ex, x, ids, w)
    assert np.isnan(got[3]).all() and np.isnan(got[11]).all()
    keep = [t for t in range(T) if t not in (3, 11)]
    assert np.array_equal(got[keep], clean[keep])
    # an expert with a NaN weight block reaches only the tokens that chose it, and weight 0 does not choose
    nm = gpu
    code, s = M.quantize(np.zeros((I, H), np.float32))
    s[5, 1] = 255
    ex.banks.gate.write_slot(1, M.tiled(code, s))
    x = f32_of(bf16(rng.standard_normal((T, H))))
    ids = np.zeros((T, 1), np.uint32)
    w = np.ones((T, 1), np.float32)
    ids[4], ids[9], w[9] = 1, 1, 0
    got = decode(gpu, ex, x, ids, w)
    assert np.isnan(got[4]).all() and (got[9] == 0).all() and np.isfinite(np.delete(got, 4, 0)).all()


@pytest.mark.parametrize("f32", [False, True])
def test_wide_ranges_within_a_block(gpu, f32):
    """Rows of very large and very small scale, and outliers of up to 2^6 times 4 in every block that half of
    the weights do not see: a value is held to 2^-19 of its block's largest, 2^-19 2^8 = 4.9e-4 of the rest."""
    rng = np.random.default_rng(8)
    T, E, H, I, k = 6, 2, 512, 64, 1
    ex = Experts(gpu, 16, E, H, I)
    x = rng.standard_normal((T, H))
    x[:, ::32] *= 64.0
    x[1] *= 2.0 ** 30
    x[2] *= 2.0 ** -40
    x = f32_of(bf16(x)) if not f32 else x.astype(np.float32)
    for e in range(E):
        for p in (0, 1):
            code, s = M.quantize((rng.standard_normal((I, H)) * 0.05).astype(np.float32))
            code[::2, ::32] = 0
            ex.w[p][e] = M.values(code, s)
            (ex.banks.gate, ex.banks.up)[p].write_slot(e, M.tiled(code, s))
    ids, w = route(rng, T, E, k)
    # the down rows see the features without outliers alone
    for e in range(E):
        code, s = M.quantize((rng.standard_normal((H, I)) * 0.05).astype(np.float32))
        code[:, 1::2] = 0
        ex.w[2][e] = M.values(code, s)
        ex.banks.down.write_slot(e, M.tiled(code, s))
    want = M.experts(x, ids, w, *ex.w)
    got = decode(gpu, ex, x, ids, w, f32=f32)
    for t in range(T):
        assert np.isfinite(want[t]).all() and rel(got[t], want[t]) < 2 * 4.9e-4, t   # gate and up


def prefill(nm, ex, x, ids, w, act="silu", out0=None, residual=False):
    T, k = ids.shape
    H = x.shape[1]
    xd = nm.DeviceBuffer.from_array(bf16(x))
    out = nm.DeviceBuffer.from_array(np.full((T, H), np.nan, np.float32) if out0 is None else out0)
    a = nm.ACT_SILU if act == "silu" else nm.ACT_GELU_PYTORCH_TANH
    nm.moe_prefill(ex.banks, xd, nm.DeviceBuffer.from_array(ids), nm.DeviceBuffer.from_array(w), T, k, out, act=a,
                   accumulate=out0 is not None, residual=residual)
    return out.download(np.float32).reshape(T, H), f32_of(xd.download(np.uint16)).reshape(T, H)


@pytest.mark.parametrize("T,E,H,I,k,act", [
    (1, 1, 32, 32, 1, "silu"), (3, 8, 160, 96, 2, "gelu"), (63, 4, 160, 96, 2, "silu"), (64, 1, 128, 128, 1, "gelu"), (65, 2, 288, 224, 1, "silu"),
    (129, 3, 512, 416, 3, "silu"), (300, 8, 672, 160, 6, "gelu"), (512, 4, 256, 1408, 2, "silu"),
    (700, 2, 1056, 96, 2, "silu"), (2048, 16, 96, 64, 8, "silu"), (200, 1, 2048, 768, 1, "silu"),
])
def test_prefill_against_64_bits(gpu, T, E, H, I, k, act):
    rng = np.random.default_rng(T + H)
    print(f"[prefill {T} {E} {H} {I} {k}]", flush=True)
    ex = Experts(gpu, 21, E, H, I)
    x = f32_of(bf16(rng.standard_normal((T, H))))
    ids, w = route(rng, T, E, k, drop=0.15 if T > 100 else 0.0, past=E)
    want = M.experts(x, ids, w, *ex.w, name=act, skip_zero=False)
    got, _ = prefill(gpu, ex, x, ids, w, act=act)
    assert rel(got, want) < REL


def test_prefill_accumulate_and_residual(gpu):
    rng = np.random.default_rng(31)
    T, E, H, I, k = 150, 4, 352, 192, 2
    ex = Experts(gpu, 22, E, H, I)
    x = f32_of(bf16(rng.standard_normal((T, H))))
    ids, w = route(rng, T, E, k)
    out0 = rng.standard_normal((T, H)).astype(np.float32)
    want = M.experts(x, ids, w, *ex.w, skip_zero=False, out0=out0)
    got, x1 = prefill(gpu, ex, x, ids, w, out0=out0, residual=True)
    assert rel(got, want) < REL
    assert np.array_equal(x1, f32_of(bf16(x + got)))   # the residual of the same sums, rounded once
    same, x2 = prefill(gpu, ex, x, ids, w, out0=out0)
    assert np.array_equal(same, got) and np.array_equal(x2, x)


def test_prefill_of_one_busy_and_many_idle_experts(gpu):
    rng = np.random.default_rng(32)
    T, E, H, I = 333, 40, 128, 96
    ex = Experts(gpu, 23, E, H, I)
    x = f32_of(bf16(rng.standard_normal((T, H))))
    ids = np.full((T, 2), 7, np.uint32)
    ids[:, 1] = 39
    ids[5, 1], ids[6] = 0, E
    w = rng.random((T, 2)).astype(np.float32)
    got, _ = prefill(gpu, ex, x, ids, w)
    assert rel(got, M.experts(x, ids, w, *ex.w, skip_zero=False)) < REL
    assert (got[6] == 0).all()


def test_results_repeat(gpu):
    rng = np.random.default_rng(33)
    T, E, H, I, k = 90, 4, 256, 160, 2
    ex = Experts(gpu, 24, E, H, I)
    x = f32_of(bf16(rng.standard_normal((T, H))))
    ids, w = route(rng, T, E, k)
    a, b = decode(gpu, ex, x, ids, w), prefill(gpu, ex, x, ids, w)[0]
    for _ in range(3):
        assert np.array_equal(decode(gpu, ex, x, ids, w), a) and np.array_equal(prefill(gpu, ex, x, ids, w)[0], b)


# ---- the framework's paths over MXFP4 banks ----------------------------------------------------


def test_layered_stack_over_mxfp4(gpu):
    """router, experts and residual of two layers, each layer checked on its own input."""
    nm = gpu
    rng = np.random.default_rng(41)
    rows, E, H, I, k = 3, 8, 256, 128, 2
    exs = [Experts(nm, 50 + l, E, H, I) for l in range(2)]
    routers = [(rng.standard_normal((E, H)) * 0.05).astype(np.float32) for _ in range(2)]
    rd = [nm.DeviceBuffer.from_array(r) for r in routers]
    x = bf16(rng.standard_normal((rows, H)))
    xd = nm.DeviceBuffer.from_array(x)
    ids, w = nm.DeviceBuffer(2 * rows * k * 4), nm.DeviceBuffer(2 * rows * k * 4)
    y = nm.DeviceBuffer(2 * rows * H * 4)
    descs = [nm.layer_desc(r, e.banks) for r, e in zip(rd, exs)]
    nm.stack_decode(descs, xd, rows, H, E, k, ids_out=ids, w_out=w, fused=False, y_out=y)
    idl, wl = ids.download(np.uint32).reshape(2, rows, k), w.download(np.float32).reshape(2, rows, k)
    yl = y.download(np.float32).reshape(2, rows, H)
    cur = f32_of(x)
    for l in range(2):
        assert rel(yl[l], M.experts(cur, idl[l], wl[l], *exs[l].w)) < REL
        cur = f32_of(bf16(cur + yl[l]))
    assert np.array_equal(f32_of(xd.download(np.uint16)).reshape(rows, H), cur)
    # without the per-layer outputs the residual is part of the combine: the same bits
    xd2 = nm.DeviceBuffer.from_array(x)
    nm.stack_decode(descs, xd2, rows, H, E, k, fused=False)
    assert np.array_equal(xd2.download(np.uint16), xd.download(np.uint16))
    with pytest.raises(nm.NaiwaError):
        nm.stack_decode(descs, xd2, rows, H, E, k, fused=True)


def test_partial_cache_over_mxfp4(gpu):
    """A layer that holds half of its experts, the misses staged from pinned host stacks of tile order."""
    nm = gpu
    rng = np.random.default_rng(43)
    E, H, I, k, usable = 8, 256, 128, 2, 4
    src = Experts(nm, 60, E, H, I)
    stacks = nm.HostExpertStacks(E, H, I, (nm.MXFP4_T,) * 3, interleaved=True)
    for p, bank in enumerate((src.banks.gate, src.banks.up, src.banks.down)):
        for e in range(E):
            stacks.view(p)[e] = bank.buffer.download(np.uint8, bank.expert_bytes, e * bank.stride)
    router = (rng.standard_normal((E, H)) * 0.05).astype(np.float32)
    rd = nm.DeviceBuffer.from_array(router)
    ring, copy = nm.policy.StagingRing(), nm.Stream()
    banks = nm.LayerBanks(usable + ring.length, H, I, (nm.MXFP4_T,) * 3, contiguous=True)
    layer = nm.policy.CachedLayer(rd.ptr, banks, stacks, E, k, usable, ring, copy.handle)
    y, ids, w = nm.DeviceBuffer(H * 4), nm.DeviceBuffer(k * 4), nm.DeviceBuffer(k * 4)
    for step in range(6):
        x = bf16(rng.standard_normal((1, H)))
        xd = nm.DeviceBuffer.from_array(x)
        nm.router_topk(xd, nm.BF16, rd, 1, H, E, k, ids, w)
        x2 = nm.DeviceBuffer.from_array(x)
        nm.policy.CachedLayer.stack_forward([layer], x2.ptr, 1, y.ptr, stream=0)
        want = M.experts(f32_of(x), ids.download(np.uint32).reshape(1, k), w.download(np.float32).reshape(1, k), *src.w)
        got = y.download(np.float32).reshape(1, H)
        assert rel(got, want) < REL, step
        assert np.array_equal(f32_of(x2.download(np.uint16)).reshape(1, H), f32_of(bf16(f32_of(x) + got)))


def test_prefill_stream_over_mxfp4(gpu):
    nm = gpu
    rng = np.random.default_rng(44)
    E, H, I, k, T = 4, 160, 96, 2, 70
    src = [Experts(nm, 70 + l, E, H, I) for l in range(2)]
    stacks = []
    for s in src:
        st = nm.HostExpertStacks(E, H, I, (nm.MXFP4_T,) * 3)
        for p, bank in enumerate((s.banks.gate, s.banks.up, s.banks.down)):
            for e in range(E):
                st.view(p)[e] = bank.buffer.download(np.uint8, bank.expert_bytes, e * bank.stride)
        stacks.append(st)
    copy = nm.Stream()
    ps = nm.prefill.PrefillStream(stacks, H, I, (nm.MXFP4_T,) * 3, 2, copy.handle)
    x = f32_of(bf16(rng.standard_normal((T, H))))
    xd = nm.DeviceBuffer.from_array(bf16(x))
    for l in range(2):
        ids, w = route(rng, T, E, k)
        out = nm.DeviceBuffer(T * H * 4)
        idd, wd = nm.DeviceBuffer.from_array(ids), nm.DeviceBuffer.from_array(w)
        ps.forward(l, xd, idd, wd, T, k, out)
        nm.synchronize()
        got = out.download(np.float32).reshape(T, H)
        assert rel(got, M.experts(x, ids, w, *src[l].w, skip_zero=False)) < REL


# ---- as callers use them -----------------------------------------------------------------------


def test_quantise_route_and_run(gpu):
    """A layer from f32 weights to its output: quantised on the device, routed, its routing counted and scored,
    decoded token by token, as a batch and as a prompt chunk, which agree."""
    nm = gpu
    rng = np.random.default_rng(80)
    T, E, H, I, k = 24, 8, 288, 160, 2
    banks = nm.LayerBanks(E, H, I, (nm.MXFP4_T,) * 3, contiguous=True)
    w64 = []
    for bank, n, kk in ((banks.gate, I, H), (banks.up, I, H), (banks.down, H, I)):
        raw = bf16(rng.standard_normal((E, n, kk)) * 0.05)
        nm.mxfp4_quantize(nm.DeviceBuffer.from_array(raw), nm.BF16, n, kk, bank.desc().base, batch=E, dst_stride=bank.stride)
        back = nm.DeviceBuffer(E * n * kk * 4)
        nm.mxfp4_dequantize(bank.desc().base, n, kk, back, nm.F32, batch=E, src_stride=bank.stride)
        v = back.download(np.float32).reshape(E, n, kk).astype(np.float64)
        for e in range(E):
            assert np.array_equal(v[e], M.values(*M.quantize(f32_of(raw[e]))))
        w64.append(list(v))
    x = f32_of(bf16(rng.standard_normal((T, H))))
    xd = nm.DeviceBuffer.from_array(bf16(x))
    router = nm.DeviceBuffer.from_array((rng.standard_normal((E, H)) * 0.1).astype(np.float32))
    ids, w, logits = nm.DeviceBuffer(T * k * 4), nm.DeviceBuffer(T * k * 4), nm.DeviceBuffer(T * E * 4)
    nm.router_topk(xd, nm.BF16, router, T, H, E, k, ids, w, logits_out=logits)
    counts, valid, probs, loss = (nm.DeviceBuffer(n * 4) for n in (E, 1, E, 1))
    nm.router_balance(logits, nm.F32, ids, T, E, k, counts, valid, probs, loss)
    idn, wn = ids.download(np.uint32).reshape(T, k), w.download(np.float32).reshape(T, k)
    lg = logits.download(np.float32).reshape(T, E).astype(np.float64)
    p = np.exp(lg - lg.max(-1, keepdims=True))
    p = (p / p.sum(-1, keepdims=True)).mean(0)
    c = np.bincount(idn.ravel(), minlength=E)
    assert np.array_equal(counts.download(np.uint32), c) and valid.download(np.uint32)[0] == T
    assert abs(loss.download(np.float32)[0] - E / (k * T) * (c * p).sum()) < 4e-6 * E
    want = M.experts(x, idn, wn, *w64, skip_zero=False)
    out = nm.DeviceBuffer(T * H * 4)
    nm.moe_prefill(banks, xd, ids, w, T, k, out)
    chunk = out.download(np.float32).reshape(T, H)
    nm.indexed_moe_fused_decode(banks, xd, nm.BF16, ids, w, T, k, out)
    batch = out.download(np.float32).reshape(T, H)
    one = nm.DeviceBuffer(H * 4)
    for t in range(T):
        nm.indexed_moe_fused_decode(banks, xd.ptr + t * H * 2, nm.BF16, ids.ptr + t * k * 4, w.ptr + t * k * 4, 1, k, one)
        assert rel(one.download(np.float32), want[t]) < REL
    assert rel(chunk, want) < REL and rel(batch, want) < REL


def test_streams_and_calls_of_changing_size(gpu):
    """Calls of many sizes one after the other on a stream of the caller's, nothing between them: each has the
    scratch of the one before, larger and smaller, and the bits of a call alone."""
    nm = gpu
    rng = np.random.default_rng(81)
    E, H, I, k = 4, 352, 224, 2
    ex = Experts(nm, 82, E, H, I)
    st = nm.Stream()
    jobs = []
    for T in (70, 1, 9, 400, 1, 33, 2):
        ids, w = route(rng, T, E, k)
        x = f32_of(bf16(rng.standard_normal((T, H))))
        jobs.append((x, ids, w, decode(nm, ex, x, ids, w), prefill(nm, ex, x, ids, w)[0]))
    bufs = [(nm.DeviceBuffer.from_array(bf16(x)), nm.DeviceBuffer.from_array(ids), nm.DeviceBuffer.from_array(w),
             nm.DeviceBuffer(x.size * 4), nm.DeviceBuffer(x.size * 4)) for x, ids, w, _, _ in jobs]
    nm.synchronize()
    for (x, ids, w, _, _), (xd, idd, wd, o1, o2) in zip(jobs, bufs):
        T = len(ids)
        nm.indexed_moe_fused_decode(ex.banks, xd, nm.BF16, idd, wd, T, k, o1, stream=st.handle)
        nm.moe_prefill(ex.banks, xd, idd, wd, T, k, o2, stream=st.handle)
    st.sync()
    for (x, _, _, d, p), (_, _, _, o1, o2) in zip(jobs, bufs):
        assert np.array_equal(o1.download(np.float32).reshape(x.shape), d)
        assert np.array_equal(o2.download(np.float32).reshape(x.shape), p)


def test_slots_past_4_gib(gpu):
    """Banks whose slots lie gigabytes apart, and a quantisation whose projections do."""
    nm = gpu
    rng = np.random.default_rng(83)
    E, H, I, k, gap = 4, 256, 96, 2, 3 << 29      # slot 3 starts at 4.5 GiB
    near = Experts(nm, 84, E, H, I)
    arena = nm.DeviceBuffer(3 * gap + (1 << 20))
    offs = (0, 1 << 18, 1 << 19)
    far = [nm.SlotBank(E, b.n, b.k, nm.MXFP4_T, base=arena.ptr + o, stride=gap)
           for b, o in zip((near.banks.gate, near.banks.up, near.banks.down), offs)]
    for b, o in zip((near.banks.gate, near.banks.up, near.banks.down), offs):
        for e in range(E):
            arena.upload(b.buffer.download(np.uint8, b.expert_bytes, e * b.stride), offset=e * gap + o)
    T = 20
    ids, w = route(rng, T, E, k)
    ids[:, 0] = 3
    ids[:, 1] = np.arange(T) % 3
    x = f32_of(bf16(rng.standard_normal((T, H))))
    want = decode(nm, near, x, ids, w), decode(nm, near, x[:1], ids[:1], w[:1]), prefill(nm, near, x, ids, w)[0]

    class Far:
        banks = nm.LayerBanks.over(*far)

    got = decode(nm, Far, x, ids, w), decode(nm, Far, x[:1], ids[:1], w[:1]), prefill(nm, Far, x, ids, w)[0]
    for a, b in zip(got, want):
        assert np.array_equal(a, b)
    n, kk = 32, 64
    raw = rng.standard_normal((2, n, kk)).astype(np.float32)
    arena.upload(raw[0], offset=0)
    arena.upload(raw[1], offset=3 * gap)
    out = nm.DeviceBuffer(2 * nm.projection_bytes(nm.MXFP4_T, n, kk))
    nm.mxfp4_quantize(arena, nm.F32, n, kk, out, batch=2, src_stride=3 * gap // 4)
    packed = out.download(np.uint8).reshape(2, -1)
    for b in range(2):
        assert np.array_equal(packed[b], M.tiled(*M.quantize(raw[b])))
    nm.mxfp4_quantize(nm.DeviceBuffer.from_array(raw), nm.F32, n, kk, arena, batch=2, dst_stride=3 * gap)
    assert np.array_equal(arena.download(np.uint8, packed.shape[1], 3 * gap), packed[1])


def test_rows_past_the_outputs_stay(gpu):
    """The bytes behind the last row of out, and x without a residual, are left as they are."""
    nm = gpu
    rng = np.random.default_rng(85)
    E, H, I, k = 3, 160, 96, 2
    ex = Experts(nm, 86, E, H, I)
    for T in (1, 5, 40):
        ids, w = route(rng, T, E, k)
        raw = bf16(rng.standard_normal((T, H)))
        xd, idd, wd = (nm.DeviceBuffer.from_array(a) for a in (raw, ids, w))
        for f in ("decode", "prefill"):
            out = nm.DeviceBuffer.from_array(np.full((T + 3, H), 9.0, np.float32))
            if f == "decode":
                nm.indexed_moe_fused_decode(ex.banks, xd, nm.BF16, idd, wd, T, k, out)
            else:
                nm.moe_prefill(ex.banks, xd, idd, wd, T, k, out)
            o = out.download(np.float32).reshape(T + 3, H)
            assert (o[T:] == 9.0).all() and (o[:T] != 9.0).all()
            assert np.array_equal(xd.download(np.uint16).reshape(T, H), raw)


class Graph:
    """What `calls` queue on a stream, captured; the library's calls allocate nothing once their scratch is as large
    as they need."""

    def __init__(self, nm, stream, calls):
        import ctypes as C
        self.hip = C.CDLL("libamdhip64.so.7")      # the runtime that the library has loaded
        self.nm, self.stream, self.graph, self.exec = nm, stream, C.c_void_p(), C.c_void_p()
        h = C.c_void_p(stream.handle)
        nm.synchronize()
        assert self.hip.hipStreamBeginCapture(h, 2) == 0
        calls()
        assert self.hip.hipStreamEndCapture(h, C.byref(self.graph)) == 0
        assert self.hip.hipGraphInstantiate(C.byref(self.exec), self.graph, None, None, C.c_size_t(0)) == 0

    def launch(self):
        import ctypes as C
        assert self.hip.hipGraphLaunch(self.exec, C.c_void_p(self.stream.handle)) == 0

    def close(self):
        self.stream.sync()
        assert self.hip.hipGraphExecDestroy(self.exec) == 0 and self.hip.hipGraphDestroy(self.graph) == 0


@pytest.mark.parametrize("T", [1, 20, 400])
def test_captured_and_replayed(gpu, T):
    """Quantisation, a decode call and a prompt chunk in one graph, replayed on new weights, inputs and routing
    between eager calls of other sizes over the same scratch."""
    nm = gpu
    rng = np.random.default_rng(90 + T)
    E, H, I, k = 4, 288, 160, 2
    ex = Experts(nm, 91, E, H, I)
    other = [f32_of(bf16(rng.standard_normal((500, H)))), *route(rng, 500, E, k)]
    xd, idd, wd = nm.DeviceBuffer(T * H * 2), nm.DeviceBuffer(T * k * 4), nm.DeviceBuffer(T * k * 4)
    raw, d, p = nm.DeviceBuffer(I * H * 2), nm.DeviceBuffer(T * H * 4), nm.DeviceBuffer(T * H * 4)

    def call(stream):
        nm.mxfp4_quantize(raw, nm.BF16, I, H, ex.banks.gate.desc().base, stream=stream)   # slot 0's gate
        nm.indexed_moe_fused_decode(ex.banks, xd, nm.BF16, idd, wd, T, k, d, stream=stream)
        nm.moe_prefill(ex.banks, xd, idd, wd, T, k, p, stream=stream)

    def eager_others():
        decode(nm, ex, *other)
        prefill(nm, ex, *other)

    def inputs():
        ids, w = route(rng, T, E, k)
        ids[0, 0] = 0
        for b, a in ((xd, bf16(rng.standard_normal((T, H)))), (idd, ids), (wd, w),
                     (raw, bf16(rng.standard_normal((I, H)) * 0.05))):
            b.upload(a)

    inputs()
    eager_others()
    st = nm.Stream()
    g = Graph(nm, st, lambda: call(st.handle))
    for _ in range(3):
        inputs()
        call(0)
        want = d.download(np.uint32), p.download(np.uint32)
        eager_others()
        for _ in range(2):
            g.launch()
            st.sync()
            assert np.array_equal(d.download(np.uint32), want[0]) and np.array_equal(p.download(np.uint32), want[1])
    g.close()


@pytest.mark.parametrize("width,E,H,I", [(64, 64, 64, 512), (64, 3, 96, 416), (63, 64, 64, 512), (57, 8, 64, 512),
                                         (64, 64, 64, 384), (48, 4, 33024, 32)])
def test_one_token_of_the_widest_rows(gpu, width, E, H, I):
    """Up to 64 experts a token, whose h fills more than LDS (from I 416 on) and goes down in tiles: all pairs,
    some of them dropped or of no slot, and nothing, over scratch that a larger call has filled."""
    nm = gpu
    rng = np.random.default_rng(width + E + I)
    print(f"[one token {width} {E} {H} {I}]", flush=True)
    ex = Experts(nm, 130, E, H, I)
    before = f32_of(bf16(rng.standard_normal((40, H)))), *route(rng, 40, E, 8)
    for case in range(3):
        x = f32_of(bf16(rng.standard_normal((1, H))))
        ids, w = route(rng, 1, E, width)
        if case == 1:
            w[0, ::5], ids[0, 2::7], ids[0, 3::11] = 0, E, 0xFFFFFFFF
        elif case == 2:
            ids[:] = E
        want = M.experts(x, ids, w, *ex.w)
        decode(nm, ex, *before)
        assert np.array_equal(got := decode(nm, ex, x, ids, w, noalloc=True), decode(nm, ex, x, ids, w))
        prefill(nm, ex, *before)
        chunk = prefill(nm, ex, x, ids, w)[0]
        if case == 2:
            assert (got == 0).all() and (chunk == 0).all()
        else:
            assert rel(got, want) < REL and rel(chunk, want) < REL


class Cached:
    """A partial-cache layer over MXFP4, its misses staged from pinned host stacks of tile order."""

    def __init__(self, nm, seed, E, H, I, k, usable):
        rng = np.random.default_rng(seed)
        self.src = Experts(nm, seed + 1, E, H, I)
        self.stacks = nm.HostExpertStacks(E, H, I, (nm.MXFP4_T,) * 3, interleaved=True)
        for p, bank in enumerate((self.src.banks.gate, self.src.banks.up, self.src.banks.down)):
            for e in range(E):
                self.stacks.view(p)[e] = bank.buffer.download(np.uint8, bank.expert_bytes, e * bank.stride)
        self.router = nm.DeviceBuffer.from_array((rng.standard_normal((E, H)) * 0.05).astype(np.float32))
        self.ring, self.copy = nm.policy.StagingRing(), nm.Stream()
        self.banks = nm.LayerBanks(usable + self.ring.length, H, I, (nm.MXFP4_T,) * 3, contiguous=True)
        self.layer = nm.policy.CachedLayer(self.router.ptr, self.banks, self.stacks, E, k, usable, self.ring,
                                           self.copy.handle)

    def state(self):
        c = self.layer.cache
        return (c.tick, c.hit_counts().tolist(), [c.slot_state(s) for s in range(c.slots)], self.ring.acquire(0))


def test_partial_cache_refuses_misses_that_it_cannot_stage(gpu):
    """The CPU path does not compute MXFP4: a step with more missed experts than ring positions, or with fewer of
    them streamed, is refused as a whole, whatever set_cpu_misses says; the policy stays and the next step is right."""
    nm = gpu
    rng = np.random.default_rng(140)
    E, H, I, k, usable, rows = 64, 128, 64, 8, 4, 6
    c = Cached(nm, 141, E, H, I, k, usable)
    x = bf16(rng.standard_normal((rows, H)))
    xd = nm.DeviceBuffer.from_array(x)
    ids, w, out = nm.DeviceBuffer(rows * k * 4), nm.DeviceBuffer(rows * k * 4), nm.DeviceBuffer(rows * H * 4)
    nm.router_topk(xd, nm.BF16, c.router, rows, H, E, k, ids, w)
    idn, wn = ids.download(np.uint32).reshape(rows, k), w.download(np.float32).reshape(rows, k)
    assert len(np.unique(idn)) > c.ring.length + usable
    for on in (True, False):
        c.layer.set_cpu_misses(on)
        for n, frac in ((rows, 1.0), (rows, 0.5), (1, 0.5), (1, 0.0)):
            before = c.state()
            with pytest.raises(nm.NaiwaError) as e:
                c.layer.forward(xd, n, out, pcie_frac=frac)
            assert e.value.rc == nm.E_UNSUPPORTED and c.state() == before, (on, n, frac)
            x2 = nm.DeviceBuffer.from_array(x)
            with pytest.raises(nm.NaiwaError) as e:
                nm.policy.CachedLayer.stack_forward([c.layer], x2.ptr, n, out.ptr, pcie_frac=frac)
            assert e.value.rc == nm.E_UNSUPPORTED and c.state() == before, (on, n, frac)
            assert np.array_equal(x2.download(np.uint16).reshape(rows, H), x)
        for t in range(2):
            info = c.layer.forward(xd.ptr + t * H * 2, 1, out)
            nm.synchronize()
            assert info["cpu"] == 0 and info["hits"] + info["staged"] == k
            got = out.download(np.float32, H)
            assert rel(got, M.experts(f32_of(x[t:t + 1]), idn[t:t + 1], wn[t:t + 1], *c.src.w)[0]) < REL


def test_partial_cache_refuses_a_call_before_the_policy_moves(gpu):
    """x or out that the experts do not take, and more rows than a call's."""
    nm = gpu
    E, H, I, k = 8, 128, 64, 2
    c = Cached(nm, 150, E, H, I, k, 4)
    xd, out = nm.DeviceBuffer.from_array(np.zeros(2 * H, np.uint16)), nm.DeviceBuffer(2 * H * 4)
    before = c.state()
    for x, rows, o in ((xd.ptr + 8, 1, out.ptr), (xd.ptr, 1, out.ptr + 4), (xd.ptr, 4097, out.ptr)):
        with pytest.raises(nm.NaiwaError) as e:
            c.layer.forward(x, rows, o)
        assert e.value.rc == nm.E_INVALID and c.state() == before
    assert c.layer.forward(xd, 2, out)["cpu"] == 0
    nm.synchronize()
    assert (out.download(np.float32) == 0).all() and c.state() != before


def test_quantize_past_the_threads_of_a_launch(gpu):
    """2^24 + 3 groups of 16 rows, 256 threads each: more threads than one launch takes.  Rows at both ends and
    about the groups where launches may meet, there and back."""
    nm = gpu
    n, k = 16 * ((1 << 24) + 3), 32
    size = nm.projection_bytes(nm.MXFP4_T, 16, k)
    if nm.mem_info()[0] < 3 * n * k * 2:
        pytest.skip("not enough free memory")
    src, dst, back = nm.DeviceBuffer(n * k * 2), nm.DeviceBuffer(n // 16 * size), nm.DeviceBuffer(n * k * 2)
    rng = np.random.default_rng(160)
    rows = {at: bf16(rng.standard_normal((16, k))) for at in (0, (1 << 23) - 1, 1 << 23, (1 << 24) - 1, 1 << 24,
                                                              (1 << 24) + 2)}
    src.zero()
    for at, r in rows.items():
        src.upload(r, offset=at * 16 * k * 2)
    nm.mxfp4_quantize(src, nm.BF16, n, k, dst)
    nm.mxfp4_dequantize(dst, n, k, back, nm.BF16)
    nm.synchronize()
    for at, r in rows.items():
        code, s = M.quantize(f32_of(r))
        assert np.array_equal(dst.download(np.uint8, size, at * size), M.tiled(code, s)), at
        got = f32_of(back.download(np.uint16, 16 * k, at * 16 * k * 2)).reshape(16, k)
        assert np.array_equal(got, M.values(code, s).astype(np.float32)), at

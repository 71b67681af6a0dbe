"""MXFP4 in numpy: the quantiser, the tile order, the GGML blocks and the experts in 64 bits,
written from the definitions in include/naiwa_mxfp4.h."""
from __future__ import annotations

import numpy as np

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])


def steps(k: int) -> int:
    return -(-k // 128)


def strip_bytes(k: int) -> int:
    return 1024 * steps(k) + 256 * -(-steps(k) // 4)


def quantize(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(codes [n, k], scale bytes [n, k / 32]) of f32 rows."""
    n, k = x.shape
    b = np.ascontiguousarray(x, np.float32).reshape(n, k // 32, 32)
    bits = b.view(np.uint32) & 0x7FFFFFFF
    e = (bits.max(-1) >> 23).astype(np.int64)
    bad = e == 255
    s = np.where(bad, 255, np.maximum(0, e - 2))
    with np.errstate(invalid="ignore", over="ignore"):
        y = np.abs(b.astype(np.float64) * 2.0 ** (127 - s)[..., None].astype(np.float64))
        # nearest magnitude, of two as near the one with the even index
        idx = np.zeros(y.shape, np.uint8)
        for i in range(7):
            mid = (E2M1[i] + E2M1[i + 1]) / 2
            idx += ((y > mid) | ((y == mid) & (i % 2 == 1))).astype(np.uint8)
    code = np.where(bad[..., None], 0, idx | (np.signbit(b).astype(np.uint8) << 3)).astype(np.uint8)
    return code.reshape(n, k), s.astype(np.uint8)


def tiled(code: np.ndarray, s: np.ndarray) -> np.ndarray:
    """Tile-order bytes."""
    n, k = code.shape
    t, size = steps(k), strip_bytes(k)
    out = np.zeros((n // 16, size), np.uint8)
    for step in range(t):
        g, last = step // 4, min(4 * (step // 4) + 4, t)
        for b in range(4):
            kb = 4 * step + b
            if kb * 32 >= k:
                continue
            c = code[:, 32 * kb:32 * kb + 32].reshape(n // 16, 16, 16, 2)
            for r in range(16):
                lane = 16 * b + r
                at = 1024 * step + 256 * g + 16 * lane
                out[:, at:at + 16] = c[:, r, :, 0] | (c[:, r, :, 1] << 4)
                out[:, 1024 * last + 256 * g + 4 * lane + step % 4] = s.reshape(n // 16, 16, -1)[:, r, kb]
    return out.reshape(-1)


def values(code: np.ndarray, s: np.ndarray) -> np.ndarray:
    """[n, k] f64."""
    n, k = code.shape
    scale = np.where(s == 255, np.nan, np.ldexp(1.0, s.astype(np.int64) - 127))
    return (E2M1[code].reshape(n, k // 32, 32) * scale[..., None]).reshape(n, k)


def ggml(code: np.ndarray, s: np.ndarray) -> np.ndarray:
    """GGML MXFP4 blocks: scale byte, then byte i holds values i (low half) and 16 + i."""
    n, k = code.shape
    c = code.reshape(n, k // 32, 2, 16)
    return np.concatenate([s[..., None], c[:, :, 0] | (c[:, :, 1] << 4)], -1).reshape(-1)


def act(name: str, g: np.ndarray) -> np.ndarray:
    if name == "silu":
        return g / (1.0 + np.exp(-g))
    return 0.5 * g * (1.0 + np.tanh(np.sqrt(2.0 / np.pi) * (g + 0.044715 * g ** 3)))


def experts(x, ids, w, gate, up, down, name="silu", skip_zero=True, out0=None):
    """sum_j w[t,j] down(act(gate x) up x) in f64; gate/up/down: lists of [I, H] / [H, I] f64."""
    out = np.zeros(x.shape) if out0 is None else out0.astype(np.float64).copy()
    x = x.astype(np.float64)
    for e in range(len(gate)):
        t, j = np.nonzero((ids == e) & ((w != 0) if skip_zero else True))
        if not len(t):
            continue
        h = act(name, x[t] @ gate[e].T) * (x[t] @ up[e].T)
        np.add.at(out, t, (h @ down[e].T) * w[t, j].astype(np.float64)[:, None])
    return out

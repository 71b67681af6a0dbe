"""Tokens sorted by expert and back, their gradients and the routed weights' gradient, against plain NumPy.

Tolerances.  The sort and the rows that move are exact.  A sum over k pairs in f32 from products that are rounded
once each (fma: not at all) errs by at most (k + 1) 2^-24 sum |w y|; a dot product of H values, added up in any order,
by H 2^-24 sum |d y|; dy by one product's 2^-24.  Each result is then rounded once, by half a step of its type.  The
router's gradient p (a - mean) errs by a few 2^-24 of p (|a| + sum p |a|): the exponential of a difference
of logits up to 20 by 20 2^-24 relative, sums of up to 128 f32 terms by no more than 8 2^-24 relative: 64 2^-24 holds both.
"""
import numpy as np
import pytest

from test_gpu_mxfp4 import Graph, bf16, f32_of

pytestmark = pytest.mark.gpu

NO = 0xFFFFFFFF
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -25}


def raw_of(x, dt):
    """Bits of x rounded to dt, and the values that they stand for in f64."""
    if dt == "f32":
        r = np.ascontiguousarray(x, np.float32)
        return r, r.astype(np.float64)
    if dt == "bf16":
        r = bf16(np.ascontiguousarray(x, np.float32))
        return r, f32_of(r).astype(np.float64)
    r = np.ascontiguousarray(x, np.float32).astype(np.float16)
    return r.view(np.uint16), r.astype(np.float64)


def values(raw, dt):
    if dt == "f32":
        return raw.astype(np.float64)
    return (f32_of(raw) if dt == "bf16" else raw.view(np.float16)).astype(np.float64)


def dtype_of(nm, dt):
    return {"f32": nm.F32, "bf16": nm.BF16, "f16": nm.F16}[dt]


def np_of(dt):
    return np.float32 if dt == "f32" else np.uint16


def close(got, want, bound, dt):
    """got within `bound` and half a step of its type of want; where want is not finite, the same kind."""
    fin = np.isfinite(want)
    assert np.array_equal(fin, np.isfinite(got))
    off = np.abs(got - want)[fin] - (bound * np.ones_like(want))[fin] - HALF[dt] * np.abs(want)[fin] * (1 + 1e-6) - TINY[dt]
    assert off.size == 0 or off.max() <= 0, off.max()


class Rows:
    """A device array of rows `ld` values apart, sentinels between and behind them."""

    def __init__(self, nm, x, dt, ld=0, shift=0):
        raw = raw_of(x, dt)[0] if x.dtype.kind == "f" else x
        self.dt, self.shape, self.ld, self.shift = dt, raw.shape, ld or raw.shape[1], shift
        self.size = np.dtype(np_of(dt)).itemsize
        wide = np.full((raw.shape[0] + 1, self.ld), 1.25, np.float32)
        wide = raw_of(wide, dt)[0]
        wide[:-1, :raw.shape[1]] = raw
        self.start = wide
        self.buf = nm.DeviceBuffer(wide.nbytes + 64)
        self.buf.upload(wide, offset=shift * self.size)

    @property
    def ptr(self):
        return self.buf.ptr + self.shift * self.size

    def raw(self):
        w = self.buf.download(np_of(self.dt), self.start.size, offset=self.shift * self.size).reshape(self.start.shape)
        assert np.array_equal(w[:, self.shape[1]:], self.start[:, self.shape[1]:])
        assert np.array_equal(w[-1], self.start[-1])
        return w[:-1, :self.shape[1]]

    def get(self):
        return values(self.raw(), self.dt)


def routing(rng, T, k, E, drop=0.0, bad=0):
    ids = np.zeros((T, k), np.uint32)
    for t in range(T):
        ids[t] = rng.permutation(E)[:k] if E >= k else rng.integers(0, E, k)
    mask = (rng.random(T) >= drop).astype(np.uint8) * 7 if drop else None
    for _ in range(bad):
        ids[rng.integers(T), rng.integers(k)] = rng.choice([E, E + 5, NO])
    return ids, mask


def sort_ref(ids, mask, E):
    T, k = ids.shape
    flat = np.where((ids >= E) | ((mask == 0)[:, None] if mask is not None else False), E, ids).ravel()
    order = np.argsort(flat, kind="stable")
    counts = np.bincount(flat.astype(np.int64), minlength=E + 1)
    offsets = np.concatenate([[0], np.cumsum(counts[:E])]).astype(np.uint32)
    n = offsets[-1]
    inv = np.full(T * k, NO, np.uint32)
    inv[order[:n]] = np.arange(n)
    live = np.ones(T, bool) if mask is None else mask != 0
    return order[:n].astype(np.uint32), inv.reshape(T, k), offsets, int((ids[live] >= E).sum())


def sort(nm, ids, mask, E, ids_ld=0):
    T, k = ids.shape
    wide = np.full((T, ids_ld or k), 12345, np.uint32)
    wide[:, :k] = ids
    d = nm.DeviceBuffer.from_array(wide if wide.size else np.zeros(4, np.uint32))
    m = None if mask is None else nm.DeviceBuffer.from_array(mask)
    perm, inv = (nm.DeviceBuffer.from_array(np.full(T * k + 1, 77, np.uint32)) for _ in range(2))
    offsets, bad = (nm.DeviceBuffer.from_array(np.full(n, 77, np.uint32)) for n in (E + 2, 1))
    nm.expert_sort(d, T, k, E, perm, inv, offsets, mask=m, bad=bad, ids_ld=ids_ld)
    p, i, o = (b.download(np.uint32) for b in (perm, inv, offsets))
    assert i[-1] == 77 and o[-1] == 77 and (p[o[E]:] == 77).all()
    return p[:o[E]], i[:-1].reshape(T, k), o[:-1], int(bad.download(np.uint32)[0])


@pytest.mark.parametrize("T,k,E,drop,bad", [
    (0, 2, 8, 0, 0), (1, 1, 1, 0, 0), (1, 8, 8, 0, 0), (3, 2, 4, 0.5, 0), (61, 2, 8, 0, 0), (64, 8, 60, 0.2, 3), (33, 4, 4096, 0, 1),
    (512, 8, 128, 0, 0), (1024, 4, 512, 0.1, 5), (1024, 4, 513, 0.1, 5), (513, 8, 128, 0.3, 0), (1366, 3, 7, 0, 40),
    (700, 6, 2049, 0.1, 2), (5000, 8, 128, 0.1, 9), (3001, 7, 4096, 0, 0), (40000, 8, 127, 0.05, 100), (140001, 8, 64, 0.5, 3),
    (9000, 1, 1, 0, 7),
])
def test_sort(gpu, T, k, E, drop, bad):
    rng = np.random.default_rng(T + 31 * E)
    ids, mask = routing(rng, T, k, E, drop, bad)
    print(f"[sort {T} {k} {E}]", flush=True)
    for got, want in zip(sort(gpu, ids, mask, E, ids_ld=k + (T % 3)), sort_ref(ids, mask, E)):
        assert np.array_equal(got, want)


@pytest.mark.parametrize("T", [9, 3000])
def test_sort_of_one_expert_and_of_none(gpu, T):
    one = np.full((T, 3), 5, np.uint32)     # the same expert for all pairs, of a token too
    for ids, mask in ((one, None), (one + 3, None), (one, np.zeros(T, np.uint8))):
        for got, want in zip(sort(gpu, ids, mask, 8), sort_ref(ids, mask, 8)):
            assert np.array_equal(got, want)


SIZES = [(1, 1, 1, "bf16"), (1, 2, 7, "f32"), (5, 3, 8, "f16"), (17, 8, 33, "bf16"), (64, 2, 128, "f16"), (33, 4, 129, "f32"),
         (100, 6, 633, "bf16"), (300, 8, 2048, "bf16"), (70, 3, 4100, "f16"), (2000, 2, 520, "f32")]


@pytest.mark.parametrize("T,k,H,dt", SIZES)
@pytest.mark.parametrize("tight", [True, False])
def test_to_experts(gpu, T, k, H, dt, tight):
    nm = gpu
    rng = np.random.default_rng(T + H)
    ids, mask = routing(rng, T, k, 16, 0.2)
    inv = sort_ref(ids, mask, 16)[1]
    inv[rng.integers(T), rng.integers(k)] = T * k          # outside the rows: in none
    x = Rows(nm, rng.standard_normal((T, H)).astype(np.float32), dt, 0 if tight else H + 3, 0 if tight else 1)
    rows = Rows(nm, np.full((T * k, H), 3.0, np.float32), dt, 0 if tight else H + 5, 0 if tight else 3)
    want = np.full((T * k, H), 3.0)
    if mask is not None:   # what a token that is in no row holds does not matter
        raw = x.start[:-1].copy()
        raw[(inv >= T * k).all(1), :H] = raw_of(np.full(1, np.nan), dt)[0]
        x.buf.upload(raw, offset=x.shift * x.size)
    for t, j in zip(*np.nonzero(inv < T * k)):
        want[inv[t, j]] = values(x.start[t, :H], dt)
    print(f"[to {T} {k} {H} {dt}]", flush=True)
    d = nm.DeviceBuffer.from_array(inv)
    nm.tokens_to_experts(x.ptr, dtype_of(nm, dt), d, T, k, H, rows.ptr, ld=x.ld, rows_ld=rows.ld)
    assert np.array_equal(rows.get(), want)


@pytest.mark.parametrize("T,k,H,dt", SIZES)
@pytest.mark.parametrize("out_f32,weighted,acc,tight", [(True, True, False, True), (False, True, True, False), (False, False, False, False),
                                                        (True, False, True, True)])
def test_from_experts(gpu, T, k, H, dt, out_f32, weighted, acc, tight):
    nm = gpu
    rng = np.random.default_rng(T + H)
    ids, mask = routing(rng, T, k, 16, 0.3)
    inv = sort_ref(ids, mask, 16)[1]
    if T > 1:
        inv[T - 1] = NO                                     # a token that no row comes back to
    od = "f32" if out_f32 else dt
    y = Rows(nm, rng.standard_normal((T * k, H)).astype(np.float32), dt, 0 if tight else H + 1, 0 if tight else 1)
    unused = np.setdiff1d(np.arange(T * k), inv.ravel())
    raw = y.start[:-1].copy()
    raw[unused, :H] = raw_of(np.full(1, np.nan), dt)[0]      # rows that are no pair's are not read
    y.buf.upload(raw, offset=y.shift * y.size)
    w = rng.random((T, k)).astype(np.float32)
    wide = np.full((T, k + 2), np.nan, np.float32)
    wide[:, :k] = w
    out = Rows(nm, rng.standard_normal((T, H)).astype(np.float32), od, 0 if tight else H + 7, 0 if tight else 1)
    start = values(out.start[:-1, :H], od)
    wd, invd = nm.DeviceBuffer.from_array(wide), nm.DeviceBuffer.from_array(inv)
    print(f"[from {T} {k} {H} {dt} {od}]", flush=True)
    nm.tokens_from_experts(y.ptr, dtype_of(nm, dt), invd, T, k, H, out.ptr, w=wd if weighted else None, w_ld=k + 2,
                           out_dtype=dtype_of(nm, od), accumulate=acc, ld=y.ld, out_ld=out.ld)
    yv = np.vstack([values(y.start[:-1, :H], dt), np.zeros((1, H))])[np.where(inv < T * k, inv, T * k)]
    f = w.astype(np.float64)[:, :, None] if weighted else 1.0
    want = (f * yv).sum(1) + (start if acc else 0)
    size = np.abs(f * yv).sum(1) + (np.abs(start) if acc else 0)
    close(out.get(), want, (k + 1) * 2.0 ** -24 * size, od)


@pytest.mark.parametrize("T,k,H,dt", SIZES)
@pytest.mark.parametrize("d_f32,weighted,tight,which", [(True, True, True, "both"), (False, True, False, "both"),
                                                        (False, False, False, "dy"), (True, True, False, "dw"),
                                                        (False, True, True, "place")])
def test_from_experts_backward(gpu, T, k, H, dt, d_f32, weighted, tight, which):
    nm = gpu
    rng = np.random.default_rng(T + H)
    ids, mask = routing(rng, T, k, 16, 0.3)
    inv = sort_ref(ids, mask, 16)[1]
    dd = "f32" if d_f32 else dt
    y = Rows(nm, rng.standard_normal((T * k, H)).astype(np.float32), dt, 0 if tight else H + 1, 0 if tight else 1)
    dout = Rows(nm, rng.standard_normal((T, H)).astype(np.float32), dd, 0 if tight else H + 2, 0 if tight else 1)
    dy = y if which == "place" else Rows(nm, np.full((T * k, H), 5.0, np.float32), dt, 0 if tight else H + 3, 0 if tight else 1)
    dw = Rows(nm, np.full((T, k), 5.0, np.float32), "f32", k + 1)
    w = rng.random((T, k)).astype(np.float32)
    wd, invd = nm.DeviceBuffer.from_array(w), nm.DeviceBuffer.from_array(inv)
    print(f"[from backward {T} {k} {H} {dt} {dd}]", flush=True)
    nm.tokens_from_experts_backward(dout.ptr, dtype_of(nm, dd), None if which == "dy" else y.ptr, dtype_of(nm, dt), invd, T, k, H,
                                    dy=None if which == "dw" else dy.ptr, dw=None if which == "dy" else dw.ptr,
                                    w=wd if weighted else None, dout_ld=dout.ld, ld=y.ld, dy_ld=dy.ld, dw_ld=dw.ld)
    dv, yv = values(dout.start[:-1, :H], dd), values(y.start[:-1, :H], dt)
    want = yv.copy() if which == "place" else np.full((T * k, H), 5.0)
    wantw = np.zeros((T, k))
    size = np.zeros((T, k))
    for t, j in zip(*np.nonzero(inv < T * k)):
        r = inv[t, j]
        wantw[t, j], size[t, j] = dv[t] @ yv[r], np.abs(dv[t]) @ np.abs(yv[r])
        want[r] = (float(w[t, j]) if weighted else 1.0) * dv[t]
    if which != "dw":
        close(dy.get(), want, 2.0 ** -24 * np.abs(want), dt)
    if which != "dy":
        close(dw.get(), wantw, H * 2.0 ** -24 * size, "f32")


def router_ref(x, ids, dw, mode, mask):
    T, E = x.shape
    k = ids.shape[1]
    d, size = np.zeros((T, E)), np.zeros((T, E))
    for t in range(T):
        if mask is not None and not mask[t]:
            continue
        on = ids[t] < E
        i, a = ids[t][on].astype(int), dw[t][on].astype(np.float64)
        if mode == 2:
            p = np.exp(x[t] - x[t].max())
            p /= p.sum()
            s = np.zeros(E)
            np.add.at(s, i, a)
            at = np.arange(E)
            g, m = s, (p[i] * np.abs(a)).sum()
            d[t] = p * (s - (p[i] * a).sum())
            size[t] = p * (np.abs(s) + m)
        elif len(i):
            p = np.exp(x[t][i] - x[t][i].max())
            p /= p.sum()
            np.add.at(d[t], i, p * (a - (p * a).sum()))
            np.add.at(size[t], i, p * (np.abs(a) + (p * np.abs(a)).sum()))
    return d, size


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (5, 8, 8), (31, 60, 4), (64, 64, 6), (33, 65, 3), (70, 127, 8), (257, 128, 8),
                                   (65, 129, 5), (40, 256, 16), (40, 100, 17), (40, 256, 32), (21, 1000, 32), (13, 1024, 1)])
@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("dt,acc", [("f32", False), ("bf16", True), ("f32", True), ("bf16", False)])
def test_router_backward(gpu, T, E, k, mode, dt, acc):
    nm = gpu
    rng = np.random.default_rng(T + E + k)
    x = Rows(nm, 2 * rng.standard_normal((T, E)).astype(np.float32), dt, E + 4 * (T % 2) + T % 3)
    xv = values(x.start[:-1, :E], dt)
    ids = np.argsort(-xv, axis=1, kind="stable")[:, :k].astype(np.uint32)
    mask = (rng.random(T) < 0.8).astype(np.uint8) if T > 5 else None
    if T > 30:
        ids[3, 0] = E + 2                                   # adds nothing
        ids[5] = NO
        ids[7, -1] = ids[7, 0]                              # named twice
    dw = Rows(nm, rng.standard_normal((T, k)).astype(np.float32), "f32", k + 1)
    wide = np.full((T, k + 2), 3, np.uint32)
    wide[:, :k] = ids
    d = Rows(nm, rng.standard_normal((T, E)).astype(np.float32), dt, x.ld)
    start = values(d.start[:-1, :E], dt)
    idd, md = nm.DeviceBuffer.from_array(wide), None if mask is None else nm.DeviceBuffer.from_array(mask)
    if mask is not None:                                    # what masked rows hold does not matter
        raw = x.start[:-1].copy()
        raw[mask == 0] = raw_of(np.full(1, np.nan), dt)[0]
        x.buf.upload(raw)
    print(f"[router {T} {E} {k} {mode} {dt} {acc}]", flush=True)
    nm.router_topk_backward(x.ptr, dtype_of(nm, dt), idd, dw.ptr, T, E, k, d.ptr, mode=mode, mask=md, accumulate=acc, ld=x.ld,
                            ids_ld=k + 2, dw_ld=k + 1, dld=d.ld)
    want, size = router_ref(xv, ids, dw.start[:-1, :k], mode, mask)
    if acc:
        want, size = start + want, size + np.abs(start)
    got = d.get()
    close(got, want, 64 * 2.0 ** -24 * size, dt)
    if mask is not None:
        assert np.array_equal(got[mask == 0], start[mask == 0] if acc else np.zeros_like(start[mask == 0]))


def test_router_backward_in_place(gpu):
    nm = gpu
    rng = np.random.default_rng(3)
    T, E, k = 50, 64, 6
    xv = rng.standard_normal((T, E)).astype(np.float32)
    ids = np.argsort(-xv, axis=1)[:, :k].astype(np.uint32)
    dw = rng.standard_normal((T, k)).astype(np.float32)
    idd, dwd = nm.DeviceBuffer.from_array(ids), nm.DeviceBuffer.from_array(dw)
    for mode in (0, 2):
        x = Rows(nm, xv, "f32")
        nm.router_topk_backward(x.ptr, nm.F32, idd, dwd, T, E, k, x.ptr, mode=mode)
        want, size = router_ref(xv.astype(np.float64), ids, dw, mode, None)
        close(x.get(), want, 64 * 2.0 ** -24 * size, "f32")


def test_router_backward_against_differences(gpu):
    """Against differences of router_topk's own weights: <dw, (w(l + h v) - w(l - h v)) / 2h> of the weights as f64 functions of
    the logits that the router returned."""
    nm = gpu
    rng = np.random.default_rng(4)
    T, H, E, k = 20, 64, 16, 4
    x = nm.DeviceBuffer.from_array(bf16(rng.standard_normal((T, H))))
    W = nm.DeviceBuffer.from_array((rng.standard_normal((E, H)) * 0.1).astype(np.float32))
    ids, w, logits = (nm.DeviceBuffer(4 * n) for n in (T * k, T * k, T * E))
    dw = rng.standard_normal((T, k)).astype(np.float32)
    dwd, d = nm.DeviceBuffer.from_array(dw), nm.DeviceBuffer(T * E * 4)
    for mode in (nm.ROUTE_SOFTMAX_TOPK_RENORM, nm.ROUTE_TOPK_SOFTMAX, nm.ROUTE_SOFTMAX_TOPK):
        nm.router_topk(x, nm.BF16, W, T, H, E, k, ids, w, mode=mode, logits_out=logits)
        nm.router_topk_backward(logits, nm.F32, ids, dwd, T, E, k, d, mode=mode)
        l0, i0 = logits.download(np.float32).reshape(T, E).astype(np.float64), ids.download(np.uint32).reshape(T, k).astype(int)

        def weights(l):
            p = np.exp(l - l.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            c = np.take_along_axis(p, i0, 1)
            return c if mode == nm.ROUTE_SOFTMAX_TOPK else c / c.sum(1, keepdims=True)

        assert np.abs(weights(l0) - w.download(np.float32).reshape(T, k)).max() < 1e-6   # the router's own weights
        v, h = rng.standard_normal((T, E)), 1e-5
        want = (dw * (weights(l0 + h * v) - weights(l0 - h * v))).sum(1) / (2 * h)
        got = (d.download(np.float32).reshape(T, E) * v).sum(1)
        # second differences of functions of size 1 leave h^2, f64 rounding 1e-16 / h; f32 gradients 1e-6
        assert np.abs(got - want).max() < 1e-5


@pytest.mark.parametrize("T", [40, 3000])
def test_captured_and_replayed(gpu, T):
    """The sort and all moves in one graph on a stream of its own, replayed on new routing between eager calls of another size."""
    nm = gpu
    k, E, H = 4, 32, 200
    rng = np.random.default_rng(T)
    st = nm.Stream()
    zeros = lambda n: nm.DeviceBuffer.from_array(np.zeros(n, np.uint32))  # noqa: E731

    class Calls:
        def __init__(self, T):
            self.T = T
            self.ids, self.x, self.w = zeros(T * k), zeros(T * H), zeros(T * k)
            self.out = [zeros(n) for n in (T * k, T * k, E + 1, T * k * H, T * H, T * k * H, T * k)]

        def fill(self):
            self.ids.upload(routing(rng, self.T, k, E)[0])
            self.x.upload(rng.standard_normal((self.T, H)).astype(np.float32))
            self.w.upload(rng.random((self.T, k)).astype(np.float32))
            nm.synchronize()

        def __call__(self, s):
            T, o = self.T, self.out
            nm.expert_sort(self.ids, T, k, E, o[0], o[1], o[2], stream=s)
            nm.tokens_to_experts(self.x, nm.F32, o[1], T, k, H, o[3], stream=s)
            nm.tokens_from_experts(o[3], nm.F32, o[1], T, k, H, o[4], w=self.w, stream=s)
            nm.tokens_from_experts_backward(o[4], nm.F32, o[3], nm.F32, o[1], T, k, H, dy=o[5], dw=o[6], w=self.w, stream=s)

        def results(self):
            nm.synchronize()
            return [b.download(np.uint32) for b in self.out]

    a, other = Calls(T), Calls(T + 2500)
    a.fill()
    a(st.handle)
    st.sync()
    g = Graph(nm, st, lambda: a(st.handle))
    for _ in range(3):
        a.fill()
        other.fill()
        other(0)
        nm.synchronize()
        g.launch()
        st.sync()
        got = a.results()
        a(0)
        assert all(np.array_equal(x, y) for x, y in zip(got, a.results()))
    g.close()

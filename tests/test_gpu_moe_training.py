"""A MoE layer's training step: router, sort, gated experts, their sum, and all gradients back to the tokens, the experts'
weights and the router's logits, one call after another, against 64 bits.

Every reference value carries a bound of its error.  Through sums the bounds add up by the absolute values, through
products and activations by their slopes and the products of both bounds; each call adds its f32 bound (test_gpu_linear,
test_gpu_tokens) and half a step where it stores fewer bits.  What a call stored is checked, and read on from."""
import numpy as np
import pytest

from test_gpu_linear import ULP, act, act_error
from test_gpu_tokens import HALF, TINY, Rows, dtype_of, raw_of, router_ref, values

pytestmark = pytest.mark.gpu


class V:
    """Values and how far the device's may be from them."""

    def __init__(self, v, e=0.0):
        self.v, self.e = np.asarray(v, np.float64), np.broadcast_to(np.asarray(e, np.float64), np.shape(v))

    def __add__(self, o):
        return V(self.v + o.v, self.e + o.e + ULP * (np.abs(self.v) + np.abs(o.v)))

    def __mul__(self, o):
        v = self.v * o.v
        return V(v, np.abs(self.v) * o.e + np.abs(o.v) * self.e + self.e * o.e + 2 * ULP * np.abs(v))

    def __getitem__(self, i):
        return V(self.v[i], self.e[i])

    def dot(self, m):
        """self @ m, m's values exact or with bounds."""
        m = m if isinstance(m, V) else V(m)
        a, b = np.abs(self.v), np.abs(m.v)
        return V(self.v @ m.v, (self.v.shape[1] + 4) * ULP * ((a + self.e) @ (b + m.e)) + self.e @ (b + m.e) + a @ m.e)

    def to(self, dt):
        """Stored: half a step of the value's size, and of the smallest ones half of theirs, which is fixed (f16: 2^-24 apart
        below 2^-14)."""
        return V(self.v, self.e + HALF[dt] * (np.abs(self.v) + self.e) + TINY[dt])

    @property
    def T(self):
        return V(self.v.T, self.e.T)


def near(got, want, what):
    """got, which has to be within the bounds of want, for what reads it next (bounds carried through several sums of sums add up
    to the values' own size); and the bounds small enough to see a wrong value: a tenth of the values' size on average at most."""
    got = got.reshape(want.v.shape).astype(np.float64)
    assert want.e.mean() < 0.1 * np.sqrt((want.v ** 2).mean()), what
    off = np.abs(got - want.v) - want.e * (1 + 1e-6) - 1e-30
    assert off.max() <= 0, (what, off.max())
    return V(got)


# T, k, E, H, I
@pytest.mark.parametrize("T,k,E,H,I", [(1, 2, 8, 64, 48), (37, 2, 8, 96, 40), (300, 6, 64, 128, 72), (2500, 2, 4, 136, 264)])
@pytest.mark.parametrize("dt,a", [("bf16", "silu"), ("f16", "gelu")])
def test_step(gpu, T, k, E, H, I, dt, a):
    nm = gpu
    rng = np.random.default_rng(T + E)
    d, code, N = dtype_of(nm, dt), {"silu": nm.ACT_SILU, "gelu": nm.ACT_GELU_PYTORCH_TANH}[a], T * k
    normal = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    zeros = lambda rows, w, t="f32": Rows(nm, np.zeros((rows, w), np.float32), t)  # noqa: E731
    buf = nm.DeviceBuffer

    def up(v, t=dt):
        raw, v = raw_of(v, t)
        return buf.from_array(raw), v

    # The router reads bf16 or f32 and makes f32 logits.
    router = normal(E, H) * 0.1
    rd = buf.from_array(router)
    tokens, xv = up(normal(T, H))
    x32 = buf.from_array(xv.astype(np.float32))
    ids, w, logits = buf(N * 4), buf(N * 4), buf(T * E * 4)
    nm.router_topk(x32, nm.F32, rd, T, H, E, k, ids, w, logits_out=logits)
    perm, inv, offsets = buf(N * 4), buf(N * 4), buf((E + 1) * 4)
    nm.expert_sort(ids, T, k, E, perm, inv, offsets)
    (gd, gv), (ud, uv), (dd, dv) = up(normal(E, I, H) * 0.2), up(normal(E, I, H) * 0.2), up(normal(E, H, I) * 0.2)
    bias = normal(E, I) * 0.1
    bd = buf.from_array(bias)
    G, U, D = nm.Weights(gd, d, E, I, H, bias=bd), nm.Weights(ud, d, E, I, H), nm.Weights(dd, d, E, H, I)
    rows, h, pre, pre_up, y, out = zeros(N, H, dt), zeros(N, I, dt), zeros(N, I, dt), zeros(N, I, dt), zeros(N, H, dt), zeros(T, H)
    nm.tokens_to_experts(tokens, d, inv, T, k, H, rows.ptr)
    nm.linear(G, rows.ptr, N, h.ptr, up=U, offsets=offsets, act=code, pre=pre.ptr, pre_up=pre_up.ptr)
    nm.linear(D, h.ptr, N, y.ptr, offsets=offsets)
    nm.tokens_from_experts(y.ptr, d, inv, T, k, H, out.ptr, w=w, out_dtype=nm.F32)

    # back: the output's gradient to every expert's rows and the weights of the sum
    dout, dov = up(normal(T, H), "f32")
    dy, dw = zeros(N, H, dt), buf(N * 4)
    nm.tokens_from_experts_backward(dout, nm.F32, y.ptr, d, inv, T, k, H, dy=dy.ptr, dw=dw, w=w)
    dpre, dpre_up, drows, dx = zeros(N, I, dt), zeros(N, I, dt), zeros(N, H, dt), zeros(T, H)
    gg, gu, gdn, gb = *(buf(E * I * H * 4) for _ in range(3)), buf(E * I * 4)
    nm.linear_input_grad(D, dy.ptr, N, dpre.ptr, offsets=offsets, act=code, pre=pre.ptr, pre_up=pre_up.ptr, dx_up=dpre_up.ptr)
    nm.linear_weight_grad(dy.ptr, h.ptr, d, N, H, I, gdn, experts=E, offsets=offsets)
    nm.linear_input_grad(G, dpre.ptr, N, drows.ptr, up=U, dy_up=dpre_up.ptr, offsets=offsets)
    nm.linear_weight_grad(dpre.ptr, rows.ptr, d, N, I, H, gg, experts=E, offsets=offsets, dbias=gb)
    nm.linear_weight_grad(dpre_up.ptr, rows.ptr, d, N, I, H, gu, experts=E, offsets=offsets)
    nm.tokens_from_experts(drows.ptr, d, inv, T, k, H, dx.ptr, out_dtype=nm.F32)
    # the router: its balance loss's gradient, then that of its weights added to it
    counts, valid, probs, loss, scale = buf(E * 4), buf(4), buf(E * 4), buf(4), buf.from_array(np.array([0.5], np.float32))
    dlogits = buf(T * E * 4)
    nm.router_balance(logits, nm.F32, ids, T, E, k, counts, valid, probs, loss)
    nm.router_balance_backward(logits, nm.F32, counts, valid, T, E, k, scale, dlogits)
    only = dlogits.download(np.float32).reshape(T, E).astype(np.float64)
    nm.router_topk_backward(logits, nm.F32, ids, dw, T, E, k, dlogits, accumulate=True)

    # the same in 64 bits
    iv, lv = ids.download(np.uint32).reshape(T, k), logits.download(np.float32).reshape(T, E).astype(np.float64)
    assert np.abs(lv - xv @ router.T.astype(np.float64)).max() < 1e-4
    z = np.take_along_axis(lv, iv.astype(int), 1)
    wv = np.exp(z - z.max(1, keepdims=True))
    wv = V(wv / wv.sum(1, keepdims=True))
    wv = V(wv.v, 64 * 2.0 ** -24 * wv.v)
    order = np.argsort(iv.reshape(-1), kind="stable")
    seg = np.searchsorted(iv.reshape(-1)[order], np.arange(E + 1))
    assert np.array_equal(offsets.download(np.uint32), seg) and np.array_equal(perm.download(np.uint32), order)
    token = order // k
    live = [(e, slice(seg[e], seg[e + 1])) for e in range(E)]
    blank = lambda width: V(np.zeros((N, width)), np.zeros((N, width)))  # noqa: E731

    def put(to, s, part):
        to.v[s] = part.v
        to.e = np.array(to.e)
        to.e[s] = part.e

    P, Q, Hd, Y = blank(I), blank(I), blank(I), blank(H)
    X = V(xv[token])
    for e, s in live:
        p, q = X[s].dot(gv[e].T) + V(np.broadcast_to(bias[e], (s.stop - s.start, I))), X[s].dot(uv[e].T)
        put(P, s, p), put(Q, s, q)
    av = act(a, P.v)[0]
    Hd = near(h.get(), (V(av, act_error(a, P.v, P.e)[0]) * Q).to(dt), "h")
    for e, s in live:
        put(Y, s, Hd[s].dot(dv[e].T).to(dt))
    Y = near(y.get(), Y, "y")
    wrow = V(wv.v.reshape(-1)[order][:, None], wv.e.reshape(-1)[order][:, None])
    terms = Y * wrow
    P, Q = near(pre.get(), P.to(dt), "pre"), near(pre_up.get(), Q.to(dt), "pre_up")
    av, slope = act(a, P.v)
    ea, es = act_error(a, P.v, P.e)
    A, S = V(av, ea), V(slope, es)
    want = V(np.zeros((T, H)), np.zeros((T, H)))
    size = np.zeros((T, H))
    for to, frm in ((want.v, terms.v), (size, np.abs(terms.v))):
        np.add.at(to, token, frm)
    want.e = np.array(want.e)
    np.add.at(want.e, token, terms.e)
    want.e += k * ULP * size
    near(out.get(), want, "out")
    dO = V(dov[token])
    dY = (dO * wrow).to(dt)
    dY = near(dy.get(), dY, "dy")
    dW = V((dO.v * Y.v).sum(1), (np.abs(dO.v) * (Y.e + H * ULP * np.abs(Y.v))).sum(1))
    got = dw.download(np.float32)
    dW = near(got[order], dW, "dw")
    dP, dQ, dX = blank(I), blank(I), blank(H)
    wants = [np.zeros((2, E, I, H)), np.zeros((2, E, I, H)), np.zeros((2, E, H, I)), np.zeros((2, E, I))]
    for e, s in live:
        g = dY[s].dot(dv[e])
        put(dP, s, (g * S[s] * Q[s]).to(dt)), put(dQ, s, (g * A[s]).to(dt))
    dP, dQ = near(dpre.get(), dP, "dpre"), near(dpre_up.get(), dQ, "dpre_up")
    for e, s in live:
        back, two = dP[s].dot(gv[e]), dQ[s].dot(uv[e])
        put(dX, s, V(back.v + two.v, back.e + two.e + I * ULP * (np.abs(back.v) + np.abs(two.v))).to(dt))
        ones = np.ones((s.stop - s.start, 1))
        for to, m in zip(wants, (dP[s].T.dot(X[s]), dQ[s].T.dot(X[s]), dY[s].T.dot(Hd[s]), dP[s].T.dot(ones))):
            to[0, e], to[1, e] = m.v.reshape(to[0, e].shape), m.e.reshape(to[1, e].shape)
    dX = near(drows.get(), dX, "drows")
    for got, to, what in zip((gg, gu, gdn, gb), wants, ("gate", "up", "down", "bias")):
        near(got.download(np.float32), V(to[0], to[1]), what)
    want, size = np.zeros((2, T, H)), np.zeros((T, H))
    np.add.at(want[0], token, dX.v), np.add.at(want[1], token, dX.e), np.add.at(size, token, np.abs(dX.v))
    near(dx.get(), V(want[0], want[1] + k * ULP * size), "dx")
    dwv = np.zeros(N)
    dwv[order] = dW.v
    r, size = router_ref(lv, iv, dwv.reshape(T, k), nm.ROUTE_SOFTMAX_TOPK_RENORM, None)
    want = V(only + r, 64 * 2.0 ** -24 * size + 2 * ULP * (np.abs(only) + np.abs(r)))
    near(dlogits.download(np.float32), want, "dlogits")

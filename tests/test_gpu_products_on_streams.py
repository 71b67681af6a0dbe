"""Long sorts and products whose sums are in parts, on several streams at once: eager calls on two of them, and a graph that was
captured on one of these and is replayed on a third.  Every stream's calls have scratch of their own."""
import ctypes as C

import numpy as np
import pytest

from test_gpu_linear import Stack
from test_gpu_tokens import raw_of, routing

pytestmark = pytest.mark.gpu


class Calls:
    """A sort of T tokens, and a gated product, an input and a weight gradient of few outputs with long sums."""

    def __init__(self, nm, seed, T, rows, n, k, m):
        rng = np.random.default_rng(seed)
        self.nm, self.sizes, up = nm, (T, rows, n, k, m), nm.DeviceBuffer.from_array
        self.W, self.U, self.V = Stack(nm, rng, 1, n, k, "bf16"), Stack(nm, rng, 1, n, k, "bf16"), Stack(nm, rng, 1, k, n, "bf16")
        self.ids = up(routing(rng, T, 4, 32)[0])
        self.x, self.a, self.b = (up(raw_of(rng.standard_normal(s).astype(np.float32), "bf16")[0]) for s in ((rows, k), (m, n), (m, rows)))
        zeros = lambda c: up(np.zeros(c, np.uint32))  # noqa: E731
        self.out = [zeros(c) for c in (T * 4, T * 4, 33, rows * n, rows * n, n * rows, n)]

    def __call__(self, s):
        nm, (T, rows, n, k, m), o = self.nm, self.sizes, self.out
        nm.expert_sort(self.ids, T, 4, 32, *o[:3], stream=s)
        nm.linear(self.W.w, self.x, rows, o[3], up=self.U.w, act=nm.ACT_SILU, out_dtype=nm.F32, stream=s)
        nm.linear_input_grad(self.V.w, self.x, rows, o[4], dx_dtype=nm.F32, stream=s)
        nm.linear_weight_grad(self.a, self.b, nm.BF16, m, n, rows, o[5], dbias=o[6], stream=s)

    def results(self):
        """What the calls left, and zeros in its place."""
        self.nm.synchronize()
        r = [b.download(np.uint32) for b in self.out]
        for b in self.out:
            b.upload(np.zeros(b.nbytes // 4, np.uint32))
        self.nm.synchronize()
        return r

    def expected(self):
        self(0)
        r = self.results()
        assert all(x.any() for x in r)
        return r


def same(a, b):
    return all(np.array_equal(x, y) for x, y in zip(a, b))


class Captured:
    """Calls captured on one stream in a mode (0: global), replayed on any."""

    def __init__(self, stream, mode, calls):
        self.hip, self.graph, self.exec, h = C.CDLL("libamdhip64.so.7"), C.c_void_p(), C.c_void_p(), C.c_void_p(stream.handle)
        assert self.hip.hipStreamBeginCapture(h, mode) == 0
        for c in calls:
            c(stream.handle)
        assert self.hip.hipStreamEndCapture(h, C.byref(self.graph)) == 0
        assert self.hip.hipGraphInstantiate(C.byref(self.exec), self.graph, None, None, C.c_size_t(0)) == 0

    def launch(self, stream):
        assert self.hip.hipGraphLaunch(self.exec, C.c_void_p(stream.handle)) == 0

    def close(self):
        assert self.hip.hipGraphExecDestroy(self.exec) == 0 and self.hip.hipGraphDestroy(self.graph) == 0


def test_two_streams_at_once(gpu):
    nm = gpu
    a = [Calls(nm, i, 2000 + i, 70 + i, 264, 30000, 9001) for i in range(4)]
    b = [Calls(nm, 9 + i, 5000 + i, 100 + i, 136, 20008, 7000) for i in range(4)]
    want = [c.expected() for c in a + b]
    s, t = nm.Stream(), nm.Stream()
    for turn in range(5):
        print(f"[two streams, turn {turn}]", flush=True)
        for x, y in zip(a, b):
            x(s.handle)
            y(t.handle)
        s.sync(), t.sync()
        for c, w in zip(a + b, want):
            assert same(c.results(), w)
    s.destroy(), t.destroy()


@pytest.mark.parametrize("mode", [0, 1, 2])
def test_a_graph_beside_eager_calls(gpu, mode):
    """The captured calls are the first of their sizes on their stream, in each mode of capture."""
    nm = gpu
    a = [Calls(nm, 20 + i, 3000 + 1000 * mode, 60 + 8 * mode + i, 264, 30000, 9001) for i in range(3)]
    b = [Calls(nm, 30 + i, 2500, 90 + i, 136, 20008, 7000) for i in range(3)]
    want = [c.expected() for c in a + b]
    s, t = nm.Stream(), nm.Stream()
    nm.synchronize()
    g = Captured(s, mode, a)
    for turn in range(4):
        print(f"[graph of mode {mode}, turn {turn}]", flush=True)
        g.launch(t)
        for c in b:
            c(s.handle)
        s.sync(), t.sync()
        for c, w in zip(a + b, want):
            assert same(c.results(), w)
    for c in b:      # and the graph on the stream that it was captured on
        c(t.handle)
    g.launch(s)
    s.sync(), t.sync()
    for c, w in zip(a + b, want):
        assert same(c.results(), w)
    g.close()
    s.destroy(), t.destroy()

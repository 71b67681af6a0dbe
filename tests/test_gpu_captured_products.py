"""Captured sorts and products whose sums are in parts, and larger calls later: a graph's addresses stay its own.  In a process of
its own, where the library's buffers are as small as the captured calls made them."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

CHILD = """
import sys
import numpy as np
import naiwa_moe as nm
from test_gpu_linear import Stack
from test_gpu_mxfp4 import Graph
from test_gpu_tokens import raw_of, routing

grow_captured = sys.argv[1] == "captured"
rng = np.random.default_rng(3)


class Calls:
    # T tokens sorted; products and gradients of `rows` rows, long sums in few tiles
    def __init__(self, T, rows, n, k):
        self.sizes = T, rows, n, k
        self.W, self.U = (Stack(nm, rng, 1, n, k, "bf16") for _ in range(2))
        up = nm.DeviceBuffer.from_array
        self.ids = up(routing(rng, T, 4, 32)[0])
        self.x, self.dy = (up(raw_of(rng.standard_normal((rows, w)).astype(np.float32), "bf16")[0]) for w in (k, n))
        zeros = lambda m: up(np.zeros(m, np.uint32))
        self.out = [zeros(m) for m in (T * 4, T * 4, 33, rows * n, rows * k, n * k, n)]

    def __call__(self, s):
        (T, rows, n, k), o = self.sizes, self.out
        nm.expert_sort(self.ids, T, 4, 32, *o[:3], stream=s)
        nm.linear(self.W.w, self.x, rows, o[3], up=self.U.w, act=nm.ACT_SILU, out_dtype=nm.F32, stream=s)
        nm.linear_input_grad(self.W.w, self.dy, rows, o[4], dx_dtype=nm.F32, stream=s)
        nm.linear_weight_grad(self.dy, self.x, nm.BF16, rows, n, k, o[5], dbias=o[6], stream=s)

    def results(self):
        nm.synchronize()
        r = [b.download(np.uint32) for b in self.out]
        for b in self.out:
            b.upload(np.zeros(b.nbytes // 4, np.uint32))
        nm.synchronize()
        return r


small, large = Calls(2000, 4000, 256, 72), Calls(30000, 9000, 1000, 264)
wide, wider = Calls(2000, 100, 136, 30000), Calls(2000, 130, 264, 40000)   # the forward's sums in parts
st = nm.Stream()
g = Graph(nm, st, lambda: (small(st.handle), wide(st.handle)))            # the first calls of the process
big = Graph(nm, st, lambda: (large(st.handle), wider(st.handle))) if grow_captured else None
print("captured", flush=True)
want = {}
for c in (large, wider, small, wide):
    c(0)
    want[c] = c.results()
    assert all(r.any() for r in want[c])
# what the larger calls would have freed, in other hands
fills = [nm.DeviceBuffer.from_array(np.full(n, 0xA5, np.uint8)) for n in (4096, 1 << 16, 1 << 18, 1 << 20, 1 << 22)
         for _ in range(16)]
for _ in range(3):
    for graph, calls in ((g, (small, wide)), (big, (large, wider))):
        if graph:
            graph.launch()
            st.sync()
            for c in calls:
                assert all(np.array_equal(a, b) for a, b in zip(c.results(), want[c]))
    for c in (large, wider):
        c(0)
        assert all(np.array_equal(a, b) for a, b in zip(c.results(), want[c]))
assert all((f.download(np.uint8) == 0xA5).all() for f in fills)
print("done", flush=True)
"""


@pytest.mark.parametrize("grow", ["eager", "captured"])
def test_larger_calls_leave_the_buffers_of_graphs(gpu, grow):
    here = os.path.dirname(os.path.abspath(__file__))
    path = [here, os.path.join(os.path.dirname(here), "naiwa-rs_amd")]
    r = subprocess.run([sys.executable, "-c", CHILD, grow], capture_output=True, text=True, timeout=100,
                       env={**os.environ, "PYTHONPATH": os.pathsep.join(path)})
    assert r.returncode == 0 and "done" in r.stdout, r.stdout + r.stderr

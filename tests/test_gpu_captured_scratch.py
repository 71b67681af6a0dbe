"""Captured calls and the library's scratch buffers: a graph holds the addresses that its calls were given, so a
larger call later may not free them.  In a process of its own, where every buffer is as small as the captured calls
made it."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

CHILD = """
import sys
import numpy as np
import naiwa_moe as nm
from test_gpu_balance import make
from test_gpu_mxfp4 import Experts, Graph, bf16, route

grow_captured = sys.argv[1] == "captured"
rng = np.random.default_rng(3)
E, H, I, k = 8, 256, 128, 2
ex = Experts(nm, 5, E, H, I)
router = nm.DeviceBuffer.from_array((rng.standard_normal((E, H)) * 0.1).astype(np.float32))


class Calls:
    # routing, a decode call, a prompt chunk and the balance loss of T tokens
    def __init__(self, T):
        self.T = T
        up = nm.DeviceBuffer.from_array
        self.x = up(bf16(rng.standard_normal((T, H))))
        ids, w = route(rng, T, E, k)
        self.ids, self.w = up(ids), up(w)
        self.logits = up(make(rng, T, E, k, 1)[0])
        zeros = lambda n: up(np.zeros(n, np.uint32))
        self.out = [zeros(T * H), zeros(T * H), zeros(E), zeros(1), zeros(E), zeros(1), zeros(T * k), zeros(T * k)]

    def __call__(self, s):
        T, o = self.T, self.out
        nm.router_topk(self.x, nm.BF16, router, T, H, E, k, o[6], o[7], stream=s)
        nm.indexed_moe_fused_decode(ex.banks, self.x, nm.BF16, self.ids, self.w, T, k, o[0], stream=s)
        nm.moe_prefill(ex.banks, self.x, self.ids, self.w, T, k, o[1], stream=s)
        nm.router_balance(self.logits, nm.F32, self.ids, T, E, k, *o[2:6], stream=s)

    def results(self):
        nm.synchronize()
        r = [b.download(np.uint32) for b in self.out]
        for b in self.out:
            b.upload(np.zeros(b.nbytes // 4, np.uint32))
        nm.synchronize()
        return r


small, large = Calls(40), Calls(3000)
st = nm.Stream()
g = Graph(nm, st, lambda: small(st.handle))              # the first calls of the process
big = Graph(nm, st, lambda: large(st.handle)) if grow_captured else None
print("captured", flush=True)
large(0)
want_large = large.results()
small(0)
want_small = small.results()
assert all(r.any() for r in want_small + want_large)
# what the larger calls would have freed, in other hands
fills = [nm.DeviceBuffer.from_array(np.full(n, 0xA5, np.uint8)) for n in (4096, 1 << 16, 1 << 18, 1 << 20, 1 << 21)
         for _ in range(16)]
for _ in range(3):
    for graph, calls, want in ((g, small, want_small), (big, large, want_large)):
        if graph:
            graph.launch()
            st.sync()
            assert all(np.array_equal(a, b) for a, b in zip(calls.results(), want))
    large(0)
    assert all(np.array_equal(a, b) for a, b in zip(large.results(), want_large))
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

"""Per-expert counts, the balance loss and its gradient against 64 bits and differences.

Tolerances: a probability errs by a few 2^-24 (its exponential, the sum, the division) and
by |logit| 2^-24 through the difference to the row's largest; sums of them are f64 past 64
rows: 2e-6 relative for logits of a few units.  The gradient p (c - sum c p) is
formed from counts less an integer m next to the sum, so it errs by a few 2^-24 of p (|c - m| +
sum p |c - m|), which is of its own size: under 1e-5 of the norm.  bf16 gradients are rounded once: 2^-8 of a value each, at
most 2^-8 of the norm.
"""
import numpy as np
import pytest

from test_gpu_mxfp4 import bf16, f32_of, rel

pytestmark = pytest.mark.gpu


def reference(x, ids, E, mask, g):
    """(counts, N, P, loss, dlogits) in f64."""
    T, k = ids.shape
    live = np.ones(T, bool) if mask is None else mask != 0
    N = int(live.sum())
    inside = ids[live].ravel()
    counts = np.bincount(inside[inside < E].astype(np.int64), minlength=E)[:E]
    z = np.zeros((T, E))
    if N:
        y = x[live].astype(np.float64)
        y = np.exp(y - y.max(-1, keepdims=True))
        z[live] = y / y.sum(-1, keepdims=True)
    P = z.sum(0) / max(N, 1)
    loss = E / (k * max(N, 1)) * (counts * P).sum()
    d = g * E / (k * max(N, 1) ** 2) * z * (counts - (z * counts).sum(-1, keepdims=True))
    return counts, N, P, loss, d


def run(nm, x, ids, E, mask, g, bf=False, ld=0, ids_ld=0, acc=None):
    T, k = ids.shape
    raw = bf16(x) if bf else np.ascontiguousarray(x, np.float32)
    wide = np.full((T, ld or E), 0x7FC0 if bf else np.nan, raw.dtype)
    wide[:, :E] = raw
    wids = np.full((T, ids_ld or k), 0xFFFFFFFF, np.uint32)
    wids[:, :k] = ids
    dt = nm.BF16 if bf else nm.F32
    up = lambda a: nm.DeviceBuffer.from_array(a if a.size else np.zeros(16, np.uint8))  # noqa: E731
    xd, idd, md = up(wide), up(wids), None if mask is None else up(mask)
    counts, valid, probs, loss = (nm.DeviceBuffer.from_array(np.full(n, 0x7FFFFFFF, np.uint32)) for n in (E, 1, E, 1))
    nm.router_balance(xd, dt, idd, T, E, k, counts, valid, probs, loss, mask=md, ld=ld, ids_ld=ids_ld)
    gd = nm.DeviceBuffer.from_array(np.array([g], np.float32))
    start = np.full((T, ld or E), 5.0, np.float32) if acc is None else np.pad(acc, ((0, 0), (0, (ld or E) - E)),
                                                                           constant_values=5.0)
    dd = up(bf16(start) if bf else start.astype(np.float32))
    nm.router_balance_backward(xd, dt, counts, valid, T, E, k, gd, dd, mask=md, ld=ld, dld=ld, accumulate=acc is not None)
    d = dd.download(np.uint16 if bf else np.float32, T * (ld or E)).reshape(T, ld or E)
    d = f32_of(d) if bf else d
    assert (d[:, E:] == 5.0).all()   # between the rows nothing is written
    return (counts.download(np.uint32, E), int(valid.download(np.uint32, 1)[0]), probs.download(np.float32, E),
            float(loss.download(np.float32, 1)[0]), d[:, :E])


def make(rng, T, E, k, valid):
    x = (rng.standard_normal((T, E)) + 0.5 * rng.standard_normal(E)).astype(np.float32)
    ids = np.argsort(-x, axis=1, kind="stable")[:, :k].astype(np.uint32)
    mask = None if valid == 1 else (rng.random(T) < valid).astype(np.uint8) * 3
    return x, ids, mask


@pytest.mark.parametrize("T,E,k,valid", [
    (1, 1, 1, 1), (1, 8, 2, 1), (5, 8, 2, 0.5), (31, 60, 4, 1), (32, 64, 8, 0.9), (33, 65, 6, 1), (64, 127, 8, 0.7),
    (255, 128, 8, 1), (1000, 129, 3, 0.8), (4097, 256, 8, 1), (300, 1000, 32, 0.9), (70, 1024, 1, 1), (20001, 8, 2, 0.95),
])
@pytest.mark.parametrize("bf", [False, True])
def test_balance_against_64_bits(gpu, T, E, k, valid, bf):
    rng = np.random.default_rng(T + E)
    x, ids, mask = make(rng, T, E, k, valid)
    if bf:
        x = f32_of(bf16(x))
    print(f"[balance {T} {E} {k} {bf}]", flush=True)
    c, n, P, loss, d = run(gpu, x, ids, E, mask, 1.5, bf=bf)
    cw, nw, Pw, lw, dw = reference(x, ids, E, mask, 1.5)
    assert n == nw and np.array_equal(c, cw)
    assert rel(P, Pw) < 2e-6 and abs(loss - lw) <= 2e-6 * abs(lw)
    if E > 1:
        assert rel(d, dw) < (2.0 ** -8 if bf else 1e-5)
    else:
        assert (d == 0).all()   # one expert: nothing to balance


def test_balance_strides_accumulate_and_bad_ids(gpu):
    rng = np.random.default_rng(2)
    T, E, k = 100, 40, 4
    x, ids, mask = make(rng, T, E, k, 0.8)
    ids[3, 1], ids[50, 0] = E, 0xFFFFFFFF
    mask[3], mask[50] = 1, 1
    acc = rng.standard_normal((T, E)).astype(np.float32)
    c, n, P, loss, d = run(gpu, x, ids, E, mask, 300.0, ld=48, ids_ld=7, acc=acc)
    cw, nw, Pw, lw, dw = reference(x, ids, E, mask, 300.0)
    assert n == nw and np.array_equal(c, cw) and rel(P, Pw) < 2e-6 and abs(loss - lw) <= 2e-6 * lw
    assert rel(d - acc, dw) < 1e-5 + 2.0 ** -24 * np.linalg.norm(acc) / np.linalg.norm(dw)
    assert np.array_equal(d[mask == 0], acc[mask == 0])


def test_balance_of_nothing(gpu):
    """No tokens, and none that is valid: zeros, and no division by them."""
    rng = np.random.default_rng(3)
    x, ids, _ = make(rng, 9, 8, 2, 1)
    for T, mask in ((0, None), (9, np.zeros(9, np.uint8))):
        c, n, P, loss, d = run(gpu, x[:T], ids[:T], 8, mask, 1.0)
        assert n == 0 and loss == 0 and (c == 0).all() and (P == 0).all() and (d == 0).all()


def test_masked_rows_are_not_read(gpu):
    rng = np.random.default_rng(4)
    x, ids, mask = make(rng, 50, 16, 2, 0.6)
    x[mask == 0] = np.nan
    ids[mask == 0] = 99
    c, n, P, loss, d = run(gpu, x, ids, 16, mask, 1.0)
    cw, nw, Pw, lw, dw = reference(x, ids, 16, mask, 1.0)
    assert np.array_equal(c, cw) and rel(P, Pw) < 2e-6 and abs(loss - lw) < 2e-6 * lw and rel(d, dw) < 1e-5


def test_extreme_logits(gpu):
    """Rows of one sure expert, of equal logits, of the largest finite values and with -inf among them."""
    E, k = 8, 2
    x = np.zeros((6, E), np.float32)
    x[0, 3] = 1e4
    x[2] = 3e38
    x[3] = -3e38
    x[4, :4] = -np.inf
    x[5, 1:] = -np.inf
    ids = np.tile(np.array([[1, 3]], np.uint32), (6, 1))
    with np.errstate(over="ignore"):
        cw, nw, Pw, lw, dw = reference(x, ids, E, None, 1.0)
    c, n, P, loss, d = run(gpu, x, ids, E, None, 1.0)
    assert rel(P, Pw) < 2e-6 and abs(loss - lw) < 2e-6 * lw and rel(d, dw) < 1e-5
    x[1, 2] = np.nan
    _, _, P, loss, d = run(gpu, x, ids, E, None, 1.0)
    assert np.isnan(P).all() and np.isnan(loss) and np.isnan(d[1]).all() and np.isfinite(np.delete(d, 1, 0)).all()


def test_gradient_against_differences(gpu):
    """Central differences of the 64-bit loss at the device's own counts."""
    rng = np.random.default_rng(5)
    T, E, k = 7, 12, 3
    x, ids, mask = make(rng, T, E, k, 0.7)
    _, _, _, _, d = run(gpu, x, ids, E, mask, 1.0)
    h = 1e-4
    num = np.zeros((T, E))
    for t in range(T):
        for e in range(E):
            a, b = x.astype(np.float64).copy(), x.astype(np.float64).copy()
            a[t, e] += h
            b[t, e] -= h
            num[t, e] = (reference(a, ids, E, mask, 1.0)[3] - reference(b, ids, E, mask, 1.0)[3]) / (2 * h)
    # the differences err by h^2 / 6 of the third derivative, at most that of the values: 2e-9; and by 2e-16 / h
    assert np.abs(d - num).max() < 1e-5 * np.abs(num).max()


@pytest.mark.parametrize("T,E,k", [(1, 8, 2), (77, 128, 8), (40000, 60, 4)])
def test_expert_counts(gpu, T, E, k):
    nm = gpu
    rng = np.random.default_rng(T)
    ids = rng.integers(0, E + 2, (T, k)).astype(np.uint32)
    mask = (rng.random(T) < 0.8).astype(np.uint8)
    for m in (None, mask):
        live = ids if m is None else ids[m != 0]
        counts, bad = nm.DeviceBuffer(E * 4), nm.DeviceBuffer.from_array(np.array([77], np.uint32))
        nm.expert_counts(nm.DeviceBuffer.from_array(ids), T, k, E, counts,
                         mask=None if m is None else nm.DeviceBuffer.from_array(m), bad=bad)
        got = counts.download(np.uint32)
        assert np.array_equal(got, np.bincount(live.ravel().astype(np.int64), minlength=E + 2)[:E])
        assert bad.download(np.uint32)[0] == (live >= E).sum()


def test_counts_of_a_prompt_seed_an_expert_cache(gpu):
    """Router, its counts, and the cache policy that takes them: the next expert to load is the busiest."""
    nm = gpu
    rng = np.random.default_rng(9)
    T, H, E, k = 200, 64, 16, 2
    x, W = bf16(rng.standard_normal((T, H))), (rng.standard_normal((E, H)) * 0.1).astype(np.float32)
    ids, w, logits = nm.DeviceBuffer(T * k * 4), nm.DeviceBuffer(T * k * 4), nm.DeviceBuffer(T * E * 4)
    nm.router_topk(nm.DeviceBuffer.from_array(x), nm.BF16, nm.DeviceBuffer.from_array(W), T, H, E, k, ids, w,
                   logits_out=logits)
    counts, valid, probs, loss = (nm.DeviceBuffer(n * 4) for n in (E, 1, E, 1))
    nm.router_balance(logits, nm.F32, ids, T, E, k, counts, valid, probs, loss)
    alone = nm.DeviceBuffer(E * 4)
    nm.expert_counts(ids, T, k, E, alone)
    c = counts.download(np.uint32)
    assert np.array_equal(alone.download(np.uint32), c) and c.sum() == T * k
    cache = nm.policy.ExpertCache(E, 4, 4)
    cache.seed_hits(c.astype(np.uint64))
    assert cache.fill_candidate() == int(np.argmax(c))
    assert loss.download(np.float32)[0] >= 1.0 - 1e-3   # chosen experts are the probable ones


def test_results_repeat(gpu):
    rng = np.random.default_rng(10)
    x, ids, mask = make(rng, 5000, 128, 8, 0.9)
    first = run(gpu, x, ids, 128, mask, 1.0)
    for _ in range(3):
        again = run(gpu, x, ids, 128, mask, 1.0)
        assert all(np.array_equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("T,E,ld", [(300, 8, 8), (77, 128, 132), (50, 60, 61), (70, 500, 500)])
@pytest.mark.parametrize("bf", [False, True])
def test_gradient_in_the_logits_place(gpu, T, E, ld, bf):
    nm = gpu
    rng = np.random.default_rng(E)
    x, ids, mask = make(rng, T, E, 4, 0.7)
    wide = np.zeros((T, ld), np.float32)
    wide[:, :E] = x
    raw, dt = (bf16(wide), nm.BF16) if bf else (wide, nm.F32)
    xd, idd, md = (nm.DeviceBuffer.from_array(a) for a in (raw, ids, mask))
    counts, valid, probs, loss, dd = (nm.DeviceBuffer.from_array(a) for a in (
        np.zeros(E, np.uint32), np.zeros(1, np.uint32), np.zeros(E, np.float32), np.zeros(1, np.float32), raw))
    gd = nm.DeviceBuffer.from_array(np.array([0.5], np.float32))
    nm.router_balance(xd, dt, idd, T, E, 4, counts, valid, probs, loss, mask=md, ld=ld)
    nm.router_balance_backward(xd, dt, counts, valid, T, E, 4, gd, dd, mask=md, ld=ld, dld=ld)
    nm.router_balance_backward(xd, dt, counts, valid, T, E, 4, gd, xd, mask=md, ld=ld, dld=ld)
    assert np.array_equal(xd.download(raw.dtype), dd.download(raw.dtype))


def test_captured_and_replayed(gpu):
    """Counts, loss and gradient in a graph, replayed on new inputs between eager calls of other sizes."""
    from test_gpu_mxfp4 import Graph

    nm = gpu
    rng = np.random.default_rng(9)
    T, E, k = 5000, 64, 6
    sets = [make(rng, T, E, k, 1)[:2] for _ in range(3)]
    big = make(rng, 2 * T, E, k, 1)[:2]

    def call(x, ids, T, stream):
        nm.router_balance(x, nm.F32, ids, T, E, k, *out[:4], stream=stream)
        nm.router_balance_backward(x, nm.F32, out[0], out[1], T, E, k, gd, out[4], stream=stream)

    out = [nm.DeviceBuffer(n * 4) for n in (E, 1, E, 1, 2 * T * E)]
    gd = nm.DeviceBuffer.from_array(np.array([1.0], np.float32))
    xd, idd = nm.DeviceBuffer.from_array(sets[0][0]), nm.DeviceBuffer.from_array(sets[0][1])
    bx, bi = nm.DeviceBuffer.from_array(big[0]), nm.DeviceBuffer.from_array(big[1])
    call(bx, bi, 2 * T, 0)           # the scratch is as large as it will be
    st = nm.Stream()
    g = Graph(nm, st, lambda: call(xd, idd, T, st.handle))
    for x, ids in sets:
        xd.upload(x)
        idd.upload(ids)
        call(xd, idd, T, 0)
        nm.synchronize()
        want = [o.download(np.uint32, n) for o, n in zip(out, (E, 1, E, 1, T * E))]
        call(bx, bi, 2 * T, 0)
        nm.synchronize()
        for _ in range(2):
            g.launch()
            st.sync()
            for o, v in zip(out, want):
                assert np.array_equal(o.download(np.uint32, v.size), v)
    g.close()


def backward(nm, x, counts, valid, k, g=1.0, bf=False, ld=0):
    """dlogits of counts and a number of tokens that the caller has, of a longer batch say."""
    T, E = x.shape
    wide = np.zeros((T, ld or E), np.float32)
    wide[:, :E] = x
    raw = bf16(wide) if bf else wide
    xd, dd = nm.DeviceBuffer.from_array(raw), nm.DeviceBuffer.from_array(np.zeros_like(raw))
    cd, vd = nm.DeviceBuffer.from_array(counts.astype(np.uint32)), nm.DeviceBuffer.from_array(np.array([valid], np.uint32))
    gd = nm.DeviceBuffer.from_array(np.array([g], np.float32))
    nm.router_balance_backward(xd, nm.BF16 if bf else nm.F32, cd, vd, T, E, k, gd, dd, ld=ld, dld=ld)
    d = dd.download(np.uint16 if bf else np.float32, raw.size).reshape(raw.shape)[:, :E]
    return f32_of(d) if bf else d


@pytest.mark.parametrize("kind,E,k,N,spread", [
    ("even", 128, 8, 32768, 2), ("even", 128, 8, 1 << 18, 2), ("even", 60, 4, 1 << 22, 50), ("even", 1000, 8, 1 << 20, 3),
    ("even", 8, 2, (1 << 30) - 1, 5),      # counts past 2^24
    ("even", 16, 2, 1 << 20, 0),           # all alike: no gradient
    ("closed", 128, 8, 32768, 2),          # a quarter of the experts closed: -inf, and chosen by nobody
    ("sure", 128, 8, 32768, 300),          # rows that are almost sure of their expert
    ("one", 64, 2, 1 << 20, 0),            # all choices of one expert
])
@pytest.mark.parametrize("bf,ld", [(False, 0), (False, 1), (True, 0)])
def test_gradient_of_nearly_even_counts(gpu, kind, E, k, N, spread, bf, ld):
    """Counts that differ by much less than they are large, as the loss makes them.

    The gradient p_j (c_j - s), s = sum p c, does not change when all counts do by an integer m.  With m next
    to s, c_j - m is exact up to 2^24 and s - m errs by a few 2^-24 of sum p |c - m|, which is of the size of the
    gradient's own c_j - s: with a probability's few 2^-24 (and |logit| 2^-24) under 1e-5 of the norm."""
    rng = np.random.default_rng(E + N % 1000 + spread)
    T = 200
    x = (rng.standard_normal((T, E)) * (8.0 if kind == "sure" else 1.0)).astype(np.float32)
    live = E - E // 4 if kind == "closed" else E
    counts = N * k // live + np.rint(rng.standard_normal(E) * spread).astype(np.int64)
    if kind == "closed":
        x[:, live:] = -np.inf
        counts[live:] = 0
    if kind == "one":
        counts[:] = 0
        counts[3] = N * k
    if bf:
        x = f32_of(bf16(x))
    z = np.exp(x.astype(np.float64) - x.max(-1, keepdims=True))
    z /= z.sum(-1, keepdims=True)
    want = E / (k * float(N) ** 2) * z * (counts - (z * counts).sum(-1, keepdims=True))
    print(f"[backward {kind} {E} {N} {bf} {ld}]", flush=True)
    d = backward(gpu, x, counts, N, k, bf=bf, ld=E + 1 if ld else 0)
    if spread == 0 and kind == "even":
        assert (d == 0).all()
    else:
        assert rel(d, want) < (2.0 ** -8 if bf else 1e-5)


FIRST_CALL_CAPTURED = """
import numpy as np
import naiwa_moe as nm
from test_gpu_balance import make, reference
from test_gpu_mxfp4 import Graph

rng = np.random.default_rng(1)
T, E, k = 5000, 64, 6
x, ids, _ = make(rng, T, E, k, 1)
xd, idd = nm.DeviceBuffer.from_array(x), nm.DeviceBuffer.from_array(ids)
out = [nm.DeviceBuffer.from_array(np.full(n, 7, np.uint32)) for n in (E, 1, E, 1)]
dirty = [nm.DeviceBuffer.from_array(np.full(1 << 16, 0xFF, np.uint8)) for _ in range(64)]
nm.synchronize()
del dirty
call = lambda s: nm.router_balance(xd, nm.F32, idd, T, E, k, *out, stream=s)
st = nm.Stream()
g = Graph(nm, st, lambda: call(st.handle))
loss = reference(x, ids, E, None, 1.0)[3]
for launch in (lambda: call(0), g.launch, lambda: call(0), g.launch, g.launch):
    out[3].upload(np.zeros(1, np.float32))
    nm.synchronize()
    launch()
    nm.synchronize()
    assert abs(out[3].download(np.float32, 1)[0] - loss) <= 2e-6 * loss, out[3].download(np.float32, 1)
    assert out[1].download(np.uint32, 1)[0] == T
g.close()
print("done", flush=True)
"""


def test_first_call_of_a_process_captured(gpu):
    """What a call keeps in its scratch needs no earlier call: the first one of a process is captured, into memory
    that held other things, and an eager call follows before the graph has run."""
    import os
    import subprocess
    import sys

    here = os.path.dirname(os.path.abspath(__file__))
    path = [here, os.path.join(os.path.dirname(here), "naiwa-rs_amd")]
    r = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED], capture_output=True, text=True, timeout=100,
                       env={**os.environ, "PYTHONPATH": os.pathsep.join(path)})
    assert r.returncode == 0 and "done" in r.stdout, r.stdout + r.stderr

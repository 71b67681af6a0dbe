"""MXFP4 on the host: sizes, the GGML conversion, the GGUF path and every refusal (no device)."""
import ctypes as C

import numpy as np
import pytest

import mxfp4_ref as M
import naiwa_moe as nm
from naiwa_moe import _lib
from naiwa_moe._lib import E_INVALID, E_TOO_LARGE, E_UNSUPPORTED, Bank


def test_projection_bytes_of_tile_order():
    L = nm.lib()
    for n, k in ((16, 32), (32, 128), (768, 2048), (2048, 1408), (48, 2880), (16, 544)):
        want = n // 16 * M.strip_bytes(k)
        assert L.naiwa_projection_bytes(nm.MXFP4_T, n, k) == want
        assert nm.projection_bytes(nm.MXFP4_T, n, k) == want
        assert nm.expert_range(nm.MXFP4_T, n, k, 3) == range(3 * want, 4 * want)
    assert L.naiwa_projection_bytes(nm.MXFP4_T, 8, 32) == -1      # rows in sixteens
    assert L.naiwa_projection_bytes(nm.MXFP4_T, 16, 48) == -1     # whole blocks
    assert L.naiwa_projection_bytes(nm.GGML_MXFP4, 16, 32) == -1  # banks hold the tile order
    with pytest.raises(ValueError):
        nm.projection_bytes(nm.MXFP4_T, 24, 32)


@pytest.mark.parametrize("n,k", [(16, 32), (32, 160), (16, 512), (48, 736), (16, 2880)])
def test_from_ggml_blocks(n, k):
    rng = np.random.default_rng(n * k)
    code = rng.integers(0, 16, (n, k), dtype=np.uint8)
    s = rng.integers(0, 256, (n, k // 32), dtype=np.uint8)
    assert np.array_equal(nm.mxfp4_from_ggml(M.ggml(code, s), n, k), M.tiled(code, s))
    with pytest.raises(ValueError):
        nm.mxfp4_from_ggml(np.zeros(17, np.uint8), n, 2 * k)


def test_from_ggml_refuses():
    f = nm.lib().naiwa_mxfp4_from_ggml
    b = np.zeros(4096, np.uint8)
    p = b.ctypes.data
    assert f(p, 8, 32, p + 2048) == E_INVALID
    assert f(p, 16, 48, p + 2048) == E_INVALID
    assert f(p, -16, 32, p + 2048) == E_INVALID
    assert f(None, 16, 32, p) == E_INVALID and f(p, 16, 32, None) == E_INVALID
    assert f(None, 0, 32, None) == 0


def _quantize(**a):
    d = dict(src=4096, dt=nm.F32, batch=1, n=16, k=64, ld=0, ss=0, dst=8192, ds=0)
    d.update(a)
    return nm.lib().naiwa_mxfp4_quantize(d["src"], d["dt"], d["batch"], d["n"], d["k"], d["ld"], d["ss"], d["dst"],
                                         d["ds"], 0)


def _dequantize(**a):
    d = dict(src=4096, dt=nm.F32, batch=1, n=16, k=64, ld=0, ss=0, dst=8192, ds=0)
    d.update(a)
    return nm.lib().naiwa_mxfp4_dequantize(d["dst"], d["batch"], d["n"], d["k"], d["ds"], d["src"], d["dt"], d["ld"],
                                           d["ss"], 0)


@pytest.mark.parametrize("call", [_quantize, _dequantize])
def test_quantize_refuses(call):
    for bad in (dict(n=8), dict(k=48), dict(batch=-1), dict(n=-16), dict(k=-32), dict(ld=56), dict(ld=-8), dict(ld=68),
                dict(batch=2, ss=64), dict(ss=-8), dict(batch=2, ds=1024), dict(ds=-16), dict(ds=1288), dict(src=None),
                dict(dst=None), dict(src=4104), dict(dst=8200), dict(batch=2, ss=1028)):
        assert call(**bad) == E_INVALID, bad
    for bad in (dict(dt=nm.Q8_0), dict(dt=nm.MXFP4_T), dict(n=1 << 32), dict(k=1 << 32), dict(n=1 << 30, k=1 << 16)):
        assert call(**bad) == E_UNSUPPORTED, bad
    assert call(batch=0) == 0 and call(n=0) == 0 and call(k=0) == 0   # nothing to do, and no device call
    assert _dequantize(dt=nm.F16) == E_UNSUPPORTED


def _bank(n, k, dtype=nm.MXFP4_T, slots=4, base=1 << 20, stride=None):
    if stride is None:
        stride = nm.slot_stride(dtype, n, k)
    return Bank(base, stride, slots, n, k, dtype)


def _decode(g, u, d, x=4096, dt=nm.BF16, ids=4096, w=4096, rows=1, width=2, act=0, out=4096, flags=0, f="ex"):
    fn = getattr(nm.lib(), "naiwa_moe_decode_" + f)
    return fn(C.byref(g), C.byref(u), C.byref(d), x, dt, ids, w, rows, width, act, out, flags, 0)


def _prefill(g, u, d, x=4096, ids=4096, w=4096, rows=1, width=2, act=0, out=4096, flags=0):
    return nm.lib().naiwa_moe_prefill(C.byref(g), C.byref(u), C.byref(d), x, ids, w, rows, width, act, out, flags, 0)


def test_expert_products_refuse():
    H, I = 256, 96
    ok = (_bank(I, H), _bank(I, H), _bank(H, I))
    shapes = [
        (_bank(I, H), _bank(I, H), _bank(H, I + 32)), (_bank(I, H + 32), _bank(I, H), _bank(H, I)),
        (_bank(I, H), _bank(I + 16, H), _bank(H, I)), (_bank(I, H, slots=5), _bank(I, H), _bank(H, I)),
        (_bank(I, H, base=None), _bank(I, H), _bank(H, I)), (_bank(I, H, base=(1 << 20) + 8), _bank(I, H), _bank(H, I)),
        (_bank(I, H, stride=1024), _bank(I, H), _bank(H, I)), (_bank(I, H, slots=0), _bank(I, H), _bank(H, I)),
        (_bank(I - 16, H), _bank(I - 16, H), _bank(H, I, stride=1 << 20)),
    ]
    for f in ("ex", "noalloc"):
        for b in shapes:
            assert _decode(*b, f=f) == E_INVALID
        # mixed formats, either way round
        assert _decode(_bank(I, H), _bank(I, H), Bank(1 << 20, 1 << 20, 4, H, I, nm.Q8_0), f=f) == E_UNSUPPORTED
        assert _decode(Bank(1 << 20, 1 << 20, 4, I, H, nm.Q8_0), Bank(1 << 20, 1 << 20, 4, I, H, nm.Q8_0), _bank(H, I),
                       f=f) == E_UNSUPPORTED
        assert _decode(Bank(1 << 20, 1 << 20, 4, I, H, nm.GGML_MXFP4), ok[1], ok[2], f=f) == E_UNSUPPORTED
        for bad, rc in ((dict(x=None), E_INVALID), (dict(out=None), E_INVALID), (dict(ids=None), E_INVALID),
                        (dict(w=None), E_INVALID), (dict(x=4104), E_INVALID), (dict(out=4100), E_INVALID),
                        (dict(dt=nm.F16), E_UNSUPPORTED), (dict(act=2), E_UNSUPPORTED), (dict(rows=-1), E_INVALID),
                        (dict(rows=4097), E_INVALID), (dict(rows=4096, width=17), E_INVALID), (dict(flags=2), E_INVALID),
                        (dict(width=65), E_UNSUPPORTED)):
            assert _decode(*ok, f=f, **bad) == rc, bad
        assert _decode(*ok, f=f, rows=0) == 0
    for b in shapes:
        assert _prefill(*b) == E_INVALID
    for bad, rc in ((dict(x=None), E_INVALID), (dict(out=None), E_INVALID), (dict(ids=None), E_INVALID),
                    (dict(w=None), E_INVALID), (dict(x=4104), E_INVALID), (dict(out=4100), E_INVALID),
                    (dict(act=2), E_UNSUPPORTED), (dict(rows=-1), E_INVALID), (dict(width=0), E_INVALID),
                    (dict(rows=65537, width=1), E_UNSUPPORTED), (dict(flags=4), E_INVALID), (dict(width=65), E_UNSUPPORTED)):
        assert _prefill(*ok, **bad) == rc, bad
    assert _prefill(*ok, rows=0) == 0
    many = (_bank(I, H, slots=4097), _bank(I, H, slots=4097), _bank(H, I, slots=4097))
    assert _decode(*many) == E_UNSUPPORTED and _prefill(*many) == E_UNSUPPORTED


def test_noalloc_admission():
    H, I = 4096, 14336
    b = (_bank(I, H), _bank(I, H), _bank(H, I))
    need = nm.lib().naiwa_moe_decode_scratch_bytes(300, 2, H, I, nm.MXFP4_T)
    assert need > 8 << 20
    assert _decode(*b, rows=300, f="noalloc") == E_TOO_LARGE
    assert nm.lib().naiwa_moe_decode_scratch_bytes(0, 2, H, I, nm.MXFP4_T) == 0
    assert nm.lib().naiwa_moe_decode_scratch_bytes(1, 2, H, I + 16, nm.MXFP4_T) == -1


def test_cpu_experts_and_fused_stack_refuse_tile_order():
    """The paths without MXFP4: the CPU misses and the one-launch stack."""
    L, H, I = nm.lib(), 256, 96
    layer = (_lib.Layer * 1)(_lib.Layer(4096, _bank(I, H), _bank(I, H), _bank(H, I), None))
    assert L.naiwa_stack_decode(layer, 1, 4096, 1, H, 4, 2, 0, 0, None, None, nm._lib.STACK_FUSED, 0) in (E_INVALID,
                                                                                                          E_UNSUPPORTED)
    b = np.zeros(1 << 20, np.uint8)
    ex = _lib.HostExperts(b.ctypes.data, b.ctypes.data, b.ctypes.data, 1 << 16, 1 << 16, 1 << 16, nm.MXFP4_T, nm.MXFP4_T,
                          nm.MXFP4_T, 4, H, I)
    x, out = np.zeros(H, np.float32), np.zeros(H, np.float32)
    ids, w = np.zeros(2, np.uint32), np.ones(2, np.float32)
    rc = L.naiwa_cpu_moe_decode(C.byref(ex), x.ctypes.data, ids.ctypes.data, w.ctypes.data, 1, 2, 0, out.ctypes.data)
    assert rc in (E_INVALID, E_UNSUPPORTED)


def test_gguf_mxfp4_stacks_are_laid_out_in_tile_order(tmp_path, monkeypatch):
    """A GGUF file's MXFP4 experts through host_stacks (pinned memory replaced: no device here)."""
    from gguf_writer import write_gguf
    from naiwa_moe import gguf, ops

    class Plain:
        def __init__(self, nbytes):
            self.a = np.zeros(nbytes, np.uint8)
            self.ptr, self.nbytes = self.a.ctypes.data, nbytes

        def view(self, dtype=np.uint8):
            return self.a.view(dtype)

    monkeypatch.setattr(ops, "PinnedBuffer", Plain)
    E, H, I = 3, 160, 64
    rng = np.random.default_rng(5)
    tensors, want = [], []
    for name, n, k in (("gate", I, H), ("up", I, H), ("down", H, I)):
        code = rng.integers(0, 16, (E, n, k), dtype=np.uint8)
        s = rng.integers(100, 140, (E, n, k // 32), dtype=np.uint8)
        blocks = np.concatenate([M.ggml(code[e], s[e]) for e in range(E)])
        tensors.append((f"blk.0.ffn_{name}_exps.weight", (k, n, E), nm.GGML_MXFP4, blocks.tobytes()))
        want.append([M.tiled(code[e], s[e]) for e in range(E)])
    path = tmp_path / "m.gguf"
    write_gguf(path, [], tensors)
    with gguf.GgufFile(path) as f:
        assert gguf.type_size(nm.GGML_MXFP4) == (32, 17)
        stacks = f.host_stacks(0)
        assert stacks.expert_bytes == [nm.projection_bytes(nm.MXFP4_T, n, k) for n, k in ((I, H), (I, H), (H, I))]
        for p in range(3):
            for e in range(E):
                assert np.array_equal(stacks.view(p)[e], want[p][e])


@pytest.mark.parametrize("rows,k,slots,H,I,by_pair", [
    (1, 64, 64, 8192, 28672, True),                                     # one token, whatever the sizes
    (2, 8, 128, 2048, 768, True), (4, 8, 128, 2048, 768, True), (6, 8, 128, 2048, 768, False),
    (4, 6, 64, 2048, 1408, True), (5, 6, 64, 2048, 1408, False), (2, 2, 8, 4096, 14336, False),
    (8, 2, 8, 1024, 2048, True), (9, 2, 8, 1024, 2048, False), (2, 1, 1, 32, 32, True), (3, 1, 1, 32, 32, False),
])
def test_few_tokens_by_pair(rows, k, slots, H, I, by_pair):
    """By the bytes that the pairs read and by how often an expert is read, not by the rows alone."""
    f = nm.lib().naiwa_mx_by_pair
    f.restype = C.c_bool
    assert f(rows, C.c_int64(rows * k), slots, H, I) == by_pair


def test_tile_list_of_one_token_is_written_whole():
    """A wave lists one token's pairs and clears the other entries, an entry a lane: at every width the list
    holds every pair and has no entry past the wave's 64 lanes (72 at width 64 were 8 that nobody wrote)."""
    f = nm.lib().naiwa_mx_tiles
    f.restype = C.c_int
    for width in range(1, 65):
        for slots in (1, 8, 64, 4096):
            t = f(1, C.c_int64(width), slots)
            assert width <= t <= 64 and t % 8 == 0, (width, slots)
    # of more tokens at most a tile a slot and one for every further 64 pairs
    for n, slots in ((2, 1), (65, 1), (66, 2), (512, 128), (65536, 4096), (8192, 4096)):
        assert f(2, C.c_int64(n), slots) >= min(n, slots) + (n - min(n, slots)) // 64


def _cached(g, u, d, H, I, top_k=2, act=0, usable=2, ring=2):
    """naiwa_cached_layer_create over made-up addresses, refused before any of them is used."""
    r = nm.policy.StagingRing()
    desc = _lib.CachedLayerDesc(4096, None, g, u, d, 1 << 20, 1 << 20, 1 << 20, 8, top_k, H, I, usable, 0, act, 0)
    h = C.c_void_p()
    rc = nm.lib().naiwa_cached_layer_create(C.byref(desc), r._h, ring, 0, C.byref(h))
    assert h.value is None
    return rc


def test_cached_layer_refuses_banks_that_its_steps_could_not_run():
    H, I = 256, 96
    ok = _bank(I, H), _bank(I, H), _bank(H, I)
    q = lambda n, k: Bank(1 << 20, 1 << 20, 4, n, k, nm.Q8_0)  # noqa: E731
    for mixed in ((ok[0], ok[1], q(H, I)), (q(I, H), ok[1], ok[2]), (q(I, H), q(I, H), ok[2]), (ok[0], q(I, H), q(H, I))):
        assert _cached(*mixed, H, I) == E_UNSUPPORTED
    assert _cached(*ok, H, I, top_k=65) == E_UNSUPPORTED and _cached(*ok, H, I, act=2) == E_UNSUPPORTED
    many = _bank(I, H, slots=5000), _bank(I, H, slots=5000), _bank(H, I, slots=5000)
    assert _cached(*many, H, I) == E_UNSUPPORTED
    assert _cached(_bank(I, H, slots=5), ok[1], ok[2], H, I) == E_INVALID
    assert _cached(_bank(I, H, base=(1 << 20) + 8), ok[1], ok[2], H, I) == E_INVALID
    assert _cached(_bank(80, H), _bank(80, H), Bank(1 << 20, 1 << 20, 4, H, 80, nm.MXFP4_T), H, 80) == E_INVALID


def test_expert_products_past_a_launch_are_refused():
    """More blocks than a launch's 2^32 threads: 4096 slots of 2^20 features, a pair each; and more blocks of
    features than a grid has along y."""
    H, I = 32, 1 << 20
    b = [_bank(n, k, slots=4096, base=1 << 40) for n, k in ((I, H), (I, H), (H, I))]
    for call in (_decode, _prefill):
        assert call(*b, rows=512, width=8) == E_UNSUPPORTED
    wide = [_bank(n, k, base=1 << 40) for n, k in (((1 << 21) + 128, H), ((1 << 21) + 128, H), (H, (1 << 21) + 128))]
    for call in (_decode, _prefill):
        assert call(*wide) == E_UNSUPPORTED


def test_from_ggml_refuses_outputs_that_it_may_not_write():
    """A read-only array (a view of a mapped file, say), one of another size or type, one over the blocks."""
    size = nm.projection_bytes(nm.MXFP4_T, 16, 32)
    mem = np.zeros(4096, np.uint8)
    blocks = mem[:16 * 17]
    fixed = np.zeros(size, np.uint8)
    fixed.flags.writeable = False
    for out in (fixed, np.zeros(size + 1, np.uint8), np.zeros(size, np.int8), np.zeros(2 * size, np.uint8)[::2],
                mem[16:16 + size]):
        with pytest.raises(ValueError):
            nm.mxfp4_from_ggml(blocks, 16, 32, out)
    assert nm.mxfp4_from_ggml(blocks, 16, 32, mem[1024:1024 + size]).size == size

"""The MXFP4 experts' operators and the router's balance loss, as measurable cases.

Four kinds of call:

- ``quantize``: a stack of projections to MXFP4 in matrix-core tile order and back
  (``mxfp4_quantize``, ``mxfp4_dequantize``);
- ``decode``: the routed experts of a decode step over MXFP4 banks
  (``indexed_moe_fused_decode``);
- ``prefill``: the routed experts of a prompt chunk over MXFP4 banks (``moe_prefill``);
- ``balance``: a router's per-expert counts and balance loss, and the loss's gradient
  (``router_balance``, ``router_balance_backward``).

MXFP4: blocks of 32 values along a row share a scale 2^(s - 127), s a byte (255: the
block is NaN); a value is a 4-bit E2M1 number times it.  Tile order: rows in strips of
16, K padded to whole steps of 128 values; of each step, lane 16 b + r holds block b (of
4) of row r as 16 bytes, value 2 i in the low half of byte i; after every 4 steps (or
what is left) come 4 scale bytes a lane, byte j of step j.

Activations are N(0, 1), weights N(0, 0.02), router logits of the scale that such
activations and routers give, with experts of unequal popularity.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
ACTS = ("silu", "gelu")
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)

# Shapes that the repository's configurations and benchmark name: hidden, intermediate, experts, top-k.
SHAPES = {
    "small": dict(hidden=1024, inter=2048, experts=8, topk=2),
    "qwen3": dict(hidden=2048, inter=768, experts=128, topk=8),
    "deepseek": dict(hidden=2048, inter=1408, experts=64, topk=6),
    "mixtral": dict(hidden=4096, inter=14336, experts=8, topk=2),
}


def _experts(name, kind, shape, rows, **more):
    c = dict(name=name, kind=kind, rows=rows, shared=0, act="silu", x="bf16", accumulate=False, residual=False, drop=0.0)
    c.update(SHAPES[shape])
    c.update(more)
    return c


def listed():
    return [
        # one expert's projection, as a program that replaces a single expert converts it
        dict(name="quantize_projection", kind="quantize", batch=1, n=768, k=2048, src="bf16", dst="f32"),
        # a layer's stacked gate projections at load time
        dict(name="quantize_stack", kind="quantize", batch=128, n=768, k=2048, src="bf16", dst="bf16"),
        # the smallest call: one token through a small 8-expert layer, where launches and latency count
        _experts("small_decode_1row", "decode", "small", 1),
        # single-user decode of a model with many small experts
        _experts("qwen3_decode_1row", "decode", "qwen3", 1),
        # an odd batch of a model with an odd intermediate size, f32 activations as a host engine hands them over
        _experts("deepseek_decode_5rows", "decode", "deepseek", 5, x="f32"),
        # a serving batch through few large experts: every expert read once for a few rows
        _experts("mixtral_decode_16rows", "decode", "mixtral", 16),
        # continuous batching: every one of many experts touched by a few rows
        _experts("qwen3_decode_96rows", "decode", "qwen3", 96),
        # a 512-token prompt chunk of a model with fine-grained and shared experts, residual added in place
        _experts("deepseek_prefill_512", "prefill", "deepseek", 512, shared=2, residual=True),
        # a whole prompt of odd length in one call
        _experts("qwen3_prefill_1999", "prefill", "qwen3", 1999),
        # a long prompt through few large experts
        _experts("mixtral_prefill_4096", "prefill", "mixtral", 4096),
        # a small training batch's router: launches and latency count
        dict(name="balance_61", kind="balance", tokens=61, experts=8, topk=2, logits="f32", valid=1.0),
        # a long batch, padded behind its sequences
        dict(name="balance_32768", kind="balance", tokens=32768, experts=128, topk=8, logits="f32", valid=0.8),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choices(["quantize", "decode", "prefill", "balance"], [2, 5, 4, 3])[0]
    if kind == "quantize":
        c = dict(kind=kind, batch=_log_uniform(rng, 1, 128), n=16 * _log_uniform(rng, 2, 256), k=32 * _log_uniform(rng, 1, 256),
                 src=rng.choice(["bf16", "f32", "f16"]), dst=rng.choice(["bf16", "f32"]))
        c["batch"] = max(1, min(c["batch"], 128 * 768 * 2048 // (2 * c["n"] * c["k"])))
        return c
    if kind == "balance":
        c = dict(kind=kind, tokens=_log_uniform(rng, 1, 32768), experts=rng.choice([8, 16, 60, 64, 127, 128]),
                 logits=rng.choice(["f32", "f32", "bf16"]), valid=rng.choice([1.0, 0.9, 0.5]))
        c["topk"] = rng.randint(1, 8)
        return c
    c = dict(kind=kind, act=rng.choice(["silu", "silu", "gelu"]), x="bf16", accumulate=rng.random() < 0.25, residual=False,
             drop=rng.choice([0.0, 0.0, 0.1, 0.4]))
    if rng.random() < 0.25:  # few large experts
        c.update(hidden=4096, inter=256 * rng.randint(24, 56), experts=8, topk=2)
    else:  # many small ones; sizes that are no multiple of a step among them
        c.update(hidden=32 * rng.randint(16, 160), experts=rng.choice([8, 16, 32, 60, 64, 128]), topk=rng.randint(1, 8),
                 inter=32 * rng.randint(8, 64))
    c["shared"] = rng.choice([0, 0, 0, 1, 2])
    if kind == "decode":
        c["rows"] = _log_uniform(rng, 1, 256)
        c["x"] = rng.choice(["bf16", "bf16", "f32"])
        return c
    c["residual"] = rng.random() < 0.5
    # at most the largest listed case's products, and the table's 65,536 pairs
    width = c["topk"] + c["shared"]
    top = 4096 * 2 * 4096 * 14336 // (width * c["hidden"] * c["inter"])
    c["rows"] = _log_uniform(rng, 48, max(64, min(4096, top, 65536 // width)))
    return c


# ---- what a program has in hand -----------------------------------------------------------


def _steps(k):
    return -(-k // 128)


def projection_bytes(n, k):
    s = _steps(k)
    return n // 16 * (1024 * s + 256 * -(-s // 4))


def _codes(x):
    """MXFP4 codes [n, k] uint8 and scale bytes [n, k / 32] uint8 of f32 rows."""
    b = x.view(x.shape[0], -1, 32)
    s = (((b.abs().amax(-1).view(torch.int32) >> 23) & 255) - 2).clamp_(min=0)
    y = torch.ldexp(b, (127 - s)[..., None])
    a = y.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code |= torch.signbit(y).to(torch.uint8) << 3
    return code.view(x.shape), s.to(torch.uint8)


def _tiled(code, s):
    """Tile-order bytes of one projection."""
    n, k = code.shape
    t = _steps(k)
    g = -(-t // 4)
    code = torch.nn.functional.pad(code, (0, 128 * t - k))
    nib = (code[:, 0::2] | (code[:, 1::2] << 4)).view(n // 16, 16, t, 4, 16).permute(0, 2, 3, 1, 4).reshape(n // 16, t, 1024)
    s = torch.nn.functional.pad(s, (0, 16 * g - k // 32)).view(n // 16, 16, g, 4, 4).permute(0, 2, 4, 1, 3).reshape(n // 16, g, 256)
    parts = []
    for i in range(g):
        parts += [nib[:, 4 * i:4 * i + 4].reshape(n // 16, -1), s[:, i]]
    return torch.cat(parts, 1).reshape(-1)


def _bank(slots, n, k, std, g):
    """[slots, stride] uint8: every slot's projection of N(0, std) weights, the stride a multiple of 256."""
    size = projection_bytes(n, k)
    bank = torch.empty(slots, -(-size // 256) * 256, dtype=torch.uint8, device=DEV)
    for e in range(slots):
        w = torch.randn(n, k, device=DEV, generator=g).mul_(std)
        bank[e, :size] = _tiled(*_codes(w))
    return bank


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(7919 * (seed + 1))
    s = {"case": case}
    if case["kind"] == "quantize":
        B, n, k = case["batch"], case["n"], case["k"]
        s["src"] = torch.empty(B, n, k, dtype=DTYPES[case["src"]], device=DEV)
        for e in range(B):
            s["src"][e] = torch.randn(n, k, device=DEV, generator=g).mul_(0.02)
        s["packed"] = torch.empty(B, -(-projection_bytes(n, k) // 256) * 256, dtype=torch.uint8, device=DEV)
        s["dst"] = torch.empty(B, n, k, dtype=DTYPES[case["dst"]], device=DEV)
        return s
    E, K = case["experts"], case["topk"]
    T = case["tokens"] if case["kind"] == "balance" else case["rows"]
    logits = torch.randn(T, E, device=DEV, generator=g) + 0.5 * torch.randn(E, device=DEV, generator=g)
    if case["kind"] == "balance":
        s["logits"] = logits.to(DTYPES[case["logits"]])
        s["ids"] = torch.topk(s["logits"].float(), K, dim=-1)[1].int()
        # padding behind the tokens, and one padded token in every 16 where there is padding
        at = torch.arange(T, device=DEV)
        pad = (at >= math.ceil(case["valid"] * T)) | (at % 16 == 15) if case["valid"] < 1 else at < 0
        s["mask"] = (~pad).to(torch.uint8)
        s["grad"] = torch.rand(1, device=DEV, generator=g) + 0.5
        s["counts"] = torch.empty(E, dtype=torch.int32, device=DEV)
        s["valid"] = torch.empty(1, dtype=torch.int32, device=DEV)
        s["probs"], s["loss"] = torch.empty(E, device=DEV), torch.empty(1, device=DEV)
        s["dlogits"] = torch.empty_like(s["logits"])
        return s
    H, I, width = case["hidden"], case["inter"], K + case["shared"]
    slots = E + case["shared"]
    s["gate"], s["up"] = _bank(slots, I, H, 0.02, g), _bank(slots, I, H, 0.02, g)
    s["down"] = _bank(slots, H, I, 0.02, g)
    top, ids = torch.topk(logits, K, dim=-1)
    s["ids"] = torch.empty(T, width, dtype=torch.int32, device=DEV)
    s["w"] = torch.ones(T, width, device=DEV)
    s["ids"][:, :K], s["w"][:, :K] = ids.int(), torch.softmax(top, -1)
    # always-on experts take the columns behind the routed ones, at weight 1
    s["ids"][:, K:] = torch.arange(E, slots, device=DEV)
    # entries that another part of the program serves: padding of weight 0 in a decode step, ids past the bank
    # in a prompt chunk
    out = torch.rand(T, K, device=DEV, generator=g) < case["drop"]
    if case["kind"] == "decode":
        s["w"][:, :K] *= ~out
        s["ids"][:, :K] *= ~out
    else:
        s["ids"][:, :K] = torch.where(out, slots, s["ids"][:, :K])
    s["x0"] = torch.randn(T, H, device=DEV, generator=g).to(DTYPES[case["x"]])
    s["x"] = s["x0"].clone()
    s["out0"] = 0.1 * torch.randn(T, H, device=DEV, generator=g)
    s["out"] = torch.zeros(T, H, device=DEV)
    s["most"] = int(torch.bincount(s["ids"].view(-1).long()).max())  # pairs of the busiest expert
    return s


# ---- one pass in plain form -----------------------------------------------------------------


def _values(bank, n, k):
    """[slots, n, k] f32 weights of tile-order banks."""
    B, t = bank.shape[0], _steps(k)
    g, whole = -(-t // 4), t // 4
    strips = bank[:, :projection_bytes(n, k)].view(B, n // 16, -1)
    full = strips[..., :whole * 4352].reshape(B, n // 16, whole, 4352)
    nib = full[..., :4096].reshape(B, n // 16, whole * 4, 1024)
    sc = full[..., 4096:]
    if whole < g:
        rest = strips[..., whole * 4352:]
        nib = torch.cat([nib, rest[..., :-256].reshape(B, n // 16, t - 4 * whole, 1024)], 2)
        sc = torch.cat([sc, rest[..., None, -256:]], 2)
    nib = nib.view(B, n // 16, t, 4, 16, 16).permute(0, 1, 4, 2, 3, 5)
    code = torch.stack([nib & 15, nib >> 4], -1).reshape(B, n, 4 * t, 32)
    sc = sc.reshape(B, n // 16, g, 4, 16, 4).permute(0, 1, 4, 2, 5, 3).reshape(B, n, 16 * g)[..., :4 * t].int()
    v = torch.tensor(E2M1, device=DEV)[code.int()]
    # 2^(s - 127) of a byte, in two factors (s = 0 alone would be subnormal), NaN for 255
    scale = torch.where(sc == 255, math.nan, torch.exp2((sc - 63).float()))
    return ((v * scale[..., None]) * 2.0 ** -64).reshape(B, n, 128 * t)[..., :k]


def _plain_quantize(s):
    case = s["case"]
    B, n, k = s["src"].shape
    x = s["src"].float().view(B, n, k // 32, 32)
    e = ((x.abs().amax(-1).view(torch.int32) >> 23) & 255) - 2
    e = e.clamp(min=0)
    y = torch.ldexp(x, (127 - e)[..., None])
    a = y.abs()
    q = 0.5 * ((a > 0.25).float() + (a >= 0.75) + (a > 1.25) + (a >= 1.75)) + (a > 2.5) + (a >= 3.5) + 2.0 * (a > 5.0)
    v = torch.ldexp(torch.copysign(q, y), (e - 127)[..., None])
    return v.view(B, n, k).to(DTYPES[case["dst"]])


def _plain_experts(s):
    case = s["case"]
    T, H, I, slots, width = case["rows"], case["hidden"], case["inter"], s["gate"].shape[0], s["ids"].shape[1]
    flat = s["ids"].view(-1).long()
    order = torch.argsort(flat, stable=True)
    e = flat[order]
    count = torch.zeros(slots + 1, dtype=torch.long, device=DEV).scatter_add_(0, flat, torch.ones_like(flat))
    place = torch.arange(T * width, device=DEV) - (torch.cumsum(count, 0) - count)[e]
    x = s["x0"].float()
    xe = torch.zeros(slots + 1, s["most"], H, device=DEV)
    xe[e, place] = x[order // width]
    xt = xe[:slots].transpose(1, 2).contiguous()
    g = torch.bmm(_values(s["gate"], I, H), xt)
    u = torch.bmm(_values(s["up"], I, H), xt)
    if case["act"] == "silu":
        a = g / (1.0 + torch.exp(-g))
    else:
        a = 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g)))
    y = torch.bmm(_values(s["down"], H, I), a * u).transpose(1, 2)
    y = torch.cat([y, torch.zeros(1, y.shape[1], H, device=DEV)])
    pairs = torch.zeros(T * width, H, device=DEV)
    pairs[order] = y[e, place] * s["w"].view(-1)[order][:, None]
    out = pairs.view(T, width, H).sum(1)
    if case["accumulate"]:
        out = s["out0"] + out
    got = {"out": out}
    if case["residual"]:
        got["x"] = (x + out).to(s["x0"].dtype)
    return got


def _plain_balance(s):
    case = s["case"]
    E, K = case["experts"], case["topk"]
    valid = s["mask"] != 0
    N = valid.sum()
    ids = torch.where(valid[:, None], s["ids"], E).view(-1).long()
    counts = torch.zeros(E + 1, dtype=torch.int32, device=DEV).scatter_add_(0, ids, torch.ones_like(ids, dtype=torch.int32))[:E]
    x = s["logits"].float()
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True) * valid[:, None]
    most = N.clamp(min=1).double()
    mean = p.double().sum(0) / most
    c = counts.double()
    loss = E / (K * most) * (c * mean).sum()
    off = counts.float() - (p * counts.float()).sum(-1, keepdim=True)
    grad = (s["grad"].double() * E / (K * most * most)).float() * p * off
    return {"counts": counts, "valid": N.int().view(1), "probs": mean.float(), "loss": loss.float().view(1),
            "dlogits": grad.to(s["logits"].dtype)}


# ---- one pass of the framework's own calls ------------------------------------------------------


def _nm():
    path = os.path.join(os.getcwd(), "naiwa-rs_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import naiwa_moe
    return naiwa_moe


def _own_banks(nm, s):
    """The layer's bank descriptors over the tensors that hold the weights, which a program makes once."""
    H, I = s["case"]["hidden"], s["case"]["inter"]
    if "banks" not in s:
        def bank(t, n, k):
            return nm.SlotBank(t.shape[0], n, k, nm.MXFP4_T, base=t.data_ptr(), stride=t.shape[1])
        s["banks"] = nm.LayerBanks.over(bank(s["gate"], I, H), bank(s["up"], I, H), bank(s["down"], H, I))
    return s["banks"]


def _own_quantize(nm, s):
    ids = {"f32": nm.F32, "bf16": nm.BF16, "f16": nm.F16}
    B, n, k = s["src"].shape
    stride = s["packed"].shape[1]
    nm.mxfp4_quantize(s["src"].data_ptr(), ids[s["case"]["src"]], n, k, s["packed"].data_ptr(), batch=B, dst_stride=stride)
    nm.mxfp4_dequantize(s["packed"].data_ptr(), n, k, s["dst"].data_ptr(), ids[s["case"]["dst"]], batch=B, src_stride=stride)
    return s["dst"]


def _own_experts(nm, s):
    case = s["case"]
    T, width = s["ids"].shape
    act = nm.ACT_SILU if case["act"] == "silu" else nm.ACT_GELU_PYTORCH_TANH
    ids, w, out = s["ids"].data_ptr(), s["w"].data_ptr(), s["out"].data_ptr()
    if case["accumulate"]:
        s["out"].copy_(s["out0"])
    if case["kind"] == "decode":
        nm.indexed_moe_fused_decode(_own_banks(nm, s), s["x0"].data_ptr(), nm.F32 if case["x"] == "f32" else nm.BF16, ids, w, T,
                                    width, out, act=act, accumulate=case["accumulate"])
        return {"out": s["out"]}
    x = s["x0"]
    if case["residual"]:
        x = s["x"]
        x.copy_(s["x0"])
    nm.moe_prefill(_own_banks(nm, s), x.data_ptr(), ids, w, T, width, out, act=act, accumulate=case["accumulate"],
                   residual=case["residual"])
    return {"out": s["out"], "x": x} if case["residual"] else {"out": s["out"]}


def _own_balance(nm, s):
    case = s["case"]
    T, E, K = case["tokens"], case["experts"], case["topk"]
    dt = nm.F32 if case["logits"] == "f32" else nm.BF16
    mask = s["mask"].data_ptr() if case["valid"] < 1 else None
    nm.router_balance(s["logits"].data_ptr(), dt, s["ids"].data_ptr(), T, E, K, s["counts"].data_ptr(), s["valid"].data_ptr(),
                      s["probs"].data_ptr(), s["loss"].data_ptr(), mask=mask)
    nm.router_balance_backward(s["logits"].data_ptr(), dt, s["counts"].data_ptr(), s["valid"].data_ptr(), T, E, K,
                               s["grad"].data_ptr(), s["dlogits"].data_ptr(), mask=mask)
    return {k: s[k] for k in ("counts", "valid", "probs", "loss", "dlogits")}


def run(state):
    kind = state["case"]["kind"]
    if own:
        nm = _nm()
        return {"quantize": _own_quantize, "balance": _own_balance}.get(kind, _own_experts)(nm, state)
    return {"quantize": _plain_quantize, "balance": _plain_balance}.get(kind, _plain_experts)(state)


# ---- what a pass cannot do without ----------------------------------------------------------


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if case["kind"] == "quantize":
        values = case["batch"] * case["n"] * case["k"]
        packed = case["batch"] * projection_bytes(case["n"], case["k"])
        return {"bytes": float(values * (size[case["src"]] + size[case["dst"]]) + 2 * packed), "flops": 2.0 * values}
    T = case["tokens"] if case["kind"] == "balance" else case["rows"]
    E, K = case["experts"], case["topk"]
    if case["kind"] == "balance":
        # the logits for the loss and for its gradient, the gradient, the ids and the mask
        return {"bytes": float(T * E * 3 * size[case["logits"]] + T * K * 4 + T), "flops": 12.0 * T * E}
    H, I, width = case["hidden"], case["inter"], K + case["shared"]
    live = width - K * case["drop"]
    expert = 2 * projection_bytes(I, H) + projection_bytes(H, I)
    touched = E * (1.0 - (1.0 - K * (1.0 - case["drop"]) / E) ** T) + case["shared"]  # distinct experts of T uniform draws
    moved = T * H * (size[case["x"]] + 4) + T * width * 8
    moved += T * H * 4 * case["accumulate"] + T * H * 2 * case["residual"]
    return {"bytes": float(touched * expert + moved), "flops": 6.0 * T * live * H * I}


# ---- the results in 64 bits -------------------------------------------------------------------


def _expert64(raw, n, k):
    """[n, k] f64 weights of one slot's tile-order bytes, group by group of four steps."""
    t = _steps(k)
    strips = raw[:projection_bytes(n, k)].view(n // 16, -1)
    table = torch.tensor(E2M1, dtype=torch.float64, device=DEV)
    w = torch.empty(n // 16, 16, 4 * t, 32, dtype=torch.float64, device=DEV)
    for i in range(0, t, 4):
        m, at = min(4, t - i), 4352 * (i // 4)
        sc = strips[:, at + 1024 * m:at + 1024 * m + 256].reshape(-1, 4, 16, 4).double()
        for j in range(m):
            nib = strips[:, at + 1024 * j:at + 1024 * (j + 1)].reshape(-1, 4, 16, 16)
            b = w[:, :, 4 * (i + j):4 * (i + j) + 4].permute(0, 2, 1, 3)
            b[..., 0::2], b[..., 1::2] = table[(nib & 15).long()], table[(nib >> 4).long()]
            b.mul_(torch.exp2(sc[..., j] - 127.0)[..., None])
    return w.view(n, 128 * t)[:, :k]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "quantize":
        return torch.cat([_nearest64(s["src"][e]) for e in range(case["batch"])]).view(s["src"].shape)
    if case["kind"] == "balance":
        return _balance64(case, s)
    act = torch.nn.functional.silu if case["act"] == "silu" else lambda v: torch.nn.functional.gelu(v, approximate="tanh")
    H, I = case["hidden"], case["inter"]
    x = s["x0"].double()
    out = s["out0"].double() if case["accumulate"] else torch.zeros_like(x)
    for e in torch.unique(s["ids"]).tolist():
        if e >= s["gate"].shape[0]:
            continue
        t, j = torch.nonzero(s["ids"] == e, as_tuple=True)
        h = act(x[t] @ _expert64(s["gate"][e], I, H).T) * (x[t] @ _expert64(s["up"][e], I, H).T)
        out.index_add_(0, t, (h @ _expert64(s["down"][e], H, I).T) * s["w"][t, j].double()[:, None])
    return {"out": out, "x": x + out} if case["residual"] else {"out": out}


def _nearest64(x):
    """The nearest of the 16 values in each block's scale, of two as near the one with the even code."""
    b = x.double().view(-1, 32)
    m = b.abs().amax(-1)
    scale = torch.where(m > 0, torch.exp2((torch.frexp(m)[1] - 3).double()), 1.0).clamp(min=2.0 ** -127)
    y = (b / scale[:, None]).clamp(-6, 6)
    a = y.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    return torch.copysign(torch.round(a / step) * step, y) * scale[:, None]


def _balance64(case, s):
    E, K = case["experts"], case["topk"]
    keep = torch.nonzero(s["mask"])[:, 0]
    N = max(1, len(keep))
    x = s["logits"].double().requires_grad_(True)
    counts = torch.bincount(s["ids"][keep].view(-1), minlength=E)
    mean = torch.softmax(x[keep], -1).sum(0) / N
    loss = E * (counts / (K * N) * mean).sum()
    loss.backward(s["grad"].double()[0])
    return {"counts": None, "valid": None, "probs": mean.detach(), "loss": loss.detach().view(1), "dlogits": x.grad}

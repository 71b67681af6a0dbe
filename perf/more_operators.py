"""Tokens sorted by expert and back, products over 16-bit weights and their gradients, as measurable cases.

Five kinds of call:

- ``sort``: a batch's routing sorted by expert, and the tokens' rows in that order
  (``expert_sort``, ``tokens_to_experts``);
- ``back``: the experts' rows back to their tokens, weighted, and the gradient of that
  (``tokens_from_experts``, ``tokens_from_experts_backward``);
- ``linear``: rows times a weight matrix, or every expert's rows times the expert's own, with bias,
  activation, gate and residual (``linear``);
- ``grads``: the gradients of such a product: rows, weights and bias (``linear_input_grad``,
  ``linear_weight_grad``);
- ``router``: the gradient of the routed weights with respect to the router's logits
  (``router_topk_backward``).

A product is out = act(x W' + b) (* (x U' + c)) + residual, W and U [experts, n, k].  Rows of expert e are
offsets[e] .. offsets[e + 1] - 1 of the sorted rows; rows behind the last one are left as they were.

Activations and gradients are N(0, 1), weights N(0, 0.02), router logits of the scale that such activations
and routers give, with experts of unequal popularity.
"""
import math
import os
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}

# Shapes that the repository's configurations and benchmark name: hidden, intermediate, experts, top-k.
SHAPES = {
    "small": dict(hidden=1024, inter=2048, experts=8, topk=2),
    "qwen3": dict(hidden=2048, inter=768, experts=128, topk=8),
    "deepseek": dict(hidden=2048, inter=1408, experts=64, topk=6),
    "mixtral": dict(hidden=4096, inter=14336, experts=8, topk=2),
}


def _tokens(name, kind, shape, tokens, **more):
    s = SHAPES[shape]
    c = dict(name=name, kind=kind, tokens=tokens, hidden=s["hidden"], experts=s["experts"], topk=s["topk"], x="bf16", valid=1.0)
    if kind == "back":
        c.update(out="bf16", accumulate=False)
    c.update(more)
    return c


def _product(name, kind, rows, n, k, **more):
    """rows: of x; with experts > 1 the rows are the pairs of rows / topk tokens."""
    c = dict(name=name, kind=kind, rows=rows, n=n, k=k, experts=1, topk=1, valid=1.0, x="bf16", act="none", gated=False, bias=False)
    if kind == "linear":
        c.update(out="bf16", residual=False, keep=False)
    else:
        c.update(dw="f32", accumulate=False)
    c.update(more)
    return c


def listed():
    return [
        # a small training batch: launches and latency count
        _tokens("sort_61", "sort", "small", 61),
        # a long training batch of many experts, padded behind its sequences
        _tokens("sort_16384", "sort", "qwen3", 16384, valid=0.9),
        # an odd batch of few tokens, experts' rows in 16 bits added to an f32 residual stream
        _tokens("back_37", "back", "deepseek", 37, out="f32", accumulate=True),
        # the long batch's way back and its gradient
        _tokens("back_16384", "back", "qwen3", 16384, valid=0.9),
        # a few rows through a projection of odd sizes, everything in the epilogue
        _product("linear_5_odd", "linear", 5, 1003, 1001, x="f16", out="f16", act="gelu", bias=True, residual=True),
        # gate and up of a decode batch of 16 tokens over few large 16-bit experts: every weight read once
        _product("linear_mixtral_16", "linear", 32, 14336, 4096, experts=8, topk=2, act="silu", gated=True),
        # gate and up of a training batch over many small experts, what the gradient needs kept
        _product("linear_qwen3_4096", "linear", 32768, 768, 2048, experts=128, topk=8, act="silu", gated=True, keep=True, valid=0.95),
        # the down projection of a dense layer over a long prompt, residual added
        _product("linear_dense_4096", "linear", 4096, 4096, 14336, bias=True, residual=True),
        # gradients of a small dense layer with a bias, for a few tokens
        _product("grads_61", "grads", 61, 2048, 1024, bias=True, act="gelu"),
        # gradients of the experts' gate and up of a training batch
        _product("grads_deepseek_4096", "grads", 24576, 1408, 2048, experts=64, topk=6, gated=True),
        # the routed weights' gradient of a small batch
        dict(name="router_61", kind="router", tokens=61, experts=8, topk=2, logits="f32", mode=1, valid=1.0, accumulate=False),
        # of a long batch, added to the balance loss's
        dict(name="router_32768", kind="router", tokens=32768, experts=128, topk=8, logits="f32", mode=0, valid=0.9, accumulate=True),
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A row's length: mostly whole steps of 64 or 8, sometimes anything."""
    step = rng.choice([64, 64, 8, 1])
    return max(1, _log_uniform(rng, lo, hi) // step) * step


def draw(rng):
    kind = rng.choices(["sort", "back", "linear", "grads", "router"], [3, 3, 5, 4, 2])[0]
    experts = rng.choice([4, 8, 16, 60, 64, 127, 128])
    c = dict(kind=kind, experts=experts, topk=rng.randint(1, min(8, experts)), valid=rng.choice([1.0, 1.0, 0.9, 0.5]))
    if kind == "router":
        c.update(tokens=_log_uniform(rng, 1, 32768), logits=rng.choice(["f32", "f32", "bf16"]), mode=rng.randint(0, 2),
                 accumulate=rng.random() < 0.5)
        return c
    c["x"] = rng.choice(["bf16", "bf16", "f16"])
    if kind in ("sort", "back"):
        c["x"] = rng.choice([c["x"], c["x"], "f32"])
        c["hidden"] = _width(rng, 64, 8192)
        top = 16384 * 8 * 2048 * 2 // (c["topk"] * c["hidden"] * SIZE[c["x"]])
        c["tokens"] = _log_uniform(rng, 1, max(2, min(32768, top)))
        if kind == "back":
            c.update(out=rng.choice(["f32", c["x"]]), accumulate=rng.random() < 0.5)
        return c
    c.update(n=_width(rng, 16, 8192), k=_width(rng, 16, 8192), act=rng.choice(["none", "silu", "gelu"]),
             gated=rng.random() < 0.5, bias=rng.random() < 0.5)
    if rng.random() < 0.4:
        c.update(experts=1, topk=1, valid=1.0)
    if c["gated"] and c["act"] == "none":
        c["act"] = "silu"
    # at most the largest listed case's work, and at most its share of the weights
    most = 4096 * 4096 * 14336 // ((6 if kind == "grads" else 2) * c["n"] * c["k"])
    while c["experts"] * c["n"] * c["k"] > 128 * 2048 * 1024:
        c["n"], c["k"] = (c["n"] // 2 + 1, c["k"]) if c["n"] > c["k"] else (c["n"], c["k"] // 2 + 1)
    tokens = _log_uniform(rng, 1, max(2, min(65536, most) // c["topk"]))
    c["rows"] = tokens * c["topk"]
    if kind == "linear":
        c.update(out=rng.choice(["f32", c["x"], c["x"]]), residual=rng.random() < 0.5, keep=rng.random() < 0.3)
    else:
        c.update(dw=rng.choice(["f32", "f32", c["x"]]), accumulate=rng.random() < 0.3)
    return c


# ---- what a program has in hand -----------------------------------------------------------


def _routing(case, tokens, g):
    """ids [T, k] int32 of the largest logits, softmax weights, mask u8 [T] (padding behind the tokens)."""
    E, K = case["experts"], case["topk"]
    logits = torch.randn(tokens, E, device=DEV, generator=g) + 0.5 * torch.randn(E, device=DEV, generator=g)
    top, ids = torch.topk(logits, K, dim=-1)
    mask = (torch.arange(tokens, device=DEV) < math.ceil(case["valid"] * tokens)).to(torch.uint8)
    return logits, ids.int(), torch.softmax(top, -1), mask


def _sorted(ids, mask, E):
    """perm [n], inv [T, k], offsets [E + 1] int32; perm's entries behind the last sorted one 0, inv -1 where left out."""
    n = ids.numel()
    flat = torch.where(mask[:, None] != 0, ids, E).view(-1).long()
    order = torch.argsort(flat, stable=True)
    counts = torch.zeros(E + 1, dtype=torch.long, device=DEV).scatter_add_(0, flat, torch.ones_like(flat))
    offsets = torch.cat([counts.new_zeros(1), torch.cumsum(counts[:E], 0)])
    place = torch.arange(n, device=DEV)
    inside = place < offsets[E]
    perm = torch.where(inside, order, 0).int()
    inv = torch.empty(n, dtype=torch.int32, device=DEV)
    inv[order] = torch.where(inside, place, -1).int()
    return perm, inv.view(ids.shape), offsets.int()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(6007 * (seed + 1))
    s = {"case": case}

    def normal(*shape, std=1.0, dtype=torch.float32):
        t = torch.empty(*shape, dtype=dtype, device=DEV)
        for part in (t if t.dim() == 3 else (t,)):
            part.copy_(torch.randn(part.shape, device=DEV, generator=g) * std)
        return t

    kind, E, K = case["kind"], case["experts"], case["topk"]
    if kind in ("linear", "grads"):
        R, n, k, x = case["rows"], case["n"], case["k"], DTYPES[case["x"]]
        if E > 1:
            _, ids, _, mask = _routing(case, R // K, g)
            s["offsets"] = _sorted(ids, mask, E)[2]
            s["most"] = int((s["offsets"][1:] - s["offsets"][:-1]).max())  # rows of the busiest expert
        else:
            s["offsets"], s["most"] = None, R
        s["w"] = normal(E, n, k, std=0.02, dtype=x)
        s["u"] = normal(E, n, k, std=0.02, dtype=x) if case["gated"] else None
        s["x"] = normal(R, k, dtype=x)
        if kind == "linear":
            s["b"] = normal(E, n, std=0.1) if case["bias"] else None
            s["c"] = normal(E, n, std=0.1) if case["bias"] and case["gated"] else None
            s["residual"] = normal(R, n, dtype=DTYPES[case["out"]]) if case["residual"] else None
            s["out"] = torch.zeros(R, n, dtype=DTYPES[case["out"]], device=DEV)
            for name in ("pre", "pre_up")[:(1 + case["gated"]) * case["keep"]]:
                s[name] = torch.zeros(R, n, dtype=x, device=DEV)
            return s
        s["dy"] = normal(R, n, dtype=x)
        s["dy_up"] = normal(R, n, dtype=x) if case["gated"] else None
        # what x = act(pre) came from, where this product's rows are another's output
        s["pre"] = normal(R, k, dtype=x) if case["act"] != "none" and not case["gated"] else None
        s["dx"] = torch.zeros(R, k, dtype=x, device=DEV)
        for name in ("w", "u")[:1 + case["gated"]]:
            s["d" + name + "0"] = normal(E, n, k, dtype=DTYPES[case["dw"]]) if case["accumulate"] else None
            s["d" + name] = torch.zeros(E, n, k, dtype=DTYPES[case["dw"]], device=DEV)
            s["db" + name] = torch.zeros(E, n, device=DEV) if case["bias"] else None
        return s
    T = case["tokens"]
    logits, ids, w, mask = _routing(case, T, g)
    s["mask"] = mask
    if kind == "router":
        s["logits"] = logits.to(DTYPES[case["logits"]])
        s["ids"] = torch.topk(s["logits"].float(), K, dim=-1)[1].int()
        s["dw"] = normal(T, K)
        s["d0"] = normal(T, E, std=0.01, dtype=s["logits"].dtype) if case["accumulate"] else None
        s["dlogits"] = torch.zeros_like(s["logits"])
        return s
    H, x = case["hidden"], DTYPES[case["x"]]
    if kind == "sort":
        s["ids"], s["x"] = ids, normal(T, H, dtype=x)
        s["perm"], s["inv"] = (torch.zeros(T * K, dtype=torch.int32, device=DEV) for _ in range(2))
        s["inv"] = s["inv"].view(T, K)
        s["offsets"] = torch.zeros(E + 1, dtype=torch.int32, device=DEV)
        s["rows"] = torch.zeros(T * K, H, dtype=x, device=DEV)
        return s
    s["inv"], s["w"] = _sorted(ids, mask, E)[1], w
    s["y"], s["dout"] = normal(T * K, H, dtype=x), normal(T, H, dtype=DTYPES[case["out"]])
    s["out0"] = normal(T, H, dtype=DTYPES[case["out"]]) if case["accumulate"] else None
    s["out"] = torch.zeros(T, H, dtype=DTYPES[case["out"]], device=DEV)
    s["dy"], s["dw"] = torch.zeros(T * K, H, dtype=x, device=DEV), torch.zeros(T, K, device=DEV)
    return s


# ---- one pass in plain form -----------------------------------------------------------------


def _plain_sort(s):
    case = s["case"]
    H, K = case["hidden"], case["topk"]
    perm, inv, offsets = _sorted(s["ids"], s["mask"], case["experts"])
    inside = torch.arange(perm.numel(), device=DEV) < offsets[-1]
    rows = torch.where(inside[:, None], s["x"][(perm // K).long()], torch.zeros(1, H, dtype=s["x"].dtype, device=DEV))
    return {"perm": perm, "inv": inv, "offsets": offsets, "rows": rows}


def _plain_back(s):
    T, K = s["inv"].shape
    flat = s["inv"].view(-1).long()
    n = flat.numel()
    at = torch.where(flat < 0, n, flat)
    y = torch.cat([s["y"].float(), torch.zeros(1, s["y"].shape[1], device=DEV)])[at].view(T, K, -1)
    out = (s["w"][:, :, None] * y).sum(1)
    if s["out0"] is not None:
        out = s["out0"].float() + out
    d = s["dout"].float()
    dw = (d[:, None, :] * y).sum(-1)
    dy = torch.zeros(n + 1, d.shape[1], device=DEV)
    dy[at] = (s["w"][:, :, None] * d[:, None, :]).view(n, -1)
    return {"out": out.to(s["out"].dtype), "dy": dy[:n].to(s["y"].dtype), "dw": dw}


def _act(name, v):
    if name == "none":
        return v
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))


def _act_slope(name, v):
    if name == "none":
        return torch.ones_like(v)
    if name == "silu":
        q = 1.0 / (1.0 + torch.exp(-v))
        return q * (1.0 + v * (1.0 - q))
    a = math.sqrt(2.0 / math.pi)
    t = torch.tanh(a * (v + 0.044715 * v * v * v))
    return 0.5 * (1.0 + t) + 0.5 * v * (1.0 - t * t) * a * (1.0 + 3.0 * 0.044715 * v * v)


def _places(s):
    """(expert, place in it, whether it is an expert's at all) of every row."""
    R = s["x"].shape[0]
    row = torch.arange(R, device=DEV)
    if s["offsets"] is None:
        return torch.zeros_like(row), row, torch.ones(R, dtype=torch.bool, device=DEV)
    o = s["offsets"].long()
    e = torch.bucketize(row, o[1:], right=True)
    inside = row < o[-1]
    e = torch.where(inside, e, 0)
    return e, torch.where(inside, row - o[e], s["most"]), inside


def _spread(s, t, where):
    """[experts, most, width] f32: every expert's rows from place 0, zeros behind."""
    out = torch.zeros(s["w"].shape[0], s["most"] + 1, t.shape[1], device=DEV)
    out[where[0], where[1]] = t.float()
    return out[:, :-1].contiguous()


def _rows(s, v, where):
    """Back to [rows, width], zeros where a row is no expert's."""
    e, at, inside = where
    return v[e, at.clamp(max=max(s["most"] - 1, 0))] * inside[:, None]


def _plain_linear(s):
    case, where = s["case"], _places(s)
    xe = _spread(s, s["x"], where)

    def product(w, b):
        v = torch.bmm(xe, w.float().transpose(1, 2).contiguous())
        return v if b is None else v + b[:, None, :]

    p = _rows(s, product(s["w"], s["b"]), where)
    v = _act(case["act"], p)
    got = {}
    if case["gated"]:
        q = _rows(s, product(s["u"], s["c"]), where)
        v = v * q
        if case["keep"]:
            got["pre_up"] = q.to(s["x"].dtype)
    if case["keep"]:
        got["pre"] = p.to(s["x"].dtype)
    v = v if s["residual"] is None else v + s["residual"].float()
    got["out"] = torch.where(where[2][:, None], v, 0.0).to(s["out"].dtype)
    return got


def _plain_grads(s):
    case, where = s["case"], _places(s)
    xt = _spread(s, s["x"], where)
    got, dx = {}, 0.0
    for name, dy in (("w", s["dy"]), ("u", s["dy_up"]))[:1 + case["gated"]]:
        de = _spread(s, dy, where)
        dx = dx + torch.bmm(de, s[name].float())
        dw = torch.bmm(de.transpose(1, 2).contiguous(), xt)
        if s["d" + name + "0"] is not None:
            dw = s["d" + name + "0"].float() + dw
        got["d" + name] = dw.to(s["d" + name].dtype)
        if case["bias"]:
            got["db" + name] = de.sum(1)
    dx = _rows(s, dx, where)
    if s["pre"] is not None:
        dx = torch.where(where[2][:, None], dx * _act_slope(case["act"], s["pre"].float()), 0.0)
    got["dx"] = dx.to(s["dx"].dtype)
    return got


def _plain_router(s):
    case = s["case"]
    ids, dw, x = s["ids"].long(), s["dw"], s["logits"].float()
    if case["mode"] == 2:  # the full softmax's own values
        p = torch.exp(x - x.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        mean = (torch.gather(p, 1, ids) * dw).sum(-1, keepdim=True)
        d = -p * mean
        d = d.scatter_add(1, ids, torch.gather(p, 1, ids) * dw)
    else:  # a softmax over the chosen
        v = torch.gather(x, 1, ids)
        w = torch.exp(v - v.amax(-1, keepdim=True))
        w = w / w.sum(-1, keepdim=True)
        d = torch.zeros_like(x).scatter_add(1, ids, w * (dw - (w * dw).sum(-1, keepdim=True)))
    d = torch.where(s["mask"][:, None] != 0, d, 0.0)
    if s["d0"] is not None:
        d = s["d0"].float() + d
    return {"dlogits": d.to(s["dlogits"].dtype)}


# ---- one pass of the framework's own calls ------------------------------------------------------


def _nm():
    path = os.path.join(os.getcwd(), "naiwa-rs_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import naiwa_moe
    return naiwa_moe


def _at(t):
    return None if t is None else t.data_ptr()


def _own_sort(nm, s):
    case = s["case"]
    T, K, H = case["tokens"], case["topk"], case["hidden"]
    dt = {"f32": nm.F32, "bf16": nm.BF16, "f16": nm.F16}[case["x"]]
    mask = _at(s["mask"]) if case["valid"] < 1 else None
    nm.expert_sort(_at(s["ids"]), T, K, case["experts"], _at(s["perm"]), _at(s["inv"]), _at(s["offsets"]), mask=mask)
    nm.tokens_to_experts(_at(s["x"]), dt, _at(s["inv"]), T, K, H, _at(s["rows"]))
    return {k: s[k] for k in ("perm", "inv", "offsets", "rows")}


def _own_back(nm, s):
    case = s["case"]
    T, K, H = case["tokens"], case["topk"], case["hidden"]
    ids = {"f32": nm.F32, "bf16": nm.BF16, "f16": nm.F16}
    dt, od = ids[case["x"]], ids[case["out"]]
    if s["out0"] is not None:
        s["out"].copy_(s["out0"])
    nm.tokens_from_experts(_at(s["y"]), dt, _at(s["inv"]), T, K, H, _at(s["out"]), w=_at(s["w"]), out_dtype=od,
                           accumulate=case["accumulate"])
    nm.tokens_from_experts_backward(_at(s["dout"]), od, _at(s["y"]), dt, _at(s["inv"]), T, K, H, _at(s["dy"]), _at(s["dw"]),
                                    w=_at(s["w"]))
    return {k: s[k] for k in ("out", "dy", "dw")}


def _own_weights(nm, s):
    """Descriptors of the weights, which a program makes once."""
    if "weights" not in s:
        case = s["case"]
        dt = nm.BF16 if case["x"] == "bf16" else nm.F16
        shape = (case["experts"], case["n"], case["k"])
        s["weights"] = (nm.Weights(_at(s["w"]), dt, *shape, bias=_at(s.get("b"))),
                        nm.Weights(_at(s["u"]), dt, *shape, bias=_at(s.get("c"))) if case["gated"] else None)
    return s["weights"]


def _own_linear(nm, s):
    case = s["case"]
    w, u = _own_weights(nm, s)
    act = {"none": nm.ACT_NONE, "silu": nm.ACT_SILU, "gelu": nm.ACT_GELU_PYTORCH_TANH}[case["act"]]
    od = {"f32": nm.F32, "bf16": nm.BF16, "f16": nm.F16}[case["out"]]
    nm.linear(w, _at(s["x"]), case["rows"], _at(s["out"]), up=u, offsets=_at(s["offsets"]), act=act, out_dtype=od,
              residual=_at(s["residual"]), pre=_at(s.get("pre")), pre_up=_at(s.get("pre_up")))
    return {k: s[k] for k in ("out", "pre", "pre_up") if k in s}


def _own_grads(nm, s):
    case = s["case"]
    w, u = _own_weights(nm, s)
    act = {"none": nm.ACT_NONE, "silu": nm.ACT_SILU, "gelu": nm.ACT_GELU_PYTORCH_TANH}[case["act"] if s["pre"] is not None else "none"]
    ids = {"f32": nm.F32, "bf16": nm.BF16, "f16": nm.F16}
    R, E, n, k = case["rows"], case["experts"], case["n"], case["k"]
    nm.linear_input_grad(w, _at(s["dy"]), R, _at(s["dx"]), up=u, dy_up=_at(s["dy_up"]), offsets=_at(s["offsets"]), act=act,
                         pre=_at(s["pre"]))
    got = {"dx": s["dx"]}
    for name, dy in (("w", s["dy"]), ("u", s["dy_up"]))[:1 + case["gated"]]:
        dw, db = s["d" + name], s["db" + name]
        if case["accumulate"]:
            dw.copy_(s["d" + name + "0"])
            if db is not None:
                db.zero_()
        nm.linear_weight_grad(_at(dy), _at(s["x"]), ids[case["x"]], R, n, k, _at(dw), experts=E, offsets=_at(s["offsets"]),
                              dw_dtype=ids[case["dw"]], dbias=_at(db), accumulate=case["accumulate"])
        got["d" + name] = dw
        if db is not None:
            got["db" + name] = db
    return got


def _own_router(nm, s):
    case = s["case"]
    dt = nm.F32 if case["logits"] == "f32" else nm.BF16
    if s["d0"] is not None:
        s["dlogits"].copy_(s["d0"])
    nm.router_topk_backward(_at(s["logits"]), dt, _at(s["ids"]), _at(s["dw"]), case["tokens"], case["experts"], case["topk"],
                            _at(s["dlogits"]), mode=case["mode"], mask=_at(s["mask"]) if case["valid"] < 1 else None,
                            accumulate=case["accumulate"])
    return {"dlogits": s["dlogits"]}


def run(state):
    kind = state["case"]["kind"]
    if own:
        calls = {"sort": _own_sort, "back": _own_back, "linear": _own_linear, "grads": _own_grads, "router": _own_router}
        return calls[kind](_nm(), state)
    calls = {"sort": _plain_sort, "back": _plain_back, "linear": _plain_linear, "grads": _plain_grads, "router": _plain_router}
    return calls[kind](state)


# ---- what a pass cannot do without ----------------------------------------------------------


def work(case):
    kind, E, K = case["kind"], case["experts"], case["topk"]
    if kind == "router":
        T, s = case["tokens"], SIZE[case["logits"]]
        chosen = K if case["mode"] != 2 and case["accumulate"] else E  # what else has to be read and written
        values = T * (min(chosen, E) * (1 + case["accumulate"]) + (K if case["mode"] != 2 else E))
        return {"bytes": float(values * s + T * K * 8 + T), "flops": 8.0 * T * (E if case["mode"] == 2 else K)}
    if kind in ("sort", "back"):
        T, H, s = case["tokens"], case["hidden"], SIZE[case["x"]]
        live = T * case["valid"]
        if kind == "sort":
            return {"bytes": float(live * H * s * (1 + K) + T * K * 12 + T + 4 * E), "flops": float(T * K)}
        so = SIZE[case["out"]]
        moved = live * K * H * s * 2 + T * H * so * (2 + case["accumulate"]) + T * K * 12
        return {"bytes": float(moved), "flops": 5.0 * live * K * H}
    R, n, k, s = case["rows"], case["n"], case["k"], SIZE[case["x"]]
    tokens, two = R // K, 1 + case["gated"]
    live = tokens * case["valid"] * K
    touched = E * (1.0 - (1.0 - K / E) ** (tokens * case["valid"])) if E > 1 else 1.0  # distinct experts of uniform draws
    if kind == "linear":
        so = SIZE[case["out"]]
        moved = live * k * s + touched * n * k * s * two + live * n * (so * (1 + case["residual"]) + s * two * case["keep"])
        return {"bytes": float(moved), "flops": 2.0 * live * n * k * two}
    moved = live * k * s * (2 + (case["act"] != "none" and not case["gated"])) + two * live * n * s
    moved += two * n * k * (touched * s + E * SIZE[case["dw"]] * (1 + case["accumulate"]))
    return {"bytes": float(moved), "flops": 4.0 * live * n * k * two}


# ---- the results in 64 bits -------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"sort": _sort64, "back": _back64, "linear": _linear64, "grads": _grads64, "router": _router64}[case["kind"]](case, s)


def _sort64(case, s):
    rows = torch.zeros(s["rows"].shape, dtype=torch.float64, device=DEV)
    ids = s["ids"].clone()
    ids[s["mask"] == 0] = case["experts"]
    at = 0
    for e in range(case["experts"]):
        t = torch.nonzero(ids == e)[:, 0]
        rows[at:at + len(t)] = s["x"][t].double()
        at += len(t)
    return {"perm": None, "inv": None, "offsets": None, "rows": rows}


def _back64(case, s):
    out = s["out0"].double() if s["out0"] is not None else torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
    dy = torch.zeros(s["dy"].shape, dtype=torch.float64, device=DEV)
    dw = torch.zeros(s["dw"].shape, dtype=torch.float64, device=DEV)
    d, w = s["dout"].double(), s["w"].double()
    for j in range(case["topk"]):
        t = torch.nonzero(s["inv"][:, j] >= 0)[:, 0]
        r = s["inv"][t, j].long()
        y = s["y"][r].double()
        out[t] += w[t, j, None] * y
        dy[r] = w[t, j, None] * d[t]
        dw[t, j] = torch.linalg.vecdot(d[t], y)
    return {"out": out, "dy": dy, "dw": dw}


def _segments(s):
    o = [0, s["x"].shape[0]] if s["offsets"] is None else s["offsets"].tolist()
    return [(e, slice(o[e], o[e + 1])) for e in range(len(o) - 1) if o[e + 1] > o[e]]


def _act64(name):
    f = torch.nn.functional
    return {"none": lambda v: v, "silu": f.silu, "gelu": lambda v: f.gelu(v, approximate="tanh")}[name]


def _linear64(case, s):
    zeros = lambda: torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)  # noqa: E731
    got = {"out": zeros()}
    for name in ("pre", "pre_up"):
        if name in s:
            got[name] = zeros()
    for e, m in _segments(s):
        x = s["x"][m].double()
        p = x @ s["w"][e].double().T
        p = p if s["b"] is None else p + s["b"][e].double()
        v = _act64(case["act"])(p)
        if "pre" in got:
            got["pre"][m] = p
        if case["gated"]:
            q = x @ s["u"][e].double().T
            q = q if s["c"] is None else q + s["c"][e].double()
            v = v * q
            if "pre_up" in got:
                got["pre_up"][m] = q
        got["out"][m] = v if s["residual"] is None else v + s["residual"][m].double()
    return got


def _grads64(case, s):
    got = {"dx": torch.zeros(s["dx"].shape, dtype=torch.float64, device=DEV)}
    names = ("w", "u")[:1 + case["gated"]]
    for name in names:
        start = s["d" + name + "0"]
        got["d" + name] = start.double() if start is not None else torch.zeros(s["dw"].shape, dtype=torch.float64, device=DEV)
        if case["bias"]:
            got["db" + name] = torch.zeros(s["db" + name].shape, dtype=torch.float64, device=DEV)
    for e, m in _segments(s):
        x = s["x"][m].double()
        for name, dy in zip(names, (s["dy"], s["dy_up"])):
            d = dy[m].double()
            got["dx"][m] += d @ s[name][e].double()
            got["d" + name][e] += d.T @ x
            if case["bias"]:
                got["db" + name][e] = d.sum(0)
        if s["pre"] is not None:
            p = s["pre"][m].double().requires_grad_(True)
            _act64(case["act"])(p).backward(got["dx"][m])
            got["dx"][m] = p.grad
    return got


def _router64(case, s):
    x = s["logits"].double().requires_grad_(True)
    ids = s["ids"].long()
    if case["mode"] == 0:  # the full softmax's chosen values over their sum
        w = torch.softmax(x, -1).gather(1, ids)
        w = w / w.sum(-1, keepdim=True)
    elif case["mode"] == 1:
        w = torch.softmax(x.gather(1, ids), -1)
    else:
        w = torch.softmax(x, -1).gather(1, ids)
    w.backward(s["dw"].double() * (s["mask"][:, None] != 0))
    return {"dlogits": x.grad if s["d0"] is None else s["d0"].double() + x.grad}

"""Workloads of the mixture-of-experts operators and of the linear with an epilogue: what a
decode step, a batched decode step and a prefill of a quantized model ask of them.

`own` false: the operators from elementary torch operations in 32 bits (the router's choice in
64); `own` true: the library's calls.  Weights are packed GGUF blocks (q8_0, q4_0, q4_1)."""
import math
import os
import sys

import torch

own = False

BLOCK = {"q8_0": 34, "q4_0": 18, "q4_1": 20}
ACTS = ("none", "silu", "gelu", "gelu_tanh", "relu", "sigmoid")


def listed():
    return [
        # the router of one decoded token: pure latency
        {"name": "route-1", "op": "route", "rows": 1, "in": 2048, "experts": 64, "top_k": 6,
         "scoring": "softmax", "bias": False, "renorm": True, "scale": 1.0, "logits": False},
        # a batched decode step that also watches its logits, an odd number of rows, sigmoid scores with a balancing bias
        {"name": "route-33-sigmoid", "op": "route", "rows": 33, "in": 3584, "experts": 128, "top_k": 8,
         "scoring": "sigmoid", "bias": True, "renorm": True, "scale": 2.5, "logits": True},
        # the router over a prompt
        {"name": "route-prompt", "op": "route", "rows": 2048, "in": 4096, "experts": 256, "top_k": 8,
         "scoring": "softmax", "bias": False, "renorm": False, "scale": 1.0, "logits": False},
        # one decoded token, many small experts
        {"name": "experts-1-small", "op": "experts", "fmt": "q4_0", "fmt_down": "q4_0", "rows": 1, "in": 2048,
         "hidden": 768, "out": 2048, "experts": 128, "top_k": 8, "empty": 0.0, "residual": True},
        # one decoded token, few large experts; the down projection kept in more bits
        {"name": "experts-1-large", "op": "experts", "fmt": "q4_0", "fmt_down": "q8_0", "rows": 1, "in": 4096,
         "hidden": 14336, "out": 4096, "experts": 8, "top_k": 2, "empty": 0.0, "residual": True},
        # a small batch; rows of 44 blocks are no multiple of 16 bytes
        {"name": "experts-7-ragged", "op": "experts", "fmt": "q8_0", "fmt_down": "q8_0", "rows": 7, "in": 2048,
         "hidden": 1408, "out": 2048, "experts": 64, "top_k": 6, "empty": 0.0, "residual": False},
        # a padded batch: a third of the slots name no expert (other ranks hold them)
        {"name": "experts-32-padded", "op": "experts", "fmt": "q4_1", "fmt_down": "q4_1", "rows": 32, "in": 3584,
         "hidden": 2560, "out": 3584, "experts": 60, "top_k": 4, "empty": 0.33, "residual": True},
        # a prompt's tokens: tens of rows for each expert
        {"name": "experts-prompt", "op": "experts", "fmt": "q4_0", "fmt_down": "q8_0", "rows": 512, "in": 2048,
         "hidden": 1024, "out": 2048, "experts": 64, "top_k": 8, "empty": 0.0, "residual": True},
        # the whole layer of a small batch, router to residual
        {"name": "layer-4", "op": "layer", "fmt": "q4_0", "fmt_down": "q4_0", "rows": 4, "in": 4096,
         "hidden": 1536, "out": 4096, "experts": 96, "top_k": 6, "residual": True,
         "scoring": "softmax", "bias": False, "renorm": True, "scale": 1.0},
        # an output projection of one token, added to the residual stream
        {"name": "epilogue-1-residual", "op": "epilogue", "fmt": "q4_0", "rows": 1, "in": 4096, "out": 4096,
         "bias": False, "act": "none", "row_scale": False, "residual": True},
        # a shared expert's down projection, gated for each row
        {"name": "epilogue-5-gated", "op": "epilogue", "fmt": "q8_0", "rows": 5, "in": 18944, "out": 3584,
         "bias": False, "act": "none", "row_scale": True, "residual": True},
        # an up projection with bias and activation over a prompt of odd length
        {"name": "epilogue-301-gelu", "op": "epilogue", "fmt": "q4_1", "rows": 301, "in": 896, "out": 4864,
         "bias": True, "act": "gelu", "row_scale": False, "residual": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A model width: mostly a multiple of 64 or 32, sometimes odd."""
    n = _log_int(rng, lo, hi)
    step = rng.choice((128, 64, 64, 32, 32, 1))
    return max(lo, n // step * step)


def _router(rng):
    experts = rng.choice((8, 16, 32, 60, 64, 96, 128, 160, 256))
    return {"experts": experts, "top_k": rng.randint(1, min(8, experts)), "scoring": rng.choice(("softmax", "sigmoid")),
            "bias": rng.random() < 0.4, "renorm": rng.random() < 0.6, "scale": rng.choice((1.0, 1.0, 2.5))}


def draw(rng):
    op = rng.choice(("route", "experts", "experts", "layer", "epilogue", "epilogue"))
    fmts = ("q8_0", "q4_0", "q4_1")
    while True:
        c = {"op": op}
        if op == "route":
            c.update(_router(rng), rows=_log_int(rng, 1, 2048), logits=rng.random() < 0.3)
            c["in"] = _width(rng, 256, 7168)
            big = c["rows"] * c["in"] * c["experts"] > 2048 * 4096 * 256
        elif op == "epilogue":
            c.update(fmt=rng.choice(fmts), rows=_log_int(rng, 1, 301), out=_width(rng, 64, 16384),
                     bias=rng.random() < 0.5, act=rng.choice(ACTS), row_scale=rng.random() < 0.4,
                     residual=rng.random() < 0.6)
            c["in"] = _width(rng, 64, 18944)
            big = c["out"] * c["in"] > 18944 * 4096 or c["rows"] * c["out"] * c["in"] > 4e9
        else:
            r = _router(rng)
            c.update(fmt=rng.choice(fmts), fmt_down=rng.choice(fmts), hidden=_width(rng, 128, 14336),
                     rows=_log_int(rng, 1, 64 if op == "layer" else 512), experts=r["experts"], top_k=r["top_k"],
                     residual=rng.random() < 0.7)
            c["in"] = _width(rng, 256, 7168)
            c["out"] = c["in"] if op == "layer" or rng.random() < 0.8 else _width(rng, 256, 7168)
            if op == "layer":
                c.update(r)
            else:
                c["empty"] = rng.choice((0.0, 0.0, 0.25, 0.6))
            weights = c["experts"] * c["hidden"] * (2 * c["in"] + c["out"])
            big = weights > 1.41e9 or c["rows"] * c["top_k"] * c["hidden"] * (2 * c["in"] + c["out"]) > 2.6e10
        if not big:
            return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _quantized(gen, fmt, rows, cols, std, dev):
    """Packed blocks of a normal weight matrix [rows, cols] (padded to whole blocks with zeros)."""
    nb = (cols + 31) // 32
    w = torch.randn(rows, nb * 32, generator=gen, device=dev) * std
    if nb * 32 > cols:
        w[:, cols:] = 0
    w = w.view(rows * nb, 32)
    if fmt == "q8_0":
        d = (w.abs().amax(1, keepdim=True) / 127).half()
        q = (w / d.float().clamp_min(1e-8)).round_().clamp_(-127, 127).to(torch.int8).view(torch.uint8)
        return torch.cat((d.view(torch.uint8), q), 1).flatten()
    if fmt == "q4_0":
        d = (w.abs().amax(1, keepdim=True) / 7).half()
        q = ((w / d.float().clamp_min(1e-8)).round_() + 8).clamp_(0, 15).to(torch.uint8)
        return torch.cat((d.view(torch.uint8), q[:, :16] | (q[:, 16:] << 4)), 1).flatten()
    m = w.amin(1, keepdim=True)
    d = ((w.amax(1, keepdim=True) - m) / 15).half()
    q = ((w - m) / d.float().clamp_min(1e-8)).round_().clamp_(0, 15).to(torch.uint8)
    return torch.cat((d.view(torch.uint8), m.half().view(torch.uint8), q[:, :16] | (q[:, 16:] << 4)), 1).flatten()


def _inputs(c, seed):
    dev = _device()
    gen = torch.Generator(device=dev).manual_seed(seed)
    rows, cin = c["rows"], c["in"]
    t = {}
    # normalised activations with a few strong channels
    strong = 1 + 7 * (torch.rand(cin, generator=gen, device=dev) < 0.01).float()
    t["x"] = torch.randn(rows, cin, generator=gen, device=dev) * strong
    if c["op"] in ("route", "layer"):
        t["router"] = torch.randn(c["experts"], cin, generator=gen, device=dev) / math.sqrt(cin)
        t["router_bias"] = torch.randn(c["experts"], generator=gen, device=dev) * 0.1 if c["bias"] else None
    if c["op"] in ("experts", "layer"):
        e, hid, out = c["experts"], c["hidden"], c["out"]
        t["gate"] = _quantized(gen, c["fmt"], e * hid, cin, 0.02, dev)
        t["up"] = _quantized(gen, c["fmt"], e * hid, cin, 0.02, dev)
        t["down"] = _quantized(gen, c["fmt_down"], e * out, hid, 0.02, dev)
    if c["op"] == "experts":
        logits = torch.randn(rows, c["experts"], generator=gen, device=dev)
        w, ids = torch.topk(torch.softmax(logits, 1), c["top_k"], 1)
        t["weights"] = (w / w.sum(1, keepdim=True)).contiguous()
        skip = torch.rand(rows, c["top_k"], generator=gen, device=dev) < c["empty"]
        t["ids"] = torch.where(skip, -1, ids).to(torch.int32).contiguous()
    if c["op"] == "epilogue":
        t["w"] = _quantized(gen, c["fmt"], c["out"], cin, 0.02, dev)
        t["bias"] = torch.randn(c["out"], generator=gen, device=dev) * 0.5 if c["bias"] else None
        t["row_scale"] = torch.rand(rows, generator=gen, device=dev) if c["row_scale"] else None
    if c["op"] != "route":
        t["residual"] = torch.randn(rows, c["out"], generator=gen, device=dev) if c["residual"] else None
    return t


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    s["kept"] = {}  # what a program keeps from one call to the next: handles, outputs, a workspace
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def _dequantized(fmt, blocks, rows, cols):
    """fp32 [rows, cols] of packed blocks [rows][ceil(cols/32)]."""
    nb = (cols + 31) // 32
    b = blocks.view(rows * nb, BLOCK[fmt])
    d = b[:, 0:2].contiguous().view(torch.float16).float()
    if fmt == "q8_0":
        w = b[:, 2:].contiguous().view(torch.int8).float() * d
    else:
        q = b[:, 2 if fmt == "q4_0" else 4:]
        q = torch.cat((q & 15, q >> 4), 1).float()
        w = (q - 8) * d if fmt == "q4_0" else q * d + b[:, 2:4].contiguous().view(torch.float16).float()
    return w.view(rows, nb * 32)[:, :cols]


def _plain_route(c, x, w, bias):
    logits = x.double() @ w.double().t()
    scores = torch.softmax(logits, 1) if c["scoring"] == "softmax" else 1 / (1 + torch.exp(-logits))
    choice = scores if bias is None else scores + bias.double()
    choice, ids = torch.sort(choice, dim=1, descending=True, stable=True)
    ids, choice = ids[:, :c["top_k"]], choice[:, :c["top_k"]]
    picked = scores.gather(1, ids)
    if c["renorm"]:
        picked = picked / picked.sum(1, keepdim=True)
    out = ids.to(torch.int32), (picked * c["scale"]).float()
    return out + (logits.float(),) if c.get("logits") else out


def _plain_experts(c, t, ids, weights):
    rows, k, e, hid, cin, out = c["rows"], c["top_k"], c["experts"], c["hidden"], c["in"], c["out"]
    held = (ids >= 0) & (ids < e)
    at = torch.where(held, ids, 0).long()
    wt = torch.where(held, weights, 0.0)
    if rows * k <= e:  # fewer (row, slot) pairs than experts: each pair takes its expert's blocks
        def of(name, fmt, n_out, n_in):
            b = t[name].view(e, -1)[at.flatten()]
            return _dequantized(fmt, b.flatten(), rows * k * n_out, n_in).view(rows * k, n_out, n_in)
        x = t["x"].repeat_interleave(k, 0).unsqueeze(2)
        g = torch.bmm(of("gate", c["fmt"], hid, cin), x).squeeze(2)
        u = torch.bmm(of("up", c["fmt"], hid, cin), x).squeeze(2)
        h = g / (1 + torch.exp(-g)) * u
        d = torch.bmm(of("down", c["fmt_down"], out, hid), h.unsqueeze(2)).view(rows, k, out)
        y = (d * wt.unsqueeze(2)).sum(1)
    else:  # every expert over every row, weighed by the row's choice
        x = t["x"].unsqueeze(0).expand(e, rows, cin)
        g = torch.bmm(x, _dequantized(c["fmt"], t["gate"], e * hid, cin).view(e, hid, cin).transpose(1, 2))
        u = torch.bmm(x, _dequantized(c["fmt"], t["up"], e * hid, cin).view(e, hid, cin).transpose(1, 2))
        share = torch.zeros(rows, e, device=wt.device).scatter_add_(1, at, wt)
        h = g / (1 + torch.exp(-g)) * u * share.t().unsqueeze(2)
        d = _dequantized(c["fmt_down"], t["down"], e * out, hid).view(e, out, hid)
        y = torch.bmm(h, d.transpose(1, 2)).sum(0)
    return y if t["residual"] is None else y + t["residual"]


def _plain_act(v, act):
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    if act == "relu":
        return torch.where(v < 0, 0.0, v)
    return 1 / (1 + torch.exp(-v)) if act == "sigmoid" else v


def _plain_epilogue(c, t):
    y = t["x"] @ _dequantized(c["fmt"], t["w"], c["out"], c["in"]).t()
    if t["bias"] is not None:
        y = y + t["bias"]
    y = _plain_act(y, c["act"])
    if t["row_scale"] is not None:
        y = y * t["row_scale"].unsqueeze(1)
    return y if t["residual"] is None else y + t["residual"]


def _mlq():
    """The library's bindings (the package folder's name has a hyphen, so it is loaded by path)."""
    if "mini_llama_b200" not in sys.modules:
        import importlib.util
        folder = os.path.join(os.getcwd(), "mini-llama_b200")
        spec = importlib.util.spec_from_file_location("mini_llama_b200", os.path.join(folder, "__init__.py"),
                                                      submodule_search_locations=[folder])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["mini_llama_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["mini_llama_b200"].mlq


def _own(s):
    m, c, keep = _mlq(), s["case"], s["kept"]
    op = c["op"]
    if not keep:
        if op in ("route", "layer"):
            keep["router"] = m.Router(s["router"], c["top_k"], bias=s["router_bias"], scoring=c["scoring"],
                                      renormalize=c["renorm"], scale=c["scale"])
        if op in ("experts", "layer"):
            keep["experts"] = m.Experts(c["fmt"], s["gate"], s["up"], s["down"], c["experts"], c["in"], c["hidden"],
                                        out_features=c["out"], fmt_down=c["fmt_down"])
        need = {"route": lambda: m.route_workspace_bytes(keep["router"], c["rows"]),
                "experts": lambda: m.experts_workspace_bytes(keep["experts"], c["rows"], c["top_k"]),
                "layer": lambda: m.layer_workspace_bytes(keep["router"], keep["experts"], c["rows"]),
                "epilogue": lambda: m.epilogue_workspace_bytes(c["fmt"], c["out"], c["in"], c["rows"])}[op]()
        keep["workspace"] = torch.empty(need, dtype=torch.uint8, device=s["x"].device)
    ws = keep["workspace"]
    if op == "route":
        logits = torch.empty(c["rows"], c["experts"], device=s["x"].device) if c["logits"] else None
        out = m.moe_route(keep["router"], s["x"], logits=logits, workspace=ws)
        return out + (logits,) if c["logits"] else out
    if op == "experts":
        return m.moe_experts(keep["experts"], s["x"], s["ids"], s["weights"], residual=s["residual"], workspace=ws)
    if op == "layer":
        return m.moe_layer(keep["router"], keep["experts"], s["x"], residual=s["residual"], workspace=ws)
    return m.linear_epilogue(c["fmt"], s["w"], c["out"], c["in"], s["x"], bias=s["bias"], activation=c["act"],
                             row_scale=s["row_scale"], residual=s["residual"], workspace=ws)


def run(state):
    if own:
        return _own(state)
    c = state["case"]
    if c["op"] == "route":
        return _plain_route(c, state["x"], state["router"], state["router_bias"])
    if c["op"] == "experts":
        return _plain_experts(c, state, state["ids"], state["weights"])
    if c["op"] == "layer":
        ids, weights = _plain_route(c, state["x"], state["router"], state["router_bias"])
        return _plain_experts(c, state, ids, weights), ids, weights
    return _plain_epilogue(c, state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    rows, cin = c["rows"], c["in"]
    b = rows * cin * 4
    f = 0.0
    if c["op"] in ("route", "layer"):
        b += c["experts"] * cin * 4 + rows * c["top_k"] * 8
        f += 2.0 * rows * c["experts"] * cin
    if c["op"] in ("experts", "layer"):
        e, k, hid, out = c["experts"], c["top_k"], c["hidden"], c["out"]
        share = k / e * (1 - c.get("empty", 0.0))
        used = e * (1 - (1 - share) ** rows)  # experts that some row names, with even routing
        b += used * (2 * hid * -(-cin // 32) * BLOCK[c["fmt"]] + out * -(-hid // 32) * BLOCK[c["fmt_down"]])
        b += rows * (k * 8 + out * 4 * (2 if c["residual"] else 1))
        f += 2.0 * rows * e * share * hid * (2 * cin + out)
    if c["op"] == "epilogue":
        out = c["out"]
        b += out * -(-cin // 32) * BLOCK[c["fmt"]] + rows * out * 4 * (2 if c["residual"] else 1)
        f += 2.0 * rows * out * cin
    return {"bytes": float(b), "flops": f}


# ---------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------
def _values64(fmt, raw, n_in):
    """Rows of packed blocks (uint8 [n, row bytes]) as float64 [n, n_in], from the block layouts."""
    n = raw.shape[0]
    raw = raw.reshape(n, -1, BLOCK[fmt])
    half = lambda o: raw[..., o:o + 2].clone().view(torch.float16).to(torch.float64)  # noqa: E731
    if fmt == "q8_0":
        v = half(0) * raw[..., 2:].clone().view(torch.int8).to(torch.float64)
    else:
        code = raw[..., BLOCK[fmt] - 16:].to(torch.int64)
        code = torch.stack((code % 16, code // 16), -2).flatten(-2).to(torch.float64)
        v = half(0) * code + (half(2) if fmt == "q4_1" else -8.0 * half(0))
    return v.reshape(n, -1)[:, :n_in]


def _exact_route(c, t):
    logits = torch.einsum("ri,ei->re", t["x"].to(torch.float64), t["router"].to(torch.float64))
    if c["scoring"] == "softmax":
        p = torch.exp(logits - logits.amax(1, keepdim=True))
        p = p / p.sum(1, keepdim=True)
    else:
        p = torch.sigmoid(logits)
    rank = p if t["router_bias"] is None else p + t["router_bias"].to(torch.float64)
    left, ids, chosen = rank.clone(), [], []
    for _ in range(c["top_k"]):
        best = left.amax(1, keepdim=True)
        at = (left == best).to(torch.int8).argmax(1, keepdim=True)  # the first of equals
        ids.append(at)
        chosen.append(p.gather(1, at))
        left.scatter_(1, at, -math.inf)
    ids, chosen = torch.cat(ids, 1), torch.cat(chosen, 1)
    if c["renorm"]:
        chosen = chosen / chosen.sum(1, keepdim=True)
    out = ids.to(torch.int32), chosen * c["scale"]
    return out + (logits,) if c.get("logits") else out


def _exact_experts(c, t, ids, weights):
    x = t["x"].to(torch.float64)
    y = torch.zeros(c["rows"], c["out"], dtype=torch.float64, device=x.device)
    hid, out = c["hidden"], c["out"]
    for e in sorted(set(ids.flatten().tolist())):
        if e < 0 or e >= c["experts"]:
            continue
        r, j = torch.nonzero(ids == e, as_tuple=True)
        rows_of = lambda name, n: t[name].view(c["experts"], n, -1)[e]  # noqa: E731
        g = x[r] @ _values64(c["fmt"], rows_of("gate", hid), c["in"]).T
        u = x[r] @ _values64(c["fmt"], rows_of("up", hid), c["in"]).T
        h = g * torch.sigmoid(g) * u
        d = h @ _values64(c["fmt_down"], rows_of("down", out), hid).T
        y.index_add_(0, r, d * weights[r, j].to(torch.float64).unsqueeze(1))
    return y if t["residual"] is None else y + t["residual"].to(torch.float64)


def _exact_epilogue(c, t):
    v = t["x"].to(torch.float64) @ _values64(c["fmt"], t["w"].view(c["out"], -1), c["in"]).T
    if t["bias"] is not None:
        v = v + t["bias"].to(torch.float64)
    act = c["act"]
    if act == "silu":
        v = v * torch.sigmoid(v)
    elif act == "gelu":
        v = v * torch.special.ndtr(v)
    elif act == "gelu_tanh":
        v = v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))
    elif act == "relu":
        v = v.clamp_min(0)
    elif act == "sigmoid":
        v = torch.sigmoid(v)
    if t["row_scale"] is not None:
        v = v * t["row_scale"].to(torch.float64)[:, None]
    return v if t["residual"] is None else v + t["residual"].to(torch.float64)


def exact(case, seed):
    c, t = case, _inputs(case, seed)
    if c["op"] == "route":
        return _exact_route(c, t)
    if c["op"] == "experts":
        return _exact_experts(c, t, t["ids"], t["weights"])
    if c["op"] == "layer":
        ids, weights = _exact_route(c, t)
        return _exact_experts(c, t, ids, weights), ids, weights
    return _exact_epilogue(c, t)

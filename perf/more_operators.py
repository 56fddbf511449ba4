"""Performance cases of the operators around products by experts.

A case is one call of
  * ``op = "route"``:    a token's experts and their weights from its scores, softmax or sigmoid, with a bias for balance and groups or without;
  * ``op = "dispatch"``: the tokens' rows sorted by expert, a row for each of a token's experts, as they are (``out = "same"``), in int8 with a scale
                         per token (``"int8"``) or in fp8 with a scale per 128 channels (``"group"``);
  * ``op = "product"``:  the product of int8 rows, sorted by expert, with their expert's int8 weights, scales per token and channel;
  * ``op = "silu"``:     silu(gate) * up between the two products, with an output in the model's type or in 8 bits (``"int8"`` and ``"fp8"`` per
                         token, ``"group"`` per 128 channels);
  * ``op = "combine"``:  the weighted sum of a token's rows that come back from its experts.

Sizes: the hidden sizes of the 7B- and 0.5B-class layers of the benchmark (3584, 896), the channels of its projections, and generic ones; token counts
from one decoding sequence to a long prompt.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
NAMES = {"bf16": "bfloat16", "fp16": "float16"}
E4M3 = torch.float8_e4m3fn


def _route(name, tokens, experts, top, scoring, dtype, bias=False, groups=1, top_groups=1, group_score="max", renormalize=True, scale=1.0):
    return {"name": name, "op": "route", "tokens": tokens, "experts": experts, "top": top, "scoring": scoring, "dtype": dtype, "bias": bias,
            "groups": groups, "top_groups": top_groups, "group_score": group_score, "renormalize": renormalize, "scale": scale}


def _dispatch(name, tokens, k, experts, top, out, dtype):
    return {"name": name, "op": "dispatch", "tokens": tokens, "k": k, "experts": experts, "top": top, "out": out, "dtype": dtype}


def _product(name, rows, experts, n, k, dtype, bias=False):
    return {"name": name, "op": "product", "rows": rows, "experts": experts, "n": n, "k": k, "dtype": dtype, "bias": bias}


def _silu(name, rows, n, out, dtype):
    return {"name": name, "op": "silu", "rows": rows, "n": n, "out": out, "dtype": dtype}


def _combine(name, tokens, n, top, dtype, shared=False):
    return {"name": name, "op": "combine", "tokens": tokens, "n": n, "top": top, "dtype": dtype, "shared": shared}


def listed():
    return [
        # a decode batch: launch and latency
        _route("route_decode16", 16, 64, 8, "softmax", "bf16"),
        # a long prompt over many experts in groups, with a bias for balance
        _route("route_prompt8192_groups", 8192, 256, 8, "sigmoid", "fp32", bias=True, groups=8, top_groups=4, group_score="top2", scale=2.5),
        # a decode batch in front of an int8 product
        _dispatch("dispatch_decode48_int8", 48, 3584, 64, 4, "int8", "bf16"),
        # a prompt of no round length on a small model, in front of a block-scaled product
        _dispatch("dispatch_prompt1999_group", 1999, 896, 60, 4, "group", "fp16"),
        # a long prompt in front of an int8 product
        _dispatch("dispatch_prompt8192_int8", 8192, 3584, 32, 4, "int8", "bf16"),
        # a decode batch of 32 sequences, each token to 8 of 64 experts: a few rows per expert, the weights' stream
        _product("product_decode_64_experts", 256, 64, 2048, 2048, "bf16"),
        # a prompt of no round length, each token to 2 of 16 experts
        _product("product_prompt_16_experts", 1998, 16, 3584, 1536, "fp16", bias=True),
        # the largest call: a long prompt, each token to 4 of 32 experts
        _product("product_prompt_32_experts", 32768, 32, 4864, 3584, "bf16"),
        # a decode batch in front of the longest reduction of the layer without experts
        _silu("silu_decode37_int8", 37, 18944, "int8", "fp16"),
        # a long prompt, each token to 4 experts
        _silu("silu_prompt32768_group", 32768, 2432, "group", "bf16"),
        # a decode batch, beside an expert that all tokens share
        _combine("combine_decode48", 48, 3584, 4, "fp16", shared=True),
        # a long prompt
        _combine("combine_prompt8192", 8192, 3584, 4, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "dispatch", "product", "silu", "combine"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "route":
        tokens, sigmoid = _log(rng, 1, 8192), rng.random() < 0.5
        case = {"op": op, "tokens": tokens, "top": rng.randint(1, 8), "scoring": "sigmoid" if sigmoid else "softmax",
                "dtype": rng.choice(["bf16", "fp16", "fp32"]), "bias": sigmoid, "renormalize": rng.random() < 0.7, "scale": rng.choice([1.0, 2.5])}
        if rng.random() < 0.4:
            groups = rng.choice([2, 4, 8])
            return {**case, "experts": groups * rng.randint(8, 32), "groups": groups, "top_groups": rng.randint(1, groups),
                    "group_score": "top2" if sigmoid else "max"}
        return {**case, "experts": _log(rng, 8, 256), "groups": 1, "top_groups": 1, "group_score": "max"}
    top = rng.randint(1, 8)
    if op == "dispatch":
        return {"op": op, "tokens": _log(rng, 1, 8192), "k": 8 * _log(rng, 64, 448), "experts": _log(rng, 8, 256), "top": top,
                "out": rng.choice(["same", "int8", "group"]), "dtype": dtype}
    if op == "silu":
        return {"op": op, "rows": _log(rng, 1, 32768), "n": 8 * _log(rng, 64, 608), "out": rng.choice(["same", "int8", "fp8", "group"]), "dtype": dtype}
    if op == "combine":
        return {"op": op, "tokens": _log(rng, 1, 8192), "n": 8 * _log(rng, 64, 448), "top": top, "dtype": dtype, "shared": rng.random() < 0.3}
    experts = _log(rng, 2, 128)
    n, k = _log(rng, 256, 4864), 16 * _log(rng, 32, 224)
    if experts > 32:  # many experts are small ones
        n, k = min(n, 2048), min(k, 2048)
    return {"op": op, "rows": _log(rng, 1, 32768), "experts": experts, "n": n, "k": k, "dtype": dtype, "bias": rng.random() < 0.3}


def _blocks(size):
    return -(-size // BLOCK)


def _activations(rows, k, gen, dev):
    """Normal values with a few channels that are much larger, as hidden states have them."""
    x = torch.randn(rows, k, generator=gen, device=dev)
    loud = torch.rand(k, generator=gen, device=dev) < 0.01
    return x * torch.where(loud, 12.0, 1.0)


def _chosen(tokens, experts, top, gen, dev):
    """Each token's experts, no one twice, some of them popular."""
    liked = torch.randn(tokens, experts, generator=gen, device=dev) + torch.randn(experts, generator=gen, device=dev)
    return liked.topk(min(top, experts), dim=1).indices.to(torch.int32)


def _offsets(rows, experts, gen, dev):
    """First rows of the experts' parts and the end of the last: popular experts, rare ones, and one in eight that nobody asked for."""
    like = torch.rand(experts, generator=gen, device=dev) + 0.3
    like = like * (torch.rand(experts, generator=gen, device=dev) > 0.125)
    like[0] += 0.3
    ends = (like.cumsum(0) / like.sum() * rows).round().to(torch.int32)
    ends[-1] = rows
    return torch.cat([torch.zeros(1, dtype=torch.int32, device=dev), ends])


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    op, dt = case["op"], DTYPES[case["dtype"]]
    s = dict(case, dt=dt)
    if op == "route":
        shape = case["tokens"], case["experts"]
        s["logits"] = (1.5 * torch.randn(shape, generator=gen, device=dev) + 0.5 * torch.randn(shape[1], generator=gen, device=dev)).to(dt)
        s["bias"] = 0.1 * torch.randn(shape[1], generator=gen, device=dev) if case["bias"] else None
        s["top"] = min(case["top"], case["experts"] // case["groups"] * case["top_groups"])
    elif op == "dispatch":
        s["x"] = _activations(case["tokens"], case["k"], gen, dev).to(dt)
        s["ids"] = _chosen(case["tokens"], case["experts"], case["top"], gen, dev)
    elif op == "silu":
        s["x"] = _activations(case["rows"], 2 * case["n"], gen, dev).to(dt)
    elif op == "combine":
        tokens, top = case["tokens"], case["top"]
        s["y"] = _activations(tokens * top, case["n"], gen, dev).to(dt)
        s["weights"] = torch.rand(tokens, top, generator=gen, device=dev).softmax(1)
        expert = _chosen(tokens, 64, top, gen, dev)
        s["places"] = expert.view(-1).argsort(stable=True).argsort().to(torch.int32).view(tokens, top)
        s["shared"] = _activations(tokens, case["n"], gen, dev).to(dt) if case["shared"] else None
    else:
        rows, experts, n, k = case["rows"], case["experts"], case["n"], case["k"]
        x = _activations(rows, k, gen, dev)
        scale = x.abs().amax(1, keepdim=True) / 127
        s["q"], s["alpha"] = (x / scale).round().to(torch.int8), scale
        s["beta"] = (torch.rand(experts, n, generator=gen, device=dev) + 0.5) * (0.06 / 127)
        s["w"] = torch.empty(experts, n, k, dtype=torch.int8, device=dev)
        for part in s["w"].view(-1, k).split(8192):
            part.copy_((torch.randn(part.shape, generator=gen, device=dev) * 32).round().clamp(-127, 127))
        s["bias"] = torch.randn(experts, n, generator=gen, device=dev).to(dt) if case["bias"] else None
        s["offsets"] = _offsets(rows, experts, gen, dev)
        s["most"] = int(s["offsets"].diff().max())  # rows of the largest expert
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------

def _route_plain(s):
    x = s["logits"].double()  # neighbours in the order of the scores differ by less than 32 bits tell apart
    score = torch.sigmoid(x) if s["scoring"] == "sigmoid" else torch.exp(x - x.amax(1, keepdim=True))
    if s["scoring"] == "softmax":
        score = score / score.sum(1, keepdim=True)
    choice = score if s["bias"] is None else score + s["bias"].double()
    if s["groups"] > 1:
        parts = choice.view(choice.shape[0], s["groups"], -1)
        best = parts.amax(2) if s["group_score"] == "max" else parts.sort(2, descending=True).values[..., :2].sum(2)
        kept = best.sort(dim=1, descending=True, stable=True).indices[:, :s["top_groups"]]
        keep = torch.zeros_like(best, dtype=torch.bool).scatter_(1, kept, True)
        choice = torch.where(keep[..., None], parts, -math.inf).view(choice.shape)
    ids = choice.sort(dim=1, descending=True, stable=True).indices[:, :s["top"]]
    w = score.gather(1, ids)
    if s["renormalize"]:
        w = w / w.sum(1, keepdim=True)
    return (w * s["scale"]).float(), ids.to(torch.int32)


def _groups_plain(x):
    rows, k = x.shape
    full = torch.nn.functional.pad(x, (0, _blocks(k) * BLOCK - k)).view(rows, -1, BLOCK)
    scale = full.abs().amax(-1).clamp_min(1e-12) / full.new_tensor(448.0)
    q = (full / scale[..., None]).clamp(-448, 448).to(E4M3)
    return q.view(rows, -1)[:, :k], scale


def _int8_plain(x):
    """The framework's int8 quantizer: scale and quotient are values of the activations' type."""
    dt, f = x.dtype, x.float()
    floor = torch.tensor(1e-5, device=x.device).to(dt).float()
    scale = (torch.maximum(f.abs().amax(1, keepdim=True), floor) / f.new_tensor(127.0)).to(dt).float()
    return (f / scale).to(dt).float().round().clamp(-128, 127).to(torch.int8), scale


def _dispatch_plain(s):
    flat = s["ids"].reshape(-1)
    order = flat.argsort(stable=True)
    places = torch.empty_like(flat)
    places[order] = torch.arange(flat.numel(), dtype=torch.int32, device=flat.device)
    counts = (flat[:, None] == torch.arange(s["experts"], device=flat.device)).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    token = order // s["ids"].shape[1]
    rows = (s["x"],) if s["out"] == "same" else _int8_plain(s["x"]) if s["out"] == "int8" else _groups_plain(s["x"].float())
    return (*(r[token] for r in rows), offsets, places.view_as(s["ids"]))


def _product_plain(s):
    a, w = s["q"].float(), s["w"].float()
    row = torch.arange(s["rows"], device=a.device)
    expert = torch.searchsorted(s["offsets"][1:], row, right=True)
    place = row - s["offsets"][expert]
    padded = a.new_zeros(w.shape[0], s["most"], s["k"])
    padded[expert, place] = a
    y = torch.bmm(padded, w.transpose(-1, -2))[expert, place] * s["alpha"] * s["beta"][expert]
    return (y if s["bias"] is None else y + s["bias"].float()[expert]).to(s["dt"])


def _silu_plain(s):
    g, u = s["x"].float().chunk(2, dim=1)
    y = g / (1 + torch.exp(-g)) * u
    if s["out"] == "same":
        return y.to(s["dt"])
    if s["out"] == "group":
        return _groups_plain(y)
    top = y.abs().amax(1, keepdim=True)
    if s["out"] == "fp8":
        scale = top.clamp_min(1e-12) / 448
        return (y / scale).clamp(-448, 448).to(E4M3), scale
    scale = top.clamp_min(1e-5) / 127
    return (y / scale).round().clamp(-128, 127).to(torch.bfloat16), scale


def _combine_plain(s):
    y = (s["y"].float()[s["places"]] * s["weights"][..., None]).sum(1)
    return (y if s["shared"] is None else y + s["shared"].float()).to(s["dt"])


# ---- the framework's calls ---------------------------------------------------------------------------------------

def _route_own(s):
    from llmqrt_amd.experts import route_to_experts
    return route_to_experts(s["logits"], s["top"], s["scoring"], s["bias"], s["groups"], s["top_groups"], s["group_score"], s["renormalize"], s["scale"])


def _dispatch_own(s):
    from llmqrt_amd import experts
    if s["out"] == "same":
        return experts.dispatch_to_experts(s["x"], s["ids"], s["experts"])
    if s["out"] == "group":
        return experts.dispatch_per_group_quantize(s["x"], s["ids"], s["experts"])
    return experts.dispatch_quantize_activation_per_token_absmax(s["x"], s["ids"], s["experts"])


def _product_own(s):
    from llmqrt_amd.sq_fp8_kernels import w8a8_int8_linear_per_channel_grouped
    return w8a8_int8_linear_per_channel_grouped(s["q"], s["w"], s["bias"], s["alpha"], s["beta"], s["offsets"], NAMES[s["dtype"]])


def _silu_own(s):
    from llmqrt_amd import activation
    if s["out"] == "same":
        return activation.silu_mul(s["x"])
    if s["out"] == "group":
        return activation.silu_mul_per_group_quantize(s["x"])
    if s["out"] == "fp8":
        return activation.silu_mul_per_token_quantize(s["x"])
    q, scale = activation.silu_mul_quantize_activation_per_token_absmax(s["x"])
    return q.to(torch.bfloat16), scale  # (computed codes: a value next to the middle between two may come out as either)


def _combine_own(s):
    from llmqrt_amd.experts import combine_from_experts
    return combine_from_experts(s["y"], s["places"], s["weights"], s["shared"])


def run(state):
    op = state["op"]
    if own:
        return {"route": _route_own, "dispatch": _dispatch_own, "product": _product_own, "silu": _silu_own, "combine": _combine_own}[op](state)
    return {"route": _route_plain, "dispatch": _dispatch_plain, "product": _product_plain, "silu": _silu_plain, "combine": _combine_plain}[op](state)


def work(case):
    op = case["op"]
    if op == "route":
        scores = case["tokens"] * case["experts"]
        size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
        return {"bytes": size * scores + (4 * case["experts"] if case["bias"] else 0) + 8 * case["tokens"] * case["top"], "flops": 4 * scores}
    if op == "dispatch":
        tokens, k, rows = case["tokens"], case["k"], case["tokens"] * min(case["top"], case["experts"])
        row = {"same": 2 * k, "int8": k + 4, "group": k + 4 * _blocks(k)}[case["out"]]
        return {"bytes": 2 * tokens * k + rows * (row + 8) + 4 * (case["experts"] + 1), "flops": 3 * tokens * k}
    if op == "silu":
        rows, n = case["rows"], case["n"]
        row = {"same": 2 * n, "int8": n + 4, "fp8": n + 4, "group": n + 4 * _blocks(n)}[case["out"]]
        return {"bytes": rows * (4 * n + row), "flops": 6 * rows * n}
    if op == "combine":
        tokens, n, top = case["tokens"], case["n"], case["top"]
        return {"bytes": 2 * tokens * n * (top + 1 + case["shared"]) + 8 * tokens * top, "flops": 2 * tokens * n * top}
    rows, n, k = case["rows"], case["n"], case["k"]
    used = min(case["experts"], rows)  # experts without rows are not read
    weights = used * (n * k + 4 * n + (2 * n if case["bias"] else 0))
    return {"bytes": rows * (k + 4) + weights + 2 * rows * n, "flops": 2 * rows * n * k}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------

def _route_exact(s):
    x = s["logits"].double()
    tokens, experts = x.shape
    score = 1 / (1 + torch.exp(-x)) if s["scoring"] == "sigmoid" else torch.softmax(x, 1)
    left = score.clone() if s["bias"] is None else score + s["bias"].double()
    each = experts // s["groups"]
    if s["groups"] > 1:
        best = torch.stack([left[:, g * each:(g + 1) * each].topk(2 if s["group_score"] == "top2" else 1, dim=1).values.sum(1)
                            for g in range(s["groups"])], 1)
        allowed = torch.zeros_like(left, dtype=torch.bool)
        row, member = torch.arange(tokens, device=x.device), torch.arange(each, device=x.device)
        for _ in range(s["top_groups"]):
            g = _first_max(best)
            best[row, g] = -math.inf
            allowed[row[:, None], g[:, None] * each + member] = True
        left = left.masked_fill(~allowed, -math.inf)
    ids = []
    for _ in range(s["top"]):
        ids.append(_first_max(left))
        left.scatter_(1, ids[-1][:, None], -math.inf)
    ids = torch.stack(ids, 1)
    w = torch.gather(score, 1, ids)
    total = w.sum(1, keepdim=True) if s["renormalize"] else 1.0
    return w / total * s["scale"], ids.to(torch.int32)


def _first_max(v):
    """Index of each row's largest value, the lowest where several are."""
    index = torch.arange(v.shape[1], device=v.device).expand_as(v)
    return torch.where(v == v.max(1, keepdim=True).values, index, v.shape[1]).min(1).values


def _groups64(y):
    out_q, out_s = torch.empty(y.shape, dtype=torch.float64, device=y.device), []
    for c in range(0, y.shape[1], BLOCK):
        part = y[:, c:c + BLOCK]
        s = torch.maximum(part.abs().max(dim=1, keepdim=True).values, part.new_tensor(1e-12)) / 448.0
        out_q[:, c:c + BLOCK] = (part / s).to(E4M3).double()
        out_s.append(s)
    return out_q, torch.cat(out_s, 1)


def _dispatch_exact(s):
    tokens, top = s["ids"].shape
    flat = s["ids"].reshape(-1).cpu().tolist()
    parts = [[] for _ in range(s["experts"])]
    for i, e in enumerate(flat):
        parts[e].append(i)
    order = [i for part in parts for i in part]
    places, offsets = [0] * len(flat), [0]
    for r, i in enumerate(order):
        places[i] = r
    for part in parts:
        offsets.append(offsets[-1] + len(part))
    dev = s["x"].device
    token = torch.tensor(order, device=dev).div(top, rounding_mode="floor")
    x = s["x"].double()
    if s["out"] == "same":
        rows = (x,)
    elif s["out"] == "group":
        rows = _groups64(x)
    else:
        least = torch.full((), 1e-5, dtype=s["dt"], device=dev).double()
        scale = (torch.maximum(x.abs().max(dim=1, keepdim=True).values, least) / 127.0).to(s["dt"]).double()
        rows = (x / scale).to(s["dt"]).double().round().clamp(-128, 127).to(torch.int8), scale
    return (*(torch.index_select(r, 0, token) for r in rows), torch.tensor(offsets, dtype=torch.int32, device=dev),
            torch.tensor(places, dtype=torch.int32, device=dev).view(tokens, top))


def _product_exact(s):
    y = torch.empty(s["rows"], s["n"], dtype=torch.float64, device=s["q"].device)
    at = s["offsets"].tolist()
    for e in range(s["experts"]):
        lo, hi = at[e], at[e + 1]
        if hi > lo:
            y[lo:hi] = s["q"][lo:hi].double() @ s["w"][e].double().t() * s["alpha"][lo:hi].double() * s["beta"][e].double()
            if s["bias"] is not None:
                y[lo:hi] += s["bias"][e].double()
    return y


def _silu_exact(s):
    x = s["x"].double()
    g, u = x[:, :s["n"]], x[:, s["n"]:]
    y = g * torch.sigmoid(g) * u
    if s["out"] == "same":
        return y
    if s["out"] == "group":
        return _groups64(y)
    top = y.abs().max(dim=1, keepdim=True).values
    if s["out"] == "fp8":
        scale = top.clamp_min(1e-12) / 448.0
        return (y / scale).to(E4M3).double(), scale
    scale = top.clamp_min(1e-5) / 127.0
    return torch.round(y / scale), scale


def _combine_exact(s):
    y = torch.zeros(s["tokens"], s["n"], dtype=torch.float64, device=s["y"].device) if s["shared"] is None else s["shared"].double()
    for j in range(s["top"]):
        y += s["weights"][:, j:j + 1].double() * s["y"].index_select(0, s["places"][:, j].long()).double()
    return y


def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _route_exact, "dispatch": _dispatch_exact, "product": _product_exact, "silu": _silu_exact, "combine": _combine_exact}[case["op"]](s)

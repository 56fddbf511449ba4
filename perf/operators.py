"""Performance cases of the operators around block-scaled fp8 (e4m3fn) products.

A case is one call of
  * ``op = "norm"``:    the residual's addition and RMSNorm, with the normalised row as it is (``out = "same"``) or in 8 bits:
                        int8 or fp8 with a scale per token (``"int8"``, ``"fp8"``), fp8 with a scale per 128 channels (``"group"``);
  * ``op = "quant"``:   the fp8 quantizer with a scale per token and 128 channels;
  * ``op = "gemm"``:    the product of such activations with weights that have a scale per block of 128 x 128;
  * ``op = "grouped"``: the same product by experts, each with its own weights and as many rows as were routed to it.

Sizes: the 7B-class layer of the benchmark (hidden 3584, feed-forward 18944), the 0.5B-class one (hidden 896), and generic ones;
token counts from one decoding sequence to a long prompt.
"""
from __future__ import annotations

import math

import torch

own = False

BLOCK = 128
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
NAMES = {"bf16": "bfloat16", "fp16": "float16"}
E4M3 = torch.float8_e4m3fn


def _norm(name, rows, k, out, dtype):
    return {"name": name, "op": "norm", "rows": rows, "k": k, "out": out, "dtype": dtype}


def _quant(name, rows, k, dtype):
    return {"name": name, "op": "quant", "rows": rows, "k": k, "dtype": dtype}


def _gemm(name, rows, n, k, dtype, bias=False):
    return {"name": name, "op": "gemm", "rows": rows, "n": n, "k": k, "dtype": dtype, "bias": bias}


def _grouped(name, rows, experts, n, k, dtype, bias=False):
    return {"name": name, "op": "grouped", "rows": rows, "experts": experts, "n": n, "k": k, "dtype": dtype, "bias": bias}


def listed():
    return [
        # one sequence decoding: the norm in front of a block-scaled projection, launch and latency
        _norm("norm_decode1_group", 1, 3584, "group", "bf16"),
        # a short prompt on a small model, the norm in front of an int8 projection
        _norm("norm_prompt333_int8", 333, 896, "int8", "fp16"),
        # a long prompt, the last norm of a model: nothing is quantized
        _norm("norm_prompt8192_same", 8192, 3584, "same", "bf16"),
        # a decode batch in front of the longest reduction
        _quant("quant_decode37", 37, 18944, "fp16"),
        # a long prompt in front of the longest reduction
        _quant("quant_prompt8192", 8192, 18944, "bf16"),
        # one sequence decoding, the narrowest projection of the layer: latency and the weights' stream
        _gemm("gemm_decode1_o", 1, 3584, 3584, "bf16"),
        # a decode batch, the widest projection: the weights' stream
        _gemm("gemm_decode48_gate_up", 48, 37888, 3584, "bf16"),
        # a mid-sized prompt of no round length, the longest reduction, with bias
        _gemm("gemm_prompt777_down", 777, 3584, 18944, "fp16", bias=True),
        # the largest call: a long prompt through the widest projection
        _gemm("gemm_prompt8192_gate_up", 8192, 37888, 3584, "bf16"),
        # a decode batch of 32 sequences, each token to 8 of 64 experts: a few rows per expert
        _grouped("grouped_decode_64_experts", 256, 64, 2048, 2048, "bf16"),
        # a prompt of no round length, each token to 2 of 16 experts
        _grouped("grouped_prompt_16_experts", 1998, 16, 3584, 1536, "fp16", bias=True),
        # a long prompt, each token to 4 of 32 experts
        _grouped("grouped_prompt_32_experts", 32768, 32, 4864, 3584, "bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "quant", "gemm", "grouped"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "norm":
        return {"op": op, "rows": _log(rng, 1, 8192), "k": 8 * _log(rng, 64, 1024), "out": rng.choice(["same", "int8", "fp8", "group"]),
                "dtype": dtype}
    if op == "quant":
        return {"op": op, "rows": _log(rng, 1, 8192), "k": 8 * _log(rng, 64, 2368), "dtype": dtype}
    bias = rng.random() < 0.3
    if op == "gemm":
        return {"op": op, "rows": _log(rng, 1, 8192), "n": _log(rng, 128, 37888), "k": 16 * _log(rng, 32, 224), "dtype": dtype, "bias": bias}
    experts = _log(rng, 2, 128)
    n, k = _log(rng, 256, 4864), 16 * _log(rng, 32, 224)
    if experts > 32:  # many experts are small ones
        n, k = min(n, 2048), min(k, 2048)
    return {"op": op, "rows": _log(rng, 1, 32768), "experts": experts, "n": n, "k": k, "dtype": dtype, "bias": bias}


def _blocks(size):
    return -(-size // BLOCK)


def _spread(scale, rows, cols):
    """A scale per BLOCK columns (``rows`` rows), or per BLOCK x BLOCK (``rows`` None), as one per element."""
    scale = scale.repeat_interleave(BLOCK, dim=-1)[..., :cols]
    return scale if rows is None else scale.repeat_interleave(BLOCK, dim=-2)[..., :rows, :]


def _activations(rows, k, gen, dev):
    """Normal values with a few channels that are much larger, as hidden states have them."""
    x = torch.randn(rows, k, generator=gen, device=dev)
    loud = torch.rand(k, generator=gen, device=dev) < 0.01
    return x * torch.where(loud, 12.0, 1.0)


def _as_codes(x, scale):
    return (x / scale).clamp(-448, 448).to(E4M3)


def _quantized(x):
    """Codes and scales of activations as a program has them in hand before a product."""
    rows, k = x.shape
    full = torch.nn.functional.pad(x, (0, _blocks(k) * BLOCK - k)).view(rows, -1, BLOCK)
    scale = full.abs().amax(-1).clamp_min(1e-12) / 448
    return _as_codes(x, _spread(scale, None, k)), scale


def _weights(shape, gen, dev):
    *lead, n, k = shape
    scale = (torch.rand(*lead, _blocks(n), _blocks(k), generator=gen, device=dev) + 0.5) * (0.06 / 448)
    w = torch.empty(*shape, dtype=E4M3, device=dev)
    for part in (w.view(-1, k) if lead else w).split(8192):  # (codes of a normal distribution whose largest values reach the format's range)
        part.copy_((torch.randn(part.shape, generator=gen, device=dev) * 110).clamp(-448, 448).to(E4M3))
    return w, scale


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
    dt, rows, k = DTYPES[case["dtype"]], case["rows"], case["k"]
    s = {"op": case["op"], "dt": dt, "dtype": NAMES[case["dtype"]], "rows": rows, "k": k, "out": case.get("out")}
    x = _activations(rows, k, gen, dev)
    if case["op"] == "norm":
        s["x"] = (0.3 * x).to(dt)
        s["residual"] = (2.0 * _activations(rows, k, gen, dev)).to(dt)
        s["weight"] = (1.0 + 0.2 * torch.randn(k, generator=gen, device=dev)).to(dt)
        return s
    if case["op"] == "quant":
        s["x"] = x.to(dt)
        return s
    n = case["n"]
    s["n"] = n
    s["q"], s["scale"] = _quantized(x)
    lead = (case["experts"],) if case["op"] == "grouped" else ()
    s["w"], s["w_scale"] = _weights((*lead, n, k), gen, dev)
    s["bias"] = torch.randn(*lead, n, generator=gen, device=dev).to(dt) if case["bias"] else None
    if lead:
        s["offsets"] = _offsets(rows, case["experts"], gen, dev)
        s["most"] = int(s["offsets"].diff().max())  # rows of the largest expert
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------

def _norm_plain(s):
    h = (s["x"].float() + s["residual"].float()).to(s["dt"])  # the residual stream is kept in the model's type, and normalised as kept
    f = h.float()
    y = f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-6) * s["weight"].float()
    if s["out"] == "same":
        return y.to(s["dt"]), h
    if s["out"] == "group":
        return (*_quant_plain(y), h)
    if s["out"] == "fp8":
        scale = y.abs().amax(-1, keepdim=True).clamp_min(1e-12) / 448
        return (y / scale).clamp(-448, 448).to(E4M3), scale, h
    scale = y.abs().amax(-1, keepdim=True).clamp_min(1e-5) / 127
    return (y / scale).round().clamp(-128, 127).to(torch.bfloat16), scale, h


def _quant_plain(x):
    rows, k = x.shape
    full = torch.nn.functional.pad(x.float(), (0, _blocks(k) * BLOCK - k)).view(rows, -1, BLOCK)
    scale = full.abs().amax(-1).clamp_min(1e-12) / 448
    q = (full / scale[..., None]).clamp(-448, 448).to(E4M3)
    return q.view(rows, -1)[:, :k], scale


def _gemm_plain(s):
    a = s["q"].float() * _spread(s["scale"], None, s["k"])
    w = s["w"].float() * _spread(s["w_scale"], s["n"], s["k"])
    y = a @ w.transpose(-1, -2)
    return (y if s["bias"] is None else y + s["bias"].float()).to(s["dt"])


def _grouped_plain(s):
    a = s["q"].float() * _spread(s["scale"], None, s["k"])
    w = s["w"].float() * _spread(s["w_scale"], s["n"], s["k"])
    row = torch.arange(s["rows"], device=a.device)
    expert = torch.searchsorted(s["offsets"][1:], row, right=True)
    place = row - s["offsets"][expert]
    padded = a.new_zeros(w.shape[0], s["most"], s["k"])
    padded[expert, place] = a
    y = torch.bmm(padded, w.transpose(-1, -2))[expert, place]
    return (y if s["bias"] is None else y + s["bias"].float()[expert]).to(s["dt"])


# ---- the framework's calls ---------------------------------------------------------------------------------------

def _norm_own(s):
    from llmqrt_amd import norm
    args = s["x"], s["residual"], s["weight"], 1e-6
    if s["out"] == "same":
        return norm.add_rmsnorm(*args)
    if s["out"] == "group":
        return norm.add_rmsnorm_per_group_quantize(*args)
    if s["out"] == "fp8":
        return norm.add_rmsnorm_per_token_quantize(*args)
    q, scale, h = norm.add_rmsnorm_quantize_activation_per_token_absmax(*args)
    return q.to(torch.bfloat16), scale, h


def _quant_own(s):
    from llmqrt_amd.quantize import per_group_quantize
    return per_group_quantize(s["x"])


def _gemm_own(s):
    from llmqrt_amd.sq_fp8_kernels import f8f8_blockwise
    return f8f8_blockwise(s["q"], s["w"].t(), s["bias"], s["scale"], s["w_scale"], s["dtype"])


def _grouped_own(s):
    from llmqrt_amd.sq_fp8_kernels import f8f8_blockwise_grouped
    return f8f8_blockwise_grouped(s["q"], s["w"], s["bias"], s["scale"], s["w_scale"], s["offsets"], s["dtype"])


def run(state):
    op = state["op"]
    if own:
        return {"norm": _norm_own, "quant": _quant_own, "gemm": _gemm_own, "grouped": _grouped_own}[op](state)
    if op == "quant":
        return _quant_plain(state["x"])
    return {"norm": _norm_plain, "gemm": _gemm_plain, "grouped": _grouped_plain}[op](state)


def work(case):
    rows, k = case["rows"], case["k"]
    groups = rows * _blocks(k)
    if case["op"] == "norm":
        # x, the residual and its sum, the weight, the normalised row and its scales
        out = {"same": 2 * rows * k, "int8": rows * k + 4 * rows, "fp8": rows * k + 4 * rows, "group": rows * k + 4 * groups}[case["out"]]
        return {"bytes": 6 * rows * k + 2 * k + out, "flops": 6 * rows * k}
    if case["op"] == "quant":
        return {"bytes": 3 * rows * k + 4 * groups, "flops": 3 * rows * k}
    n, experts = case["n"], case.get("experts", 1)
    used = min(experts, rows)  # experts without rows are not read
    weights = used * (n * k + 4 * _blocks(n) * _blocks(k) + (2 * n if case["bias"] else 0))
    return {"bytes": rows * k + 4 * groups + weights + 2 * rows * n, "flops": 2 * rows * n * k}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------

def _groups64(y):
    out_q, out_s = torch.empty(y.shape, dtype=torch.float64, device=y.device), []
    for c in range(0, y.shape[1], BLOCK):
        part = y[:, c:c + BLOCK]
        s = torch.maximum(part.abs().max(dim=1, keepdim=True).values, part.new_tensor(1e-12)) / 448.0
        out_q[:, c:c + BLOCK] = (part / s).to(E4M3).double()
        out_s.append(s)
    return out_q, torch.cat(out_s, 1)


def _dequantized64(q, s):
    a = q.double()
    for b in range(s.shape[-1]):
        a[:, b * BLOCK:(b + 1) * BLOCK] *= s[:, b:b + 1].double()
    return a


def _weights64(w, s):
    v = w.double()
    for i in range(s.shape[0]):
        v[i * BLOCK:(i + 1) * BLOCK] *= s[i].double().repeat_interleave(BLOCK)[:v.shape[1]]
    return v


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quant":
        return _groups64(s["x"].double())
    if case["op"] == "norm":
        h = (s["x"].double() + s["residual"].double()).to(s["dt"]).double()
        y = h / torch.sqrt((h * h).sum(1, keepdim=True) / s["k"] + 1e-6) * s["weight"].double()
        if s["out"] == "same":
            return y, h
        if s["out"] == "group":
            return (*_groups64(y), h)
        top = y.abs().max(dim=1, keepdim=True).values
        if s["out"] == "fp8":
            scale = top.clamp_min(1e-12) / 448.0
            return (y / scale).to(E4M3).double(), scale, h
        scale = top.clamp_min(1e-5) / 127.0
        return torch.round(y / scale), scale, h
    a = _dequantized64(s["q"], s["scale"])
    if case["op"] == "gemm":
        y = torch.cat([a @ _weights64(w, ws).t() for w, ws in zip(s["w"].split(4096), s["w_scale"].split(4096 // BLOCK))], 1)
        return y if s["bias"] is None else y + s["bias"].double()
    y = torch.empty(s["rows"], s["n"], dtype=torch.float64, device=a.device)
    at = s["offsets"].tolist()
    for e in range(case["experts"]):
        if at[e + 1] > at[e]:
            y[at[e]:at[e + 1]] = a[at[e]:at[e + 1]] @ _weights64(s["w"][e], s["w_scale"][e]).t()
            if s["bias"] is not None:
                y[at[e]:at[e + 1]] += s["bias"][e].double()
    return y

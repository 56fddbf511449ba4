"""Around products by experts: which experts a token goes to, its rows' way to them in the form that their product takes, and back.

No counterpart in the reference.  The products themselves are ``sq_fp8_kernels.w8a8_int8_linear_per_channel_grouped`` and ``f8f8_blockwise_grouped``; what
``activation.silu_mul`` makes of the first one's rows is what the second one takes.  Nothing here is read back by the host, so a captured run follows the
routing of its replay.  None of these calls has a backward pass.
"""
from __future__ import annotations

import operator

import torch

from . import _abi
from ._native import host
from .quantize import _apart, _as_rows

_SCORING = {"softmax": 0, "sigmoid": 1}
_GROUP_SCORE = {"max": 0, "top2": 1}
MAX_ROUTED_EXPERTS, MAX_DISPATCHED_EXPERTS, MAX_TOP_K, MAX_GROUPS = 1024, 4096, 64, 64
_MAX_ROWS = 0x7fff0000


def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def route_to_experts(logits: torch.Tensor, top_k: int, scoring: str = "softmax", bias: torch.Tensor | None = None, num_groups: int = 1,
                     top_groups: int = 1, group_score: str = "max", renormalize: bool = True, scale: float = 1.0):
    """The ``top_k`` experts of each token and their weights: -> (weights fp32 [.., top_k], experts int32 [.., top_k]), largest first.

    ``logits`` [.., experts] in bf16, fp16 or fp32; s = softmax(logits) or sigmoid(logits) in fp32.  Chosen are the largest c = s + ``bias`` (fp32 [experts], for
    balance; it takes part in the choice alone), ties going to the lowest expert; the weights are their s, divided by their sum if ``renormalize``, times
    ``scale``.  With ``num_groups`` > 1 only the experts of the ``top_groups`` groups of neighbours with the largest score take part: the largest c of the group
    (``group_score`` "max") or the sum of its two largest ("top2"; where masks leave one expert of a group, that one's c alone).
    An expert whose logit or bias is -inf is never chosen; a place that is left over has expert -1 and weight 0, and goes nowhere in the functions below.
    The order is that of the exact scores: the logits' own, or with a bias or "top2" groups that of scores in 64 bits, where those closer than 64 bits tell apart
    are ties.  A token with a NaN (or, for softmax, +inf) among its logits gets experts in range, none twice; its softmax weights are NaN."""
    if scoring in _SCORING and group_score in _GROUP_SCORE:
        y = host().route(logits, bias, top_k, _SCORING[scoring], num_groups, top_groups, _GROUP_SCORE[group_score], bool(renormalize), scale)
        if y is not None:
            return y
    return _route_general(logits, top_k, scoring, bias, num_groups, top_groups, group_score, renormalize, scale)


@torch.no_grad()
def _route_general(logits, top_k, scoring, bias, num_groups, top_groups, group_score, renormalize, scale):
    what = "route_to_experts"
    _check(scoring in _SCORING, f"{what}: scoring must be one of {list(_SCORING)}, got {scoring!r}")
    _check(group_score in _GROUP_SCORE, f"{what}: group_score must be one of {list(_GROUP_SCORE)}, got {group_score!r}")
    _check(isinstance(logits, torch.Tensor) and logits.is_cuda and logits.dim() >= 1, f"{what}: logits must be a GPU tensor [.., experts]")
    _check(logits.dtype in (torch.bfloat16, torch.float16, torch.float32), f"{what}: logits must be bf16, fp16 or fp32, got {logits.dtype}")
    E, top_k, num_groups, top_groups = logits.shape[-1], operator.index(top_k), operator.index(num_groups), operator.index(top_groups)
    _check(1 <= E <= MAX_ROUTED_EXPERTS, f"{what}: 1 to {MAX_ROUTED_EXPERTS} experts, got {E}")
    _check(1 <= num_groups <= MAX_GROUPS and E % num_groups == 0, f"{what}: num_groups must divide the experts, at most {MAX_GROUPS}, got {num_groups}")
    _check(1 <= top_groups <= num_groups, f"{what}: top_groups must be 1 to num_groups, got {top_groups}")
    _check(1 <= top_k <= min(MAX_TOP_K, E // num_groups * top_groups),
           f"{what}: top_k must be 1 to {MAX_TOP_K} and at most the experts of the groups that take part, got {top_k}")
    if bias is not None:
        _check(isinstance(bias, torch.Tensor) and bias.dtype == torch.float32 and bias.device == logits.device and tuple(bias.shape) == (E,),
               f"{what}: bias must be fp32 [experts] on the GPU of the logits")
        bias = bias.detach().contiguous()
    dev = logits.device
    rows = logits.detach().reshape(-1, E)
    if rows.stride(1) != 1 or (rows.shape[0] > 1 and rows.stride(0) < E):
        rows = rows.contiguous()
    T = rows.shape[0]
    _check(T <= _MAX_ROWS // top_k, f"{what}: too many tokens")
    weights = torch.empty((*logits.shape[:-1], top_k), dtype=torch.float32, device=dev)
    ids = torch.empty((*logits.shape[:-1], top_k), dtype=torch.int32, device=dev)
    if T:
        with torch.cuda.device(dev):
            _abi.check(_abi.lib().llmq_route_experts(
                _SCORING[scoring], rows.data_ptr(), _abi.dtype_code(rows.dtype), T, E, rows.stride(0) if T > 1 else E, _abi.ptr(bias), num_groups, top_groups,
                _GROUP_SCORE[group_score], top_k, int(bool(renormalize)), float(scale), weights.data_ptr(), ids.data_ptr(), _abi.stream_of(rows)), what)
    return weights, ids


# outputs of llmq_dispatch_experts
_SAME, _I8_TOKEN, _FP8_GROUP = 0, 1, 3


@torch.no_grad()
def _dispatch_general(x, experts, num_experts, first_expert, out):
    what = "dispatch to experts"
    num_experts, first_expert = operator.index(num_experts), operator.index(first_expert)
    _check(1 <= num_experts <= MAX_DISPATCHED_EXPERTS, f"{what}: 1 to {MAX_DISPATCHED_EXPERTS} experts, got {num_experts}")
    _check(0 <= first_expert <= 0x7fff0000, f"{what}: first_expert must not be negative, got {first_expert}")
    _check(x.dim() >= 1 and experts.dim() == x.dim() and experts.shape[:-1] == x.shape[:-1] and experts.device == x.device,
           f"{what}: experts must be [.., top_k] for activations [.., K], on their GPU")
    _check(experts.dtype in (torch.int32, torch.int64), f"{what}: experts must be int32 or int64, got {experts.dtype}")
    top = experts.shape[-1]
    _check(1 <= top <= MAX_TOP_K, f"{what}: 1 to {MAX_TOP_K} experts per token, got {top}")
    _check(x.shape[-1] > 0, f"{what}: the activations have no channels")
    rows = _apart(_as_rows(x.detach()))
    T, K = rows.shape
    _check(T <= _MAX_ROWS // top, f"{what}: too many tokens")
    ids = experts.detach().reshape(-1, top)
    if ids.dtype != torch.int32:
        ids = ids.clamp(-1, 0x7fffffff).to(torch.int32)  # (what does not fit goes nowhere, before and after)
    ids = ids.contiguous()
    dev, n = x.device, T * top
    scale = None
    if out == _SAME:
        sorted_rows = torch.empty((n, K), dtype=x.dtype, device=dev)
    else:
        sorted_rows = torch.empty((n, K), dtype=torch.int8 if out == _I8_TOKEN else torch.float8_e4m3fn, device=dev)
        scale = torch.empty((n, 1 if out == _I8_TOKEN else (K + 127) // 128), dtype=torch.float32, device=dev)
    offsets = torch.empty(num_experts + 1, dtype=torch.int32, device=dev)
    places = torch.empty(experts.shape, dtype=torch.int32, device=dev)
    ws = torch.empty(_abi.lib().llmq_dispatch_experts_workspace_bytes(T, top, num_experts), dtype=torch.uint8, device=dev)
    with torch.cuda.device(dev):
        _abi.check(_abi.lib().llmq_dispatch_experts(
            out, rows.data_ptr(), _abi.dtype_code(rows.dtype), T, K, rows.stride(0) if T > 1 else K, ids.data_ptr(), top, first_expert, num_experts,
            sorted_rows.data_ptr(), _abi.ptr(scale), offsets.data_ptr(), places.data_ptr(),
            ws.data_ptr() or None, ws.numel(), _abi.stream_of(rows)), "llmq_dispatch_experts")
    return (sorted_rows, offsets, places) if scale is None else (sorted_rows, scale, offsets, places)


def dispatch_to_experts(x: torch.Tensor, experts: torch.Tensor, num_experts: int, first_expert: int = 0):
    """A row for each of a token's experts, sorted by expert and within an expert by token: -> (rows [tokens * top_k, K], offsets int32 [num_experts + 1],
    places int32 [.., top_k]).

    ``x`` [.., K] in bf16 or fp16; ``experts`` int32 or int64 [.., top_k], counted from ``first_expert`` (of a GPU that holds a part of the experts); ids outside
    its ``num_experts`` go nowhere.  Rows offsets[e] .. offsets[e + 1] - 1 belong to expert e; those from offsets[num_experts] on are not written.
    ``places`` says where a token's copies are (-1: nowhere), for ``combine_from_experts``."""
    y = host().dispatch(x, experts, num_experts, first_expert, _SAME)
    return _dispatch_general(x, experts, num_experts, first_expert, _SAME) if y is None else y


def dispatch_quantize_activation_per_token_absmax(x: torch.Tensor, experts: torch.Tensor, num_experts: int, first_expert: int = 0):
    """dispatch_to_experts with rows in int8, the bits of ``quantize.quantize_activation_per_token_absmax_f32``, quantized once per token:
    -> (int8 rows, fp32 scales [rows, 1], offsets, places)."""
    y = host().dispatch(x, experts, num_experts, first_expert, _I8_TOKEN)
    return _dispatch_general(x, experts, num_experts, first_expert, _I8_TOKEN) if y is None else y


def dispatch_per_group_quantize(x: torch.Tensor, experts: torch.Tensor, num_experts: int, first_expert: int = 0):
    """dispatch_to_experts with rows in e4m3fn, the bits of ``quantize.per_group_quantize``, quantized once per token:
    -> (codes, fp32 scales [rows, ceil(K / 128)], offsets, places)."""
    y = host().dispatch(x, experts, num_experts, first_expert, _FP8_GROUP)
    return _dispatch_general(x, experts, num_experts, first_expert, _FP8_GROUP) if y is None else y


def combine_from_experts(y: torch.Tensor, places: torch.Tensor, weights: torch.Tensor, shared: torch.Tensor | None = None) -> torch.Tensor:
    """out[t] = sum_j weights[t, j] * y[places[t, j]] (+ shared[t]), fp32 sums in the order of j, rounded once: -> [.., N] in y's type.

    ``y`` [rows, N] in bf16 or fp16; ``places`` int32 [.., top_k] (-1, or any other that is no row: adds nothing); ``weights`` [.., top_k] floating point;
    ``shared`` [.., N] in y's type: what every token adds, the output of an expert that all share."""
    out = host().combine(y, places, weights, shared)
    return _combine_general(y, places, weights, shared) if out is None else out


@torch.no_grad()
def _combine_general(y, places, weights, shared):
    what = "combine_from_experts"
    _check(y.is_cuda and y.dim() == 2 and y.dtype in (torch.bfloat16, torch.float16), f"{what}: y must be a GPU tensor [rows, N] in bf16 or fp16")
    _check(places.dtype == torch.int32 and places.dim() >= 1 and places.device == y.device, f"{what}: places must be int32 [.., top_k] on the GPU of y")
    _check(weights.is_floating_point() and weights.shape == places.shape and weights.device == y.device,
           f"{what}: weights must be floating point and as many as places, on the GPU of y")
    top, N = places.shape[-1], y.shape[1]
    _check(1 <= top <= MAX_TOP_K, f"{what}: 1 to {MAX_TOP_K} experts per token, got {top}")
    _check(N % 8 == 0, f"{what}: the last dimension must be a multiple of 8")
    lead = places.shape[:-1]
    out = torch.empty((*lead, N), dtype=y.dtype, device=y.device)
    if shared is not None:
        _check(shared.dtype == y.dtype and shared.device == y.device and tuple(shared.shape) == (*lead, N),
               f"{what}: shared must be [.., N] in the type and on the GPU of y")
    T = out.numel() // N if N else 0
    if T == 0:
        return out
    _check(T <= _MAX_ROWS // top, f"{what}: too many tokens")
    rows = _apart(_as_rows(y.detach())) if y.numel() else y
    add = None if shared is None else _apart(_as_rows(shared.detach()))
    p, w = places.contiguous(), weights.detach().to(torch.float32).contiguous()
    with torch.cuda.device(y.device):
        _abi.check(_abi.lib().llmq_combine_experts(
            rows.data_ptr() or None, _abi.dtype_code(y.dtype), rows.shape[0], N, rows.stride(0) if rows.shape[0] > 1 else N, p.data_ptr(), w.data_ptr(), T, top,
            _abi.ptr(add), add.stride(0) if add is not None and T > 1 else N, out.data_ptr(), _abi.stream_of(y)), "llmq_combine_experts")
    return out

"""RMSNorm, alone or fused with the per-token activation quantizer of the Linear that follows it.

``RMSNorm`` has the constructor and forward of the reference module
(nn_models/modules/nonlinear/norm.py:4-16).  The fused functions replace the pair
"norm, then quantize inside the next Linear" (nn_models/modules/nonlinear/block.py:68,76 followed by
linear_sq.py:55-65 or linear_fp8.py:40-63) by one kernel that reads the activations once.
"""
from __future__ import annotations

import torch
from torch import nn

from . import _abi
from ._native import host
from .quantize import _apart, _as_rows


def _check_weight(x: torch.Tensor, weight: torch.Tensor) -> torch.Tensor:
    if weight.dtype != x.dtype or weight.device != x.device or weight.numel() != x.shape[-1]:
        raise RuntimeError("RMSNorm weight must be a [K] tensor with the dtype and device of the activations")
    return weight.contiguous()


@torch.no_grad()
def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, _inv_dump: torch.Tensor | None = None):
    """weight * (fp32(x) * rsqrt(mean(fp32(x)^2) + eps)).to(x.dtype), one kernel."""
    rows = _as_rows(x)
    w = _check_weight(rows, weight)
    M, K = rows.shape
    y = torch.empty((M, K), dtype=rows.dtype, device=rows.device)
    if M:
        _abi.check(_abi.lib().llmq_rmsnorm(rows.data_ptr(), _abi.dtype_code(rows.dtype), M, K,
                                           rows.stride(0) if M > 1 else K, w.data_ptr(), float(eps), y.data_ptr(),
                                           _abi.ptr(_inv_dump), _abi.stream_of(rows)), "llmq_rmsnorm")
    return y.view(x.shape)


def _fused(x, weight, eps, fp8, scale_dtype, return_normed, inv_dump):
    rows = _as_rows(x)
    w = _check_weight(rows, weight)
    M, K = rows.shape
    dev = rows.device
    q = torch.empty((M, K), dtype=torch.float8_e4m3fn if fp8 else torch.int8, device=dev)
    scale = torch.empty((M, 1), dtype=torch.float32 if fp8 else scale_dtype, device=dev)
    y = torch.empty((M, K), dtype=rows.dtype, device=dev) if return_normed else None
    if M:
        L = _abi.lib()
        ldx = rows.stride(0) if M > 1 else K
        if fp8:
            _abi.check(L.llmq_rmsnorm_quant_fp8_per_token(
                rows.data_ptr(), _abi.dtype_code(rows.dtype), M, K, ldx, w.data_ptr(), float(eps), _abi.ptr(y),
                q.data_ptr(), scale.data_ptr(), _abi.ptr(inv_dump), _abi.stream_of(rows)),
                "llmq_rmsnorm_quant_fp8_per_token")
        else:
            _abi.check(L.llmq_rmsnorm_quant_i8_per_token(
                rows.data_ptr(), _abi.dtype_code(rows.dtype), M, K, ldx, w.data_ptr(), float(eps), _abi.ptr(y),
                q.data_ptr(), scale.data_ptr(), _abi.dtype_code(scale_dtype), _abi.ptr(inv_dump),
                _abi.stream_of(rows)), "llmq_rmsnorm_quant_i8_per_token")
    out = (q.view(x.shape), scale.view(*x.shape[:-1], 1))
    return out + (y.view(x.shape),) if return_normed else out


@torch.no_grad()
def rmsnorm_quantize_activation_per_token_absmax(x, weight, eps: float = 1e-6, scale_dtype=None,
                                                 return_normed: bool = False, _inv_dump=None):
    """RMSNorm followed by quantize_activation_per_token_absmax, fused.

    -> (int8 like x, scales [.., 1] in x.dtype or ``scale_dtype``=torch.float32[, normalised activations])."""
    return _fused(x, weight, eps, False, scale_dtype or x.dtype, return_normed, _inv_dump)


@torch.no_grad()
def rmsnorm_per_token_quantize(x, weight, eps: float = 1e-6, return_normed: bool = False, _inv_dump=None):
    """RMSNorm followed by per_token_quantize (e4m3fn, fp32 scales), fused."""
    return _fused(x, weight, eps, True, torch.float32, return_normed, _inv_dump)


# outputs of llmq_add_rmsnorm
_SAME, _I8_TOKEN, _FP8_TOKEN, _FP8_GROUP = range(4)


def _same_rows(t: torch.Tensor, x: torch.Tensor, what: str) -> torch.Tensor:
    if t.dtype != x.dtype or t.device != x.device or t.shape != x.shape:
        raise RuntimeError(f"{what} must have the shape, dtype and device of the activations")
    return _apart(_as_rows(t))


def _partly_over(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two sets of rows of one shape and type share elements without being the same (different strides: whether their ranges meet)."""
    if a.data_ptr() < b.data_ptr():
        a, b = b, a
    M, K = a.shape
    apart = (a.data_ptr() - b.data_ptr()) // a.element_size()
    if M == 1:
        return 0 < apart < K
    ld = b.stride(0)
    if a.stride(0) != ld:
        return apart < (M - 1) * ld + K
    rows, columns = divmod(apart, ld)  # how many a lies behind b
    return apart > 0 and (columns < K and rows < M or ld - columns < K and rows + 1 < M)


def _add_norm(x, residual, weight, eps, out, return_normed=False, inplace=False):
    y = host().add_norm(x, residual, weight, eps, out, return_normed, inplace)
    if y is not None:
        return y
    if inplace and residual is not None:
        _abi.check_writable(residual, "the residual")
    return _add_norm_general(x, residual, weight, eps, out, return_normed, inplace)


@torch.no_grad()
def _add_norm_general(x, residual, weight, eps, out, return_normed, inplace):
    if inplace and residual is None:
        raise RuntimeError("inplace needs a residual")
    rows = _apart(_as_rows(x))
    w = _check_weight(rows, weight)
    M, K = rows.shape
    dev = rows.device
    res = h = None
    if residual is not None:
        res = _same_rows(residual, x, "the residual")
        if not inplace:
            h = torch.empty((M, K), dtype=rows.dtype, device=dev)
        elif res.data_ptr() != residual.data_ptr():
            raise RuntimeError("a residual that is updated in place needs rows of one stride that is a multiple of 16 bytes, 16-byte aligned")
        elif M and _partly_over(rows, res):
            raise RuntimeError("a residual that is updated in place must be the activations or lie apart from them")
        else:
            h = res
    groups = (K + 127) // 128
    q = scale = y = None
    if out != _SAME:
        q = torch.empty((M, K), dtype=torch.int8 if out == _I8_TOKEN else torch.float8_e4m3fn, device=dev)
        scale = torch.empty((M, groups if out == _FP8_GROUP else 1), dtype=torch.float32, device=dev)
    if out == _SAME or return_normed:
        y = torch.empty((M, K), dtype=rows.dtype, device=dev)
    if M:
        with torch.cuda.device(dev):
            _abi.check(_abi.lib().llmq_add_rmsnorm(
                out, rows.data_ptr(), _abi.dtype_code(rows.dtype), M, K, rows.stride(0) if M > 1 else K, _abi.ptr(res),
                res.stride(0) if res is not None and M > 1 else K, _abi.ptr(h), h.stride(0) if h is not None and M > 1 else K, w.data_ptr(), float(eps),
                _abi.ptr(y), _abi.ptr(q), _abi.ptr(scale), _abi.stream_of(rows)), "llmq_add_rmsnorm")
        if inplace:
            torch.autograd.graph.increment_version(residual)
    result = [] if q is None else [q.view(x.shape), scale.view(*x.shape[:-1], scale.shape[-1])]
    if y is not None:
        result.append(y.view(x.shape))
    if h is not None:
        result.append(residual if inplace else h.view(x.shape))
    return tuple(result)


def add_rmsnorm(x, residual, weight, eps: float = 1e-6, inplace: bool = False):
    """The residual's addition and RMSNorm in one pass: h = (x + residual).to(x.dtype), y = (h * rsqrt(mean(h^2) + eps) * weight) in fp32,
    rounded once to x.dtype.  -> (y, h).  ``inplace`` writes h over the residual (and returns it), as torch's in-place operations do: its version is
    raised, and a residual that requires grad is refused outside no_grad.  There the residual may be x itself, and may not overlap it otherwise."""
    if residual is None:
        raise RuntimeError("add_rmsnorm needs a residual (rmsnorm is the form without)")
    return _add_norm(x, residual, weight, eps, _SAME, inplace=inplace)


def add_rmsnorm_quantize_activation_per_token_absmax(x, residual, weight, eps: float = 1e-6, return_normed: bool = False, inplace: bool = False):
    """add_rmsnorm with y quantized to int8 per token: -> (int8 like x, fp32 scales [.., 1][, y], h).  scale = max(absmax, 1e-5) / 127.

    y is quantized as it is in fp32.  (The pair without a residual, rmsnorm_quantize_activation_per_token_absmax, rounds the normalised
    row, y, scale and quotients to x.dtype, as its reference does.)"""
    if residual is None:
        raise RuntimeError("add_rmsnorm_quantize_activation_per_token_absmax needs a residual")
    return _add_norm(x, residual, weight, eps, _I8_TOKEN, return_normed, inplace)


def add_rmsnorm_per_token_quantize(x, residual, weight, eps: float = 1e-6, return_normed: bool = False, inplace: bool = False):
    """add_rmsnorm with y quantized to e4m3fn per token: -> (codes, fp32 scales [.., 1][, y], h).  scale = max(absmax, 1e-12) / 448."""
    if residual is None:
        raise RuntimeError("add_rmsnorm_per_token_quantize needs a residual")
    return _add_norm(x, residual, weight, eps, _FP8_TOKEN, return_normed, inplace)


def add_rmsnorm_per_group_quantize(x, residual, weight, eps: float = 1e-6, return_normed: bool = False, inplace: bool = False):
    """add_rmsnorm with y quantized to e4m3fn per token and 128 channels, for a block-scaled Linear: -> (codes, fp32 scales
    [.., ceil(K / 128)][, y], h)."""
    if residual is None:
        raise RuntimeError("add_rmsnorm_per_group_quantize needs a residual (rmsnorm_per_group_quantize is the form without)")
    return _add_norm(x, residual, weight, eps, _FP8_GROUP, return_normed, inplace)


def rmsnorm_per_group_quantize(x, weight, eps: float = 1e-6, return_normed: bool = False):
    """RMSNorm with an output in e4m3fn per token and 128 channels, without a residual: -> (codes, fp32 scales [.., ceil(K / 128)][, y])."""
    return _add_norm(x, None, weight, eps, _FP8_GROUP, return_normed)


class RMSNorm(nn.Module):
    """Drop-in for the reference RMSNorm: same constructor (a ready weight tensor, eps) and forward."""

    def __init__(self, weight, eps=1e-6):
        super().__init__()
        self.weight = weight
        self.variance_epsilon = eps

    def forward(self, hidden_states):
        y = host().rmsnorm(hidden_states, self.weight, self.variance_epsilon)
        return rmsnorm(hidden_states, self.weight, self.variance_epsilon) if y is None else y

    def forward_add(self, hidden_states, residual, quantize: str | None = None, return_normed: bool = False, inplace: bool = False):
        """The residual's addition in front of the norm, in the same pass: add_rmsnorm (``quantize`` None) or its form for the Linear that follows:
        "int8" (SqW8A8BBF16OBF16PerChannel), "fp8" (FP8DynamicLinear per token), "fp8_block" (FP8BlockLinear)."""
        kinds = {None: _SAME, "int8": _I8_TOKEN, "fp8": _FP8_TOKEN, "fp8_block": _FP8_GROUP}
        if quantize not in kinds or residual is None:
            raise RuntimeError(f"forward_add needs a residual, and quantize one of {list(kinds)}")
        return _add_norm(hidden_states, residual, self.weight, self.variance_epsilon, kinds[quantize], return_normed and quantize is not None, inplace)

    def forward_quantized(self, hidden_states, fp8: bool = False, return_normed: bool = False):
        """Normalise and quantize per token in one pass, for a W8A8 / FP8 Linear that accepts (q, scale)."""
        if not return_normed:
            out = host().rmsnorm_quant(hidden_states, self.weight, self.variance_epsilon, fp8)
            if out is not None:
                return out
        if fp8:
            return rmsnorm_per_token_quantize(hidden_states, self.weight, self.variance_epsilon, return_normed)
        return rmsnorm_quantize_activation_per_token_absmax(hidden_states, self.weight, self.variance_epsilon,
                                                            torch.float32, return_normed)

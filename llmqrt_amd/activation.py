"""The gated activation between two Linear modules, silu(gate) * up, alone or with the quantizer of the second one in the same pass.

No counterpart in the reference, whose modules call torch's.  ``x`` [.., 2 N] holds the gates in its first N channels and what they scale in the others, as the
output of gate and up projections joined by ``fused_utils.fuse_linears`` does.  Arithmetic is fp32 from x to the output's one rounding or its codes.  None of
these calls has a backward pass.
"""
from __future__ import annotations

import torch

from . import _abi
from ._native import host
from .quantize import _apart, _as_rows

# outputs of llmq_silu_mul
_SAME, _I8_TOKEN, _FP8_TOKEN, _FP8_GROUP = range(4)


@torch.no_grad()
def _silu_mul_general(x, out):
    if x.dim() < 1 or x.shape[-1] % 16:
        raise RuntimeError("silu_mul needs gates and factors side by side, a multiple of 8 channels of each")
    rows = _apart(_as_rows(x.detach()))
    M, N = rows.shape[0], rows.shape[1] // 2
    dev = x.device
    lead = x.shape[:-1]
    groups = (N + 127) // 128
    scale = None
    if out == _SAME:
        y = torch.empty((*lead, N), dtype=x.dtype, device=dev)
    else:
        y = torch.empty((*lead, N), dtype=torch.int8 if out == _I8_TOKEN else torch.float8_e4m3fn, device=dev)
        scale = torch.empty((*lead, groups if out == _FP8_GROUP else 1), dtype=torch.float32, device=dev)
    if M and N:
        with torch.cuda.device(dev):
            _abi.check(_abi.lib().llmq_silu_mul(out, rows.data_ptr(), _abi.dtype_code(rows.dtype), M, N, rows.stride(0) if M > 1 else 2 * N, y.data_ptr(),
                                                _abi.ptr(scale), _abi.stream_of(rows)), "llmq_silu_mul")
    return y if scale is None else (y, scale)


def silu_mul(x: torch.Tensor) -> torch.Tensor:
    """silu(x[.., :N]) * x[.., N:], rounded once to x's type: -> [.., N]."""
    y = host().silu_mul(x, _SAME)
    return _silu_mul_general(x, _SAME) if y is None else y


def silu_mul_quantize_activation_per_token_absmax(x: torch.Tensor):
    """silu_mul quantized to int8 per token, as it is in fp32: -> (int8 [.., N], fp32 scales [.., 1]).  scale = max(absmax, 1e-5) / 127."""
    y = host().silu_mul(x, _I8_TOKEN)
    return _silu_mul_general(x, _I8_TOKEN) if y is None else y


def silu_mul_per_token_quantize(x: torch.Tensor):
    """silu_mul quantized to e4m3fn per token: -> (codes [.., N], fp32 scales [.., 1]).  scale = max(absmax, 1e-12) / 448."""
    y = host().silu_mul(x, _FP8_TOKEN)
    return _silu_mul_general(x, _FP8_TOKEN) if y is None else y


def silu_mul_per_group_quantize(x: torch.Tensor):
    """silu_mul quantized to e4m3fn per token and 128 channels, for a block-scaled Linear: -> (codes [.., N], fp32 scales [.., ceil(N / 128)])."""
    y = host().silu_mul(x, _FP8_GROUP)
    return _silu_mul_general(x, _FP8_GROUP) if y is None else y

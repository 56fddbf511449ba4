"""Block-scaled FP8 (OCP e4m3fn) Linear modules: one scale per token and 128 channels of the activations, formed in the forward pass, and one per
128 x 128 block of the weight.

The reference refuses group-wise FP8 (``group_size`` must be 0, nn_models/modules/linear/linear_fp8.py:160-163); buffer names follow its FP8
modules.  The weight is kept in e4m3fn, as checkpoints of this format store it (checkpoint.py reads their names).
"""
from __future__ import annotations

import torch

from .._native import host
from ..quantize import per_group_quantize, quantize_weight_per_block
from ..sq_fp8_kernels import f8f8_blockwise, f8f8_blockwise_grouped
from .linear_base import LinearBase

__all__ = ["FP8BlockLinear", "FP8BlockGroupedLinear"]

BLOCK = 128
_NAMES = {torch.bfloat16: "bfloat16", torch.float16: "float16"}


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


def _check_plain(module) -> None:
    """A module whose weight is codes has scales beside it, which a quantizer of the codes would lose."""
    if getattr(module, "weight_scale", None) is not None or module.weight.dtype.itemsize < 2:
        raise RuntimeError(f"{type(module).__name__} is quantized already: a weight to be quantized must be a floating-point one without scales")


class _FP8BlockBase(LinearBase):
    def _init_block(self, lead, in_features, out_features, bias, dev, dtype):
        if in_features % 16:
            raise RuntimeError(f"block-scaled fp8 needs in_features that are a multiple of 16, got {in_features}")
        if dtype not in _NAMES:
            raise RuntimeError(f"block-scaled fp8 modules work in bf16 or fp16, got {dtype}")
        self.dtype = dtype
        self.in_features = in_features
        self.out_features = out_features
        self.group_size = BLOCK
        self.register_buffer("weight", torch.zeros((*lead, out_features, in_features), dtype=torch.float8_e4m3fn, device=dev))
        self.register_buffer("weight_scale", torch.ones((*lead, _blocks(out_features), _blocks(in_features)), dtype=torch.float32, device=dev))
        self.register_buffer("bias", torch.zeros((*lead, out_features), dtype=dtype, device=dev) if bias else None)

    def _apply(self, fn, *args, **kwargs):
        kept = self.weight, self.weight_scale

        def moved(t):  # .half() and .bfloat16() are for the bias and the outputs: codes and scales keep their types
            u = fn(t)
            return t.to(u.device) if u.dtype != t.dtype and any(t is k for k in kept) else u
        like = fn(torch.empty(0, dtype=self.dtype, device=self.weight.device))  # the type that a module without a bias is converted to
        out = super()._apply(moved, *args, **kwargs)
        if like.dtype in _NAMES:
            self.dtype = like.dtype
        return out

    @torch.no_grad()
    def set_weight(self, weight, bias=None):
        """Quantize a floating-point weight (and take a bias) of the module's shape."""
        if weight.shape != self.weight.shape or (bias is not None) != (self.bias is not None):
            raise RuntimeError(f"weight must be {list(self.weight.shape)}, with a bias if the module has one")
        if weight.dtype.itemsize < 2 or (bias is not None and bias.shape != self.bias.shape):
            raise RuntimeError("a weight to be quantized must have 16 bits or more, and a bias the module's shape")
        q, s = quantize_weight_per_block(weight.to(self.weight.device))
        self.weight.copy_(q)
        self.weight_scale.copy_(s)
        if bias is not None:
            self.bias.copy_(bias)

    def extra_repr(self):
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, dtype={self.dtype}"


class FP8BlockLinear(_FP8BlockBase):
    def __init__(self, in_features, out_features, bias, dev="cuda:0", dtype=torch.bfloat16):
        super().__init__()
        self._init_block((), in_features, out_features, bias, dev, dtype)

    @classmethod
    def from_linear(cls, module: torch.nn.Linear, w_bit=8, group_size=BLOCK, init_only=True, dtype=torch.bfloat16, per_tensor=False):
        if w_bit != 8 or group_size != BLOCK:
            raise RuntimeError(f"block-scaled fp8 has 8 bits and groups of {BLOCK}, got {w_bit} and {group_size}")
        if not init_only:
            _check_plain(module)
        lin = cls(module.in_features, module.out_features, module.bias is not None, module.weight.device, dtype)
        if not init_only:
            lin.set_weight(module.weight.data, None if module.bias is None else module.bias.data)
        return lin

    def forward(self, x):
        b = self._buffers
        y = host().fp8_block_linear(x, b["weight"], b["weight_scale"], b["bias"])
        return self._forward_general(x) if y is None else y

    @torch.no_grad()
    def _forward_general(self, x):
        assert x.device == self.weight.device, "when fp8 linear fwd, input and qweight must be same device!"
        if x.shape[-1] != self.in_features:
            raise RuntimeError(f"the input has {x.shape[-1]} channels, the module {self.in_features}")
        out_shape = (*x.shape[:-1], self.out_features)
        if x.numel() == 0:
            return torch.empty(out_shape, dtype=x.dtype, device=x.device)
        q, s = per_group_quantize(x.reshape(-1, self.in_features))
        return f8f8_blockwise(q, self.weight.t(), self.bias, s, self.weight_scale, _NAMES[x.dtype]).view(out_shape)

    def forward_quantized(self, qinput, x_scale):
        """Forward for activations already quantized per token and 128 channels (e4m3fn qinput [.., K], fp32 scales [.., ceil(K / 128)] or
        [tokens, ceil(K / 128)]), e.g. by the fused norm; the result is in the module's dtype."""
        b = self._buffers
        y = host().fp8_block(qinput, x_scale, b["weight"], b["weight_scale"], b["bias"], self.dtype)
        if y is None:
            if x_scale.dim() != 2 and x_scale.shape[:-1] != qinput.shape[:-1]:
                raise RuntimeError("x_scale must hold one scale per token and 128 channels, [.., ceil(K / 128)]")
            y = f8f8_blockwise(qinput.reshape(-1, qinput.shape[-1]), self.weight.t(), self.bias, x_scale.reshape(-1, x_scale.shape[-1]), self.weight_scale,
                               _NAMES[self.dtype]).view(*qinput.shape[:-1], self.out_features)
        return y


class FP8BlockGroupedLinear(_FP8BlockBase):
    """The Linear modules of several experts in one: rows sorted by expert, each part with its expert's weight."""

    def __init__(self, num_experts, in_features, out_features, bias=False, dev="cuda:0", dtype=torch.bfloat16):
        super().__init__()
        self.num_experts = num_experts
        self._init_block((num_experts,), in_features, out_features, bias, dev, dtype)

    @classmethod
    def from_linears(cls, modules, dtype=None):
        """The experts' nn.Linear modules, whose weights are quantized here (``dtype`` of the outputs: bf16 unless given), or their FP8BlockLinear
        modules, as a checkpoint fills them, whose codes and scales are taken as they are (``dtype``: theirs unless given)."""
        modules = list(modules)
        if not modules:
            raise RuntimeError("from_linears needs the modules of one expert or more")
        first = modules[0]
        codes = isinstance(first, FP8BlockLinear)
        if any(isinstance(m, FP8BlockLinear) != codes or (codes and dtype is None and m.dtype != first.dtype) for m in modules):
            raise RuntimeError("the experts must be modules of one kind and type")
        if any(m.weight.shape != first.weight.shape or (m.bias is None) != (first.bias is None) for m in modules):
            raise RuntimeError("the experts must have the same shape, and all or none of them a bias")
        if not codes:
            for m in modules:
                _check_plain(m)
        lin = cls(len(modules), first.in_features, first.out_features, first.bias is not None, first.weight.device,
                  dtype or (first.dtype if codes else torch.bfloat16))
        if codes:
            for e, m in enumerate(modules):
                for name in ("weight", "weight_scale", "bias"):
                    if m._buffers[name] is not None:
                        lin._buffers[name][e].copy_(m._buffers[name])
            return lin
        lin.set_weight(torch.stack([m.weight.data for m in modules]), None if first.bias is None else torch.stack([m.bias.data for m in modules]))
        return lin

    def forward(self, x, offsets, out=None):
        """``x`` [M, K], sorted by expert; ``offsets``: int32 [num_experts + 1] on the GPU, the experts' first rows and the end of the last.  Rows of
        no expert are not written (sq_fp8_kernels.f8f8_blockwise_grouped)."""
        b = self._buffers
        y = host().fp8_block_grouped(x, None, b["weight"], b["weight_scale"], b["bias"], offsets, x.dtype, out)
        if y is not None:
            return y
        if x.dim() != 2 or x.shape[1] != self.in_features or x.dtype not in _NAMES:
            raise RuntimeError(f"the input must be [rows, {self.in_features}] in bf16 or fp16")
        q, s = per_group_quantize(x)
        return f8f8_blockwise_grouped(q, self.weight, self.bias, s, self.weight_scale, offsets, _NAMES[x.dtype], out)

    def forward_quantized(self, qinput, x_scale, offsets, out=None):
        """The same for rows already quantized per token and 128 channels; the result is in the module's dtype."""
        return f8f8_blockwise_grouped(qinput, self.weight, self.bias, x_scale, self.weight_scale, offsets, _NAMES[self.dtype], out)

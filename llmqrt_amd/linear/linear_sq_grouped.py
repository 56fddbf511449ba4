"""SmoothQuant W8A8 Linear modules of several experts in one: int8 weights with a scale per expert and output channel, activation scales per row.

The reference has no experts; buffer names follow its W8A8 modules (nn_models/modules/linear/linear_sq.py:155-214)."""
from __future__ import annotations

import torch

from ..quantize import quantize_activation_per_token_absmax_f32
from ..sq_fp8_kernels import w8a8_int8_linear_per_channel_grouped
from .linear_base import LinearBase
from .linear_sq import SqW8A8BBF16OBF16PerChannel

__all__ = ["SqW8A8GroupedLinear"]

_NAMES = {torch.bfloat16: "bfloat16", torch.float16: "float16"}


class SqW8A8GroupedLinear(LinearBase):
    """The Linear modules of several experts: rows sorted by expert, each part with its expert's weight."""

    def __init__(self, num_experts, in_features, out_features, bias=False, dev="cuda:0", dtype=torch.bfloat16):
        super().__init__()
        if in_features % 16 or in_features >= 1 << 17:
            raise RuntimeError(f"W8A8 by experts needs in_features that are a multiple of 16 below 131072, got {in_features}")
        if dtype not in _NAMES:
            raise RuntimeError(f"W8A8 modules by experts work in bf16 or fp16, got {dtype}")
        self.num_experts, self.in_features, self.out_features, self.dtype = num_experts, in_features, out_features, dtype
        self.register_buffer("qweight", torch.zeros((num_experts, out_features, in_features), dtype=torch.int8, device=dev))
        self.register_buffer("weight_scale", torch.ones((num_experts, out_features), dtype=torch.float32, device=dev))
        self.register_buffer("bias", torch.zeros((num_experts, out_features), dtype=dtype, device=dev) if bias else None)

    def _apply(self, fn, *args, **kwargs):
        kept = self.weight_scale

        def moved(t):  # .half() and .bfloat16() are for the bias and the outputs: scales stay fp32
            u = fn(t)
            return t.to(u.device) if t is kept and u.dtype != t.dtype else u
        like = fn(torch.empty(0, dtype=self.dtype, device=self.qweight.device))  # the type that a module without a bias is converted to
        out = super()._apply(moved, *args, **kwargs)
        if like.dtype in _NAMES:
            self.dtype = like.dtype
        return out

    @classmethod
    @torch.no_grad()
    def from_linears(cls, modules, dtype=None):
        """The experts' nn.Linear modules, whose weights are quantized here per output channel (``dtype`` of the outputs: bf16 unless given), or their
        SqW8A8BBF16OBF16PerChannel modules, whose codes and scales are taken as they are (``dtype``: theirs unless given)."""
        modules = list(modules)
        if not modules:
            raise RuntimeError("from_linears needs the modules of one expert or more")
        first = modules[0]
        codes = isinstance(first, SqW8A8BBF16OBF16PerChannel)
        if any(isinstance(m, SqW8A8BBF16OBF16PerChannel) != codes or (codes and dtype is None and m.dtype != first.dtype) for m in modules):
            raise RuntimeError("the experts must be modules of one kind and type")
        if any((m.in_features, m.out_features) != (first.in_features, first.out_features) or (m.bias is None) != (first.bias is None) for m in modules):
            raise RuntimeError("the experts must have the same shape, and all or none of them a bias")
        if not codes and any(not isinstance(m, torch.nn.Linear) or m.weight.dtype.itemsize < 2 for m in modules):
            raise RuntimeError("from_linears takes nn.Linear modules with floating-point weights, or SqW8A8BBF16OBF16PerChannel modules")
        dtype = dtype or (first.dtype if codes else torch.bfloat16)
        dev = first.qweight.device if codes else first.weight.device
        lin = cls(len(modules), first.in_features, first.out_features, first.bias is not None, dev, dtype)
        for e, m in enumerate(modules):
            q = m if codes else SqW8A8BBF16OBF16PerChannel.from_linear(m, 8, 0, init_only=False, dtype=dtype)
            lin.qweight[e].copy_(q.qweight)
            lin.weight_scale[e].copy_(q.weight_scale.view(-1))
            if lin.bias is not None:
                lin.bias[e].copy_(q.bias)
        return lin

    def forward(self, x, offsets, out=None):
        """``x`` [M, K] in bf16 or fp16, sorted by expert; ``offsets``: int32 [num_experts + 1] on the GPU, the experts' first rows and the end of the last.
        Rows of no expert are not written (sq_fp8_kernels.w8a8_int8_linear_per_channel_grouped).  -> [M, N] in x's type."""
        if x.dim() != 2 or x.shape[1] != self.in_features or x.dtype not in _NAMES or not x.is_cuda:
            raise RuntimeError(f"the input must be [rows, {self.in_features}] in bf16 or fp16 on a GPU")
        with torch.cuda.device(x.device):  # (the quantizer launches on the current one)
            q, s = quantize_activation_per_token_absmax_f32(x)
        return w8a8_int8_linear_per_channel_grouped(q, self.qweight, self.bias, s, self.weight_scale, offsets, _NAMES[x.dtype], out)

    def forward_quantized(self, qinput, x_scale, offsets, out=None):
        """The same for rows already quantized per token (int8 and fp32 scales [M, 1]); the result is in the module's dtype."""
        return w8a8_int8_linear_per_channel_grouped(qinput, self.qweight, self.bias, x_scale, self.weight_scale, offsets, _NAMES[self.dtype], out)

    def extra_repr(self):
        return (f"num_experts={self.num_experts}, in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, "
                f"dtype={self.dtype}")

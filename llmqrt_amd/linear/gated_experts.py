"""The feed-forward layer of several experts on quantized weights: routing, dispatch, gate and up projections, gated activation, down projection, combine.

No counterpart in the reference.  Nothing is read back by the host between the steps, and no activation is quantized twice: dispatch and activation give
the next product its codes and scales."""
from __future__ import annotations

import torch

from ..activation import silu_mul_per_group_quantize, silu_mul_quantize_activation_per_token_absmax
from ..experts import combine_from_experts, dispatch_per_group_quantize, dispatch_quantize_activation_per_token_absmax, route_to_experts
from .linear_fp8_block import FP8BlockGroupedLinear
from .linear_sq_grouped import SqW8A8GroupedLinear

__all__ = ["GatedExperts"]

_KINDS = {SqW8A8GroupedLinear: (dispatch_quantize_activation_per_token_absmax, silu_mul_quantize_activation_per_token_absmax),
          FP8BlockGroupedLinear: (dispatch_per_group_quantize, silu_mul_per_group_quantize)}


class GatedExperts(torch.nn.Module):
    """``gate_up``: the experts' gate and up projections joined, [2 I, K] each, ``down``: their down projections [K', I], K' a multiple of 8; both
    SqW8A8GroupedLinear or both FP8BlockGroupedLinear.  ``score_bias``: fp32 [experts of the router] or None; ``routing``: the other arguments of route_to_experts
    (scoring, num_groups, top_groups, group_score, renormalize, scale).  ``first_expert``: the router's number of the first expert here, where a GPU holds a part
    of them; its output is then its part of the sum."""

    def __init__(self, gate_up, down, top_k, score_bias=None, first_expert=0, **routing):
        super().__init__()
        if type(gate_up) not in _KINDS or type(down) is not type(gate_up):
            raise RuntimeError("gate_up and down must both be SqW8A8GroupedLinear or both FP8BlockGroupedLinear")
        if gate_up.num_experts != down.num_experts or gate_up.out_features != 2 * down.in_features or gate_up.out_features % 16:
            raise RuntimeError("gate_up and down must have as many experts, and gate_up twice the channels that down takes, a multiple of 8")
        if down.out_features % 8:
            raise RuntimeError(f"down must have a multiple of 8 output channels, got {down.out_features}")
        if gate_up.dtype != down.dtype:
            raise RuntimeError("gate_up and down must have one dtype")
        unknown = set(routing) - {"scoring", "num_groups", "top_groups", "group_score", "renormalize", "scale"}
        if unknown:
            raise RuntimeError(f"unknown routing arguments {sorted(unknown)}")
        self.gate_up, self.down = gate_up, down
        self.top_k, self.first_expert, self.routing = top_k, first_expert, routing
        self.register_buffer("score_bias", score_bias)

    def _apply(self, fn, *args, **kwargs):
        kept = self.score_bias

        def moved(t):  # .half() and .bfloat16() are for the activations: scores stay fp32
            u = fn(t)
            return t.to(u.device) if t is kept and u.dtype != t.dtype else u
        return super()._apply(moved, *args, **kwargs)

    def forward(self, x, logits, shared=None):
        """``x`` [.., K] in the modules' dtype, ``logits`` [.., experts of the router]; ``shared`` [.., K'] is added to the result (an expert that all tokens
        share).  -> [.., K']."""
        if x.dtype != self.gate_up.dtype or x.shape[-1] != self.gate_up.in_features:
            raise RuntimeError(f"the input must be [.., {self.gate_up.in_features}] in {self.gate_up.dtype}")
        if logits.shape[:-1] != x.shape[:-1]:
            raise RuntimeError("logits must be [.., experts] for activations [.., K]")
        dispatch, activate = _KINDS[type(self.gate_up)]
        weights, experts = route_to_experts(logits, self.top_k, bias=self.score_bias, **self.routing)
        q, s, offsets, places = dispatch(x, experts, self.gate_up.num_experts, self.first_expert)
        q, s = activate(self.gate_up.forward_quantized(q, s, offsets))
        return combine_from_experts(self.down.forward_quantized(q, s, offsets), places, weights, shared)

    def extra_repr(self):
        return ", ".join([f"top_k={self.top_k}", f"first_expert={self.first_expert}", *(f"{k}={v!r}" for k, v in self.routing.items())])

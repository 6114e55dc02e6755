"""Inference modules with 8-bit integer weights (``ops.int8_linear``,
``ops.moe_int8_forward``), made from a ``Linear`` (``astrai/model/components/
linear.py:7-24``) or a trained MoE layer (``mlp.py:28-100``, or ``ScoredMoE``).

A weight is quantised once, by output channel; activations are quantised token
by token in every call. The codes and scales are buffers, so ``state_dict``
saves and loads them; scales keep 32 bits when the module is cast. There is no
backward: the modules refuse inputs that need a gradient.
"""

from __future__ import annotations

import torch
import torch.nn as nn
from torch import Tensor

from astrai_amd.extension import ops
from astrai_amd.model.components.linear import Linear
from astrai_amd.model.components.mlp import DeepSeekMoE
from astrai_amd.model.components.scored_moe import keep_float32


def _check_input(x: Tensor, who: str) -> None:
    if x.device.type != "cuda":
        raise RuntimeError(f"{who} runs on the HIP kernels and needs a ROCm device tensor, got {x.device}")
    if torch.is_grad_enabled() and x.requires_grad:
        raise RuntimeError(f"{who} is for inference: it has no backward")


class Int8Linear(nn.Module):
    """``x . weight^T (+ bias)`` in 8-bit integers, in x's dtype."""

    def __init__(self, in_dim: int, out_dim: int, bias: bool = False):
        super().__init__()
        self.in_dim = in_dim
        self.register_buffer("weight", torch.zeros(out_dim, ops.int8_row_bytes(in_dim), dtype=torch.int8))
        self.register_buffer("weight_scale", torch.zeros(out_dim))
        self.register_buffer("bias", torch.zeros(out_dim) if bias else None)

    @classmethod
    @torch.no_grad()
    def from_linear(cls, linear: Linear | nn.Linear) -> "Int8Linear":
        """The int8 form of a Linear on the GPU (its weight is not kept)."""
        out_dim, in_dim = linear.weight.shape
        made = cls.__new__(cls)
        nn.Module.__init__(made)
        made.in_dim = in_dim
        q, scale = ops.quantize_rows(linear.weight.detach().contiguous())
        made.register_buffer("weight", q)
        made.register_buffer("weight_scale", scale)
        made.register_buffer("bias", None if linear.bias is None else linear.bias.detach().clone())
        return made.train(linear.training)

    def _apply(self, *args, **kwargs):
        keep_float32(self, ("weight_scale",), super()._apply, *args, **kwargs)
        return self

    def forward(self, x: Tensor) -> Tensor:
        _check_input(x, "Int8Linear")
        if x.shape[-1] != self.in_dim:  # (rows of codes are padded: their bytes do not tell)
            raise ValueError(f"Int8Linear of {self.in_dim} columns got {x.shape[-1]}")
        lead = x.shape[:-1]
        bias = self.bias if self.bias is None or self.bias.dtype == x.dtype else self.bias.to(x.dtype)
        out = ops.int8_linear(x.reshape(-1, x.shape[-1]).contiguous(), self.weight, self.weight_scale, bias)
        return out.view(*lead, out.shape[-1])


class Int8MoE(nn.Module):
    """A MoE layer whose experts run in 8-bit integers; router and routing stay
    those of the layer it was made from."""

    SCALES = ("gate_scale", "up_scale", "down_scale", "balance_bias")

    def __init__(self, dim: int, dim_ffn: int, n_routed_experts: int, n_shared_experts: int = 1,
                 n_activated_experts: int = 2, routing: ops.Routing | None = None, router: nn.Module | None = None):
        super().__init__()
        self.dim, self.dim_ffn = dim, dim_ffn
        self.n_routed_experts, self.n_shared_experts = n_routed_experts, n_shared_experts
        self.n_activated_experts, self.routing = n_activated_experts, routing
        self.router = Linear(dim, n_routed_experts) if router is None else router
        e = n_routed_experts + n_shared_experts
        for name, n, k in (("gate", dim_ffn, dim), ("up", dim_ffn, dim), ("down", dim, dim_ffn)):
            self.register_buffer(name, torch.zeros(e, n, ops.int8_row_bytes(k), dtype=torch.int8))
            self.register_buffer(name + "_scale", torch.zeros(e, n))
        self.register_buffer("balance_bias", None if routing is None else torch.zeros(n_routed_experts))

    @classmethod
    @torch.no_grad()
    def from_layer(cls, layer: DeepSeekMoE) -> "Int8MoE":
        """The int8 form of a layer on the GPU. Routed and shared experts must
        have the same shape; the router module is shared with the layer, the
        experts' weights are not kept."""
        routed = layer._expert_weights(layer.routed_experts)
        shared = layer._expert_weights(layer.shared_experts)
        dim_ffn = routed[0][0].shape[0]
        routing, bias = layer._routing()
        with torch.device("meta"):
            made = cls(layer.dim, dim_ffn, layer.n_routed_experts, layer.n_shared_experts, layer.n_activated_experts,
                       routing, layer.router)
        for name, ws in zip(("gate", "up", "down"), map(list.__add__, routed, shared)):
            shape = made._buffers[name].shape
            q = torch.empty(shape, dtype=torch.int8, device=ws[0].device)
            scale = torch.empty(shape[:2], device=ws[0].device)
            for i, w in enumerate(ws):  # (one at a time: no second copy of all the weights)
                if w.shape[0] != shape[1] or ops.int8_row_bytes(w.shape[1]) != shape[2]:
                    raise RuntimeError(f"Int8MoE: expert weight {i} has shape {tuple(w.shape)}, others differ")
                q[i], scale[i] = ops.quantize_rows(w.detach().contiguous())
            made._buffers[name], made._buffers[name + "_scale"] = q, scale
        made._buffers["balance_bias"] = None if bias is None else bias.detach().clone()
        return made.train(layer.training)

    def _apply(self, *args, **kwargs):
        keep_float32(self, self.SCALES, super()._apply, *args, **kwargs)
        return self

    def experts(self) -> ops.Int8Experts:
        return ops.Int8Experts(self.gate, self.up, self.down, self.gate_scale, self.up_scale, self.down_scale)

    def forward(self, x: Tensor) -> Tensor:
        _check_input(x, "Int8MoE")
        lead = x.shape[:-1]
        x2 = x.reshape(-1, x.shape[-1]).contiguous()
        with torch.no_grad():
            logits = self.router(x2)
        out = ops.moe_int8_forward(x2, logits, self.experts(), self.n_activated_experts, self.n_shared_experts,
                                   self.routing, self.balance_bias)
        return out.view(*lead, out.shape[-1])


def quantize_moe(model: nn.Module) -> int:
    """Replaces every ``DeepSeekMoE`` (and ``ScoredMoE``) inside ``model`` by its
    ``Int8MoE``, for inference; returns how many. The model's own module cannot
    be replaced: ``Int8MoE.from_layer`` makes its int8 form."""
    found = [(parent, name, child) for parent in model.modules() for name, child in parent._modules.items()
             if isinstance(child, DeepSeekMoE)]
    for parent, name, child in found:
        parent._modules[name] = Int8MoE.from_layer(child)
    return len(found)

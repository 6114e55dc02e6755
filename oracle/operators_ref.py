"""Plain 64-bit forms of the routing by scores and of the 8-bit products, for the
tests: elementary torch operations in float64, on the CPU or the GPU. The
reference (``astrai/model/components/mlp.py``) has no counterpart: parity
unpinned, the formulas are those of ``include/astrai_moe.h``.
"""

from __future__ import annotations

import math

import torch


def choose(logits, top_k, routing, bias=None):
    """(scores [T, E], chosen [T, K] with ties to the lower index, live [T, K])
    for logits without NaN (softmax: and without +inf)."""
    l = logits.double()
    t, e = l.shape
    if routing.score == "sigmoid":
        s = torch.sigmoid(l)
    else:
        top = l.amax(-1, keepdim=True)
        p = torch.exp(l - torch.where(torch.isinf(top), torch.zeros_like(top), top))
        s = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    key = s if bias is None else s + bias.double()
    key = torch.where((l == -math.inf) | torch.isnan(key), torch.full_like(key, -math.inf), key)
    if routing.n_groups > 1:
        parts = key.view(t, routing.n_groups, -1)
        value = parts.topk(routing.group_top, dim=-1).values.sum(-1)
        kept = torch.sort(value, dim=-1, descending=True, stable=True).indices[:, :routing.topk_groups]
        keep = torch.zeros_like(value, dtype=torch.bool).scatter_(1, kept, True)
        key = parts.masked_fill(~keep.unsqueeze(-1), -math.inf).reshape(t, e)
    values, order = torch.sort(key, dim=-1, descending=True, stable=True)
    return s, order[:, :top_k], values[:, :top_k] > -math.inf


def weights(s, chosen, live, routing):
    """Routing weights, differentiable in ``s``."""
    v = torch.where(live, s.gather(1, chosen), torch.zeros((), dtype=s.dtype, device=s.device))
    if routing.renormalise:
        total = v.sum(-1, keepdim=True)
        v = torch.where(total > 0, v / torch.where(total > 0, total, torch.ones_like(total)), torch.zeros_like(v))
    return v * routing.scale


def route_grad(logits, top_k, routing, bias, dw):
    """Gradient of the logits (float64 autograd through the chosen scores)."""
    l = logits.double().requires_grad_(True)
    _, chosen, live = choose(logits, top_k, routing, bias)
    if routing.score == "sigmoid":
        s = torch.sigmoid(l)
    else:
        off = torch.isinf(l).all(-1, keepdim=True)
        s = torch.softmax(torch.where(off, torch.zeros_like(l), l), dim=-1)
        s = torch.where(off, torch.zeros_like(s), s)
    weights(s, chosen, live, routing).backward(dw.double())
    return torch.nan_to_num(l.grad, nan=0.0)


def histogram(chosen, n_experts):
    t = chosen.shape[0]
    hot = torch.zeros(-(-t // 32) * 32, n_experts, dtype=torch.int32, device=chosen.device)
    hot[:t].scatter_(1, chosen, 1)
    return hot.view(-1, 32, n_experts).sum(1, dtype=torch.int32)


def quantize(x):
    """(codes, scales) as float64 of the rows of finite x; a scale is a float32."""
    x = x.double()
    most = x.abs().amax(-1, keepdim=True)
    return torch.round(x * 127.0 / torch.where(most > 0, most, torch.ones_like(most))), (most / 127.0).float().double()


def int8_linear(x, w, w_scale, bias=None):
    """x [M, K], w [N, >= K] codes -> float64 [M, N] (not rounded)."""
    q, s = quantize(x)
    y = (q @ w[:, :x.shape[1]].double().t()) * s * w_scale.double()
    return y if bias is None else y + bias.double()


def int8_mlp(x, gate, up, down, gate_scale, up_scale, down_scale):
    """One SwiGLU expert in 8 bits, h and the output rounded to x's dtype."""
    g, u = int8_linear(x, gate, gate_scale), int8_linear(x, up, up_scale)
    h = (g * torch.sigmoid(g) * u).to(x.dtype)
    return int8_linear(h, down, down_scale).to(x.dtype)


def int8_layer(x, chosen, w, experts, n_shared=0):
    """Weighted experts plus the mean of the shared ones in float64."""
    out = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    n = experts.gate.shape[0] - n_shared
    for e in range(n):
        token, slot = (chosen == e).nonzero(as_tuple=True)
        if token.numel():
            y = int8_mlp(x[token], *(t[e] for t in experts))
            out.index_add_(0, token, y.double() * w[token, slot].double().unsqueeze(1))
    for e in range(n_shared):
        out += int8_mlp(x, *(t[n + e] for t in experts)).double() / n_shared
    return out

"""MoE layer whose router chooses by scores (``ops.moe_route_scores``).

The reference's ``DeepSeekMoE`` knows softmax scores, renormalised, without
groups or a bias (``astrai/model/components/mlp.py:84-87``) and keeps its
``topk_method`` unused (``mlp.py:45``). ``ScoredMoE`` is the same layer, with
the same children and ``state_dict`` keys plus ``balance_bias``, for routers of
softmax or sigmoid scores, groups of experts, plain or renormalised weights and
a scale, whose bias evens out the experts' loads without a loss of its own.
Registered as ``"moe_scored"``; routing, experts and backward run on the HIP
kernels as in ``DeepSeekMoE``.
"""

from __future__ import annotations

import torch
from torch import Tensor

from astrai_amd.extension import ops
from astrai_amd.model.components.autograd import ScoredRouteWeights
from astrai_amd.model.components.mlp import DeepSeekMoE, FFNFactory


def keep_float32(module: torch.nn.Module, names: tuple[str, ...], apply, *args, **kwargs) -> None:
    """``apply`` (the module's inherited ``_apply``), after which the buffers
    ``names`` have moved, but kept their 32 bits."""
    before = {n: module._buffers[n] for n in names if module._buffers.get(n) is not None}
    apply(*args, **kwargs)
    for n, old in before.items():
        new = module._buffers[n]
        if new.dtype != old.dtype:
            module._buffers[n] = old.to(device=new.device)


@FFNFactory.register("moe_scored")
class ScoredMoE(DeepSeekMoE):
    """``DeepSeekMoE`` routing by ``score_func`` ("softmax" or "sigmoid") of the
    router's logits: ``topk_groups`` of ``n_groups`` groups of experts stay (by
    their ``group_top`` best experts), the best experts of these by score plus
    ``balance_bias`` are chosen, and their scores, over their sum with
    ``renormalise`` and times ``route_scale``, are the weights.

    ``balance_bias`` (float32, zeros at first) is no parameter: with
    ``track_load`` set, training forwards add up the experts' loads, and
    ``update_balance(rate)`` moves the bias against them."""

    def __init__(
        self,
        dim: int,
        dim_ffn: int,
        n_routed_experts: int,
        n_shared_experts: int = 1,
        n_activated_experts: int = 2,
        topk_method: str = "greedy",
        n_layers: int = 1,
        score_func: str = "softmax",
        n_groups: int = 1,
        topk_groups: int = 1,
        group_top: int = 1,
        renormalise: bool = True,
        route_scale: float = 1.0,
        track_load: bool = False,
    ):
        super().__init__(dim, dim_ffn, n_routed_experts, n_shared_experts, n_activated_experts, topk_method, n_layers)
        self.routing = ops.Routing(score_func, n_groups, topk_groups, group_top, renormalise, route_scale)
        ops._check_routing(self.routing, n_routed_experts, n_activated_experts)
        self.register_buffer("balance_bias", torch.zeros(n_routed_experts, dtype=torch.float32))
        self.track_load = track_load
        self.load: Tensor | None = None  # tokens per expert since the last update_balance

    def _apply(self, *args, **kwargs):
        keep_float32(self, ("balance_bias",), super()._apply, *args, **kwargs)
        if self.load is not None:
            self.load = self.load.to(self.balance_bias.device)
        return self

    def _routing(self) -> tuple[ops.Routing, Tensor]:
        return self.routing, self.balance_bias

    def _route_autograd(self, logits: Tensor, dtype: torch.dtype) -> tuple[Tensor, Tensor, Tensor]:
        topk_w, topk_idx, chunk_hist = ScoredRouteWeights.apply(logits, self.balance_bias, self.n_activated_experts,
                                                                self.routing, dtype)
        if self.track_load and self.training:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("track_load: a captured graph's replays would not be counted; capture with track_load off")
            load = ops.moe_expert_load(chunk_hist)
            self.load = load if self.load is None else self.load.add_(load)
        return topk_w, topk_idx, chunk_hist

    @torch.no_grad()
    def update_balance(self, rate: float, group=None) -> Tensor | None:
        """Moves ``balance_bias`` by ``rate`` up for experts that got fewer
        tokens than the mean since the last call and down for those that got
        more; returns the loads it went by (None, and no change, without
        tracked forwards). ``group``: a process group over whose ranks the
        loads are summed first (``torch.distributed.group.WORLD`` for all);
        every rank of it calls, also one that tracked no forward."""
        load, self.load = self.load, None
        if load is None:
            if group is None:
                return None
            load = torch.zeros(self.balance_bias.shape, dtype=torch.int32, device=self.balance_bias.device)
        if group is not None:
            if torch.distributed.get_backend(group) == "gloo":  # (sums host tensors)
                host = load.cpu()
                torch.distributed.all_reduce(host, group=group)
                load.copy_(host)
            else:
                torch.distributed.all_reduce(load, group=group)
        ops.moe_balance_bias(self.balance_bias, load, rate, out=self.balance_bias)
        return load

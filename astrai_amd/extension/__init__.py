"""MoE expert-forward kernels (HIP, gfx950) behind AstrAI's extension-loading
contract.

Public API:
    - ``moe_route``        router softmax / top-k / renormalisation
    - ``moe_permute``      expert-major token permutation + GEMM tile list
    - ``moe_gemm_gate_up`` grouped gate/up projection with fused SwiGLU
    - ``moe_gemm_down``    grouped down projection with fused routing weight
    - ``moe_combine``      weighted un-permute, shared-expert mean and add
    - ``moe_routed_forward`` the five above in sequence
    - ``moe_route_scores`` routing by softmax or sigmoid scores with a bias for
      balance, groups and a scale (``Routing``); ``moe_route_scores_grad``,
      ``moe_expert_load`` and ``moe_balance_bias`` for its training
    - ``quantize_rows``, ``int8_linear``, ``moe_int8_forward`` products in 8-bit
      integers: a Linear's, and the experts' (``Int8Experts``)

``is_available(name)`` and ``KERNEL_NAMES`` follow the reference's
``astrai/extension/__init__.py``.
"""

from astrai_amd.extension.loader import KERNEL_NAMES, is_available
from astrai_amd.extension.ops import (
    Int8Experts,
    Routing,
    expert_weight_table,
    int8_linear,
    moe_balance_bias,
    moe_combine,
    moe_dense_mlp,
    moe_expert_load,
    moe_gemm_down,
    moe_gemm_gate_up,
    moe_int8_forward,
    moe_permute,
    moe_route,
    moe_route_scores,
    moe_route_scores_grad,
    moe_routed_forward,
    quantize_rows,
    select_block_m,
)

__all__ = [
    "KERNEL_NAMES",
    "is_available",
    "Int8Experts",
    "Routing",
    "expert_weight_table",
    "int8_linear",
    "moe_balance_bias",
    "moe_combine",
    "moe_dense_mlp",
    "moe_expert_load",
    "moe_gemm_down",
    "moe_gemm_gate_up",
    "moe_int8_forward",
    "moe_permute",
    "moe_route",
    "moe_route_scores",
    "moe_route_scores_grad",
    "moe_routed_forward",
    "quantize_rows",
    "select_block_m",
]

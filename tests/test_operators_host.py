"""Refusals of the scores' and the 8-bit entry points that need no GPU: the C ABI
turns every bad argument into an error before any device work (the dummy pointers
below are never dereferenced), and the plain 64-bit forms against small cases
worked by hand."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from astrai_amd.extension import loader, ops
from oracle import operators_ref as R

BF16, F32 = 1, 0


def _routing(score=1, n_groups=1, topk_groups=1, group_top=1, renormalise=1, scale=1.0):
    return ctypes.byref(loader.CRouting(score, n_groups, topk_groups, group_top, renormalise, scale))


def _refused(rc, words):
    assert rc == -1 and words in loader.last_error(), loader.last_error()


def test_route_scores_refuses_before_any_device_work():
    lib = loader.library()

    def call(routing, n_tokens=4, e=64, k=4, dtype=F32, wdtype=F32, p=16):
        return lib.astrai_moe_route_scores(p, dtype, None, routing, n_tokens, e, k, wdtype, p, p, p, None)

    _refused(call(None), "null routing")
    _refused(call(_routing(score=2)), "score")
    _refused(call(_routing(n_groups=7)), "divide")
    _refused(call(_routing(n_groups=0)), "divide")
    _refused(call(_routing(n_groups=8, topk_groups=9)), "topk_groups")
    _refused(call(_routing(n_groups=8, topk_groups=0)), "topk_groups")
    _refused(call(_routing(n_groups=32, topk_groups=1)), "fewer than top_k")
    _refused(call(_routing(group_top=3)), "group_top")
    _refused(call(_routing(n_groups=64, topk_groups=8, group_top=2)), "group_top")
    _refused(call(_routing(scale=math.nan)), "finite")
    _refused(call(_routing(), e=0), "n_experts")
    _refused(call(_routing(), e=1025), "n_experts")
    _refused(call(_routing(), k=33), "top_k")
    _refused(call(_routing(), dtype=2), "dtype")
    _refused(call(_routing(), wdtype=5), "dtype")
    _refused(call(_routing(), n_tokens=-1), "n_tokens")
    _refused(call(_routing(), p=None), "null buffer")
    assert call(_routing(), n_tokens=0, p=None) == 0
    grad = lib.astrai_moe_route_scores_grad
    _refused(grad(16, F32, 16, 16, None, F32, _routing(), 4, 64, 4, 16, None), "null buffer")
    _refused(grad(16, F32, 16, 16, 16, 9, _routing(), 4, 64, 4, 16, None), "dtype")
    _refused(lib.astrai_moe_expert_load(16, 4, 2000, 16, None), "n_experts")
    _refused(lib.astrai_moe_expert_load(None, 4, 8, 16, None), "null buffer")
    _refused(lib.astrai_moe_balance_bias(16, 16, 8, math.inf, 16, None), "finite")
    _refused(lib.astrai_moe_balance_bias(16, 16, 0, 0.1, 16, None), "n_experts")
    _refused(lib.astrai_moe_balance_bias(None, 16, 8, 0.1, 16, None), "null buffer")


def test_forward_scores_refuses_before_any_device_work():
    lib = loader.library()
    sizes = (4, 8, 2, 1, 64, 64)
    need = lib.astrai_moe_forward_workspace_bytes(*sizes, BF16, 0)
    assert need > 0

    def call(routing, ldtype=F32, sizes=sizes, ws=256, nbytes=need, packed=None, x=16):
        return lib.astrai_moe_forward_scores(x, 16, ldtype, None, routing, 16, 16, 16, packed, None, BF16, *sizes, ws, nbytes,
                                             16, None)

    _refused(call(None), "null routing")
    _refused(call(_routing(score=5)), "score")
    _refused(call(_routing(n_groups=3)), "divide")
    _refused(call(_routing(), ldtype=7), "dtype")
    _refused(call(_routing(scale=math.inf)), "finite")
    _refused(call(_routing(), packed=16), "packed")
    _refused(call(_routing(), x=None), "null buffer")
    _refused(call(_routing(), nbytes=need - 1), "")
    _refused(call(_routing(), sizes=(4, 8, 9, 1, 64, 64)), "top_k")
    assert call(_routing(), sizes=(0, 8, 2, 1, 64, 64)) == 0


def test_int8_refuses_before_any_device_work():
    lib = loader.library()
    assert [lib.astrai_moe_int8_row_bytes(k) for k in (0, 1, 16, 17)] == [0, 16, 16, 32]
    assert [ops.int8_row_bytes(k) for k in (1, 16, 17)] == [16, 16, 32]
    _refused(lib.astrai_moe_quantize_rows(16, 3, 4, 8, 16, 16, None), "dtype")
    _refused(lib.astrai_moe_quantize_rows(16, F32, 4, 131073, 16, 16, None), "inner size")
    _refused(lib.astrai_moe_quantize_rows(16, F32, -1, 8, 16, 16, None), "n_rows")
    _refused(lib.astrai_moe_quantize_rows(16, F32, 1, 8, 8, 16, None), "16-byte")
    _refused(lib.astrai_moe_quantize_rows(None, F32, 1, 8, 16, 16, None), "null buffer")
    need = lib.astrai_moe_int8_linear_workspace_bytes(4, 64, 32, BF16)
    assert need > 0
    _refused(lib.astrai_moe_int8_linear_workspace_bytes(4, 0, 32, BF16), "inner size")

    def linear(dtype=BF16, w=16, m=4, k=64, n=32, ws=256, nbytes=need, out=16):
        return lib.astrai_moe_int8_linear(16, dtype, w, 16, None, m, k, n, ws, nbytes, out, None)

    _refused(linear(dtype=4), "dtype")
    _refused(linear(w=8), "16-byte")
    _refused(linear(ws=128), "256-byte")
    _refused(linear(nbytes=need - 1), "workspace holds")
    _refused(linear(out=None), "null buffer")
    _refused(linear(n=(1 << 22) + 1), "outputs")
    assert linear(m=0) == 0
    sizes = (4, 8, 2, 1, 64, 96)
    need = lib.astrai_moe_int8_forward_workspace_bytes(*sizes, BF16)
    assert need > 0
    _refused(lib.astrai_moe_int8_forward_workspace_bytes(4, 8, 32, 1, 64, 96, BF16), "top_k")
    _refused(lib.astrai_moe_int8_forward_workspace_bytes(1 << 30, 8, 2, 1, 64, 96, BF16), "2^31")

    def forward(routing=_routing(), ldtype=F32, bias=None, w=16, ws=256, nbytes=need, sizes=sizes, x=16):
        return lib.astrai_moe_int8_forward(x, BF16, 16, ldtype, bias, routing, w, 16, 16, 16, 16, 16, *sizes, ws, nbytes,
                                           16, None)

    _refused(forward(routing=None), "without a routing")
    _refused(forward(routing=None, ldtype=BF16, bias=16), "without a routing")
    _refused(forward(routing=_routing(score=7)), "score")
    _refused(forward(w=24), "16-byte")
    _refused(forward(ws=64), "256-byte")
    _refused(forward(nbytes=need - 1), "workspace holds")
    _refused(forward(x=None), "null buffer")
    _refused(forward(sizes=(4, 8, 2, -1, 64, 96)), "n_shared")
    _refused(forward(sizes=(4, 1024, 2, 1, 64, 96)), "n_experts")
    _refused(forward(sizes=(4, 8, 2, 1, 64, 200000)), "inner size")
    assert forward(sizes=(0, 8, 2, 1, 64, 96)) == 0


def test_wrappers_refuse_cpu_tensors_and_bad_routings():
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.moe_route_scores(x, 2)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.quantize_rows(x)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.int8_linear(x, x, x)
    with pytest.raises(ValueError, match="ROCm device"):
        ops.moe_int8_forward(x, x, None, 2)
    for routing in (ops.Routing("greedy"), ops.Routing(n_groups=3), ops.Routing(n_groups=64, topk_groups=1),
                    ops.Routing(group_top=0), ops.Routing(scale=math.inf)):
        with pytest.raises(ValueError):
            ops._check_routing(routing, 64, 2)


def test_plain_routing_by_hand():
    """Four experts in two groups, sigmoid scores 0.5, 0.75, 0.6, 0.6 (logits 0,
    log 3, log 1.5 twice)."""
    logits = torch.tensor([[0.0, math.log(3), math.log(1.5), math.log(1.5)]], dtype=torch.float64)
    pick = lambda k, r, b=None: R.choose(logits, k, r, b)[1].tolist()  # noqa: E731
    assert pick(3, ops.Routing("sigmoid")) == [[1, 2, 3]]
    # groups by their best expert: the first; by their best two: 1.25 against 1.2, the first again
    assert pick(2, ops.Routing("sigmoid", 2, 1, 1)) == [[1, 0]]
    assert pick(2, ops.Routing("sigmoid", 2, 1, 2)) == [[1, 0]]
    # a bias of 0.1 on expert 3 turns both
    bias = torch.tensor([0.0, 0.0, 0.0, 0.2])
    assert pick(2, ops.Routing("sigmoid", 2, 1, 1), bias) == [[3, 2]]
    s, chosen, live = R.choose(logits, 2, ops.Routing("sigmoid", 2, 1, 2), bias)
    w = R.weights(s, chosen, live, ops.Routing("sigmoid", scale=2.0))
    torch.testing.assert_close(w, torch.tensor([[1.0, 1.0]], dtype=torch.float64))  # the weights know no bias
    logits[0, :3] = -math.inf
    s, chosen, live = R.choose(logits, 3, ops.Routing("softmax"))
    assert chosen.tolist() == [[3, 0, 1]] and live.tolist() == [[True, False, False]]
    assert R.weights(s, chosen, live, ops.Routing()).tolist() == [[1.0, 0.0, 0.0]]


def test_plain_product_by_hand():
    x = torch.tensor([[1.0, -2.0, 0.5], [0.0, 0.0, 0.0]])
    q, s = R.quantize(x)
    assert q.tolist() == [[64.0, -127.0, 32.0], [0.0, 0.0, 0.0]] and s[0, 0] == (torch.tensor(2.0) / 127).double() and s[1, 0] == 0
    w = torch.tensor([[1, 2, 3, 99]], dtype=torch.int8)
    y = R.int8_linear(x, w, torch.tensor([0.5]))
    assert y[0, 0].item() == pytest.approx((64 - 254 + 96) * 0.5 * 2 / 127, rel=1e-7) and y[1, 0] == 0

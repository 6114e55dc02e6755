"""Routing by scores (``ops.moe_route_scores``), its gradient, the experts' loads
and the balance bias against the plain 64-bit forms of ``oracle/operators_ref.py``.

The choice is compared for equality: the kernel decides in 64 bits, as the plain
form does, so that only scores closer than 1e-15 could part them. Tolerances:

* float32 weights: exp of l - max, |l - max| < 32, has a relative error of at most
  32 * 2^-24 from the argument and 2 * 2^-24 of its own; sums and quotients of up
  to 32 positive terms add at most 36 * 2^-24: 70 * 2^-24 < 2^-17;
* rounding to bf16 adds half a step, 2^-8 of the value;
* a gradient is a sum of terms of the size of its largest intermediate ds: an
  absolute 2^-16 of max |ds| next to the rounding of its type.
"""

from __future__ import annotations

import math

import pytest
import torch

from astrai_amd.extension import ops
from oracle import operators_ref as R

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
REL = 2.0 ** -17

# (tokens, experts, top_k, routing)
CASES = [
    (1, 1, 1, ops.Routing("softmax")),
    (1, 8, 2, ops.Routing("sigmoid")),
    (31, 60, 4, ops.Routing("softmax", renormalise=False)),
    (32, 64, 6, ops.Routing("sigmoid", scale=2.5)),
    (33, 64, 8, ops.Routing("sigmoid", 8, 4, 2, True, 2.5)),
    (100, 96, 5, ops.Routing("softmax", 6, 3, 1)),
    (257, 160, 6, ops.Routing("softmax", 8, 3, 1, True, 16.0)),
    (500, 128, 8, ops.Routing("sigmoid", 16, 2, 2)),
    (130, 100, 7, ops.Routing("sigmoid", 5, 2, 2)),
    (77, 256, 8, ops.Routing("sigmoid", 8, 4, 2, True, 2.5)),
    (65, 384, 10, ops.Routing("softmax")),
    (40, 1024, 32, ops.Routing("sigmoid", 32, 8, 2)),
    (40, 1000, 32, ops.Routing("softmax", 1000, 40, 1)),
    (9, 70, 3, ops.Routing("sigmoid", 35, 2, 2)),
    (4097, 64, 6, ops.Routing("sigmoid")),
]


def _inputs(gpu, t, e, dtype, masked, with_bias, seed=0):
    gen = torch.Generator().manual_seed(seed)
    logits = torch.randn(t, e, generator=gen) * 2.0
    if masked:
        logits[torch.rand(t, e, generator=gen) < 0.3] = -math.inf
        logits[torch.rand(t, generator=gen) < 0.2] = -math.inf
    bias = torch.randn(e, generator=gen) * 0.1 if with_bias else None
    return logits.to(dtype).to(gpu), bias.to(gpu) if with_bias else None


def _check_route(got, logits, top_k, routing, bias, weight_dtype):
    s, chosen, live = R.choose(logits, top_k, routing, bias)
    assert torch.equal(got.topk_idx.long(), chosen)
    assert torch.equal(got.chunk_hist, R.histogram(chosen, logits.shape[1]))
    w = R.weights(s, chosen, live, routing)
    assert got.topk_w.dtype == weight_dtype
    err = (got.topk_w.double() - w).abs()
    assert (err <= (REL + HALF[weight_dtype]) * w.abs()).all(), err.max()
    return s, chosen, live


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype,weight_dtype", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16),
                                                (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("t,e,k,routing", CASES)
def test_route_scores(gpu, t, e, k, routing, dtype, weight_dtype, masked):
    for with_bias in (False, True):
        logits, bias = _inputs(gpu, t, e, dtype, masked, with_bias)
        got = ops.moe_route_scores(logits, k, routing, bias, weight_dtype)
        _check_route(got, logits, k, routing, bias, weight_dtype)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_equal_scores_go_to_the_lower_expert(gpu, score):
    for e, routing in ((64, ops.Routing(score)), (256, ops.Routing(score, 8, 4, 2)), (96, ops.Routing(score, 6, 2, 1))):
        logits = torch.zeros(40, e, device=gpu)
        logits[1::2, e // 2:] = 1.0
        got = ops.moe_route_scores(logits, 6, routing)
        assert got.topk_idx[0].tolist() == list(range(6))
        assert got.topk_idx[1].tolist() == list(range(e // 2, e // 2 + 6))
        torch.testing.assert_close(got.topk_w, torch.full_like(got.topk_w, 1 / 6))


def test_scores_closer_than_a_float_are_told_apart(gpu):
    """Two biases a 2^-30 apart on equal logits, and logits whose sigmoids round
    to the same float: the larger one first, in either place."""
    for lo, hi in ((3, 50), (50, 3)):
        bias = torch.zeros(64, device=gpu)
        bias[hi], bias[lo] = 2.0 ** -30 + 2.0 ** -40, 2.0 ** -30
        got = ops.moe_route_scores(torch.zeros(5, 64, device=gpu), 2, ops.Routing("sigmoid"), bias)
        assert got.topk_idx.tolist() == [[hi, lo]] * 5
        logits = torch.full((5, 64), -1.0, device=gpu)
        logits[:, hi], logits[:, lo] = 20.5, 20.25
        got = ops.moe_route_scores(logits, 2, ops.Routing("sigmoid"))
        assert got.topk_idx.tolist() == [[hi, lo]] * 5


def test_rows_without_a_live_expert(gpu):
    for routing in (ops.Routing("softmax"), ops.Routing("sigmoid", 8, 3, 2)):
        logits = torch.full((3, 64), -math.inf, device=gpu)
        logits[1, 7] = 0.5  # one live expert for four slots
        bias = torch.ones(64, device=gpu)
        got = ops.moe_route_scores(logits, 4, routing, bias)
        assert got.topk_idx[0].tolist() == [0, 1, 2, 3] and got.topk_w[0].tolist() == [0.0] * 4
        live = got.topk_idx[1].tolist()
        if routing.n_groups == 1:
            assert live == [7, 0, 1, 2] and got.topk_w[1].tolist() == [1.0, 0.0, 0.0, 0.0]
        assert len(set(live)) == 4


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_odd_logits_and_biases(gpu, score):
    """NaN, infinities and biases that are none: valid distinct experts, NaN
    weights only in the rows that say so; neighbours are left alone."""
    logits = torch.randn(6, 64, device=gpu)
    logits[1, 3], logits[2, 5], logits[3, 9] = math.nan, math.inf, -math.inf
    plain = ops.moe_route_scores(logits[4:].contiguous(), 4, ops.Routing(score, 8, 4, 2))
    bias = torch.zeros(64, device=gpu)
    got = ops.moe_route_scores(logits, 4, ops.Routing(score, 8, 4, 2), bias)
    assert torch.isnan(got.topk_w[1]).all() and got.topk_idx[1].tolist() == [0, 1, 2, 3]
    if score == "softmax":
        assert torch.isnan(got.topk_w[2]).all()
    else:
        assert got.topk_idx[2, 0] == 5 and torch.isfinite(got.topk_w[2]).all()
    assert torch.isfinite(got.topk_w[3]).all()
    assert torch.equal(got.topk_idx[4:], plain.topk_idx) and torch.equal(got.topk_w[4:], plain.topk_w)
    bias[0], bias[1], bias[2], bias[9] = math.nan, math.inf, -math.inf, -math.inf
    got = ops.moe_route_scores(logits, 4, ops.Routing(score, 8, 4, 2), bias)
    idx = got.topk_idx.cpu()
    assert ((idx >= 0) & (idx < 64)).all() and all(len(set(r.tolist())) == 4 for r in idx)


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype,weight_dtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                                (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("t,e,k,routing", CASES)
def test_route_scores_grad(gpu, t, e, k, routing, dtype, weight_dtype, masked):
    logits, bias = _inputs(gpu, t, e, dtype, masked, True, seed=1)
    dw = torch.randn(t, k, generator=torch.Generator().manual_seed(2)).to(weight_dtype).to(gpu)
    r = ops.moe_route_scores(logits, k, routing, bias, weight_dtype)
    got = ops.moe_route_scores_grad(logits, r.topk_idx, r.topk_w, dw, routing)
    ref = R.route_grad(logits, k, routing, bias, dw)
    s, chosen, live = R.choose(logits, k, routing, bias)
    v = torch.where(live, s.gather(1, chosen), 0.0)
    total = v.sum(-1, keepdim=True)
    # |ds| s is at most |scale| 2 max |dw| (renormalised: s / S <= 1)
    size = abs(routing.scale) * 2.0 * dw.double().abs().amax(-1, keepdim=True)
    size = size * (torch.where(total > 0, v / total.clamp_min(1e-300), 0.0).amax(-1, keepdim=True)
                   if routing.renormalise else v.amax(-1, keepdim=True))
    assert got.dtype == dtype
    err = (got.double() - ref).abs()
    assert (err <= (REL + HALF[dtype]) * ref.abs() + 2.0 ** -16 * size).all(), (err - HALF[dtype] * ref.abs()).max()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_gradient_of_weights_that_cannot_change(gpu, score):
    """Renormalised, the weight of one expert alone is constant: no gradient, not a
    rounding's worth. The same where the others are off, and for equal dw; and of a
    softmax nothing at the experts that were not chosen."""
    logits, _ = _inputs(gpu, 300, 384, torch.float32, False, False)
    dw = torch.randn(300, 4, generator=torch.Generator().manual_seed(2)).to(gpu)
    for k, lo in ((1, logits), (3, logits.masked_fill(torch.arange(384, device=gpu) != 5, -math.inf))):
        r = ops.moe_route_scores(lo, k, ops.Routing(score, scale=2.5))
        assert (ops.moe_route_scores_grad(lo, r.topk_idx, r.topk_w, dw[:, :k].contiguous(), ops.Routing(score, scale=2.5)) == 0).all()
    r = ops.moe_route_scores(logits, 4, ops.Routing(score))
    assert (ops.moe_route_scores_grad(logits, r.topk_idx, r.topk_w, dw[:, :1].expand(-1, 4).contiguous(), ops.Routing(score)) == 0).all()
    got = ops.moe_route_scores_grad(logits, r.topk_idx, r.topk_w, dw, ops.Routing(score))
    assert (got.scatter(1, r.topk_idx.long(), 0.0) == 0).all() and (got != 0).any(1).all()


def test_gradient_of_a_weight_near_one(gpu):
    """One expert far above the others: its gradient is small, and keeps its digits
    (every factor of the formula in differences within 2^-17 of its own size)."""
    logits, _ = _inputs(gpu, 200, 64, torch.float32, False, False)
    logits[:, 7] = 25.0
    dw = torch.randn(200, 4, generator=torch.Generator().manual_seed(2)).to(gpu)
    routing = ops.Routing("softmax")
    r = ops.moe_route_scores(logits, 4, routing)
    got = ops.moe_route_scores_grad(logits, r.topk_idx, r.topk_w, dw, routing)
    w = torch.softmax(logits.double().gather(1, r.topk_idx.long()), -1)
    terms = w.unsqueeze(2) * w.unsqueeze(1) * (dw.double().unsqueeze(2) - dw.double().unsqueeze(1))
    want = terms.sum(2)
    err = (got.gather(1, r.topk_idx.long()).double() - want).abs()
    assert (err <= 2.0 ** -17 * terms.abs().sum(2)).all()


def test_gradient_against_differences(gpu):
    """dw . d(weights) along random directions, by central differences of the
    64-bit weights at the kernel's choice."""
    for routing in (ops.Routing("sigmoid", scale=2.5), ops.Routing("softmax"), ops.Routing("softmax", renormalise=False)):
        gen = torch.Generator().manual_seed(3)
        logits = torch.randn(16, 24, generator=gen).to(gpu)
        dw = torch.randn(16, 5, generator=gen).to(gpu)
        r = ops.moe_route_scores(logits, 5, routing)
        got = ops.moe_route_scores_grad(logits, r.topk_idx, r.topk_w, dw, routing).double()
        chosen, live = r.topk_idx.long(), torch.ones(16, 5, dtype=torch.bool, device=gpu)

        def value(l):
            s = torch.sigmoid(l) if routing.score == "sigmoid" else torch.softmax(l, -1)
            return (R.weights(s, chosen, live, routing) * dw.double()).sum(-1)

        for _ in range(4):
            d = torch.randn(16, 24, generator=gen).double().to(gpu)
            h = 1e-5
            slope = (value(logits.double() + h * d) - value(logits.double() - h * d)) / (2 * h)
            # differences: h^2 times third derivatives (< 100); the kernel's float: 24 terms of 2^-20
            assert ((got * d).sum(-1) - slope).abs().max() < 1e-4


def test_load_and_balance_bias(gpu):
    for t, e, k in ((0, 8, 2), (1, 8, 2), (1000, 64, 6), (5000, 1024, 32)):
        logits, bias = _inputs(gpu, t, e, torch.float32, False, True, seed=4)
        r = ops.moe_route_scores(logits, k, ops.Routing("sigmoid"), bias)
        load = ops.moe_expert_load(r.chunk_hist)
        want = torch.bincount(r.topk_idx.long().view(-1), minlength=e).to(torch.int32)
        assert torch.equal(load, want)
        moved = ops.moe_balance_bias(bias, load, 0.01)
        step = torch.sign((want.sum() - e * want.long()).double()) * 0.01
        # one float addition of a rounded rate
        assert ((moved.double() - bias.double() - step).abs() <= 2.0 ** -24 * (bias.abs().double() + 0.02)).all()
        before = bias.clone()
        assert ops.moe_balance_bias(bias, load, 0.01, out=bias) is bias and torch.equal(bias, moved)
        assert torch.equal(ops.moe_balance_bias(before, load, 0.0), before)


def test_balance_bias_evens_out_the_loads(gpu):
    """A router that prefers four experts spreads out once the bias has moved far
    enough, as the plain form's does: same choices every step."""
    gen = torch.Generator().manual_seed(5)
    logits = torch.randn(512, 16, generator=gen)
    logits[:, :4] += 1.5
    logits, bias, routing = logits.to(gpu), torch.zeros(16, device=gpu), ops.Routing("sigmoid")
    first = None
    for _ in range(60):
        r = ops.moe_route_scores(logits, 2, routing, bias)
        assert torch.equal(r.topk_idx.long(), R.choose(logits, 2, routing, bias)[1])
        load = ops.moe_expert_load(r.chunk_hist)
        first = load if first is None else first
        bias = ops.moe_balance_bias(bias, load, 0.01)
    assert load.max() < first.max() // 2


def test_logits_off_16_byte_boundaries(gpu):
    for e, dtype in ((64, torch.bfloat16), (256, torch.float32)):
        logits, bias = _inputs(gpu, 50, e, dtype, False, True)
        buf = torch.zeros(50 * e + 1, dtype=dtype, device=gpu)
        buf[1:] = logits.view(-1)
        shifted = torch.zeros(e + 1, device=gpu)
        shifted[1:] = bias
        a = ops.moe_route_scores(logits, 4, ops.Routing("sigmoid", 8, 4, 2), bias)
        b = ops.moe_route_scores(buf[1:].view(50, e), 4, ops.Routing("sigmoid", 8, 4, 2), shifted[1:])
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_near_ties_in_every_place(gpu):
    """Biases that put neighbours of the order, the border of the choice and the
    border of the groups within 2^-24 of each other: still the 64-bit choice."""
    gen = torch.Generator().manual_seed(8)
    for e, routing in ((64, ops.Routing("sigmoid")), (128, ops.Routing("sigmoid", 8, 3, 2)),
                       (256, ops.Routing("softmax", 8, 4, 1)), (512, ops.Routing("sigmoid", 16, 4, 2))):
        logits = (torch.randn(300, 1, generator=gen) + 1e-6 * torch.randn(300, e, generator=gen)).to(gpu)
        bias = (torch.randn(e, generator=gen) * 2.0 ** -26).to(gpu)
        _check_route(ops.moe_route_scores(logits, 6, routing, bias), logits, 6, routing, bias, torch.float32)


@pytest.mark.parametrize("e,groups,kept", [(32, 4, 2), (64, 8, 3), (64, 4, 2), (128, 2, 1), (256, 8, 4), (256, 2, 1),
                                           (256, 16, 5), (192, 6, 2), (512, 2, 1), (512, 16, 4), (1024, 2, 1),
                                           (1024, 32, 8), (160, 8, 3), (96, 32, 9)])
@pytest.mark.parametrize("top", [1, 2])
def test_groups_of_every_width(gpu, e, groups, kept, top):
    """Groups of part of a lane's experts up to half of all lanes', coarse logits with
    many exact ties, with and without a bias, some experts off."""
    gen = torch.Generator().manual_seed(e + groups)
    for score in ("sigmoid", "softmax"):
        routing = ops.Routing(score, groups, kept, top)
        for dtype in (torch.bfloat16, torch.float32):
            for bias in (None, torch.zeros(e, device=gpu), torch.randn(e, generator=gen).to(gpu)):
                logits = torch.randn(70, e, generator=gen).to(torch.bfloat16).to(dtype)
                logits[torch.rand(70, e, generator=gen) < 0.1] = -math.inf
                logits = logits.to(gpu)
                _check_route(ops.moe_route_scores(logits, 3, routing, bias), logits, 3, routing, bias, dtype)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_logits_that_differ_in_their_last_bits(gpu, score):
    """Neighbours a unit in the last place apart, at every size: the larger first,
    also of group maxima."""
    gen = torch.Generator().manual_seed(4)
    for e, routing in ((64, ops.Routing(score)), (128, ops.Routing(score, 8, 3, 1)), (60, ops.Routing(score, 6, 2, 1)),
                       (256, ops.Routing(score, 8, 4, 2))):
        base = torch.randn(200, 1, generator=gen)
        steps = torch.randint(-20, 20, (200, e), generator=gen, dtype=torch.int32)
        logits = (base.view(torch.int32) + steps).view(torch.float32).to(gpu)
        _check_route(ops.moe_route_scores(logits, 6, routing), logits, 6, routing, None, torch.float32)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_logits_at_the_ends_of_their_range(gpu, score):
    """Masks of the lowest float and scores that are 0 or 1 in 64 bits: the order of the
    logits, weight 0 where the score is 0."""
    for dtype in (torch.float32, torch.bfloat16):
        low = torch.finfo(dtype).min
        logits = torch.full((4, 64), low, dtype=dtype, device=gpu)
        logits[0, 9] = logits[0, 3] = 0.5
        logits[1, 40], logits[1, 7] = -800.0, -900.0
        logits[2, 5], logits[2, 6] = 60.0, 62.0
        r = ops.moe_route_scores(logits, 3, ops.Routing(score))
        assert r.topk_idx.tolist() == [[3, 9, 0], [40, 7, 0], [6, 5, 0], [0, 1, 2]]
        assert torch.isfinite(r.topk_w).all() and (r.topk_w[0, :2] == 0.5).all() and (r.topk_w[0, 2] == 0).all()
        g = ops.moe_route_scores_grad(logits, r.topk_idx, r.topk_w, torch.ones_like(r.topk_w), ops.Routing(score))
        assert (g == 0).all()


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_scores_below_every_float_keep_their_share(gpu, score):
    """Chosen experts (by the bias alone) whose scores are 1e-45 to 1e-275: the weights
    and their gradient are those of 64 bits."""
    gen = torch.Generator().manual_seed(9)
    logits = torch.randn(100, 64, generator=gen)
    logits[:, 10:14] = -torch.rand(100, 1, generator=gen) * 500.0 - 120.0 + torch.randn(100, 4, generator=gen) * 5.0
    logits, bias = logits.to(gpu), torch.zeros(64, device=gpu)
    bias[10:14] = torch.tensor([40.0, 30.0, 20.0, 10.0], device=gpu)
    routing = ops.Routing(score, scale=2.5)
    r = ops.moe_route_scores(logits, 4, routing, bias)
    _check_route(r, logits, 4, routing, bias, torch.float32)
    dw = torch.randn(100, 4, generator=gen).to(gpu)
    got = ops.moe_route_scores_grad(logits, r.topk_idx, r.topk_w, dw, routing)
    l = logits.double().gather(1, r.topk_idx.long())
    w = torch.softmax(l, -1)  # (a sigmoid of these is exp(l), and 1 - s is 1)
    terms = w.unsqueeze(2) * w.unsqueeze(1) * (dw.double().unsqueeze(2) - dw.double().unsqueeze(1)) * 2.5
    err = (got.gather(1, r.topk_idx.long()).double() - terms.sum(2)).abs()
    # a difference d of logits, at most 40, is rounded by |d| 2^-24 < 2^-18, which is the
    # relative error of its exponential; r is a quotient of two such (2^-17), a term a
    # product of two r
    assert (err <= 2.0 ** -15 * terms.abs().sum(2) + 1e-38).all()


def test_large_biases_that_cancel_in_a_group(gpu):
    """Group values whose parts are far larger than their sums: rounded in 32 bits they
    lose what tells the groups apart."""
    gen = torch.Generator().manual_seed(6)
    for e, groups in ((64, 8), (160, 8)):
        per = e // groups
        bias = torch.full((e,), -4096.0)
        bias[::per], bias[1::per] = 4096.0, -4095.0
        logits = torch.randn(200, e, generator=gen).to(gpu)
        routing = ops.Routing("sigmoid", groups, 3, 2)
        bias = bias.to(gpu)
        _check_route(ops.moe_route_scores(logits, 4, routing, bias), logits, 4, routing, bias, torch.float32)


def test_captured_training_side_replays(gpu):
    """Routing, gradient, load and the bias's step in one graph: every replay on new
    logits as the eager calls, with eager work of other sizes in between."""
    routing = ops.Routing("sigmoid", 8, 4, 2, True, 2.5)
    gen = torch.Generator().manual_seed(3)
    logits, bias = torch.randn(700, 128, generator=gen).to(gpu), torch.zeros(128, device=gpu)
    dw = torch.randn(700, 8, generator=gen).to(gpu)

    def step(b):
        r = ops.moe_route_scores(logits, 8, routing, b)
        g = ops.moe_route_scores_grad(logits, r.topk_idx, r.topk_w, dw, routing)
        load = ops.moe_expert_load(r.chunk_hist)
        return (*r, g, load, ops.moe_balance_bias(b, load, 0.01, out=b))

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        step(bias.clone())
        with torch.cuda.graph(graph, stream=stream):
            got = step(bias)
    torch.cuda.current_stream().wait_stream(stream)
    eager = torch.zeros(128, device=gpu)
    for i in range(4):
        logits.copy_(torch.randn(700, 128, generator=gen))
        graph.replay()
        want = step(eager)
        for a, b in zip(got, want):
            assert torch.equal(a, b), i
        ops.moe_route_scores(torch.randn(50 + i, 60, device=gpu), 4)
        torch.cuda.synchronize()
    assert (bias != 0).any()


def test_no_tokens(gpu):
    r = ops.moe_route_scores(torch.empty(0, 64, device=gpu), 4)
    assert r.topk_idx.shape == (0, 4) and r.chunk_hist.shape == (0, 64)
    assert ops.moe_route_scores_grad(torch.empty(0, 64, device=gpu), r.topk_idx, r.topk_w, r.topk_w).shape == (0, 64)


def test_route_scores_refusals(gpu):
    logits = torch.zeros(4, 64, device=gpu)
    bad = [dict(routing=ops.Routing("tanh")), dict(routing=ops.Routing(n_groups=7)),
           dict(routing=ops.Routing(n_groups=8, topk_groups=9)), dict(routing=ops.Routing(n_groups=32, topk_groups=1)),
           dict(routing=ops.Routing(n_groups=64, topk_groups=8, group_top=2)), dict(routing=ops.Routing(group_top=3)),
           dict(routing=ops.Routing(scale=math.inf)), dict(bias=torch.zeros(63, device=gpu)),
           dict(bias=torch.zeros(64, dtype=torch.bfloat16, device=gpu)), dict(bias=torch.zeros(64)),
           dict(weight_dtype=torch.float16)]
    for kwargs in bad:
        with pytest.raises(ValueError):
            ops.moe_route_scores(logits, 4, **kwargs)
    for k in (0, 33, 65):
        with pytest.raises(ValueError, match="top_k"):
            ops.moe_route_scores(logits, k)
    with pytest.raises(ValueError, match="contiguous"):
        ops.moe_route_scores(logits.t(), 2)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        ops.moe_route_scores(logits.half(), 2)
    r = ops.moe_route_scores(logits, 4)
    for args in ((r.topk_idx.long(), r.topk_w, r.topk_w), (r.topk_idx, r.topk_w[:2], r.topk_w),
                 (r.topk_idx, r.topk_w, r.topk_w.bfloat16())):
        with pytest.raises(ValueError):
            ops.moe_route_scores_grad(logits, *args)
    with pytest.raises(ValueError):
        ops.moe_expert_load(r.chunk_hist.long())
    load = ops.moe_expert_load(r.chunk_hist)
    for args in ((torch.zeros(63, device=gpu), load, 0.1), (torch.zeros(64, device=gpu), load, math.nan),
                 (torch.zeros(64, device=gpu).double(), load, 0.1)):
        with pytest.raises(ValueError):
            ops.moe_balance_bias(*args)


@pytest.mark.parametrize("t,e,k,routing", [(33, 64, 8, ops.Routing("sigmoid", 8, 4, 2)), (700, 160, 6, ops.Routing())])
def test_captured_routing_replays(gpu, t, e, k, routing):
    """Choice, gradient, load and bias captured in one graph: every replay equals
    the eager calls, with eager work between and on refilled inputs."""
    logits, bias = _inputs(gpu, t, e, torch.float32, False, True)
    dw = torch.randn(t, k, device=gpu)

    def step():
        r = ops.moe_route_scores(logits, k, routing, bias)
        load = ops.moe_expert_load(r.chunk_hist)
        return (*r, ops.moe_route_scores_grad(logits, r.topk_idx, r.topk_w, dw, routing), load,
                ops.moe_balance_bias(bias, load, 0.01))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        logits.copy_(_inputs(gpu, t, e, torch.float32, i % 2 == 1, False, seed=10 + i)[0])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)

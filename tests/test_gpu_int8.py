"""Products in 8-bit integers against the plain 64-bit forms of
``oracle/operators_ref.py``.

Codes are compared for equality, sums of code products are exact. Tolerances of a
dense product: the sum's conversion, the scales' product, the multiplication and
the bias' addition round once each, 4 * 2^-24 of |product| + |bias|; then half a
step of the output's type.

Of an expert: a bf16 h whose 32-bit value is next to a border between two bf16
values (within 2^-20 of it, a share of 2^-20 / 2^-9 = 2^-11 of the values) may
round to the other one, a step of 2^-7 of it, which moves its code by at most one
(127 * 2^-7 < 1). A code is a step of 1/127 of the row's largest |h|, itself at
most 8 times its rms here, so the h behind the down product is off by
sqrt(2^-11) * 8 / 127 = 1.4e-3 of its norm at most, and so is the output. The
roundings of y and of the output to bf16 add 2^-8 each: 2^-8 * 2 + 1.4e-3 < 1e-2. An fp32 h
is rounded once from 64 bits: its codes are the plain form's, and 2^-18 covers the
few roundings of the sums after them.
"""

from __future__ import annotations

import math

import pytest
import torch

from astrai_amd.extension import ops
from oracle import operators_ref as R

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
LAYER_REL = {torch.bfloat16: 1e-2, torch.float32: 2.0 ** -18}
DTYPES = [torch.bfloat16, torch.float32]


def _randn(gpu, *shape, seed=0, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).to(gpu)


# -- quantisation -----------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 15), (3, 16), (5, 17), (7, 64), (64, 100), (33, 513), (4, 1000), (9, 1024),
                                    (300, 2048), (2, 4097), (5, 8192), (3, 14336), (1, 20001), (1, 131072)])
def test_quantize_rows(gpu, rows, k, dtype):
    x = _randn(gpu, rows, k, seed=k, dtype=dtype)
    x[0, k // 2] *= 6.0
    q, scale = ops.quantize_rows(x)
    want, s = R.quantize(x)
    assert q.shape == (rows, -(-k // 16) * 16) and (q[:, k:] == 0).all()
    assert torch.equal(q[:, :k].double(), want)
    assert torch.equal(scale, s.squeeze(-1).float())


@pytest.mark.parametrize("dtype", DTYPES)
def test_values_at_the_border_of_two_codes(gpu, dtype):
    """max / 2 is 63.5 codes for every max, and a max of 254 steps has every half:
    halves go to the even code."""
    most = torch.arange(1, 256).double()
    x = torch.stack([most, most / 2, -most / 2, most / 4], 1).to(dtype).to(gpu)
    q, _ = ops.quantize_rows(x)
    assert torch.equal(q[:, :4].double(), R.quantize(x)[0])
    assert (q[:, 1] == 64).all() and (q[:, 2] == -64).all()
    x = torch.cat([torch.tensor([254.0]), torch.arange(-253.0, 254.0, 2.0)]).unsqueeze(0).to(dtype).to(gpu)
    q, _ = ops.quantize_rows(x)
    n = torch.arange(-253, 254, 2).double() / 2
    assert torch.equal(q[0, 1:255].cpu().double(), torch.round(n))


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_out_of_the_ordinary(gpu, dtype):
    big, small = torch.finfo(dtype).max, torch.finfo(dtype).tiny
    x = torch.zeros(10, 40, dtype=dtype, device=gpu)
    x[1, 3] = math.inf
    x[2, 39] = math.nan
    x[3, 5], x[3, 6] = -math.inf, 1.0
    x[4, ::3], x[4, 1] = big, -big / 2
    x[5, ::2], x[5, 1] = small, small / 2
    x[6, 7], x[6, 8] = small / 64, -small / 128  # denormal
    x[7, 0], x[7, 1] = big, small
    x[8, 0], x[8, 1] = -0.0, 0.0
    x[9] = torch.linspace(-3, 3, 40).to(dtype)
    q, scale = ops.quantize_rows(x)
    assert (q[:4] == 0).all() and scale[0] == 0 and torch.isnan(scale[1:4]).all()
    ok = [4, 5, 6, 7, 8, 9]
    want, s = R.quantize(x[ok])
    assert torch.equal(q[ok, :40].double(), want)
    assert torch.equal(scale[ok], s.squeeze(-1).float())


def test_quantize_rows_takes_stacks_and_none(gpu):
    x = _randn(gpu, 3, 5, 33)
    q, scale = ops.quantize_rows(x)
    assert q.shape == (3, 5, 48) and scale.shape == (3, 5)
    assert torch.equal(q.view(15, 48), ops.quantize_rows(x.view(15, 33))[0])
    q, scale = ops.quantize_rows(torch.empty(0, 7, device=gpu))
    assert q.shape == (0, 16) and scale.shape == (0,)


# -- the dense product --------------------------------------------------------------


def _weight(gpu, n, k, seed):
    return ops.quantize_rows(_randn(gpu, n, k, seed=seed, std=0.02))


SHAPES = [(1, 1, 1), (1, 16, 8), (2, 17, 9), (1, 64, 64), (1, 4096, 1000), (5, 100, 130), (16, 128, 256), (17, 130, 72),
          (31, 256, 264), (33, 1000, 2664), (64, 512, 1024), (65, 2047, 1001), (100, 128, 8), (127, 272, 136),
          (129, 704, 576), (200, 1408, 2048), (256, 256, 512), (300, 4096, 520), (333, 2880, 776), (513, 640, 1032),
          (1030, 144, 2056), (2100, 520, 264)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_int8_linear(gpu, m, k, n, dtype):
    x = _randn(gpu, m, k, seed=1, dtype=dtype)
    w, ws = _weight(gpu, n, k, 2)
    if w.shape[1] > k:
        w[:, k:] = 55  # what lies behind a weight row's last column does not matter
    for bias in (None, _randn(gpu, n, seed=3, dtype=dtype)):
        got = ops.int8_linear(x, w, ws, bias)
        want = R.int8_linear(x, w, ws, bias)
        size = R.int8_linear(x, w, ws).abs() + (0 if bias is None else bias.double().abs())
        assert got.shape == (m, n) and got.dtype == dtype
        err = (got.double() - want).abs()
        assert (err <= 4 * 2.0 ** -24 * size + HALF[dtype] * want.abs()).all(), (err / size.clamp_min(1e-30)).max()


def test_sums_at_the_limit_of_32_bits(gpu):
    """Codes of 127 against -128 over the longest row: -2130706432 = 127 * -128 * 131072 - ... stays exact."""
    k = ops.INT8_MAX_K
    x = torch.ones(2, k, device=gpu)
    x[1] = -1.0
    w = torch.full((16, k), -128, dtype=torch.int8, device=gpu)
    w[1::2] = 127
    got = ops.int8_linear(x, w, torch.ones(16, device=gpu))
    scale = (torch.ones(1) / 127).double().item()
    for r, sign in ((0, 1.0), (1, -1.0)):
        for c, v in ((0, -128), (1, 127)):
            want = sign * 127.0 * v * k * scale
            assert abs(got[r, c].item() - want) <= 4 * 2.0 ** -24 * abs(want)


@pytest.mark.parametrize("m", [3, 200, 700])
def test_rows_that_hold_no_number(gpu, m):
    """A row with a NaN or an infinity comes out NaN, a row of zeros as the bias,
    and neither touches its neighbours."""
    x = _randn(gpu, m, 640, dtype=torch.bfloat16)
    w, ws = _weight(gpu, 264, 640, 2)
    bias = _randn(gpu, 264, seed=3, dtype=torch.bfloat16)
    clean = ops.int8_linear(x, w, ws, bias)
    x[0, 5], x[2] = math.nan, 0.0
    if m > 100:
        x[m - 1, 0] = -math.inf
    got = ops.int8_linear(x, w, ws, bias)
    assert torch.isnan(got[0]).all() and torch.equal(got[2], bias) and torch.equal(got[1], clean[1])
    assert torch.equal(got[3:m - 1], clean[3:m - 1])
    if m > 100:
        assert torch.isnan(got[m - 1]).all()


@pytest.mark.parametrize("m,k,n", [(1, 512, 520), (70, 1000, 264), (600, 512, 1032)])
def test_out_is_written_where_it_belongs(gpu, m, k, n):
    """``out`` inside a larger buffer: nothing before or behind it changes."""
    x = _randn(gpu, m, k, dtype=torch.bfloat16)
    w, ws = _weight(gpu, n, k, 2)
    buf = torch.full((m + 2, n), 7.0, dtype=torch.bfloat16, device=gpu)
    got = ops.int8_linear(x, w, ws, out=buf[1:m + 1])
    assert torch.equal(got, ops.int8_linear(x, w, ws)) and got.data_ptr() == buf[1:].data_ptr()
    assert (buf[0] == 7).all() and (buf[m + 1] == 7).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", [(1, 512, 520), (20, 640, 264), (70, 1000, 264), (600, 512, 1032), (300, 512, 1000)])
def test_operands_off_16_byte_boundaries(gpu, m, k, n, dtype):
    """x, out, bias and scales that start one value behind a boundary: the same
    bits as aligned ones, and no neighbour of out written."""
    def shifted(t, fill=0.0):
        buf = torch.full((t.numel() + 2,), fill, dtype=t.dtype, device=gpu)
        buf[1:-1] = t.reshape(-1)
        return buf, buf[1:-1].view(t.shape)

    x = _randn(gpu, m, k, dtype=dtype)
    w, ws = _weight(gpu, n, k, 2)
    bias = _randn(gpu, n, seed=3, dtype=dtype)
    want = ops.int8_linear(x, w, ws, bias)
    buf, out = shifted(torch.zeros_like(want), 7.0)
    got = ops.int8_linear(shifted(x)[1], w, shifted(ws)[1], shifted(bias)[1], out=out)
    assert torch.equal(got, want) and buf[0] == 7.0 and buf[-1] == 7.0
    q, s = ops.quantize_rows(shifted(x)[1])
    want_q, want_s = ops.quantize_rows(x)
    assert torch.equal(q, want_q) and torch.equal(s, want_s)


def test_codes_past_4_gib(gpu):
    """Rows whose codes lie past 32-bit offsets have the bits that they have alone: a
    Linear's, which are counted from their tile, and a layer's, which are gathered."""
    k, m, n = 131072, 2 ** 15 + 70, 40
    some = torch.tensor([0, 1, 31, 16383, 16384, 2 ** 15 - 1, 2 ** 15, 2 ** 15 + 69], device=gpu)
    x = torch.empty(m, k, dtype=torch.bfloat16, device=gpu)
    gen = torch.Generator(gpu).manual_seed(1)
    for i in range(0, m, 4096):
        x[i:i + 4096].normal_(generator=gen)
    w, ws = _weight(gpu, n, k, 2)
    few = x[some].contiguous()
    assert torch.equal(ops.int8_linear(x, w, ws)[some], ops.int8_linear(few, w, ws))
    experts = _experts(gpu, 2, k, 24)
    logits = torch.randn(m, 2, generator=gen, device=gpu)
    got = ops.moe_int8_forward(x, logits, experts, 1, routing=ops.Routing("sigmoid"))[some]
    want = ops.moe_int8_forward(few, logits[some].contiguous(), experts, 1, routing=ops.Routing("sigmoid"))
    assert torch.equal(got, want)


def test_rows_do_not_depend_on_their_company(gpu):
    """Exact sums: a row's bits are the same in every batch, whatever kernel its
    size takes."""
    w, ws = _weight(gpu, 1032, 1000, 2)
    x = _randn(gpu, 3000, 1000, dtype=torch.bfloat16)
    whole = ops.int8_linear(x, w, ws)
    for m in (1, 2, 16, 40, 64, 100, 129, 256, 300, 700, 1500):
        assert torch.equal(ops.int8_linear(x[:m].contiguous(), w, ws), whole[:m]), m


# -- experts --------------------------------------------------------------------------


def _experts(gpu, n, dim, dim_ffn, seed=0):
    parts = [ops.quantize_rows(_randn(gpu, n, a, b, seed=seed + i, std=0.02 if i < 2 else 0.05))
             for i, (a, b) in enumerate(((dim_ffn, dim), (dim_ffn, dim), (dim, dim_ffn)))]
    return ops.Int8Experts(*(q for q, _ in parts), *(s for _, s in parts))


def _layer(x, logits, experts, top_k, n_shared, routing, bias):
    s, chosen, live = R.choose(logits, top_k, routing, bias)
    w = R.weights(s, chosen, live, routing).to(x.dtype)
    return R.int8_layer(x, chosen, w, experts, n_shared)


# (tokens, dim, dim_ffn, experts, top_k, shared, routing)
LAYERS = [
    (1, 64, 64, 4, 1, 0, ops.Routing()),
    (1, 512, 1024, 8, 2, 1, ops.Routing("sigmoid", scale=2.5)),
    (3, 100, 37, 5, 2, 2, ops.Routing()),
    (17, 129, 136, 8, 3, 1, ops.Routing("softmax", renormalise=False)),
    (32, 512, 1024, 8, 2, 0, ops.Routing()),
    (33, 704, 576, 16, 4, 1, ops.Routing("sigmoid", 4, 2, 2, True, 2.5)),
    (64, 256, 384, 64, 8, 0, ops.Routing("sigmoid", 8, 4, 2)),
    (130, 1000, 2664, 8, 2, 2, ops.Routing()),
    (333, 2048, 1408, 16, 4, 1, ops.Routing()),
    (700, 512, 1024, 8, 2, 1, ops.Routing("softmax", 4, 2)),
    (1500, 640, 520, 4, 2, 0, ops.Routing("sigmoid")),
    (4096, 512, 1024, 8, 2, 1, ops.Routing()),
    (300, 256, 256, 1, 1, 1, ops.Routing()),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,dim,dim_ffn,e,k,shared,routing", LAYERS)
def test_int8_layer(gpu, t, dim, dim_ffn, e, k, shared, routing, dtype):
    x = _randn(gpu, t, dim, seed=1, dtype=dtype)
    logits, bias = _randn(gpu, t, e, seed=2), _randn(gpu, e, seed=3, std=0.1)
    experts = _experts(gpu, e + shared, dim, dim_ffn)
    got = ops.moe_int8_forward(x, logits, experts, k, shared, routing, bias)
    want = _layer(x, logits, experts, k, shared, routing, bias)
    assert got.shape == x.shape and got.dtype == dtype
    assert (got.double() - want).norm() <= LAYER_REL[dtype] * want.norm()
    # and no single value is far off: 32 codes of the largest term of the down product
    assert (got.double() - want).abs().max() <= 8 * LAYER_REL[dtype] * want.abs().max()


@pytest.mark.parametrize("t", [5, 40, 900])
def test_one_expert_takes_every_token(gpu, t):
    x = _randn(gpu, t, 256, dtype=torch.bfloat16)
    logits = torch.zeros(t, 8, device=gpu)
    logits[:, 5] = 9.0
    experts = _experts(gpu, 8, 256, 320)
    got = ops.moe_int8_forward(x, logits, experts, 1, routing=ops.Routing())
    want = R.int8_mlp(x, *(p[5] for p in experts)).double()
    assert (got.double() - want).norm() <= LAYER_REL[torch.bfloat16] * want.norm()


def test_switched_off_experts_and_padding_rows(gpu):
    """Tokens with every expert off come out as zeros, whatever their rows hold
    that is finite; tokens with one live expert for two slots get that one."""
    x = _randn(gpu, 50, 256, dtype=torch.bfloat16)
    x[10:20] = 1e30
    logits = _randn(gpu, 50, 8, seed=2)
    logits[10:20] = -math.inf
    logits[20:25, 1:] = -math.inf
    experts = _experts(gpu, 8, 256, 320)
    got = ops.moe_int8_forward(x, logits, experts, 2, routing=ops.Routing())
    assert (got[10:20] == 0).all() and torch.isfinite(got).all()
    want = R.int8_mlp(x[20:25], *(p[0] for p in experts)).double()
    assert (got[20:25].double() - want).norm() <= LAYER_REL[torch.bfloat16] * want.norm()


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_reference_routing(gpu, dtype):
    """Without a routing: moe_route's choice and weights."""
    t, dim, e, k, shared = 100, 256, 8, 2, 1
    x, logits = _randn(gpu, t, dim, dtype=dtype), _randn(gpu, t, e, seed=2, dtype=dtype)
    experts = _experts(gpu, e + shared, dim, 320)
    got = ops.moe_int8_forward(x, logits, experts, k, shared)
    r = ops.moe_route(logits, k)
    want = R.int8_layer(x, r.topk_idx.long(), r.topk_w, experts, shared)
    assert (got.double() - want).norm() <= LAYER_REL[dtype] * want.norm()


def test_tokens_do_not_depend_on_their_company(gpu):
    experts = _experts(gpu, 9, 512, 520)
    x, logits = _randn(gpu, 2000, 512, dtype=torch.bfloat16), _randn(gpu, 2000, 8, seed=2)
    whole = ops.moe_int8_forward(x, logits, experts, 2, 1, ops.Routing())
    for t in (1, 16, 33, 100, 400, 1000):
        part = ops.moe_int8_forward(x[:t].contiguous(), logits[:t].contiguous(), experts, 2, 1, ops.Routing())
        assert torch.equal(part, whole[:t]), t


def test_no_tokens(gpu):
    experts = _experts(gpu, 4, 64, 64)
    x = torch.empty(0, 64, dtype=torch.bfloat16, device=gpu)
    assert ops.moe_int8_forward(x, torch.empty(0, 4, device=gpu), experts, 2, routing=ops.Routing()).shape == (0, 64)
    w, ws = _weight(gpu, 8, 64, 0)
    assert ops.int8_linear(x, w, ws).shape == (0, 8)


@pytest.mark.parametrize("t", [1, 48, 600])
def test_captured_forward_replays(gpu, t):
    """A linear and a layer captured together, replayed on refilled inputs with
    eager calls between: every replay equals the eager calls."""
    x, logits = _randn(gpu, t, 512, dtype=torch.bfloat16), _randn(gpu, t, 8, seed=2)
    experts = _experts(gpu, 9, 512, 1024)
    w, ws = _weight(gpu, 512, 512, 9)

    def step():
        y = ops.int8_linear(x, w, ws)
        return y, ops.moe_int8_forward(y, logits, experts, 2, 1, ops.Routing())

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        x.copy_(_randn(gpu, t, 512, seed=20 + i, dtype=torch.bfloat16))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, step()):
            assert torch.equal(a, b)


def test_calls_on_two_streams(gpu):
    """Overlapping calls on two streams, each with its own workspace."""
    experts = _experts(gpu, 8, 512, 1024)
    xs = [_randn(gpu, 300, 512, seed=s, dtype=torch.bfloat16) for s in (1, 2)]
    logits = _randn(gpu, 300, 8, seed=3)
    want = [ops.moe_int8_forward(x, logits, experts, 2, routing=ops.Routing()) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.moe_int8_forward(xs[i], logits, experts, 2, routing=ops.Routing()))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert torch.equal(g, want[i])


def test_int8_refusals(gpu):
    x = _randn(gpu, 4, 64, dtype=torch.bfloat16)
    w, ws = _weight(gpu, 24, 64, 0)
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        ops.quantize_rows(x.half())
    with pytest.raises(ValueError, match="row length"):
        ops.quantize_rows(torch.empty(2, ops.INT8_MAX_K + 1, device=gpu))
    with pytest.raises(ValueError, match="row length"):
        ops.quantize_rows(torch.empty(2, 0, device=gpu))
    bad = [(x, w[:, :48].contiguous(), ws), (x, w.float(), ws), (x, w, ws[:8]), (x, w, ws.bfloat16()), (x.t(), w, ws),
           (x, w.cpu(), ws), (x, w, ws, ws), (x[:, :40].contiguous(), w, ws),
           (x, torch.empty(24 * 64 + 16, dtype=torch.int8, device=gpu)[8:8 + 24 * 64].view(24, 64), ws)]
    for args in bad:
        with pytest.raises(ValueError):
            ops.int8_linear(*args)
    square, sq = _weight(gpu, 64, 64, 0)
    with pytest.raises(ValueError, match="overlap"):
        ops.int8_linear(x, square, sq, out=x)
    with pytest.raises(ValueError, match="out must be"):
        ops.int8_linear(x, w, ws, out=torch.empty(4, 23, dtype=torch.bfloat16, device=gpu))
    experts = _experts(gpu, 5, 64, 96)
    logits = torch.zeros(4, 4, device=gpu)
    good = dict(x=x, logits=logits, experts=experts, top_k=2, n_shared=1, routing=ops.Routing())
    ops.moe_int8_forward(**good)
    for change in (dict(n_shared=0), dict(n_shared=2), dict(n_shared=-1), dict(top_k=0), dict(top_k=5), dict(top_k=32),
                   dict(logits=logits[:2]), dict(routing=None), dict(bias=torch.zeros(3, device=gpu)),
                   dict(experts=experts._replace(up=experts.up[:, :80].contiguous())),
                   dict(experts=experts._replace(down_scale=experts.gate_scale)),
                   dict(experts=experts._replace(gate=experts.gate.float()))):
        with pytest.raises(ValueError):
            ops.moe_int8_forward(**{**good, **change})

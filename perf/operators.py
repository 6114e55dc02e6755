"""Timed cases of the routing by scores, the 8-bit product and the 8-bit experts.

Three operators:

* ``"route"``: experts chosen by softmax or sigmoid scores with a bias for
  balance, groups of experts, top-k and renormalised weights; with ``train``
  also the logits' gradient, the experts' loads and the updated bias;
* ``"linear"``: ``x [M, K] . w [N, K]^T`` in 8-bit integers with a scale for
  each token (taken from x in the call) and each output channel, and a bias;
* ``"experts"``: a layer of routed SwiGLU experts (and shared ones) whose
  products run in 8-bit integers, from the router's logits to the output.

``run`` computes them in torch's elementary operations, or, where ``own`` is
set, with the calls a program makes of the package.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_RATE = 1e-3  # step of the balance bias


def _route(name, tokens, experts, top_k, score, groups=1, kept=1, group_top=1, bias=False, renorm=True, scale=1.0,
           dtype="fp32", weights="bf16", masked=0.0, train=False):
    c = {"op": "route", "tokens": tokens, "experts": experts, "top_k": top_k, "score": score, "groups": groups,
         "kept": kept, "group_top": group_top, "bias": bias, "renorm": renorm, "scale": scale, "dtype": dtype,
         "weights": weights, "masked": masked, "train": train}
    return {"name": name, **c} if name else c


def _linear(name, rows, k, n, dtype="bf16", bias=False):
    c = {"op": "linear", "rows": rows, "k": k, "n": n, "dtype": dtype, "bias": bias}
    return {"name": name, **c} if name else c


def _experts(name, tokens, dim, dim_ffn, experts, top_k, shared=0, dtype="bf16", score="softmax", groups=1, kept=1,
             group_top=1, bias=False, scale=1.0, skew=0.0):
    c = {"op": "experts", "tokens": tokens, "dim": dim, "dim_ffn": dim_ffn, "experts": experts, "top_k": top_k,
         "shared": shared, "dtype": dtype, "score": score, "groups": groups, "kept": kept, "group_top": group_top,
         "bias": bias, "renorm": True, "scale": scale, "skew": skew}
    return {"name": name, **c} if name else c


def listed():
    return [
        # a decoding batch through a router of many experts in groups: launches and latency
        _route("route_decode_64_e128", 64, 128, 8, "sigmoid", groups=8, kept=4, group_top=2, bias=True, scale=2.5),
        # a chunk of a prompt, softmax scores as they are, some experts switched off and some tokens padding
        _route("route_chunk_333_e60", 333, 60, 4, "softmax", renorm=False, dtype="bf16", masked=0.1),
        # prompts prefilled together, the largest router
        _route("route_prefill_16384_e256", 16384, 256, 8, "sigmoid", groups=8, kept=4, group_top=2, bias=True,
               scale=2.5),
        # a training step's routing: weights, the logits' gradient, loads and the new bias
        _route("route_train_8192_e64", 8192, 64, 6, "sigmoid", bias=True, dtype="bf16", train=True),
        # the same of softmax scores whose best groups are taken by their best expert
        _route("route_train_700_e160", 700, 160, 6, "softmax", groups=8, kept=3, dtype="fp32", weights="fp32",
               train=True),
        # one token through a wide projection: its weights stream once
        _linear("linear_1_wide", 1, 4096, 14336),
        # a ragged chunk through a projection with bias whose sizes are no multiples of 64, in fp32
        _linear("linear_333_ragged_fp32", 333, 1000, 2664, dtype="fp32", bias=True),
        # prompts prefilled together through a wide projection
        _linear("linear_8192_wide", 8192, 4096, 14336),
        # one sequence decoding through a small layer with a shared expert
        _experts("experts_1_small", 1, 512, 1024, 8, 2, shared=1),
        # a decode batch over 128 experts in groups: nearly every expert has a few rows
        _experts("experts_64_e128", 64, 4096, 1536, 128, 8, score="sigmoid", groups=8, kept=4, group_top=2, bias=True,
                 scale=2.5),
        # a ragged chunk of a prompt through fine-grained experts with a shared one, the router skewed
        _experts("experts_333_e64_skewed", 333, 2048, 1408, 64, 6, shared=1, skew=1.2),
        # eight prompts prefilled together through the wide layer
        _experts("experts_16384_wide", 16384, 4096, 14336, 8, 2),
    ]


# (experts, groups, kept) of drawn routers
_ROUTERS = [(8, 1, 1), (16, 4, 2), (60, 1, 1), (64, 1, 1), (64, 8, 3), (96, 6, 3), (128, 8, 4), (160, 8, 3), (256, 8, 4),
            (384, 1, 1)]
# (dim, dim_ffn, experts, top_k, most tokens) of drawn layers
_LAYERS = [(512, 1024, 8, 2, 16384), (704, 576, 16, 4, 16384), (1000, 2664, 8, 2, 8192), (2048, 1408, 64, 6, 16384),
           (2880, 2880, 32, 4, 16384), (4096, 1536, 128, 8, 8192), (4096, 14336, 8, 2, 8192)]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["route", "route", "linear", "linear", "experts", "experts"])
    if kind == "route":
        e, groups, kept = rng.choice(_ROUTERS)
        top_k = rng.randint(1, min(10, kept * (e // groups)))
        return _route("", _log_int(rng, 1, 16384), e, top_k, rng.choice(["softmax", "sigmoid"]), groups, kept,
                      rng.choice([1, 2]) if groups > 1 else 1, rng.choice([True, False]), rng.choice([True, True, False]),
                      rng.choice([1.0, 2.5]), rng.choice(["bf16", "fp32"]), rng.choice(["bf16", "fp32"]),
                      rng.choice([0.0, 0.0, 0.1]), rng.choice([True, False]))
    if kind == "linear":
        step = rng.choice([1, 8, 64])
        k, n = (step * _log_int(rng, max(1, 64 // step), 8192 // step) for _ in range(2))
        return _linear("", _log_int(rng, 1, 8192), k, n, rng.choice(["bf16", "bf16", "fp32"]), rng.choice([True, False]))
    dim, ffn, e, top_k, most = rng.choice(_LAYERS)
    groups = 4 if e >= 16 and rng.random() < 0.5 else 1
    return _experts("", _log_int(rng, 1, most), dim, ffn, e, top_k, rng.choice([0, 0, 1, 2]),
                    "fp32" if dim <= 1000 and rng.random() < 0.5 else "bf16", rng.choice(["softmax", "sigmoid"]), groups,
                    max(1, groups // 2), 1 if groups == 1 else rng.choice([1, 2]), rng.choice([True, False]),
                    rng.choice([1.0, 2.5]), rng.choice([0.0, 0.0, 1.2]))


# -- inputs ---------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape, std=1.0, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=gen)


def _logits(gen, case, dtype):
    """Router logits ~ N(0, 1.5); ``skew``: less for each expert of a random
    ranking; ``masked``: this share of the experts is off (-inf) for a token,
    and a third of it of the tokens are padding with every expert off."""
    t, e = case["tokens"], case["experts"]
    logits = _normal(gen, t, e, std=1.5)
    if case.get("skew"):
        rank = torch.randperm(e, generator=gen, device="cuda") + 1
        logits -= case["skew"] * torch.log(rank.float())
    logits = logits.to(dtype)
    if case.get("masked"):
        off = torch.rand(t, e, generator=gen, device="cuda") < case["masked"]
        off |= torch.rand(t, 1, generator=gen, device="cuda") < case["masked"] / 3
        logits = logits.masked_fill(off, -math.inf)
    return logits


def _int8_weight(gen, rows, k, out=None):
    """Codes of a weight [rows, k] quantised by rows, as rows of a whole number
    of 16 bytes with zeros behind column k, and its scales: normal values, the
    largest of a row about four standard deviations out."""
    kp = -(-k // 16) * 16
    q = torch.zeros(rows, kp, dtype=torch.int8, device="cuda") if out is None else out
    q[:, :k] = _normal(gen, rows, k, std=127 / 4, dtype=torch.bfloat16).round_().clamp_(-127, 127)
    scale = (1.0 + 0.1 * torch.rand(rows, generator=gen, device="cuda")) * (0.02 * 4 / 127)
    return q, scale


def _activations(gen, rows, k, dtype):
    """~ N(0, 1) with a few channels five times as large."""
    x = _normal(gen, rows, k)
    x[:, torch.randperm(k, generator=gen, device="cuda")[:max(1, k // 128)]] *= 5.0
    return x.to(dtype)


def prepare(case, seed):
    gen, op = _gen(seed), case["op"]
    state = {"case": case}
    if op == "route":
        state["logits"] = _logits(gen, case, _DTYPES[case["dtype"]])
        state["dw"] = _normal(gen, case["tokens"], case["top_k"], dtype=_DTYPES[case["weights"]])
    elif op == "linear":
        state["x"] = _activations(gen, case["rows"], case["k"], _DTYPES[case["dtype"]])
        state["w"], state["w_scale"] = _int8_weight(gen, case["n"], case["k"])
        state["bias"] = _normal(gen, case["n"], dtype=_DTYPES[case["dtype"]]) if case["bias"] else None
        return state
    else:
        state["logits"] = _logits(gen, case, torch.float32)
        d, f, e = case["dim"], case["dim_ffn"], case["experts"] + case["shared"]
        state["x"] = _activations(gen, case["tokens"], d, _DTYPES[case["dtype"]])
        for name, n, k in (("gate", f, d), ("up", f, d), ("down", d, f)):
            w = torch.zeros(e, n, -(-k // 16) * 16, dtype=torch.int8, device="cuda")
            s = torch.empty(e, n, device="cuda")
            for i in range(e):
                s[i] = _int8_weight(gen, n, k, out=w[i])[1]
            state[name], state[name + "_scale"] = w, s
    state["bias"] = _normal(gen, case["experts"], std=0.05) if case["bias"] else None
    if case.get("train") and state["bias"] is None:
        state["bias"] = torch.zeros(case["experts"], device="cuda")
    return state


# -- one pass -------------------------------------------------------------------


def run(state):
    if own:
        return _run_own(state)
    return {"route": _plain_route, "linear": _plain_linear, "experts": _plain_experts}[state["case"]["op"]](state)


def _run_own(state):
    from astrai_amd.extension import ops

    c = state["case"]
    if c["op"] == "linear":
        return ops.int8_linear(state["x"], state["w"], state["w_scale"], state["bias"])
    routing = ops.Routing(c["score"], c["groups"], c["kept"], c["group_top"], c["renorm"], c["scale"])
    if c["op"] == "experts":
        experts = ops.Int8Experts(state["gate"], state["up"], state["down"], state["gate_scale"], state["up_scale"],
                                  state["down_scale"])
        return ops.moe_int8_forward(state["x"], state["logits"], experts, c["top_k"], c["shared"], routing, state["bias"])
    r = ops.moe_route_scores(state["logits"], c["top_k"], routing, state["bias"], weight_dtype=_DTYPES[c["weights"]])
    got = {"idx": r.topk_idx, "w": r.topk_w, "chunk_hist": r.chunk_hist}
    if c["train"]:
        got["dlogits"] = ops.moe_route_scores_grad(state["logits"], r.topk_idx, r.topk_w, state["dw"], routing)
        got["load"] = ops.moe_expert_load(r.chunk_hist)
        got["bias"] = ops.moe_balance_bias(state["bias"], got["load"], _RATE)
    return got


def _choose(c, logits, bias):
    """(scores in 64 bits [T, E], chosen experts [T, K], which of them are live)."""
    l = logits.double()
    off = l == -math.inf
    if c["score"] == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-l))
    else:
        top = l.amax(-1, keepdim=True)
        p = torch.exp(l - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        s = p / torch.where(total == 0.0, 1.0, total)
    key = s if bias is None else s + bias.double()
    key = key.masked_fill(off, -math.inf)
    t, e = key.shape
    if c["groups"] > 1:
        per = e // c["groups"]
        best = torch.sort(key.view(t, c["groups"], per), dim=-1, descending=True).values[..., :c["group_top"]].sum(-1)
        kept = torch.sort(best, dim=-1, descending=True, stable=True).indices[:, :c["kept"]]
        out = torch.ones(t, c["groups"], dtype=torch.bool, device=key.device).scatter_(1, kept, False)
        key = key.masked_fill(out.repeat_interleave(per, dim=1), -math.inf)
    values, order = torch.sort(key, dim=-1, descending=True, stable=True)
    return s, order[:, :c["top_k"]], values[:, :c["top_k"]] > -math.inf


def _weights(c, s, chosen, live):
    """Routing weights in 32 bits: (weights, scores at the chosen experts, their sum)."""
    v = torch.where(live, s.gather(1, chosen), 0.0).float()
    total = v.sum(-1, keepdim=True)
    safe = torch.where(total == 0.0, 1.0, total)
    return (v / safe if c["renorm"] else v) * c["scale"], v, safe


def _plain_route(state):
    c, logits, bias = state["case"], state["logits"], state["bias"]
    s, chosen, live = _choose(c, logits, bias)
    w, v, total = _weights(c, s, chosen, live)
    t, e = logits.shape
    chunk = torch.arange(t, device=logits.device).div(32, rounding_mode="floor").unsqueeze(1)
    hist = torch.zeros(-(-t // 32) * e, dtype=torch.int32, device=logits.device)
    hist = hist.scatter_add_(0, (chunk * e + chosen).view(-1), torch.ones_like(chosen, dtype=torch.int32).view(-1))
    got = {"idx": chosen.to(torch.int32), "w": w.to(_DTYPES[c["weights"]]), "chunk_hist": hist.view(-1, e)}
    if c["train"]:
        ds = state["dw"].float() * c["scale"]
        if c["renorm"]:
            ds = (ds - (ds * v).sum(-1, keepdim=True) / total) / total
        ds = torch.where(live, ds, 0.0)
        s32 = s.float()
        dp = torch.zeros_like(s32).scatter_(1, chosen, ds)
        if c["score"] == "sigmoid":
            dl = dp * s32 * (1.0 - s).float()
        else:
            dl = s32 * (dp - (dp * s32).sum(-1, keepdim=True))
        got["dlogits"] = dl.to(logits.dtype)
        load = got["chunk_hist"].sum(0, dtype=torch.int32)
        got["load"] = load
        got["bias"] = bias + _RATE * torch.sign(load.sum() - e * load.long()).float()
    return got


def _quantise(x):
    """Codes of the rows of x (as 32-bit floats) and their scales."""
    x = x.double()
    most = x.abs().amax(-1, keepdim=True)
    q = torch.round(x * 127.0 / torch.where(most == 0.0, 1.0, most)).float()
    return q, (most / 127.0).float()


def _product(xq, xs, w, ws, k):
    """In 32 bits, which hold the sums of code products; the scales are applied
    in 64, since what follows may be next to a border between two codes."""
    return (xq @ w[:, :k].float().t()).double() * (xs.double() * ws.double())


def _plain_linear(state):
    c, x = state["case"], state["x"]
    xq, xs = _quantise(x)
    y = _product(xq, xs, state["w"], state["w_scale"], c["k"]).float()
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(x.dtype)


def _plain_experts(state):
    c, x = state["case"], state["x"]
    s, chosen, live = _choose(c, state["logits"], state["bias"])
    # a routing weight and an expert's output are values of the layer's type
    w = _weights(c, s, chosen, live)[0].to(x.dtype).float()
    d, f, e, shared = c["dim"], c["dim_ffn"], c["experts"], c["shared"]
    xq, xs = _quantise(x)

    def expert(i, rows, scales):
        g = _product(rows, scales, state["gate"][i], state["gate_scale"][i], d)
        u = _product(rows, scales, state["up"][i], state["up_scale"][i], d)
        h = (g / (1.0 + torch.exp(-g)) * u).to(x.dtype)
        return _product(*_quantise(h), state["down"][i], state["down_scale"][i], f).to(x.dtype).float()

    out = torch.zeros(x.shape, device=x.device)
    order = torch.sort(chosen.reshape(-1), stable=True).indices
    counts = torch.bincount(chosen.reshape(-1), minlength=e).tolist()
    at = 0
    for i, n in enumerate(counts):
        if n:
            slot = order[at:at + n]
            token = slot.div(c["top_k"], rounding_mode="floor")
            out.index_add_(0, token, expert(i, xq[token], xs[token]) * w.view(-1, 1)[slot])
            at += n
    for i in range(shared):
        out += expert(e + i, xq, xs) / shared
    return out.to(x.dtype)


# -- what a pass cannot do without ------------------------------------------------


def work(case):
    size = {"bf16": 2, "fp32": 4}
    if case["op"] == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        nbytes = t * e * size[case["dtype"]] + t * k * (4 + size[case["weights"]]) + -(-t // 32) * e * 4
        if case["train"]:
            # logits read once, their gradient written, the weights' gradient read, load and bias
            nbytes += t * e * size[case["dtype"]] + t * k * size[case["weights"]] + 12 * e
        return {"bytes": nbytes, "flops": (20.0 if case["train"] else 10.0) * t * e}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": size[case["dtype"]] * (m * k + m * n) + n * k + 4 * n, "flops": 2.0 * m * k * n}
    t, d, f, e, k, s = (case[n] for n in ("tokens", "dim", "dim_ffn", "experts", "top_k", "shared"))
    live = e * (1.0 - (1.0 - k / e) ** t) + s  # experts that meet a token: expected under even routing
    return {"bytes": size[case["dtype"]] * 2 * t * d + 4 * t * e + live * (3 * d * f + 4 * (2 * f + d)),
            "flops": 6.0 * t * (k + s) * d * f}


# -- the operators in 64 bits -----------------------------------------------------


def _route64(c, logits, bias):
    """Scores, chosen experts and their liveness with numpy, one pick at a time
    (the first of equal values is numpy's argmax)."""
    l = logits.double().cpu().numpy()
    off = np.isneginf(l)
    with np.errstate(invalid="ignore", over="ignore"):
        if c["score"] == "sigmoid":
            s = np.where(l >= 0, 1.0 / (1.0 + np.exp(-np.abs(l))), np.exp(-np.abs(l)) / (1.0 + np.exp(-np.abs(l))))
        else:
            shift = np.max(l, axis=1, keepdims=True)
            p = np.where(off, 0.0, np.exp(l - np.where(np.isfinite(shift), shift, 0.0)))
            s = p / np.maximum(p.sum(1, keepdims=True), 1e-300)
    s = np.where(off, 0.0, s)
    key = s + (0.0 if bias is None else bias.double().cpu().numpy())
    key = np.where(off, -np.inf, key)
    t, e = key.shape
    rows = np.arange(t)
    if c["groups"] > 1:
        parts = key.reshape(t, c["groups"], -1).copy()
        value = np.zeros((t, c["groups"]))
        for _ in range(c["group_top"]):
            value += parts.max(-1)
            np.put_along_axis(parts, parts.argmax(-1)[..., None], -np.inf, -1)
        keep = np.zeros((t, c["groups"]), dtype=bool)
        for _ in range(c["kept"]):
            best = np.where(keep, -np.inf, value).argmax(1)
            dead = np.isneginf(np.where(keep, -np.inf, value).max(1))
            best = np.where(dead, np.argmin(keep, axis=1), best)
            keep[rows, best] = True
        key = np.where(np.repeat(keep, e // c["groups"], axis=1), key, -np.inf)
    chosen = np.zeros((t, c["top_k"]), dtype=np.int64)
    live = np.zeros((t, c["top_k"]), dtype=bool)
    taken = np.zeros((t, e), dtype=bool)
    for k in range(c["top_k"]):
        left = np.where(taken, -np.inf, key)
        best = left.argmax(1)
        live[:, k] = left[rows, best] > -np.inf
        best = np.where(live[:, k], best, np.argmin(taken, axis=1))
        taken[rows, best] = True
        chosen[:, k] = best
    v = np.where(live, np.take_along_axis(s, chosen, 1), 0.0)
    total = v.sum(1, keepdims=True)
    total = np.where(total == 0.0, 1.0, total)
    w = c["scale"] * (v / total if c["renorm"] else v)
    return s, chosen, live, v, total, w


def _exact_route(c, state):
    s, chosen, live, v, total, w = _route64(c, state["logits"], state["bias"])
    t, e = s.shape
    hist = np.zeros((-(-t // 32), e), dtype=np.int32)
    np.add.at(hist, (np.repeat(np.arange(t) // 32, c["top_k"]), chosen.reshape(-1)), 1)
    got = {"idx": torch.from_numpy(chosen.astype(np.int32)), "w": torch.from_numpy(w), "chunk_hist": torch.from_numpy(hist)}
    if c["train"]:
        ds = c["scale"] * state["dw"].double().cpu().numpy()
        if c["renorm"]:
            ds = (ds - (ds * v).sum(1, keepdims=True) / total) / total
        ds = np.where(live, ds, 0.0)
        if c["score"] == "sigmoid":
            at_chosen = np.take_along_axis(state["logits"].double().cpu().numpy(), chosen, 1)
            at_chosen = np.where(live, at_chosen, 0.0)
            slope = np.exp(-np.abs(at_chosen)) / (1.0 + np.exp(-np.abs(at_chosen))) ** 2
            dl = np.zeros((t, e))
            np.put_along_axis(dl, chosen, ds * slope, 1)
        else:
            dl = -s * (ds * v).sum(1, keepdims=True)
            np.put_along_axis(dl, chosen, np.take_along_axis(dl, chosen, 1) + ds * v, 1)
        load = hist.sum(0)
        got["dlogits"] = torch.from_numpy(dl)
        got["load"] = torch.from_numpy(load.astype(np.int32))
        step = np.sign(load.sum() - e * load.astype(np.int64))
        got["bias"] = torch.from_numpy(state["bias"].double().cpu().numpy() + _RATE * step)
    return got


def _codes(x):
    """Codes of the rows of x and their scales, which are 32-bit values; a value at
    a border between two codes is decided exactly (254 x against (2 n + 1) max:
    both fit 64 bits)."""
    x = x.double()
    most = x.abs().amax(dim=1, keepdim=True)
    safe = torch.where(most > 0, most, torch.ones_like(most))
    n = torch.floor(x * 127.0 / safe)
    twice, border = 2.0 * 127.0 * x, (2.0 * n + 1.0) * safe
    up = (twice > border) | ((twice == border) & (torch.remainder(n, 2.0) == 1.0))
    return n + up.double(), (most / 127.0).float().double()


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "route":
        return _exact_route(case, state)
    x = state["x"]
    if case["op"] == "linear":
        q, s = _codes(x)
        y = (q @ state["w"][:, :case["k"]].double().t()) * (s * state["w_scale"].double())
        return y + state["bias"].double() if case["bias"] else y
    _, chosen, _, _, _, w = _route64(case, state["logits"], state["bias"])
    chosen = torch.from_numpy(chosen).cuda()
    w = torch.from_numpy(w).cuda().to(x.dtype).double()
    d, f, e = case["dim"], case["dim_ffn"], case["experts"]
    q, s = _codes(x)

    def mlp(i, q, s):
        def times(q, s, name, k):
            return (q @ state[name][i][:, :k].double().t()) * (s * state[name + "_scale"][i].double())

        g, u = times(q, s, "gate", d), times(q, s, "up", d)
        h = (g * torch.sigmoid(g) * u).to(x.dtype)
        return times(*_codes(h), "down", f).to(x.dtype).double()

    out = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    for i in range(e):
        token, slot = (chosen == i).nonzero(as_tuple=True)
        if token.numel():
            out.index_add_(0, token, mlp(i, q[token], s[token]) * w[token, slot].unsqueeze(1))
    for i in range(case["shared"]):
        out += mlp(e + i, q, s) / case["shared"]
    return out

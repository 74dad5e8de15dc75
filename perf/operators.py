"""Measured cases of two operators: the fused linear layer and the routing of tokens to experts.

``linear(x, weight, bias, activation, residual)`` is ``activation(x @ weight.T + bias) + residual`` rounded once; its
gated activations split the weight's rows into a gate half and an up half.  ``route_experts(logits, top_k, ...)`` turns
router logits into the chosen experts of every token and their weights.  Where ``own`` is false both are computed in
their plain form (elementary torch operations in 32 bits, the routing's comparisons in 64).
"""

from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_GATED = ("silu_and_mul", "gelu_tanh_and_mul")
_ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh") + _GATED


def _linear(name, m, n, k, dtype="bf16", activation="none", bias=False, residual=False, out="same", pitch=0):
    """``n`` counts the output's columns: a gated weight has ``2 n`` rows.  ``pitch``: unused elements after every row
    of x, as in a slice of a wider activation buffer."""
    return {"name": name, "op": "linear", "m": m, "n": n, "k": k, "dtype": dtype, "activation": activation, "bias": bias,
            "residual": residual, "out": out, "pitch": pitch}


def _route(name, tokens, experts, top_k, dtype="fp32", scoring="softmax", bias=False, num_groups=1, top_groups=1,
           group_top=1, renormalize=False, scale=1.0, masked=0):
    """``masked``: the last experts of every row have a logit of -inf (a table padded to a rounder size)."""
    return {"name": name, "op": "route", "tokens": tokens, "experts": experts, "top_k": top_k, "dtype": dtype,
            "scoring": scoring, "bias": bias, "num_groups": num_groups, "top_groups": top_groups, "group_top": group_top,
            "renormalize": renormalize, "scale": scale, "masked": masked}


def listed():
    return [
        # the router's own product for one decoded token: latency, and logits wanted in fp32
        _linear("linear_router_1", 1, 128, 4096, out="fp32"),
        # one token through the down projection of a 70B-class layer, the residual stream added on the way out
        _linear("linear_down_1", 1, 8192, 28672, residual=True),
        # a few sequences through a small biased layer with sizes that fit no tile, fp16
        _linear("linear_bias_gelu_7", 7, 5001, 1288, dtype="fp16", activation="gelu", bias=True),
        # a decode batch through the same layer's gate and up projections with the gated activation
        _linear("linear_gate_up_16", 16, 28672, 8192, activation="silu_and_mul"),
        # a speculative or chunked step: more rows than a decode batch, too few to fill prefill tiles
        _linear("linear_mid_200", 200, 8192, 8192, residual=True),
        # a ragged prompt through an uneven biased layer, x a slice of a wider buffer
        _linear("linear_ragged_1003", 1003, 4999, 4104, dtype="fp16", activation="gelu_tanh", bias=True, residual=True, pitch=24),
        # prompt processing: gate and up projections of an 8B-class layer
        _linear("linear_gate_up_4096", 4096, 14336, 4096, activation="silu_and_mul"),
        # prompt processing: a square projection with the residual stream, the largest case
        _linear("linear_prefill_8192", 8192, 8192, 8192, residual=True),
        # one decoded token: sigmoid scores, a balance bias, the best 4 of 8 groups
        _route("route_groups_1", 1, 256, 8, scoring="sigmoid", bias=True, num_groups=8, top_groups=4, group_top=2,
               renormalize=True, scale=2.5),
        # groups that are no power of two, a few padding experts without tokens
        _route("route_ragged_777", 777, 160, 6, dtype="fp16", num_groups=8, top_groups=3, scale=16.0, masked=4),
        # the MoE layer's own step: 8192 tokens over 128 experts, softmax then top-8
        _route("route_softmax_8192", 8192, 128, 8),
        # a long prompt batch through the grouped router
        _route("route_groups_65536", 65536, 256, 8, scoring="sigmoid", bias=True, num_groups=8, top_groups=4, group_top=2,
               renormalize=True, scale=2.5),
    ]


_MOST_FLOPS, _MOST_BYTES = 1.1e12, 9.4e8  # of the largest listed cases


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    if rng.random() < 0.62:
        while True:
            activation = rng.choice(_ACTIVATIONS)
            m = rng.choice([1, _log_int(rng, 1, 32), _log_int(rng, 1, 512), _log_int(rng, 1, 16384)])
            n = _log_int(rng, 16, 32768)
            if rng.random() < 0.6:
                n = max(16, n // 8 * 8)  # most layers' widths are round; the others stay odd
            k = 8 * _log_int(rng, 8, 3584)
            case = _linear("", m, n, k, dtype=rng.choice(["bf16", "fp16"]), activation=activation, bias=rng.random() < 0.5,
                           residual=rng.random() < 0.5, out=rng.choice(["same", "same", "fp32"]),
                           pitch=rng.choice([0, 0, 8 * rng.randint(1, 16)]))
            del case["name"]
            w = work(case)
            if w["flops"] <= _MOST_FLOPS and w["bytes"] <= _MOST_BYTES:
                return case
    size = rng.choice([_log_int(rng, 1, 64), 8 * rng.randint(1, 8)])
    num_groups = rng.choice([1, 1, 2, 4, 8, rng.randint(3, 16)])
    experts = max(8, min(512, size * num_groups if num_groups > 1 else _log_int(rng, 8, 512)))
    num_groups = num_groups if experts % num_groups == 0 else 1
    top_groups = rng.randint(1, num_groups)
    per_group = experts // num_groups
    top_k = min(rng.randint(1, 12), top_groups * per_group)
    case = _route("", _log_int(rng, 1, 65536), experts, top_k, dtype=rng.choice(["bf16", "fp16", "fp32"]),
                  scoring=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, num_groups=num_groups,
                  top_groups=top_groups, group_top=rng.choice([1, 2]) if per_group >= 2 and num_groups > 1 else 1,
                  renormalize=rng.random() < 0.5, scale=rng.choice([1.0, 2.5, 16.0]),
                  masked=rng.choice([0, 0, rng.randint(0, experts // 2)]))
    del case["name"]
    return case


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))

    def normal(*shape, dtype, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).mul_(std).to(dtype)

    dtype = _DTYPES[case["dtype"]]
    state = dict(case)
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        rows = 2 * n if case["activation"] in _GATED else n
        out = dtype if case["out"] == "same" else _DTYPES[case["out"]]
        state.update(
            x=normal(m, k + case["pitch"], dtype=dtype)[:, :k],
            weight=normal(rows, k, dtype=dtype, std=k**-0.5),
            bias=normal(rows, dtype=dtype, std=0.5) if case["bias"] else None,
            residual=normal(m, n, dtype=out) if case["residual"] else None,
            out_dtype=out,
        )
        return state
    tokens, experts = case["tokens"], case["experts"]
    logits = normal(tokens, experts, dtype=dtype, std=1.5)
    if case["masked"]:
        logits[:, experts - case["masked"]:] = -math.inf
    state.update(logits=logits, bias=normal(experts, dtype=torch.float32, std=0.1) if case["bias"] else None)
    return state


def run(state):
    if own:
        import helion_b200 as hb

        if state["op"] == "linear":
            return hb.linear(state["x"], state["weight"], state["bias"], activation=state["activation"],
                             residual=state["residual"], out_dtype=state["out_dtype"])
        return hb.route_experts(state["logits"], state["top_k"], scoring=state["scoring"], bias=state["bias"],
                                num_groups=state["num_groups"], top_groups=state["top_groups"],
                                group_top=state["group_top"], renormalize=state["renormalize"], scale=state["scale"])
    return _plain_linear(state) if state["op"] == "linear" else _plain_route(state)


# ---------------------------------------------------------------- plain forms
def _plain_linear(s):
    y = s["x"].float() @ s["weight"].float().t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    act = s["activation"]
    up = None
    if act in _GATED:
        y, up = y[:, : s["n"]], y[:, s["n"]:]
        act = act[: -len("_and_mul")]
    if act == "relu":
        y = torch.where(y > 0, y, torch.zeros_like(y))
    elif act == "silu":
        y = y / (1 + torch.exp(-y))
    elif act == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    elif act == "gelu_tanh":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    if up is not None:
        y = y * up
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["out_dtype"])


def _plain_route(s):
    # in 64 bits: two experts' scores next to each other decide which indices come out
    logits = s["logits"].double()
    tokens, experts = logits.shape
    live = logits > -math.inf
    if s["scoring"] == "softmax":
        top = logits.max(-1, keepdim=True).values
        e = torch.where(live, torch.exp(logits - top), torch.zeros_like(logits))
        scores = torch.where(live, e / e.sum(-1, keepdim=True), torch.zeros_like(logits))
    else:
        scores = 1 / (1 + torch.exp(-logits))
    low = torch.full_like(logits, -math.inf)
    choice = scores + s["bias"].double() if s["bias"] is not None else scores
    rank = torch.where(live, choice if s["bias"] is not None else logits, low)  # without a bias the logits decide
    kept = torch.ones_like(live)
    groups, size = s["num_groups"], experts // s["num_groups"]
    if groups > 1:
        by_group = torch.where(live, choice, low) if s["group_top"] > 1 else rank
        best = by_group.view(tokens, groups, size).sort(dim=-1, descending=True).values[..., : s["group_top"]]
        any_live = best[..., 0] > -math.inf
        score = torch.where(best > -math.inf, best, torch.zeros_like(best)).sum(-1)
        score = torch.where(any_live, score, torch.full_like(score, -math.inf))
        order = score.sort(dim=-1, descending=True, stable=True).indices[:, : s["top_groups"]]
        chosen = torch.zeros(tokens, groups, dtype=torch.bool, device=logits.device).scatter_(1, order, True)
        kept = chosen[:, :, None].expand(tokens, groups, size).reshape(tokens, experts)
    # experts of dropped groups come after everything else, masked experts of kept groups included
    by_rank = rank.sort(dim=-1, descending=True, stable=True).indices
    last = (~kept).gather(1, by_rank).sort(dim=-1, stable=True).indices
    picked = by_rank.gather(1, last)[:, : s["top_k"]]
    weights = scores.gather(1, picked)
    if s["renormalize"]:
        total = weights.sum(-1, keepdim=True)
        weights = torch.where(total > 0, weights / total, torch.zeros_like(weights))
    return (weights * s["scale"]).float(), picked


# ---------------------------------------------------------------------- exact
def exact(case, seed):
    """The operators' definitions in 64 bits, output column block by column block and pick by pick."""
    s = prepare(case, seed)
    if case["op"] == "linear":
        m, n = case["m"], case["n"]
        x = s["x"].to(torch.float64)
        out = torch.empty(m, n, dtype=torch.float64, device="cuda")

        def product(lo, hi):
            p = torch.mm(x, s["weight"][lo:hi].to(torch.float64).T)
            return p if s["bias"] is None else p.add_(s["bias"][lo:hi].to(torch.float64))

        inner = {
            "none": lambda v: v,
            "relu": lambda v: v.clamp_min(0),
            "silu": lambda v: v * torch.sigmoid(v),
            "gelu": lambda v: v * torch.special.ndtr(v),
            "gelu_tanh": lambda v: v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v**3)),
        }
        act = inner[case["activation"].replace("_and_mul", "")]
        for lo in range(0, n, 4096):
            hi = min(n, lo + 4096)
            v = act(product(lo, hi))
            out[:, lo:hi] = v * product(n + lo, n + hi) if case["activation"] in _GATED else v
        if s["residual"] is not None:
            out += s["residual"].to(torch.float64)
        return out
    z = s["logits"].to(torch.float64)
    t, e = z.shape
    dead = torch.isneginf(z)
    prob = torch.sigmoid(z) if case["scoring"] == "sigmoid" else torch.softmax(z, -1).nan_to_num(0.0)
    biased = prob if s["bias"] is None else prob + s["bias"].to(torch.float64)
    key = (z if s["bias"] is None else biased).masked_fill(dead, -math.inf)
    index = torch.arange(e, device="cuda").expand(t, e)

    def first_max(v, idx):
        best = v.amax(-1, keepdim=True)
        return best, torch.where(v == best, idx, v.shape[-1]).amin(-1, keepdim=True)

    open_ = torch.ones(t, e, dtype=torch.bool, device="cuda")
    if case["num_groups"] > 1:
        g, size = case["num_groups"], e // case["num_groups"]
        left = (key if case["group_top"] == 1 else biased.masked_fill(dead, -math.inf)).reshape(t, g, size).clone()
        total = torch.zeros(t, g, dtype=torch.float64, device="cuda")
        for i in range(case["group_top"]):
            best, at = first_max(left, torch.arange(size, device="cuda").expand(t, g, size))
            total += best.squeeze(-1).masked_fill(torch.isneginf(best.squeeze(-1)), -math.inf if i == 0 else 0.0)
            left.scatter_(-1, at, -math.inf)
        taken = torch.zeros(t, g, dtype=torch.bool, device="cuda")
        gidx = torch.arange(g, device="cuda").expand(t, g)
        for _ in range(case["top_groups"]):
            # a dead group (-inf) still comes before one that is taken
            best = total.masked_fill(taken, -math.inf).amax(-1, keepdim=True)
            at = torch.where((total == best) & ~taken, gidx, g).amin(-1, keepdim=True)
            taken.scatter_(1, at, True)
        open_ = taken.repeat_interleave(size, dim=1)
    picks = []
    for _ in range(case["top_k"]):
        best = key.masked_fill(~open_, -math.inf).amax(-1, keepdim=True)
        at = torch.where((key == best) & open_, index, e).amin(-1, keepdim=True)
        open_ = open_.scatter(1, at, False)
        picks.append(at)
    picks = torch.cat(picks, 1)
    w = prob.gather(1, picks)
    if case["renormalize"]:
        w = (w / w.sum(-1, keepdim=True)).nan_to_num(0.0)
    return w * case["scale"], picks


def work(case):
    item = {"bf16": 2, "fp16": 2, "fp32": 4}
    if case["op"] == "linear":
        m, n, k, size = case["m"], case["n"], case["k"], item[case["dtype"]]
        rows = 2 * n if case["activation"] in _GATED else n
        out = size if case["out"] == "same" else item[case["out"]]
        nbytes = (m + rows) * k * size + m * n * out * (2 if case["residual"] else 1) + (rows * size if case["bias"] else 0)
        return {"bytes": nbytes, "flops": 2 * m * rows * k}
    t, e = case["tokens"], case["experts"]
    nbytes = t * e * item[case["dtype"]] + t * case["top_k"] * (4 + 8) + (4 * e if case["bias"] else 0)
    return {"bytes": nbytes, "flops": 4 * t * e}  # a score, a sum and two comparisons for every logit

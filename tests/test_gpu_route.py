"""Expert routing against its definition in 64 bits: picks exactly, weights to a few units in the last place."""

from __future__ import annotations

import math

import pytest
import torch

import helion_b200 as hb
from helion_b200 import _lib
from helion_b200 import dist as D
from helion_b200 import moe as M
from linear_reference import check as check_linear
from route_reference import route

pytestmark = pytest.mark.gpu
DEV = "cuda"


def compare(logits, top_k, **kw):
    w, e = hb.route_experts(logits, top_k, **kw)
    rw, re = route(logits, top_k, **kw)
    assert w.dtype is torch.float32 and e.dtype is torch.int64
    assert torch.equal(e.cpu(), re)
    # fp32: logit - top is rounded (half a unit of up to |d|, which the exponential turns into |d| 2^-24 of its value), the
    # exponential and the division are off by 2 units and the sum of up to 1024 terms by 10 additions and a tree; the
    # smallest results are denormal
    d = 2.0 * logits.float().masked_fill(torch.isinf(logits), 0).abs().amax(1, keepdim=True).cpu().double() + 32
    assert ((w.cpu().double() - rw).abs() <= d * 2.0**-23 * rw + 2.0**-140 * abs(kw.get("scale", 1.0))).all()
    return w, e


CONFIGS = [
    (8, 2, {}),
    (1, 1, {}),
    (33, 5, dict(scoring="sigmoid")),
    (60, 4, dict(renormalize=True)),
    (64, 6, dict(renormalize=True, scale=2.5, bias=True)),
    (128, 8, {}),
    (128, 8, dict(scoring="sigmoid", bias=True, renormalize=True)),
    (160, 6, dict(num_groups=8, top_groups=3, scale=16.0)),
    (160, 6, dict(num_groups=8, top_groups=3, group_top=2)),
    (256, 8, dict(scoring="sigmoid", bias=True, num_groups=8, top_groups=4, group_top=2, renormalize=True, scale=2.5)),
    (256, 8, dict(bias=True, num_groups=4, top_groups=1)),
    (96, 12, dict(scoring="sigmoid", num_groups=32, top_groups=4, group_top=1)),
    (62, 4, dict(num_groups=31, top_groups=2, group_top=2, bias=True)),
    (257, 32, dict(bias=True)),
    (512, 10, dict(scoring="sigmoid", bias=True, num_groups=16, top_groups=4, group_top=2)),
    (1024, 32, dict(num_groups=2, top_groups=1, renormalize=True)),
    (1000, 7, dict(scoring="sigmoid", bias=True)),
    (32, 32, dict(bias=True, renormalize=True)),
]


def make(tokens, experts, dtype, kw, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + experts)
    logits = (torch.randn(tokens, experts, generator=g, device=DEV) * 2).to(dtype)
    kw = dict(kw)
    if kw.get("bias"):
        kw["bias"] = torch.randn(experts, generator=g, device=DEV) * 0.1
    return logits, kw


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("experts,top_k,kw", CONFIGS)
def test_configs(experts, top_k, kw, dtype):
    for tokens in (1, 50):
        logits, k = make(tokens, experts, dtype, kw)
        compare(logits, top_k, **k)


@pytest.mark.parametrize("experts,top_k,kw", CONFIGS)
def test_masked_experts_and_empty_rows(experts, top_k, kw):
    logits, k = make(24, experts, torch.float32, kw, seed=1)
    g = torch.Generator(device=DEV).manual_seed(5)
    logits[torch.rand(24, experts, generator=g, device=DEV) < 0.7] = -math.inf
    logits[3] = -math.inf  # nothing left
    logits[4] = -math.inf
    logits[4, experts // 2] = 0.5  # one left
    w, e = compare(logits, top_k, **k)
    assert (w[3] == 0).all() and torch.isfinite(w).all()
    assert all(len(set(r)) == top_k for r in e.tolist())


@pytest.mark.parametrize("kw", [{}, dict(scoring="sigmoid"), dict(renormalize=True), dict(scoring="sigmoid", renormalize=True),
                                dict(bias=True, renormalize=True), dict(num_groups=8, top_groups=2, group_top=2)])
def test_extreme_logits(kw):
    logits, k = make(16, 64, torch.float32, kw, seed=2)
    logits *= torch.logspace(-3, 2.5, 16, device=DEV)[:, None]
    logits[5] -= 95.0  # sigmoid scores that are denormal in fp32
    logits[6] = -1e4 * torch.arange(64, device=DEV)
    logits[7] = 3.0e38
    logits[8, ::2] = -3.0e38
    if k.get("scoring") == "sigmoid" or kw.get("renormalize"):
        logits[6] = -10.0 * torch.arange(64, device=DEV)
    compare(logits, 6, **k)


def test_ties_go_to_the_lowest_index():
    logits = torch.zeros(5, 256, device=DEV)
    logits[1] = torch.arange(256, device=DEV) % 3
    logits[2, 100:] = 1.0
    logits[3] = -0.0
    logits[3, ::2] = 0.0  # equal to -0
    for kw in ({}, dict(scoring="sigmoid"), dict(bias=torch.zeros(256, device=DEV)),
               dict(scoring="sigmoid", bias=torch.full((256,), 0.25, device=DEV), num_groups=8, top_groups=4, group_top=2)):
        compare(logits, 8, **kw)


MANY = [
    (32, 2, {}),
    (64, 6, dict(renormalize=True, bias=True)),
    (64, 8, dict(scoring="sigmoid", bias=True, num_groups=8, top_groups=4, group_top=2, renormalize=True, scale=2.5)),
    (96, 4, dict(bias=True)),
    (128, 8, {}),
    (128, 8, dict(scoring="sigmoid", num_groups=4, top_groups=2, group_top=2)),
    (128, 1, dict(num_groups=8, top_groups=1, renormalize=True)),
    (160, 6, dict(num_groups=8, top_groups=3, scale=16.0)),
    (192, 8, dict(scoring="sigmoid", bias=True, num_groups=8, top_groups=4, group_top=2)),
    (200, 5, dict(scoring="sigmoid", renormalize=True)),
    (256, 8, dict(scoring="sigmoid", bias=True, num_groups=8, top_groups=4, group_top=2, renormalize=True, scale=2.5)),
    (256, 8, dict(num_groups=2, top_groups=1)),
    (256, 8, dict(num_groups=8, top_groups=1, group_top=2, bias=True)),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("experts,top_k,kw", MANY)
def test_many_tokens(experts, top_k, kw, dtype):
    """Large batches take another form: every token as in a small batch and as in the definition, whatever the row
    holds (masked experts, the type's lowest value as a mask, ties, NaN, nothing at all)."""
    tokens = 16403
    logits, k = make(tokens, experts, dtype, kw, seed=7)
    g = torch.Generator(device=DEV).manual_seed(experts)
    logits[100:200][torch.rand(100, experts, generator=g, device=DEV) < 0.6] = -math.inf
    logits[200:300][torch.rand(100, experts, generator=g, device=DEV) < 0.3] = torch.finfo(dtype).min
    logits[300:340] = 0.25
    logits[340:360] = torch.randint(0, 3, (20, experts), generator=g, device=DEV).to(dtype)
    logits[360, 5], logits[361, 1::2], logits[362] = math.nan, math.nan, -math.inf
    logits[363, 3] = math.inf
    logits[364, : experts - 1] = -math.inf
    logits[365] = torch.finfo(dtype).max
    logits[400:420] *= 40
    w, e = hb.route_experts(logits, top_k, **k)
    # a warp per token, 5000 at a time
    parts = [hb.route_experts(logits[i : i + 5000], top_k, **k) for i in range(0, tokens, 5000)]
    we, ee = torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts])
    assert torch.equal(e, ee)
    assert torch.equal(torch.isnan(w), torch.isnan(we))
    assert ((w - we).abs() <= 2.0**-19 * we.abs() + 1e-38).logical_or(torch.isnan(we)).all()
    keep = torch.tensor([i for i in range(420) if i not in (360, 361, 363)] + [tokens - 2, tokens - 1], device=DEV)
    compare(logits[keep], top_k, **k)  # (the small form)
    rw, re = route(logits[keep], top_k, **k)
    assert torch.equal(e[keep].cpu(), re)
    # not contiguous: the same answers from a pitched view, aligned and not
    wide = torch.full((tokens, experts + 24), math.nan, dtype=dtype, device=DEV)
    for at in (8, 3):
        wide[:, at : at + experts] = logits
        w2, e2 = hb.route_experts(wide[:, at : at + experts], top_k, **k)
        assert torch.equal(e2, e) and ((w2 - w).abs() <= 2.0**-19 * w.abs() + 1e-38).logical_or(torch.isnan(w)).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_choices_closer_than_fp32_can_tell(scoring):
    """Biases that make pairs of choices meet to within 2^-26: the picks are still those of exact arithmetic."""
    g = torch.Generator().manual_seed(3)
    flips = 0
    for trial in range(40):
        logits = torch.randn(64, generator=g, dtype=torch.float64).float()
        score = torch.softmax(logits.double(), 0) if scoring == "softmax" else torch.sigmoid(logits.double())
        bias = (0.75 - score).float()  # every choice is 0.75 but for the bias's own rounding
        row = logits[None].to(DEV)
        kw = dict(scoring=scoring, bias=bias.to(DEV))
        _, e = compare(row, 8, **kw)
        compare(row, 8, **kw, num_groups=8, top_groups=3, group_top=2)
        fp32 = (torch.softmax(logits, 0) if scoring == "softmax" else torch.sigmoid(logits)) + bias
        flips += fp32.sort(descending=True, stable=True).indices[:8].tolist() != e[0].tolist()
    assert flips > 0  # the case is one that fp32 alone gets wrong


@pytest.mark.parametrize("experts,kw", [(64, dict(scoring="sigmoid")), (200, dict(scoring="softmax", renormalize=True)),
                                        (64, dict(scoring="sigmoid", num_groups=8, top_groups=4, group_top=2)),
                                        (96, dict(scoring="softmax", num_groups=4, top_groups=3))])
def test_two_neighbouring_picks_closer_than_fp32_can_tell(experts, kw):
    """One pair of choices, at every place among the picks and across their end, made to meet to within 2^-25."""
    g = torch.Generator().manual_seed(experts)
    rows, biases = [], []
    k = 6
    for trial in range(80):
        logits = torch.randn(experts, generator=g)
        bias = torch.randn(experts, generator=g) * 0.2
        score = torch.softmax(logits.double(), 0) if kw["scoring"] == "softmax" else torch.sigmoid(logits.double())
        order = (score + bias.double()).sort(descending=True).indices
        i = trial % (k + 1)
        hi, lo = order[i], order[i + 1]
        bias[lo] = (score[hi] + bias[hi].double() - score[lo]).float()  # exact but for the bias's own rounding
        rows.append(logits), biases.append(bias)
    flips = 0
    for logits, bias in zip(rows, biases):
        _, e = compare(logits[None].to(DEV), k, bias=bias.to(DEV), **kw)
        fp32 = (torch.softmax(logits, 0) if kw["scoring"] == "softmax" else torch.sigmoid(logits)) + bias
        flips += fp32.sort(descending=True, stable=True).indices[:k].tolist() != e[0].tolist()
    assert flips > 0


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,groups,biased", [(64, 8, True), (60, 6, True), (256, 8, True), (64, 8, False), (60, 6, False)])
def test_neighbouring_groups_closer_than_fp32_can_tell(experts, groups, biased, scoring):
    """The last group that stays and the first that goes meet to within a rounding, in sums of two choices."""
    g = torch.Generator().manual_seed(experts + groups)
    size, keep = experts // groups, groups // 2
    for trial in range(30):
        logits = torch.randn(experts, generator=g)
        bias = torch.randn(experts, generator=g) * 0.1 if biased else None
        score = torch.softmax(logits.double(), 0) if scoring == "softmax" else torch.sigmoid(logits.double())
        choice = (score + bias.double() if biased else score).view(groups, size)
        best = choice.sort(1, descending=True).values[:, :2].sum(1)
        order = best.sort(descending=True).indices
        a, b = order[keep - 1], order[keep]
        if biased:
            top = int(choice[b].argmax()) + int(b) * size
            bias[top] = (bias[top].double() + best[a] - best[b]).float()
        else:  # the same two logits in both groups, in other places: a tie, and a last-place step away from one
            pair = logits.view(groups, size)[a].sort(descending=True).values[:2]
            logits.view(groups, size)[b] = -3.0
            logits.view(groups, size)[b, 1], logits.view(groups, size)[b, 3] = pair[1], pair[0]
            if trial % 3:
                step = torch.tensor(math.inf if trial % 3 == 1 else -math.inf)
                logits.view(groups, size)[b, 3] = torch.nextafter(pair[0], step)
        kw = dict(scoring=scoring, num_groups=groups, top_groups=keep, group_top=2)
        compare(logits[None].to(DEV), 5, bias=None if bias is None else bias.to(DEV), **kw)
        compare(logits[None].to(DEV), 5, bias=None if bias is None else bias.to(DEV), **{**kw, "group_top": 1})


@pytest.mark.parametrize("seed", range(6))
def test_nan_and_infinite_logits(seed):
    logits = torch.randn(6, 96, generator=torch.Generator().manual_seed(seed)).to(DEV)
    logits[1, 7] = math.nan
    logits[2] = math.nan
    logits[3, 9] = math.inf
    for scoring in ("softmax", "sigmoid"):
        for kw in ({}, dict(num_groups=8, top_groups=3, group_top=2), dict(num_groups=6, top_groups=2),
                   dict(bias=torch.zeros(96, device=DEV), renormalize=True)):
            w, e = hb.route_experts(logits, 6, scoring=scoring, **kw)
            assert torch.isnan(w[1]).all() and torch.isnan(w[2]).all()
            if scoring == "softmax":
                assert torch.isnan(w[3]).all()
            else:  # a score of 1, whatever the group makes of it
                assert torch.equal(e[3:4].cpu(), route(logits[3:4], 6, scoring=scoring, **kw)[1]) and torch.isfinite(w[3]).all()
            assert torch.isfinite(w[[0, 4, 5]]).all()
            assert ((e >= 0) & (e < 96)).all() and all(len(set(r)) == 6 for r in e.tolist())
    bias = torch.zeros(96, device=DEV)
    bias[40] = math.nan
    for kw in ({}, dict(num_groups=8, top_groups=1), dict(num_groups=6, top_groups=2, group_top=2)):
        w, e = hb.route_experts(logits, 6, scoring="sigmoid", bias=bias, **kw)
        assert torch.isnan(w).all() and all(len(set(r)) == 6 for r in e.tolist())
    # infinite biases force an expert in or keep it out
    bias[40], bias[41] = math.inf, -math.inf
    clean = torch.randn(6, 96, generator=torch.Generator().manual_seed(seed + 50)).to(DEV)
    for kw in ({}, dict(num_groups=8, top_groups=2), dict(num_groups=6, top_groups=2, group_top=2)):
        w, e = compare(clean, 6, scoring="sigmoid", bias=bias, **kw)
        assert (e[:, 0] == 40).all() and (e != 41).all()


def test_strides_empty_and_repeat():
    logits, kw = make(300, 160, torch.bfloat16, dict(bias=True, num_groups=8, top_groups=3))
    want = hb.route_experts(logits, 6, **kw)
    wide = torch.full((300, 171), math.nan, dtype=torch.bfloat16, device=DEV)
    wide[:, 3:163] = logits
    for view in (wide[:, 3:163], logits.t().contiguous().t()):
        assert all(torch.equal(a, b) for a, b in zip(hb.route_experts(view, 6, **kw), want))
    strided = torch.stack([kw["bias"], kw["bias"]], 1)[:, 1]
    assert all(torch.equal(a, b) for a, b in zip(hb.route_experts(logits, 6, **{**kw, "bias": strided}), want))
    row = logits[:1].expand(5, -1)
    w, e = hb.route_experts(row, 6, **kw)
    assert torch.equal(w, want[0][:1].expand(5, -1)) and torch.equal(e, want[1][:1].expand(5, -1))
    w, e = hb.route_experts(logits[:0], 6, **kw)
    assert w.shape == e.shape == (0, 6)


def test_large_batch_graph_and_operator():
    logits, kw = make(70001, 64, torch.bfloat16, dict(scoring="sigmoid", bias=True, renormalize=True, num_groups=8, top_groups=4, group_top=2))
    w, e = hb.route_experts(logits, 6, **kw)
    pick = torch.tensor([0, 1, 9471, 9472, 40000, 70000], device=DEV)
    rw, re = route(logits[pick], 6, **kw)
    assert torch.equal(e[pick].cpu(), re)
    w2, e2 = torch.ops.helion_b200.moe_route_experts(logits, 6, "sigmoid", kw["bias"], 8, 4, 2, True, 1.0)
    assert torch.equal(w, w2) and torch.equal(e, e2)
    torch.library.opcheck(torch.ops.helion_b200.moe_route_experts, (logits[:9], 6, "sigmoid", kw["bias"], 8, 4, 2, True, 1.0),
                          test_utils=("test_schema", "test_faketensor"))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gw, ge = hb.route_experts(logits, 6, **kw)
    logits.copy_(logits.flip(0))
    graph.replay()
    assert torch.equal(gw, w.flip(0)) and torch.equal(ge, e.flip(0))


def test_agrees_with_softmax_top_k():
    logits = torch.randn(4096, 128, device=DEV)
    w, e = hb.route_experts(logits, 8)
    w0, e0 = M.route_top_k(logits, 8)
    assert torch.equal(e, e0) and ((w - w0).abs() <= 16 * 2.0**-23 * w0).all()


# ---------------------------------------------------------------- together with the layers that use them
ROUTING = dict(scoring="sigmoid", num_groups=4, top_groups=2, group_top=2, renormalize=True, scale=2.5)


def _moe_problem(t, h, inter, e, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(t, h, generator=g).to(torch.bfloat16).to(DEV)
    w_gu = M.quantize_expert_weights((torch.randn(e, 2 * inter, h, generator=g) * 0.02).to(DEV))
    w_d = M.quantize_expert_weights((torch.randn(e, h, inter, generator=g) * 0.02).to(DEV))
    bias = (torch.randn(e, generator=g) * 0.1).to(DEV)
    return x, M.interleave_gate_up(w_gu), w_d, hb.Routing(bias=bias, **ROUTING), g


def test_moe_layer_with_routing():
    t, h, inter, e, k = 72, 256, 128, 16, 4
    x, w_gu, w_d, routing, g = _moe_problem(t, h, inter, e)
    logits = torch.randn(t, e, generator=g).to(DEV)
    got = {}
    y = M.nvfp4_moe(x, logits, k, w_gu, w_d, routing=routing, intermediates=got)
    weights, experts = routing(logits, k)
    assert torch.equal(got["weights"], weights) and torch.equal(got["experts"], experts)
    assert torch.equal(M.nvfp4_moe(x, logits, k, w_gu, w_d, routing=routing), y)  # through the registered operator
    # the same layer from its parts
    sched = M.build_schedule(experts, e)
    o = M.grouped_matmul(got["a2"], got["sf2"], w_d, sched, got["g2"])
    want = torch.zeros(t, h, dtype=torch.float64, device=DEV)
    for s in range(k):
        rows = sched.row_of_pair.view(t, k)[:, s].long()
        want += weights[:, s : s + 1].double() * o[rows].double()
    # fp32 sum of k terms (k units of the largest partial sum) and one rounding to bf16
    mag = torch.zeros_like(want)
    for s in range(k):
        mag += (weights[:, s : s + 1].double() * o[sched.row_of_pair.view(t, k)[:, s].long()].double()).abs()
    assert ((y.double() - want).abs() <= 2.0**-8 * 1.01 * want.abs() + 2 * k * 2.0**-24 * mag + 1e-30).all()
    # twice the scale is twice the result, and no routing is softmax and top-k as before
    twice = hb.Routing(**{**routing.__dict__, "scale": 5.0})
    assert torch.equal(M.nvfp4_moe(x, logits, k, w_gu, w_d, routing=twice), 2 * y)
    base = {}
    M.nvfp4_moe(x, logits, k, w_gu, w_d, intermediates=base)
    assert torch.equal(base["experts"], M.route_top_k(logits, k)[1]) and torch.equal(base["weights"], M.route_top_k(logits, k)[0])


def test_expert_parallel_ranks_with_routing():
    world, t_local, h, inter, e, k = 2, 48, 256, 128, 8, 2
    x, w_gu, w_d, routing, g = _moe_problem(world * t_local, h, inter, e, seed=4)
    logits = torch.randn(world * t_local, e, generator=g).to(DEV)
    single = M.nvfp4_moe(x, logits, k, w_gu, w_d, routing=routing)
    nbytes = D.ExpertParallel.buffer_bytes(world, t_local, h, k, e)
    buffers = [torch.zeros(nbytes, dtype=torch.uint8, device=DEV) for _ in range(world)]
    dev = torch.device(DEV, torch.cuda.current_device())
    ranks = [D.ExpertParallel(dev, t_local, h, k, e, _emulate=(world, r, buffers)) for r in range(world)]

    def shard(b, r):
        sl = slice(r * e // world, (r + 1) * e // world)
        return M.GroupedNvfp4Weight(b.packed[sl].contiguous(), b.scales[sl].contiguous(), b.global_scale[sl].contiguous(), b.gate_up_interleaved)

    for r, ep in enumerate(ranks):
        sl = slice(r * t_local, (r + 1) * t_local)
        ep.dispatch(x[sl].contiguous(), logits[sl].contiguous(), routing)
    torch.cuda.synchronize()
    for r, ep in enumerate(ranks):
        ep.run_experts(shard(w_gu, r), shard(w_d, r))
    torch.cuda.synchronize()
    got = torch.cat([ep.combine() for ep in ranks])
    assert _lib.load().hb200_device_status(1) == 0
    # sums per rank first (11 significant bits), then over ranks, one rounding to bf16: a last-place flip at most
    floor = single.float().pow(2).mean().sqrt()
    assert float(((got.float() - single.float()).abs() / torch.maximum(single.float().abs(), floor)).max()) <= 2.0**-7


@pytest.mark.parametrize("t", [1, 40, 700])
def test_moe_block_from_router_to_shared_expert(t):
    """Router product, routing, NVFP4 experts, shared expert with the routed result as its residual: one layer, eager
    and captured, each step against its own formula."""
    h, inter, e, k = 512, 256, 16, 4
    x, w_gu, w_d, routing, g = _moe_problem(t, h, inter, e, seed=9)
    w_r = (torch.randn(e, h, generator=g) / h**0.5).to(torch.bfloat16).to(DEV)
    s_gu = (torch.randn(2 * inter, h, generator=g) / h**0.5).to(torch.bfloat16).to(DEV)
    s_d = (torch.randn(h, inter, generator=g) / inter**0.5).to(torch.bfloat16).to(DEV)

    def block():
        logits = hb.linear(x, w_r, out_dtype=torch.float32)
        routed = M.nvfp4_moe(x, logits, k, w_gu, w_d, routing=routing)
        hidden = hb.linear(x, s_gu, activation="silu_and_mul")
        return logits, routed, hidden, hb.linear(hidden, s_d, residual=routed)

    logits, routed, hidden, y = block()
    check_linear(logits, x, w_r)
    compare(logits, k, **routing.__dict__)
    check_linear(hidden, x, s_gu, activation="silu_and_mul")
    check_linear(y, hidden, s_d, residual=routed)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block()
    new = torch.randn(t, h, generator=g).to(torch.bfloat16).to(DEV)
    x.copy_(new)
    graph.replay()
    captured = [o.clone() for o in out]
    assert all(torch.equal(a, b) for a, b in zip(captured, block()))
    torch.cuda.synchronize()
    assert _lib.load().hb200_device_status(1) == 0


def test_block_traces_as_one_graph():
    """Router product, routing and a residual product under torch.compile with changing numbers of tokens."""
    g = torch.Generator().manual_seed(2)
    w_r = torch.randn(32, 256, generator=g).to(torch.bfloat16).to(DEV)
    w = (torch.randn(256, 256, generator=g) / 16).to(torch.bfloat16).to(DEV)
    routing = hb.Routing(bias=torch.randn(32, generator=g).to(DEV) * 0.1, **ROUTING)

    def block(x):
        weights, experts = routing(hb.linear(x, w_r, out_dtype=torch.float32), 4)
        return weights, experts, hb.linear(x, w, activation="silu", residual=x)

    compiled = torch.compile(block, backend="aot_eager", fullgraph=True, dynamic=True)
    with torch.no_grad():
        for t in (5, 9, 300):
            x = torch.randn(t, 256, generator=g).to(torch.bfloat16).to(DEV)
            assert all(torch.equal(a, b) for a, b in zip(compiled(x), block(x)))

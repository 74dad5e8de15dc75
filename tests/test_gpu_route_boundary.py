"""The end of the expert router's picks: equal inputs there, masks that are large but finite, scores that saturate."""

from __future__ import annotations

import math

import pytest
import torch

import helion_b200 as hb
from route_exact import picks
from route_reference import route

pytestmark = pytest.mark.gpu
DEV = "cuda"


def check(logits, top_k, **kw):
    """Indices against the definition, row by row where there are few of them."""
    _, e = hb.route_experts(logits, top_k, **kw)
    want = route(logits, top_k, **kw)[1] if logits.shape[0] <= 64 else picks(logits, top_k, **kw).cpu()
    wrong = (e.cpu() != want).any(1).nonzero().flatten().tolist()
    assert not wrong, f"{len(wrong)} rows, the first {wrong[0]}: {e[wrong[0]].tolist()}, not {want[wrong[0]].tolist()}"


def tied_rows(tokens, experts, dtype, top_k, mask, seed, step=0.25):
    """Logits on a grid, so that the last pick often has its equal behind it; the tail is padding with a finite mask."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    logits = (torch.randn(tokens, experts, generator=g, device=DEV) * 1.5 / step).round() * step
    logits = logits.to(dtype)
    if mask is not None:
        logits[:, experts - max(1, experts // 8):] = mask
        rows = torch.arange(0, tokens, 2, device=DEV)  # the first experts are equals around the place where the picks end
        if top_k < experts - max(1, experts // 8):
            logits[rows, top_k] = logits[rows, top_k - 1]
    return logits


# (experts, top_k, settings)
CONFIGS = [
    (16, 2, {}),
    (32, 4, dict(scoring="sigmoid")),
    (64, 6, dict(renormalize=True)),
    (128, 8, {}),
    (128, 8, dict(scoring="sigmoid", bias=0.25)),
    (256, 8, dict(scoring="sigmoid", bias=0.5, num_groups=8, top_groups=4, group_top=2)),
    (160, 6, dict(num_groups=8, top_groups=3)),
    (384, 10, dict(scoring="sigmoid", bias=0.0)),
    (1000, 32, {}),
]


def settings(experts, kw):
    kw = dict(kw)
    if "bias" in kw:
        kw["bias"] = torch.full((experts,), kw["bias"], device=DEV)
    return kw


def masks(dtype):
    return (None, -1e4, -65504.0) if dtype is torch.float16 else (None, -1e4, -1e9, -1e20)


def test_a_tie_at_the_end_hides_nothing():
    rows = [3, 1, 1, 9, 2, 4, 5, 6, 7, 8, 0, -1, -2, -3, -4, -1e9]
    check(torch.tensor([rows], device=DEV, dtype=torch.float32), 2)
    # scores that a step of 2^-24 cannot tell apart: two of them equal, the largest behind them
    check(torch.tensor([[17.0, 17.0, 18.0]], device=DEV), 1, scoring="sigmoid", bias=torch.zeros(3, device=DEV))
    # the last pick and the one behind it are equal, and both belong before the pick that stands in front of them
    check(torch.tensor([[16.75, 17.0, 17.0, 3.0]], device=DEV), 2, scoring="sigmoid", bias=torch.zeros(4, device=DEV))
    logits = torch.zeros(3, 64, device=DEV)  # one value alone, and one expert above or below it by a little
    logits[1, 63], logits[2, 0] = 2.0**-20, -(2.0**-20)
    for kw in ({}, dict(scoring="sigmoid"), dict(scoring="sigmoid", bias=torch.full((64,), 0.5, device=DEV))):
        check(logits, 5, **kw)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("experts,top_k,kw", CONFIGS)
def test_ties_and_finite_masks(experts, top_k, kw, dtype):
    for i, mask in enumerate(masks(dtype)):
        check(tied_rows(48, experts, dtype, top_k, mask, 10 * i + experts), top_k, **settings(experts, kw))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,top_k", [(24, 3), (64, 6), (256, 8)])
def test_saturated_scores_under_a_constant_bias(experts, top_k, scoring):
    """Sigmoids next to 1 and softmax tails next to 0: fp32 choices are all alike, the 64-bit ones are not."""
    g = torch.Generator(device=DEV).manual_seed(experts)
    grid = torch.randint(0, 24, (48, experts), generator=g, device=DEV) * 0.25
    logits = 15.0 + grid if scoring == "sigmoid" else grid - 20.0
    if scoring == "softmax":
        logits[:, experts // 2] = 4.0
    check(logits, top_k, scoring=scoring, bias=torch.full((experts,), 0.25, device=DEV))


MANY = [
    (32, 2, {}),
    (64, 6, dict(renormalize=True)),
    (64, 8, dict(scoring="sigmoid", bias=0.5, num_groups=8, top_groups=4, group_top=2)),
    (128, 8, {}),
    (128, 1, dict(scoring="sigmoid", bias=0.25)),
    (192, 8, dict(scoring="sigmoid", bias=0.25, num_groups=8, top_groups=4)),
    (256, 8, dict(scoring="sigmoid")),
    (256, 6, dict(scoring="sigmoid", bias=0.0, num_groups=8, top_groups=4, group_top=2)),
    (256, 5, dict(num_groups=8, top_groups=3)),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("experts,top_k,kw", MANY)
def test_ties_and_finite_masks_in_large_batches(experts, top_k, kw, dtype):
    for i, mask in enumerate(masks(dtype)):
        logits = tied_rows(16403, experts, dtype, top_k, mask, 10 * i + experts)
        logits[5000:6000] = 0.0  # rows of padding, all of one value
        logits[6000:6500, ::2] = -1.0
        check(logits, top_k, **settings(experts, kw))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,top_k", [(64, 6), (256, 8)])
def test_saturated_scores_in_large_batches(experts, top_k, scoring):
    g = torch.Generator(device=DEV).manual_seed(experts)
    grid = torch.randint(0, 24, (16403, experts), generator=g, device=DEV) * 0.25
    logits = 15.0 + grid if scoring == "sigmoid" else grid - 20.0
    if scoring == "softmax":
        logits[:, experts // 2] = 4.0
    check(logits, top_k, scoring=scoring, bias=torch.full((experts,), 0.25, device=DEV))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_three_choices_within_rounding_at_the_bottom_of_the_range(scoring):
    """As many lanes with experts as picks and one more, and a third choice next to the smallest of the lanes' best: the
    last pick, the one left behind and that one meet to within 2^-25."""
    g = torch.Generator().manual_seed(5)
    behind = 0
    for trial in range(200):
        live = [0, 1, 2, 4]  # two experts to a lane: 0 leads, 1 shares its lane
        logits = torch.full((64,), -math.inf)
        logits[live] = torch.randn(4, generator=g)
        score = torch.softmax(logits.double(), 0) if scoring == "softmax" else torch.sigmoid(logits.double())
        bias = torch.zeros(64)
        bias[live] = (0.75 - score[live]).float()
        bias[0] += 0.25
        exact = score + bias.double()
        behind += int(exact[1] > min(exact[2], exact[4]))
        check(logits[None].to(DEV), 2, scoring=scoring, bias=bias.to(DEV))
    assert behind > 50  # the third one belongs among the picks often enough


@pytest.mark.parametrize("tokens", [3, 16403])
@pytest.mark.parametrize("experts,groups", [(64, 8), (24, 8), (60, 12), (256, 32)])
def test_group_scores_beyond_fp32(experts, groups, tokens):
    """Sums of two choices that fp32 cannot hold, upwards and downwards: the larger sum is still the larger."""
    g = torch.Generator(device=DEV).manual_seed(experts)
    logits = torch.randn(tokens, experts, generator=g, device=DEV)
    logits[1] = 0.5
    size = experts // groups
    for sign in (1, -1):
        bias = torch.zeros(groups, size, device=DEV)
        bias[1], bias[2] = sign * 3e38, sign * 2e38
        bias[4] = 3.2e38  # (the largest where they are positive, alone in its group where they are negative)
        if sign < 0:
            bias[[0, *range(3, groups)]] = -3.2e38
        for top_k in (2, size):
            check(logits, top_k, scoring="sigmoid", bias=bias.flatten(), num_groups=groups, group_top=2)


@pytest.mark.parametrize("tokens", [48, 16403])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("size,lead", [(8, 100.0), (8, 1e4), (8, 1e8), (5, 1e4), (2, 1e6), (32, 1e4)])
def test_group_scores_that_cancel(size, lead, scoring, tokens):
    """Two choices of opposite sign whose sum is what the groups differ by: far less than the choices' own rounding."""
    groups = 8
    g = torch.Generator(device=DEV).manual_seed(size)
    logits = torch.randn(tokens, groups * size, generator=g, device=DEV)
    bias = torch.full((groups, size), -2 * lead, device=DEV)
    bias[:, 0], bias[:, -1] = lead, -lead  # each group's best two; their sum is that of two scores
    check(logits, 2, scoring=scoring, bias=bias.flatten(), num_groups=groups, top_groups=3, group_top=2)

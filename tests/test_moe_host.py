"""Argument checks of the NVFP4 MoE layer (no GPU: fake tensors)."""

from __future__ import annotations

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import helion_b200 as hb
from helion_b200 import dist as D
from helion_b200 import moe as M


def problem(tokens=6, experts=8, hidden=256, inter=128):
    def weight(n, k):
        return M.GroupedNvfp4Weight(torch.empty(experts, n, k // 2, dtype=torch.uint8, device="cuda"),
                                    torch.empty(experts, n * k // 16, device="cuda").to(torch.float8_e4m3fn),
                                    torch.empty(experts, device="cuda"))

    x = torch.empty(tokens, hidden, dtype=torch.bfloat16, device="cuda")
    return x, torch.empty(tokens, experts, device="cuda"), weight(2 * inter, hidden), weight(hidden, inter)


@pytest.mark.parametrize("settings", [dict(scoring=""), dict(scoring="", num_groups=4, top_groups=2, scale=2.5),
                                      dict(scoring="relu"), dict(scoring=None)])
def test_an_unknown_scoring_is_refused_on_every_path(settings):
    with FakeTensorMode():
        x, logits, w_gu, w_d = problem()
        for kw in ({}, {"intermediates": {}}):
            with pytest.raises(ValueError, match="scoring must be"):
                M.nvfp4_moe(x, logits, 2, w_gu, w_d, routing=hb.Routing(**settings), **kw)
        with pytest.raises(ValueError, match="scoring must be"):
            hb.Routing(**settings)(logits, 2)


def test_settings_without_a_scoring_are_refused_by_the_registered_operator():
    with FakeTensorMode():
        x, logits, w_gu, w_d = problem()
        bundles = (w_gu.packed, w_gu.scales, w_gu.global_scale, False, w_d.packed, w_d.scales, w_d.global_scale)
        assert torch.ops.helion_b200.nvfp4_moe(x, logits, 2, *bundles).shape == x.shape
        assert M.nvfp4_moe(x, logits, 2, w_gu, w_d, routing=hb.Routing("sigmoid", renormalize=True)).shape == x.shape
        for kw in (dict(route_bias=torch.empty(8, device="cuda")), dict(num_groups=2, top_groups=1), dict(group_top=2),
                   dict(renormalize=True), dict(route_scale=2.5)):
            with pytest.raises(ValueError, match="scoring must be"):
                torch.ops.helion_b200.nvfp4_moe(x, logits, 2, *bundles, **kw)


@pytest.mark.parametrize("routing", [None, hb.Routing("sigmoid")])
@pytest.mark.parametrize("shape", [(5, 8), (7, 8), (1, 8), (6, 9), (48,)])
def test_logits_that_do_not_fit_tokens_and_experts_are_refused(shape, routing):
    """Other rows than x has, or experts without weights: the row tables would be read where nothing was written."""
    with FakeTensorMode():
        x, _, w_gu, w_d = problem()
        for kw in ({}, {"intermediates": {}}):
            with pytest.raises(ValueError, match=r"router_logits must be \[6, 8\]"):
                M.nvfp4_moe(x, torch.empty(shape, device="cuda"), 2, w_gu, w_d, routing=routing, **kw)
        with pytest.raises(ValueError, match="one device"):
            M.nvfp4_moe(x, torch.empty(6, 8, device="cuda:1"), 2, w_gu, w_d, routing=routing)


@pytest.mark.parametrize("routing", [None, hb.Routing("sigmoid")])
@pytest.mark.parametrize("shape", [(5, 8), (7, 8), (6, 9), (48,)])
def test_expert_parallel_refuses_logits_that_do_not_fit(shape, routing):
    tokens, hidden, top_k, experts = 6, 256, 2, 8
    buffers = [torch.zeros(D.ExpertParallel.buffer_bytes(2, tokens, hidden, top_k, experts), dtype=torch.uint8) for _ in range(2)]
    rank = D.ExpertParallel(torch.device("cpu"), tokens, hidden, top_k, experts, _emulate=(2, 0, buffers))
    with pytest.raises(ValueError, match=r"router_logits must be \[6, 8\]"):
        rank.dispatch(torch.zeros(tokens, hidden, dtype=torch.bfloat16), torch.zeros(shape), routing)

"""Calls of the fused linear layer at the edges of what its documentation allows."""

from __future__ import annotations

import math

import pytest
import torch

import helion_b200 as hb
from linear_reference import GATED
from linear_reference import activate

pytestmark = pytest.mark.gpu
DEV = "cuda"
ACTIVATIONS = ("none", "relu", "silu", "gelu", "gelu_tanh", *GATED)


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n", [(1, 24), (40, 200), (300, 7136), (2048, 1024)])
@pytest.mark.parametrize("activation", ACTIVATIONS)
def test_activations_at_both_infinities(m, n, activation, out):
    """Sums of +inf and -inf through every activation: what the formula makes of them, NaN included."""
    base, gated = activation.removesuffix("_and_mul"), activation in GATED
    x = torch.zeros(m, 64, dtype=torch.bfloat16, device=DEV)
    weight = torch.zeros(2 * n if gated else n, 64, dtype=torch.bfloat16, device=DEV)
    v = torch.tensor([math.inf, -math.inf, math.nan, -3e38, 3e38, -20000.0, -0.0, 1.0], device=DEV).repeat(n // 8 + 1)[:n]
    bias = torch.cat([v, torch.full((n,), 0.5, device=DEV)]) if gated else v
    y = hb.linear(x, weight, bias, activation=activation, out_dtype=out)
    want = activate(v.double(), base) * (0.5 if gated else 1.0)
    assert torch.equal(torch.isnan(y), torch.isnan(want).expand(m, -1))
    # what is finite here is 0, 1 or so and +-3e38: the epilogue's 2^-20 and one rounding
    ok = torch.isfinite(want)
    step = torch.finfo(out).eps / 2 + 2.0**-19
    assert ((y.double() - want).abs() <= step * want.abs() + 2.0**-126).logical_or(~ok).all()
    assert torch.equal(y[:, torch.isinf(want)].double(), want[torch.isinf(want)].expand(m, -1))


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
@pytest.mark.parametrize("shape", [(5, 64), (2, 3, 64)])
def test_traced_calls_run_their_kernels(shape):
    g = torch.Generator(device=DEV).manual_seed(1)
    w = torch.randn(24, 64, generator=g, device=DEV).to(torch.bfloat16)

    def block(x):
        y = hb.linear(x, w, activation="silu", residual=x[..., :24])
        return (y, *hb.route_experts(hb.linear(x, w, out_dtype=torch.float32).flatten(0, -2), 3, scoring="sigmoid"))

    traced = torch.jit.trace(block, (torch.randn(shape, generator=g, device=DEV).to(torch.bfloat16),))
    for _ in range(2):
        x = torch.randn(shape, generator=g, device=DEV).to(torch.bfloat16)
        junk = [torch.full_like(t, 7) for t in block(x)]  # (what an output that nothing writes would hold)
        del junk
        assert all(torch.equal(a, b) for a, b in zip(traced(x), block(x)))

"""What the fused linear layer and the expert router see of tracers and derivatives: host logic, on plain stand-ins for
the kernels (no GPU)."""

from __future__ import annotations

import pytest
import torch

import helion_b200 as hb
from helion_b200 import fused_linear
from helion_b200 import routing


@pytest.fixture(autouse=True)
def stand_ins(monkeypatch):
    def linear(x, weight, bias, residual, activation, out_dtype):
        y = x.float() @ weight.float().t()
        return (y if residual is None else y + residual.float()).to(out_dtype)

    def route(logits, top_k, *settings):
        weights, experts = torch.softmax(logits.float(), 1).topk(top_k)
        return weights, experts

    monkeypatch.setattr(fused_linear, "_linear_cuda", linear)
    monkeypatch.setattr(routing, "_route_cuda", route)


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning", "ignore::DeprecationWarning")
@pytest.mark.parametrize("shape", [(3, 16), (2, 3, 16)])
def test_a_trace_records_the_operators(shape):
    w = torch.randn(8, 16).to(torch.bfloat16)
    linear = torch.jit.trace(lambda x: hb.linear(x, w, residual=x[..., :8]) * 2, (torch.randn(shape).to(torch.bfloat16),))
    assert "helion_b200::linear" in str(linear.graph)
    x = torch.randn(shape).to(torch.bfloat16)
    assert torch.equal(linear(x), hb.linear(x, w, residual=x[..., :8]) * 2)
    route = torch.jit.trace(lambda logits: hb.route_experts(logits, 2), (torch.randn(4, 8),))
    assert "helion_b200::moe_route_experts" in str(route.graph)
    logits = torch.randn(7, 8)
    assert all(torch.equal(a, b) for a, b in zip(route(logits), hb.route_experts(logits, 2)))


def test_forward_mode_derivatives_are_refused():
    """Neither operator has one; without a word the tangent would be lost."""
    w, x = torch.randn(8, 16).to(torch.bfloat16), torch.randn(3, 16).to(torch.bfloat16)
    logits = torch.randn(4, 8)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: hb.linear(dual, w), lambda: hb.linear(x, w, residual=dual[:, :8]),
                     lambda: hb.route_experts(torch.autograd.forward_ad.make_dual(logits, logits), 2)):
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call()
        assert hb.linear(x, w).shape == (3, 8)  # nothing to lose
    for transform in (lambda f: torch.func.jvp(f, (x,), (x,)), lambda f: torch.func.jacfwd(f)(x),
                      lambda f: torch.func.jvp(lambda v: torch.vmap(f)(v), (x,), (x,))):
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            transform(lambda v: hb.linear(v, w))
    with pytest.raises(RuntimeError, match="no forward-mode derivative"):
        torch.func.jvp(lambda v: hb.route_experts(v, 2)[0], (logits,), (logits,))
    # without a tangent of their own they run, in any nesting
    assert torch.func.vmap(lambda v: hb.linear(v, w))(x).shape == (3, 8)
    inner = torch.func.jvp(lambda v: v + torch.vmap(lambda u: hb.linear(u, w))(x), (x[:, :8],), (x[:, :8],))
    assert torch.equal(inner[1], x[:, :8])
    outer = torch.vmap(lambda u: torch.func.jvp(lambda v: v + hb.linear(u, w), (u[:8],), (u[:8],))[1])(x)
    assert torch.equal(outer, x[:, :8])

"""Argument checks of the fused linear layer and of the expert router, and their C entry points' refusals (no GPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

import helion_b200 as hb
from helion_b200 import _lib
from helion_b200.fused_linear import _ARGS
from helion_b200.routing import _ARGS as _ROUTE_ARGS


def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize(
    "error,match,args,kwargs",
    [
        (ValueError, "activation must be one of", (_t(2, 16), _t(8, 16)), {"activation": "swish"}),
        (TypeError, "operands of one type", (_t(2, 16, dtype=torch.float32), _t(8, 16, dtype=torch.float32)), {}),
        (TypeError, "operands of one type", (_t(2, 16), _t(8, 16, dtype=torch.float16)), {}),
        (TypeError, "out_dtype must be", (_t(2, 16), _t(8, 16)), {"out_dtype": torch.float16}),
        (ValueError, "weight .rows, K.", (_t(2, 16), _t(8, 2, 16)), {}),
        (ValueError, "does not match x", (_t(2, 16), _t(8, 24)), {}),
        (ValueError, "positive multiple of 8", (_t(2, 12), _t(8, 12)), {}),
        (ValueError, "positive multiple of 8", (_t(2, 0), _t(8, 0)), {}),
        (ValueError, "gate half", (_t(2, 16), _t(7, 16)), {"activation": "silu_and_mul"}),
        (ValueError, "bias must be .8.", (_t(2, 16), _t(8, 16), _t(7)), {}),
        (ValueError, "bias must be .8.", (_t(2, 16), _t(8, 16), _t(1, 8)), {}),
        (TypeError, "bias must be", (_t(2, 16), _t(8, 16), _t(8, dtype=torch.float16)), {}),
        (ValueError, "residual must be", (_t(2, 16), _t(8, 16)), {"residual": _t(1, 8)}),
        (ValueError, "residual must be", (_t(2, 16), _t(8, 16)), {"residual": _t(2, 8), "activation": "silu_and_mul"}),
        (TypeError, "residual must be", (_t(2, 16), _t(8, 16)), {"residual": _t(2, 8), "out_dtype": torch.float32}),
        (ValueError, "one device", (_t(2, 16), _t(8, 16).to("meta")), {}),
        (RuntimeError, "no CPU fallback", (_t(2, 16), _t(8, 16)), {}),
    ],
)
def test_linear_refusals(error, match, args, kwargs):
    with pytest.raises(error, match=match):
        hb.linear(*args, **kwargs)


def test_linear_traces_under_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(3, 5, 64, dtype=torch.float16, device="cuda")
        w = torch.empty(26, 64, dtype=torch.float16, device="cuda")
        y = hb.linear(x, w, activation="gelu_and_mul", residual=torch.empty(3, 5, 13, device="cuda"), out_dtype=torch.float32)
        assert y.shape == (3, 5, 13) and y.dtype is torch.float32
        with pytest.raises(ValueError, match="does not match"):
            hb.linear(x, w[:, :32])


def test_linear_entry_point_rejects_bad_arguments_before_any_cuda_call():
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 15) // 16 * 16

    def call(x=p, w=p, bias=None, res=None, out=p, m=4, n=8, k=16, ldx=16, ldw=16, ldr=8, ldo=8, act=0, bias_f32=0):
        return lib.hb200_linear(_ARGS.pack(x or 0, w or 0, bias or 0, res or 0, out or 0, m, n, k, ldx, ldw, ldr, ldo, act, 0, 1,
                                           bias_f32, 0, 0), None)

    bad, unsupported = _lib.HB200_ERR_INVALID_ARGUMENT, _lib.HB200_ERR_UNSUPPORTED
    assert call(x=None) == bad and call(w=None) == bad and call(out=None) == bad
    assert call(m=0) == bad and call(n=0) == bad and call(k=0) == bad
    assert call(ldx=8) == bad and call(ldw=8) == bad and call(ldo=4) == bad and call(res=p, ldr=-8) == bad
    assert call(act=5) == bad and call(act=-1) == bad
    assert call(k=12) == unsupported and call(ldx=20) == unsupported and call(ldw=20) == unsupported
    assert call(x=p + 2) == unsupported and call(w=p + 8) == unsupported
    assert call(out=p + 1) == bad and call(bias=p + 2, bias_f32=1) == bad and call(res=p + 1) == bad
    assert call(m=1 << 30) == unsupported
    assert lib.hb200_linear(None, None) == bad


@pytest.mark.parametrize(
    "error,match,logits,top_k,kwargs",
    [
        (ValueError, "tokens, experts", torch.zeros(8), 2, {}),
        (TypeError, "bfloat16, float16 or float32", torch.zeros(4, 8, dtype=torch.float64), 2, {}),
        (ValueError, "1024 experts", torch.zeros(4, 1025), 2, {}),
        (ValueError, "1024 experts", torch.zeros(4, 0), 1, {}),
        (ValueError, "scoring", torch.zeros(4, 8), 2, {"scoring": "relu"}),
        (ValueError, "num_groups", torch.zeros(4, 8), 2, {"num_groups": 3}),
        (ValueError, "num_groups", torch.zeros(4, 66), 2, {"num_groups": 33}),
        (ValueError, "num_groups", torch.zeros(4, 8), 2, {"num_groups": 0}),
        (ValueError, "top_groups", torch.zeros(4, 8), 2, {"num_groups": 4, "top_groups": 5}),
        (ValueError, "top_groups", torch.zeros(4, 8), 2, {"top_groups": 0}),
        (ValueError, "group_top", torch.zeros(4, 8), 2, {"num_groups": 4, "group_top": 3}),
        (ValueError, "group_top", torch.zeros(4, 8), 1, {"num_groups": 8, "group_top": 2}),
        (ValueError, "top_k", torch.zeros(4, 8), 0, {}),
        (ValueError, "top_k", torch.zeros(4, 8), 9, {}),
        (ValueError, "top_k", torch.zeros(4, 64), 33, {}),
        (ValueError, "top_k", torch.zeros(4, 8), 3, {"num_groups": 4, "top_groups": 1}),
        (ValueError, "bias must be .8.", torch.zeros(4, 8), 2, {"bias": torch.zeros(7)}),
        (TypeError, "bias must be float32", torch.zeros(4, 8), 2, {"bias": torch.zeros(8, dtype=torch.bfloat16)}),
        (ValueError, "one device", torch.zeros(4, 8), 2, {"bias": torch.zeros(8, device="meta")}),
        (RuntimeError, "no CPU fallback", torch.zeros(4, 8), 2, {}),
    ],
)
def test_route_refusals(error, match, logits, top_k, kwargs):
    with pytest.raises(error, match=match):
        hb.route_experts(logits, top_k, **kwargs)
    with pytest.raises(error, match=match):
        hb.Routing(**kwargs)(logits, top_k)


def test_route_traces_under_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        w, e = hb.route_experts(torch.empty(5, 64, device="cuda", dtype=torch.bfloat16), 6, num_groups=8, top_groups=2)
        assert w.shape == e.shape == (5, 6) and w.dtype is torch.float32 and e.dtype is torch.int64


def test_route_entry_point_rejects_bad_arguments_before_any_cuda_call():
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 15) // 16 * 16

    def call(logits=p, dtype=2, tokens=4, experts=8, ld=8, k=2, scoring=0, groups=1, top_groups=1, group_top=1, w=p, c=p):
        return lib.hb200_moe_route_experts(_ROUTE_ARGS.pack(logits or 0, 0, w or 0, c or 0, tokens, experts, ld, k, groups, top_groups,
                                                            group_top, dtype, scoring, 0, 1.0), None)

    bad = _lib.HB200_ERR_INVALID_ARGUMENT
    assert call(logits=None) == bad and call(w=None) == bad and call(c=None) == bad
    assert call(dtype=3) == bad and call(scoring=2) == bad and call(tokens=-1) == bad
    assert call(experts=0) == bad and call(experts=1025) == bad and call(ld=-1) == bad
    assert call(k=0) == bad and call(k=9) == bad and call(groups=3) == bad and call(groups=4, top_groups=5) == bad
    assert call(groups=4, k=3) == bad and call(group_top=3) == bad and call(groups=8, group_top=2, k=1) == bad
    assert call(tokens=0) == 0 and lib.hb200_moe_route_experts(None, None) == bad


def test_reference_router_in_small():
    """The tests' own reference: values worked out by hand."""
    from route_reference import route_row

    w, p = route_row([0.0, 2.0, 1.0, -1.0], 2, "softmax", None, 2, 1, 1, True, 1.0)
    assert p == [1, 0] and abs(w[0] - 1 / (1 + 2.718281828459045**-2)) < 1e-12 and abs(sum(w) - 1) < 1e-12
    w, p = route_row([0.0, 0.0, 0.0, 0.0], 2, "sigmoid", [0.0, 0.1, 0.1, 0.0], 1, 1, 1, False, 4.0)
    assert p == [1, 2] and w == [2.0, 2.0]
    w, p = route_row([float("-inf")] * 4, 3, "softmax", None, 2, 2, 2, True, 1.0)
    assert p == [0, 1, 2] and w == [0.0, 0.0, 0.0]

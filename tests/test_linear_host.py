"""Argument checks of the fused linear layer and of the expert router, and their C entry points' refusals (no GPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

import helion_b200 as hb
from helion_b200 import _lib


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
        return lib.hb200_linear(x, w, bias, res, out, m, n, k, ldx, ldw, ldr, ldo, act, 0, 1, bias_f32, 0, None)

    bad, unsupported = _lib.HB200_ERR_INVALID_ARGUMENT, _lib.HB200_ERR_UNSUPPORTED
    assert call(x=None) == bad and call(w=None) == bad and call(out=None) == bad
    assert call(m=0) == bad and call(n=0) == bad and call(k=0) == bad
    assert call(ldx=8) == bad and call(ldw=8) == bad and call(ldo=4) == bad and call(res=p, ldr=-8) == bad
    assert call(act=5) == bad and call(act=-1) == bad
    assert call(k=12) == unsupported and call(ldx=20) == unsupported and call(ldw=20) == unsupported
    assert call(x=p + 2) == unsupported and call(w=p + 8) == unsupported
    assert call(out=p + 1) == bad and call(bias=p + 2, bias_f32=1) == bad and call(res=p + 1) == bad
    assert call(m=1 << 30) == unsupported

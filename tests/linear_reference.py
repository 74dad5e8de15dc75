"""The fused linear layer in 64 bits, and how far a result may be from it."""

from __future__ import annotations

import math

import torch

GATED = ("silu_and_mul", "gelu_and_mul", "gelu_tanh_and_mul")
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
# the largest slope of each activation: an error e of its argument moves the result by at most slope * e
SLOPE = {"none": 1.0, "relu": 1.0, "silu": 1.1, "gelu": 1.13, "gelu_tanh": 1.13}


def activate(v: torch.Tensor, name: str) -> torch.Tensor:
    if name == "relu":
        return v.clamp_min(0)
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "gelu":
        return v * torch.special.ndtr(v)
    if name == "gelu_tanh":
        return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v**3))
    return v


def linear(x, weight, bias, activation, residual, out_dtype):
    """``(y, bound)``: the exact result and the largest error that fp32 sums, the fp32 epilogue and one rounding to
    ``out_dtype`` can leave.

    The tensor core adds 16 products to the accumulator at a time and may truncate: K / 16 additions (and up to 32
    within the first and last and over the partial sums of a split K range), each off by at most 2^-23 of a running
    sum that never exceeds sum |x w|.  For fp32 outputs a chain of such additions covers at most 640 elements of K; the
    chains' sums (of 256 elements at least) are added to nearest, each addition off by 2^-24.  The epilogue's
    exponential is off by a few units, scaled by its argument."""
    k = weight.shape[1]
    xd, wd = x.double().reshape(-1, k), weight.double()
    v = xd @ wd.t()
    additions = k / 16 if out_dtype is not torch.float32 else min(k, 640) / 16 + k / 512
    err = (additions + 32) * 2.0**-23 * (xd.abs() @ wd.abs().t())
    if bias is not None:
        v = v + bias.double()
        err = err + 2.0**-24 * v.abs()
    base = activation.removesuffix("_and_mul")
    up = None
    if activation in GATED:
        n = v.shape[1] // 2
        (v, up), (err, up_err) = (v[:, :n], v[:, n:]), (err[:, :n], err[:, n:])
    a = activate(v, base)
    err = SLOPE[base] * err
    if base != "none":
        err = err + 2.0**-20 * a.abs() * (1 + v.abs()) + 2.0**-23 * v.abs()
    if up is not None:
        err = err * (up.abs() + up_err) + a.abs() * up_err + 2.0**-24 * (a * up).abs()
        a = a * up
    if residual is not None:
        a = a + residual.double().reshape(a.shape)
        err = err + 2.0**-24 * a.abs()
    y = a.reshape(*x.shape[:-1], a.shape[-1])
    err = err.reshape(y.shape)
    return y, err + 1.01 * HALF_STEP[out_dtype] * (y.abs() + err) + 2.0**-25


def check(got, x, weight, bias=None, activation="none", residual=None):
    ref, bound = linear(x, weight, bias, activation, residual, got.dtype)
    assert got.shape == ref.shape
    excess = ((got.double() - ref).abs() - bound).max().item() if got.numel() else 0.0
    assert excess <= 0, f"off by {excess} more than the bound"

"""Linear layer with bias, activation (plain or gated) and residual in the matrix product's epilogue.

The un-quantised projections around the quantised operators of this package: a router's logits in fp32, the shared
expert of an MoE layer, biased or residual projections that stay in bf16 / fp16.  Inference only, like every operator
here: no autograd formula is registered.
"""

from __future__ import annotations

import torch
from torch import Tensor
from torch.utils._python_dispatch import _get_current_dispatch_mode

from . import _lib
from .ops import _require_cuda

# name -> (code of the C ABI, gated)
_ACTIVATIONS = {
    "none": (0, False),
    "relu": (1, False),
    "silu": (2, False),
    "gelu": (3, False),
    "gelu_tanh": (4, False),
    "silu_and_mul": (2, True),
    "gelu_and_mul": (3, True),
    "gelu_tanh_and_mul": (4, True),
}
_OPERAND_DTYPES = (torch.bfloat16, torch.float16)


def _check(x: Tensor, weight: Tensor, bias: Tensor | None, residual: Tensor | None, activation: str,
           out_dtype: torch.dtype) -> int:
    """Validates a call; returns the number of output columns."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {', '.join(_ACTIVATIONS)}; got {activation!r}")
    if x.dtype not in _OPERAND_DTYPES or weight.dtype != x.dtype:
        raise TypeError(f"linear takes bfloat16 or float16 operands of one type, got {x.dtype} and {weight.dtype}")
    if out_dtype not in (x.dtype, torch.float32):
        raise TypeError(f"out_dtype must be {x.dtype} or torch.float32, got {out_dtype}")
    if x.dim() < 1 or weight.dim() != 2:
        raise ValueError(f"linear expects x [..., K] and weight [rows, K]; got {tuple(x.shape)} and {tuple(weight.shape)}")
    rows, k = weight.shape
    if x.shape[-1] != k:
        raise ValueError(f"weight {tuple(weight.shape)} does not match x {tuple(x.shape)}")
    if k == 0 or k % 8:
        raise ValueError(f"K must be a positive multiple of 8, got {k}")
    n = rows
    if _ACTIVATIONS[activation][1]:
        if rows % 2:
            raise ValueError(f"{activation} needs a gate half and an up half of the weight's rows; got {rows} rows")
        n = rows // 2
    if bias is not None:
        if bias.dim() != 1 or bias.shape[0] != rows:
            raise ValueError(f"bias must be [{rows}], got {tuple(bias.shape)}")
        if bias.dtype not in (x.dtype, torch.float32):
            raise TypeError(f"bias must be {x.dtype} or torch.float32, got {bias.dtype}")
    if residual is not None:
        if residual.shape != (*x.shape[:-1], n):
            raise ValueError(f"residual must be {(*x.shape[:-1], n)}, got {tuple(residual.shape)}")
        if residual.dtype != out_dtype:
            raise TypeError(f"residual must be {out_dtype} (the output's type), got {residual.dtype}")
    for t in (weight, bias, residual):
        if t is not None and t.device != x.device:
            raise ValueError(f"all tensors must be on one device, got {x.device} and {t.device}")
    return n


def _tma_rows(t: Tensor) -> tuple[Tensor, int]:
    """``t [rows, K]`` as the kernels' bulk copies can read it (unit stride along K, 16-byte aligned rows that do not
    overlap), and its row pitch; anything else is copied."""
    rows, k = t.shape
    pitch = t.stride(0) if rows > 1 else k
    if t.stride(1) != 1 or pitch < k or pitch % 8 or t.data_ptr() % 16:
        return t.contiguous() if not t.is_contiguous() else t.clone(), k
    return t, pitch


def _linear_cuda(x: Tensor, weight: Tensor, bias: Tensor | None, residual: Tensor | None, activation: str,
                 out_dtype: torch.dtype) -> Tensor:
    n = _check(x, weight, bias, residual, activation, out_dtype)
    _require_cuda(x, weight, bias, residual)
    out = torch.empty((*x.shape[:-1], n), dtype=out_dtype, device=x.device)
    if out.numel() == 0:
        return out
    index = x.get_device()
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            _launch(out, x, weight, bias, residual, activation, n, index)
    else:
        _launch(out, x, weight, bias, residual, activation, n, index)
    return out


def _launch(out: Tensor, x: Tensor, weight: Tensor, bias: Tensor | None, residual: Tensor | None, activation: str, n: int,
            index: int) -> None:
    k = weight.shape[1]
    x2, ldx = _tma_rows(x if x.dim() == 2 else x.reshape(-1, k))
    w2, ldw = _tma_rows(weight)
    m = x2.shape[0]
    ldr = 0
    if residual is not None:
        residual = residual if residual.dim() == 2 else residual.reshape(-1, n)
        if n > 1 and residual.stride(1) != 1:
            residual = residual.contiguous()
        ldr = residual.stride(0)
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    code, gated = _ACTIVATIONS[activation]
    _lib.call(
        "hb200_linear", x2.data_ptr(), w2.data_ptr(), None if bias is None else bias.data_ptr(),
        None if residual is None else residual.data_ptr(), out.data_ptr(), m, n, k, ldx, ldw, ldr, n, code, gated,
        x.dtype is torch.bfloat16, bias is not None and bias.dtype is torch.float32, out.dtype is torch.float32,
        torch._C._cuda_getCurrentRawStream(index),
    )


@torch.library.custom_op("helion_b200::linear", mutates_args=())
def _linear_op(x: Tensor, weight: Tensor, bias: Tensor | None, residual: Tensor | None, activation: str,
               out_dtype: torch.dtype) -> Tensor:
    return _linear_cuda(x, weight, bias, residual, activation, out_dtype)


@_linear_op.register_fake
def _(x, weight, bias, residual, activation, out_dtype):
    n = _check(x, weight, bias, residual, activation, out_dtype)
    return x.new_empty((*x.shape[:-1], n), dtype=out_dtype)


def _plain(*tensors: Tensor | None) -> bool:
    """Whether a call can go straight to the kernel: nothing traces, and no subclass or gradient is involved."""
    if torch.compiler.is_compiling() or _get_current_dispatch_mode() is not None:
        return False
    grad = torch.is_grad_enabled()
    return all(t is None or (type(t) in (Tensor, torch.nn.Parameter) and not (grad and t.requires_grad)) for t in tensors)


def linear(x: Tensor, weight: Tensor, bias: Tensor | None = None, *, activation: str | None = None,
           residual: Tensor | None = None, out_dtype: torch.dtype | None = None) -> Tensor:
    """``activation(x @ weight.T + bias) + residual`` in one kernel, rounded once (``torch.ops.helion_b200.linear``).

    ``x [..., K]`` and ``weight [N, K]`` are bf16 or fp16 (one type); the products are summed in fp32, and bias,
    activation and residual are applied to the fp32 sum.  ``bias [N]``: the operands' type or fp32.
    ``residual [..., N]``: the output's type, any row pitch.  ``out_dtype``: the operands' type (default) or
    ``torch.float32``.

    ``activation``: ``None`` / ``"none"``, ``"relu"``, ``"silu"``, ``"gelu"`` (erf), ``"gelu_tanh"``, or a gated one,
    ``"silu_and_mul"``, ``"gelu_and_mul"``, ``"gelu_tanh_and_mul"``: ``weight [2 N, K]`` (and ``bias [2 N]``) then
    hold the gate rows first and the up rows second, as the package's ``silu_and_mul`` producers take them, and the
    result ``[..., N]`` is ``activation(gate) * up + residual``.

    ``K`` must be a multiple of 8.  Operands whose rows are not 16-byte aligned or have no unit stride along K are
    copied first.  Runs on the current stream of ``x``'s device; needs no workspace, so calls on several streams and
    captured graphs are independent of each other.  Infinities and NaN spread as in the formula.
    """
    activation = activation or "none"
    out_dtype = out_dtype or x.dtype
    if _plain(x, weight, bias, residual):  # a registered operator's dispatch costs more than a small call's kernel
        return _linear_cuda(x, weight, bias, residual, activation, out_dtype)
    _check(x, weight, bias, residual, activation, out_dtype)
    return _linear_op(x, weight, bias, residual, activation, out_dtype)

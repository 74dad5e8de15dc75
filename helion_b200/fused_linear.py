"""Linear layer with bias, activation (plain or gated) and residual in the matrix product's epilogue.

The un-quantised projections around the quantised operators of this package: a router's logits in fp32, the shared
expert of an MoE layer, biased or residual projections that stay in bf16 / fp16.  Inference only, like every operator
here: no autograd formula is registered.
"""

from __future__ import annotations

import struct

import torch
from torch import Tensor
from torch import is_grad_enabled as _is_grad_enabled
from torch._C import _are_functorch_transforms_active as _in_transform
from torch._C import _functorch
from torch._C import _is_tracing
from torch.autograd import forward_ad as _forward_ad
from torch.compiler import is_compiling as _is_compiling
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
_cuda_getDevice = getattr(torch._C, "_cuda_getDevice", None)  # (absent in a build without CUDA, where nothing gets there)
_cuda_getCurrentRawStream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_PLAIN = (Tensor, torch.nn.Parameter)
_ARGS = struct.Struct("=12q6i")  # hb200_linear_args (a bytes object passes through ctypes at a fifth of 18 values' cost)
_pack = _ARGS.pack


def _check(x: Tensor, weight: Tensor, bias: Tensor | None, residual: Tensor | None, activation: str,
           out_dtype: torch.dtype) -> tuple[int, int, int, bool, torch.Size]:
    """Validates a call; returns the number of output columns, the weight's rows, the activation's code and gating, and
    x's shape."""
    kind = _ACTIVATIONS.get(activation)
    if kind is None:
        raise ValueError(f"activation must be one of {', '.join(_ACTIVATIONS)}; got {activation!r}")
    code, gated = kind
    dtype, device, x_shape, w_shape = x.dtype, x.device, x.shape, weight.shape
    if (dtype is not torch.bfloat16 and dtype is not torch.float16) or weight.dtype is not dtype:
        raise TypeError(f"linear takes bfloat16 or float16 operands of one type, got {dtype} and {weight.dtype}")
    if out_dtype is not dtype and out_dtype is not torch.float32:
        raise TypeError(f"out_dtype must be {dtype} or torch.float32, got {out_dtype}")
    if len(x_shape) < 1 or len(w_shape) != 2:
        raise ValueError(f"linear expects x [..., K] and weight [rows, K]; got {tuple(x_shape)} and {tuple(w_shape)}")
    rows, k = w_shape
    if x_shape[-1] != k:
        raise ValueError(f"weight {tuple(w_shape)} does not match x {tuple(x_shape)}")
    if k == 0 or k % 8:
        raise ValueError(f"K must be a positive multiple of 8, got {k}")
    n = rows
    if gated:
        if rows % 2:
            raise ValueError(f"{activation} needs a gate half and an up half of the weight's rows; got {rows} rows")
        n = rows // 2
    if weight.device != device:
        raise ValueError(f"all tensors must be on one device, got {device} and {weight.device}")
    if bias is not None:
        if bias.shape != (rows,):
            raise ValueError(f"bias must be [{rows}], got {tuple(bias.shape)}")
        if bias.dtype is not dtype and bias.dtype is not torch.float32:
            raise TypeError(f"bias must be {dtype} or torch.float32, got {bias.dtype}")
        if bias.device != device:
            raise ValueError(f"all tensors must be on one device, got {device} and {bias.device}")
    if residual is not None:
        if residual.shape != (*x_shape[:-1], n):
            raise ValueError(f"residual must be {(*x_shape[:-1], n)}, got {tuple(residual.shape)}")
        if residual.dtype is not out_dtype:
            raise TypeError(f"residual must be {out_dtype} (the output's type), got {residual.dtype}")
        if residual.device != device:
            raise ValueError(f"all tensors must be on one device, got {device} and {residual.device}")
    return n, rows, code, gated, x_shape


def _tma_rows(t: Tensor, rows: int, k: int) -> tuple[Tensor, int, int]:
    """``t [rows, K]`` as the kernels' bulk copies can read it (unit stride along K, 16-byte aligned rows that do not
    overlap), its row pitch and its address; anything else is copied."""
    pitch, unit = t.stride()
    if rows == 1:
        pitch = k
    address = t.data_ptr()
    if unit != 1 or pitch < k or pitch % 8 or address % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        return t, k, t.data_ptr()
    return t, pitch, address


_entry = None
_allocate = getattr(getattr(getattr(torch._C, "_dynamo", None), "guards", None), "_empty_strided_cuda", None)


def _empty(size: tuple[int, ...], stride: tuple[int, ...], dtype: torch.dtype) -> Tensor:
    """Uninitialised tensor on the current CUDA device.  Straight to the allocator where this torch offers it (0.8 us;
    1.5 through ``torch.empty_strided``, 1.9 through ``new_empty``: a fifth of a small call's host time)."""
    if _allocate is not None:
        return _allocate(size, stride, dtype)
    return torch.empty_strided(size, stride, dtype=dtype, device="cuda")


def _linear_cuda(x: Tensor, weight: Tensor, bias: Tensor | None, residual: Tensor | None, activation: str,
                 out_dtype: torch.dtype) -> Tensor:
    global _entry
    n, rows, code, gated, x_shape = _check(x, weight, bias, residual, activation, out_dtype)
    index = x.get_device()
    if index < 0:
        _require_cuda(x)
    if _cuda_getDevice() != index:
        with torch.cuda.device(index):
            return _linear_cuda(x, weight, bias, residual, activation, out_dtype)
    if len(x_shape) == 2:
        m, k = x_shape
        out = _empty((m, n), (n, 1), out_dtype)
    else:
        out = x.new_empty((*x_shape[:-1], n), dtype=out_dtype)
        k = x_shape[-1]
        x = x.reshape(-1, k)
        m = x.shape[0]
    if m == 0 or n == 0:
        return out
    x, ldx, x_ptr = _tma_rows(x, m, k)
    weight, ldw, w_ptr = _tma_rows(weight, rows, k)
    ldr = res_ptr = bias_ptr = 0
    if residual is not None:
        if residual.dim() != 2:
            residual = residual.reshape(m, n)
        ldr, unit = residual.stride()
        if unit != 1 and n > 1:
            residual = residual.contiguous()
            ldr = n
        res_ptr = residual.data_ptr()
    bias_f32 = False
    if bias is not None:
        bias = bias.contiguous()
        bias_ptr, bias_f32 = bias.data_ptr(), bias.dtype is torch.float32
    if _entry is None:
        _entry = _lib.load().hb200_linear
    status = _entry(
        _pack(x_ptr, w_ptr, bias_ptr, res_ptr, out.data_ptr(), m, n, k, ldx, ldw, ldr, n, code, gated,
              x.dtype is torch.bfloat16, bias_f32, out_dtype is torch.float32, 0),
        _cuda_getCurrentRawStream(index),
    )
    if status:
        _lib.check(status, "hb200_linear")
    return out


@torch.library.custom_op("helion_b200::linear", mutates_args=())
def _linear_op(x: Tensor, weight: Tensor, bias: Tensor | None, residual: Tensor | None, activation: str,
               out_dtype: torch.dtype) -> Tensor:
    return _linear_cuda(x, weight, bias, residual, activation, out_dtype)


@_linear_op.register_fake
def _(x, weight, bias, residual, activation, out_dtype):
    n = _check(x, weight, bias, residual, activation, out_dtype)[0]
    return x.new_empty((*x.shape[:-1], n), dtype=out_dtype)


def _direct(*tensors: Tensor | None) -> bool:
    """Whether a call can go straight to its kernel: nothing traces (``torch.jit.trace`` would record the output's
    allocation alone) or transforms (the tensors of a ``torch.func`` transform look plain but have no address), and no
    subclass or gradient is involved.  The dispatch of a registered operator written in Python costs more host time than
    a small call's kernel runs."""
    if _is_compiling() or _is_tracing() or _get_current_dispatch_mode() is not None or _in_transform():
        return False
    grad = _is_grad_enabled()
    for t in tensors:
        if t is not None and (type(t) not in _PLAIN or (grad and t.requires_grad)):
            return False
    return True


def _refuse_tangents(name: str, *tensors: Tensor | None) -> None:
    """Inside a forward-mode level: an operator without a derivative would drop its inputs' tangents without a word."""
    for t in tensors:
        while t is not None and _functorch.is_batchedtensor(t):
            t = _functorch.get_unwrapped(t)
        if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"helion_b200::{name} has no forward-mode derivative")


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
    captured graphs are independent of each other.  Infinities and NaN spread as in the formula.  Gradients are refused:
    in ``backward``, and forward-mode ones in the call.
    """
    activation = activation or "none"
    out_dtype = out_dtype or x.dtype
    if _forward_ad._current_level >= 0:
        _refuse_tangents("linear", x, weight, bias, residual)
    if _direct(x, weight, bias, residual):
        return _linear_cuda(x, weight, bias, residual, activation, out_dtype)
    _check(x, weight, bias, residual, activation, out_dtype)
    return _linear_op(x, weight, bias, residual, activation, out_dtype)

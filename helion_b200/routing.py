"""Routing of tokens to experts beyond softmax-then-top-k: sigmoid scores, a balance bias, groups, renormalised weights."""

from __future__ import annotations

from dataclasses import dataclass
import functools
import struct

import torch
from torch import Tensor

from . import _lib
from .fused_linear import _cuda_getCurrentRawStream
from .fused_linear import _cuda_getDevice
from .fused_linear import _direct
from .fused_linear import _empty
from .fused_linear import _forward_ad
from .fused_linear import _refuse_tangents
from .ops import _require_cuda

_SCORINGS = {"softmax": 0, "sigmoid": 1}
_ARGS = struct.Struct("=11q3if")  # hb200_route_args
_pack = _ARGS.pack
_LOGIT_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _check_settings(experts: int, top_k: int, scoring: str, num_groups: int, top_groups: int, group_top: int) -> None:
    if not 1 <= experts <= 1024:
        raise ValueError(f"1 to 1024 experts are supported, got {experts}")
    if scoring not in _SCORINGS:
        raise ValueError(f"scoring must be 'softmax' or 'sigmoid'; got {scoring!r}")
    if not 1 <= num_groups <= 32 or experts % num_groups:
        raise ValueError(f"num_groups must be in 1..32 and divide the {experts} experts; got {num_groups}")
    if not 1 <= top_groups <= num_groups:
        raise ValueError(f"top_groups must be in 1..{num_groups}, got {top_groups}")
    size = experts // num_groups
    if group_top not in (1, 2) or group_top > size:
        raise ValueError(f"group_top must be 1 or 2 and at most a group's {size} experts; got {group_top}")
    if not 1 <= top_k <= min(32, top_groups * size):
        raise ValueError(f"top_k must be in 1..{min(32, top_groups * size)}, got {top_k}")


_check_settings_once = functools.lru_cache(maxsize=64)(_check_settings)  # a model's settings: looked at once


def _check(router_logits: Tensor, top_k: int, scoring: str, bias: Tensor | None, num_groups: int, top_groups: int,
           group_top: int) -> None:
    if router_logits.dim() != 2:
        raise ValueError("router_logits must be [tokens, experts]")
    experts = router_logits.shape[1]
    if router_logits.dtype not in _LOGIT_DTYPES:
        raise TypeError(f"router_logits must be bfloat16, float16 or float32, got {router_logits.dtype}")
    # (under tracing a size may be a symbol, which has no hash)
    check = _check_settings if torch.compiler.is_compiling() or type(experts) is not int else _check_settings_once
    check(experts, top_k, scoring, num_groups, top_groups, group_top)
    if bias is not None:
        if bias.shape != (experts,):
            raise ValueError(f"bias must be [{experts}], got {tuple(bias.shape)}")
        if bias.dtype is not torch.float32:
            raise TypeError(f"bias must be float32, got {bias.dtype}")
        if bias.device != router_logits.device:
            raise ValueError(f"all tensors must be on one device, got {router_logits.device} and {bias.device}")


_entry = None


def _route_cuda(router_logits: Tensor, top_k: int, scoring: str, bias: Tensor | None, num_groups: int, top_groups: int,
                group_top: int, renormalize: bool, scale: float) -> tuple[Tensor, Tensor]:
    global _entry
    _check(router_logits, top_k, scoring, bias, num_groups, top_groups, group_top)
    index = router_logits.get_device()
    if index < 0:
        _require_cuda(router_logits)
    if _cuda_getDevice() != index:
        with torch.cuda.device(index):
            return _route_cuda(router_logits, top_k, scoring, bias, num_groups, top_groups, group_top, renormalize, scale)
    tokens, experts = router_logits.shape
    weights = _empty((tokens, top_k), (top_k, 1), torch.float32)
    chosen = _empty((tokens, top_k), (top_k, 1), torch.int64)
    if tokens == 0:
        return weights, chosen
    pitch, unit = router_logits.stride()
    if unit != 1 and experts > 1:
        router_logits = router_logits.contiguous()
        pitch = experts
    bias_ptr = 0
    if bias is not None:
        bias = bias.contiguous()
        bias_ptr = bias.data_ptr()
    if _entry is None:
        _entry = _lib.load().hb200_moe_route_experts
    status = _entry(
        _pack(router_logits.data_ptr(), bias_ptr, weights.data_ptr(), chosen.data_ptr(), tokens, experts, pitch, top_k,
              num_groups, top_groups, group_top, _LOGIT_DTYPES[router_logits.dtype], _SCORINGS[scoring], renormalize, scale),
        _cuda_getCurrentRawStream(index),
    )
    if status:
        _lib.check(status, "hb200_moe_route_experts")
    return weights, chosen


@torch.library.custom_op("helion_b200::moe_route_experts", mutates_args=())
def _route_op(router_logits: Tensor, top_k: int, scoring: str, bias: Tensor | None, num_groups: int, top_groups: int,
              group_top: int, renormalize: bool, scale: float) -> tuple[Tensor, Tensor]:
    return _route_cuda(router_logits, top_k, scoring, bias, num_groups, top_groups, group_top, renormalize, scale)


@_route_op.register_fake
def _(router_logits, top_k, scoring, bias, num_groups, top_groups, group_top, renormalize, scale):
    _check(router_logits, top_k, scoring, bias, num_groups, top_groups, group_top)
    shape = (router_logits.shape[0], top_k)
    return router_logits.new_empty(shape, dtype=torch.float32), router_logits.new_empty(shape, dtype=torch.int64)


def route_experts(router_logits: Tensor, top_k: int, *, scoring: str = "softmax", bias: Tensor | None = None,
                  num_groups: int = 1, top_groups: int = 1, group_top: int = 1, renormalize: bool = False,
                  scale: float = 1.0) -> tuple[Tensor, Tensor]:
    """Chosen experts of every token and their weights, in one kernel (``torch.ops.helion_b200.moe_route_experts``).

    ``router_logits [T, E]`` in bf16, fp16 or fp32, any row pitch.  Returns ``(weights [T, top_k] fp32, experts
    [T, top_k] int64)`` in descending order of choice, equal choices by ascending index: what ``moe.build_schedule``
    and the grouped GEMMs take.

    * score: ``softmax`` over the experts or ``sigmoid`` of each logit, in fp32.
    * choice: the score plus ``bias [E]`` (fp32, a load-balancing bias); it decides which experts are picked but never
      enters the weights.
    * groups: the experts in ``num_groups`` equal runs; a group's score is the sum of its best ``group_top`` (1 or 2)
      choices, and only the best ``top_groups`` groups' experts can be picked.
    * weights: the picked experts' scores, divided by their sum with ``renormalize``, times ``scale``.

    The picks are those of an evaluation in 64 bits: where two choices are too close for fp32 they are compared in 64, and
    what is equal there goes by ascending index.
    A logit of ``-inf`` masks an expert: it counts in no sum, is picked only when nothing else is left (ascending
    index) and gets weight 0; a row with every expert masked gets weights 0.  A row with a NaN (or, under softmax, a
    logit of ``+inf``) gets NaN weights and distinct experts.  A large finite logit in place of ``-inf`` is a logit like
    any other: right, but without a bias many such rows are decided in 64 bits throughout (65536 x 256 with the last 32 at
    -1e9: 440 us, at ``-inf`` 36).  ``E <= 1024``, ``top_k <= 32``, ``num_groups <= 32``.
    """
    args = (router_logits, top_k, scoring, bias, num_groups, top_groups, group_top, renormalize, scale)
    if _forward_ad._current_level >= 0:
        _refuse_tangents("moe_route_experts", router_logits, bias)
    if _direct(router_logits, bias):
        return _route_cuda(*args)
    _check(*args[:7])
    return _route_op(*args)


@dataclass(frozen=True)
class Routing:
    """The settings of :func:`route_experts` that belong to a model, for the MoE layers that take them
    (``moe.nvfp4_moe``, ``dist.ExpertParallel``); called with ``(router_logits, top_k)`` it routes, so it also is a
    router for ``dist.expert_parallel_moe``."""

    scoring: str = "softmax"
    bias: Tensor | None = None
    num_groups: int = 1
    top_groups: int = 1
    group_top: int = 1
    renormalize: bool = False
    scale: float = 1.0

    def __call__(self, router_logits: Tensor, top_k: int) -> tuple[Tensor, Tensor]:
        return route_experts(router_logits, top_k, scoring=self.scoring, bias=self.bias, num_groups=self.num_groups,
                             top_groups=self.top_groups, group_top=self.group_top, renormalize=self.renormalize,
                             scale=self.scale)

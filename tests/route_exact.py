"""Picks of the expert router from their definition in 64 bits, all rows at once (indices only)."""

from __future__ import annotations

import math

import torch


def picks(logits, top_k, *, scoring="softmax", bias=None, num_groups=1, top_groups=1, group_top=1, **_):
    z = logits.double()
    tokens, experts = z.shape
    dead = z == -math.inf
    score = torch.sigmoid(z) if scoring == "sigmoid" else torch.softmax(z, 1).nan_to_num(0.0)
    choice = z if bias is None else score + bias.double()
    by_group = choice if bias is not None or group_top == 1 else score
    choice, by_group = choice.masked_fill(dead, -math.inf), by_group.masked_fill(dead, -math.inf)
    closed = torch.zeros_like(dead)
    if num_groups > 1:
        best = by_group.view(tokens, num_groups, -1).sort(2, descending=True).values[..., :group_top]
        total = best.masked_fill(best == -math.inf, 0.0).sum(2).masked_fill(best[..., 0] == -math.inf, -math.inf)
        order = total.sort(dim=1, descending=True, stable=True).indices[:, :top_groups]
        kept = torch.zeros(tokens, num_groups, dtype=torch.bool, device=z.device).scatter_(1, order, True)
        closed = ~kept.repeat_interleave(experts // num_groups, 1)
    by_choice = choice.sort(dim=1, descending=True, stable=True).indices
    last = closed.gather(1, by_choice).sort(dim=1, stable=True).indices  # closed experts behind all open ones
    return by_choice.gather(1, last)[:, :top_k]

"""Expert routing from its definition, in 64 bits, one row at a time."""

from __future__ import annotations

import math

import torch


def route_row(logits: list[float], top_k: int, scoring: str, bias: list[float] | None, num_groups: int, top_groups: int,
              group_top: int, renormalize: bool, scale: float) -> tuple[list[float], list[int]]:
    e = len(logits)
    live = [v > -math.inf for v in logits]
    if scoring == "softmax":
        top = max(logits)
        terms = [math.exp(v - top) if ok else 0.0 for v, ok in zip(logits, live)]
        total = math.fsum(terms)
        score = [t / total if total else 0.0 for t in terms]
    else:
        score = [(1 / (1 + math.exp(-v)) if v >= 0 else math.exp(v) / (1 + math.exp(v))) if ok else 0.0
                 for v, ok in zip(logits, live)]
    choice = [s + b for s, b in zip(score, bias)] if bias is not None else list(logits)
    of_group = choice if bias is not None or group_top == 1 else score
    choice = [c if ok else -math.inf for c, ok in zip(choice, live)]
    size = e // num_groups
    groups = []
    for g in range(num_groups):
        best = sorted((of_group[i] for i in range(g * size, (g + 1) * size) if choice[i] > -math.inf), reverse=True)
        groups.append(math.fsum(best[:group_top]) if best else -math.inf)
    kept = sorted(range(num_groups), key=lambda g: (-groups[g], g))[:top_groups]
    open_ = [i for i in range(e) if i // size in kept]
    picks = sorted(open_, key=lambda i: (-choice[i], i))[:top_k]
    # the weights as ratios of scores that do not underflow
    if renormalize:
        best = max(logits[i] for i in picks)
        if best == -math.inf:
            w = [0.0] * top_k
        else:
            shift = best if scoring == "softmax" else min(best, 0.0)
            def raw_of(v: float) -> float:
                if v == -math.inf:
                    return 0.0
                if scoring == "softmax":
                    return math.exp(v - shift)
                return 1 / (1 + math.exp(-v)) if v >= 0 else math.exp(v - shift) / (1 + math.exp(v))

            raw = [raw_of(logits[i]) for i in picks]
            w = [r / math.fsum(raw) for r in raw]
    else:
        w = [score[i] for i in picks]
    return [v * scale for v in w], picks


def route(logits, top_k, *, scoring="softmax", bias=None, num_groups=1, top_groups=1, group_top=1, renormalize=False, scale=1.0):
    b = None if bias is None else bias.double().cpu().tolist()
    rows = [route_row(r, top_k, scoring, b, num_groups, top_groups, group_top, renormalize, scale)
            for r in logits.double().cpu().tolist()]
    return (torch.tensor([w for w, _ in rows], dtype=torch.float64).reshape(-1, top_k),
            torch.tensor([p for _, p in rows], dtype=torch.int64).reshape(-1, top_k))

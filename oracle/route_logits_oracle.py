"""CPU restatement, in 64 bits and a row at a time, of routing from logits
(moe_route_logits): the choice by groups, the weights, and the weights' gradient.

TEST INFRASTRUCTURE ONLY.  Only tests/ may import this module, as the
checker; the product path (vllm-cmp170hx_amd/) never does.

No reference code computes this; it is pinned by hand-made rows, by the
gradient against differences of the weights, and by moe_route's own oracle
where the two agree (tests/test_oracle_route_logits.py).
"""

from __future__ import annotations

import numpy as np

NOTHING = np.float32(-708.396)


def scores(row: np.ndarray, sigmoid: bool):
    """(scores, masked, poisoned) of one row of float64 logits."""
    bad = np.isnan(row) if sigmoid else ~(row < np.inf)
    l = np.where(bad, -np.inf, row)
    with np.errstate(over="ignore", invalid="ignore"):
        if sigmoid:
            s = np.where(l >= 0, 1 / (1 + np.exp(-np.abs(l))), np.exp(-np.abs(l)) / (1 + np.exp(-np.abs(l))))
            masked = ~(l >= NOTHING)
        else:
            top = l.max() if np.isfinite(l.max()) else 0.0
            e = np.exp(l - top)
            s = e / e.sum() if e.sum() > 0 else e
            masked = ~((l - top).astype(np.float32) >= NOTHING)
    return s, masked | bad, bool(bad.any())


def complements(row: np.ndarray) -> np.ndarray:
    """1 - sigmoid of each logit, its opposite's sigmoid (1 - s is 0 from logits of 37 on)."""
    return scores(-row, True)[0]


def choice(row, topk, sigmoid, bias=None, groups=1, topk_groups=1):
    """The row's experts in order, -1 where none is left."""
    s, masked, _ = scores(row, sigmoid)
    key = row.astype(np.float64).copy() if bias is None else s + bias.astype(np.float64)
    key = np.where(masked | ~(key > -np.inf), -np.inf, key)
    per = len(row) // groups
    if topk_groups < groups:
        rank = []
        for g in range(groups):
            k = np.sort(key[g * per:(g + 1) * per])[::-1]
            k = k[k > -np.inf][:1 if bias is None else 2]
            rank.append((-k.sum() if len(k) else np.inf, g))
        opened = [g for r, g in sorted(rank)[:topk_groups] if r < np.inf]
        key = np.where(np.isin(np.arange(len(row)) // per, opened), key, -np.inf)
    order = sorted((e for e in range(len(row)) if key[e] > -np.inf), key=lambda e: (-key[e], e))[:topk]
    return np.array(order + [-1] * (topk - len(order)), np.int32)


def weigh(row, ids, sigmoid, renormalize, scale):
    """The weights of the chosen (ids, -1: none), from logarithms of the scores."""
    s, _, poisoned = scores(row, sigmoid)
    held = ids >= 0
    w = np.zeros(len(ids))
    l = row[ids[held]]
    if renormalize and held.any():
        log = -np.logaddexp(0, -l) if sigmoid else l
        z = np.exp(log - log.max())
        w[held] = z / z.sum()
    else:
        w[held] = s[ids[held]]
    return np.where(held, np.nan, 0.0) if poisoned else w * scale


def gradient(row, ids, w, up, sigmoid, renormalize, scale):
    """dL/dlogits of the row, dL/dw = up."""
    s, _, _ = scores(row, sigmoid)
    held = ids >= 0
    out = np.zeros(len(row))
    if not held.any() or scale == 0:
        return out
    e, w, up = ids[held], w[held], up[held]
    mean = (w * up).sum()
    if renormalize:
        out[e] = w * (up - mean / scale) * (complements(row)[e] if sigmoid else 1)
    elif sigmoid:
        out[e] = w * complements(row)[e] * up
    else:
        out = -s * mean
        out[e] += w * up
    return out


def route(logits, topk, sigmoid=True, bias=None, groups=1, topk_groups=1, renormalize=True, scale=1.0, padding=None):
    """(ids [M, topk] int32, weights [M, topk] float64)."""
    l = logits.astype(np.float64)
    ids = np.full((len(l), topk), -1, np.int32)
    weights = np.zeros((len(l), topk))
    for t in range(len(l)):
        if padding is not None and padding[t]:
            continue
        ids[t] = choice(l[t], topk, sigmoid, bias, groups, topk_groups)
        weights[t] = weigh(l[t], ids[t], sigmoid, renormalize, scale)
    return ids, weights

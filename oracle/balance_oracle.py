"""CPU statement of the router's load-balance loss and its gradient, FP64 NumPy.

TEST INFRASTRUCTURE ONLY.  Only tests/ may import this module;
the product path (vllm-cmp170hx_amd/) never does.

Pinned by even routing giving 1, by all rows on one expert, and the gradient by
central differences of the loss (tests/test_oracle_balance.py).
"""

from __future__ import annotations

import numpy as np


def counts(ids, experts, padding=None):
    kept = ids if padding is None else ids[~padding]
    flat = kept.reshape(-1)
    flat = flat[(flat >= 0) & (flat < experts)]
    return np.bincount(flat, minlength=experts).astype(np.int64)


def probabilities(l, sigmoid):
    """(p, slope): dp_e/dl_e = slope_e (1 - ...) as the gradient below uses it."""
    l = np.asarray(l, np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        if sigmoid:
            z = 1 / (1 + np.exp(-l))
            back = 1 / (1 + np.exp(l))
        else:
            top = l.max(1, keepdims=True)
            z = np.exp(l - np.where(np.isneginf(top), 0, top))
            back = np.ones_like(z)
        s = z.sum(1, keepdims=True)
        p = np.where(s == 0, 0, z / np.where(s == 0, 1, s))
    return p, p * back


def loss_and_grad(logits, ids, sigmoid=False, padding=None):
    """-> (loss, counts, dloss/dlogits) with the counts constant."""
    M, E = logits.shape
    kept = np.ones(M, bool) if padding is None else ~padding
    n = int(kept.sum())
    c = counts(ids, E, padding)
    grad = np.zeros((M, E))
    if n == 0:
        return 0.0, c, grad
    f = c * (E / (n * ids.shape[1]))
    p, d = probabilities(logits[kept], sigmoid)
    r = p @ f
    grad[kept] = d * (f - r[:, None]) / n
    return float(r.mean()), c, grad

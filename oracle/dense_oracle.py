"""CPU restatement, in 64 bits, of the dense linear layer and its gradient, with the
bounds of what FP32 sums and the roundings between may be off by.

TEST INFRASTRUCTURE ONLY.  Only tests/ may import this module, as the
checker; the product path (vllm-cmp170hx_amd/) never does.

No reference code computes this; the slopes are pinned by differences
(tests/test_oracle_dense.py).
"""

from __future__ import annotations

import numpy as np
from scipy import special

GATED = "swiglu"


def sigmoid(v):
    return special.expit(v)


def activate(name, z):
    if name == "relu":
        return np.maximum(z, 0)
    if name == "gelu":
        return 0.5 * z * special.erfc(-z / np.sqrt(2))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + np.tanh(np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3)))
    if name == "silu":
        return z * sigmoid(z)
    return z


def slope(name, z):
    if name == "relu":
        return (~(z <= 0)).astype(np.float64)  # (1 at a NaN, which relu keeps)
    if name == "gelu":
        return special.ndtr(z) + z * np.exp(-z * z / 2) / np.sqrt(2 * np.pi)
    if name == "gelu_tanh":
        u = np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3)
        t = np.tanh(u)
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * np.sqrt(2 / np.pi) * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        s = sigmoid(z)
        return s * (1 + z * (1 - s))
    return np.ones_like(z)


# The largest of each activation's second derivative, and 1.13 the largest slope.
BEND = {None: 0.0, "relu": 0.0, "gelu": 0.8, "gelu_tanh": 0.81, "silu": 0.5, GATED: 0.5}
STEEP = 1.13


def sum_error(a, b):
    """FP32 sums of the exact products of a's and b's rows on the matrix cores: 16 products at a
    time, each addition off by a step of 2^-23 of a partial sum (up to the magnitudes' sum)."""
    return (a.shape[-1] / 16 + 24) * 2.0 ** -23 * (np.abs(a) @ np.abs(b).T)


def products(x, w, bias):
    z = x @ w.T + (0 if bias is None else bias)
    off = sum_error(x, w) + 2.0 ** -23 * (np.abs(z) + (0 if bias is None else np.abs(bias)))
    return z, off


def forward(x, w, bias, activation, residual, limit=np.inf):
    """(y, what FP32 may be off by before y is rounded)."""
    z, off = products(x, w, bias)
    if activation == GATED:
        n = len(w) // 2
        g, u = np.minimum(z[:, :n], limit), np.clip(z[:, n:], -limit, limit)
        h = activate("silu", g)
        # e^-g is off by 2^-22 and |g| 2^-23 of it, a few roundings
        y = h * u
        tol = STEEP * off[:, :n] * np.abs(u) + np.abs(h) * off[:, n:] + off[:, :n] * off[:, n:] * 2 + np.abs(y) * (2.0 ** -20 + np.abs(g) * 2.0 ** -22)
    else:
        y = activate(activation, z)
        # (erfc: 16 steps; the cubic's argument to e is off by four roundings, up to |2 u| 2^-21)
        arg = np.abs(z) + (2 * np.abs(z) ** 3 if activation == "gelu_tanh" else np.abs(z) ** 2 if activation == "gelu" else 0)
        tol = STEEP * off + np.abs(y) * (2.0 ** -19 + np.minimum(arg, 200.0) * 2.0 ** -21) * (activation not in (None, "relu")) + 1e-37
    if residual is not None:
        y = y + residual
        tol = tol + 2.0 ** -24 * (np.abs(y) + np.abs(residual))
    return y, tol


def backward(x, w, bias, activation, dy, eps, limit=np.inf):
    """({"x", "w", "bias"}: (gradient, what it may be off by before it is rounded to its type),
    dz), where dz is rounded with steps of eps (relative, half of which is lost)."""
    z, off = products(x, w, bias)
    half = eps / 2
    off_z = off
    if activation == GATED:
        n = len(w) // 2
        g, u = np.minimum(z[:, :n], limit), np.clip(z[:, n:], -limit, limit)
        in_g, in_u = z[:, :n] <= limit, np.abs(z[:, n:]) <= limit
        og, ou = off_z[:, :n], off_z[:, n:]
        h, s = activate("silu", g), slope("silu", g)
        dz = np.concatenate([dy * u * s * in_g, dy * h * in_u], 1)
        tol = np.concatenate([np.abs(dy) * (np.abs(u) * 0.5 * og + STEEP * ou + 0.5 * og * ou), np.abs(dy) * STEEP * og], 1)
        # values at the very limit may fall to either side
        edge = np.concatenate([np.abs(dy * u * s) * (np.abs(z[:, :n] - limit) <= off[:, :n]),
                               np.abs(dy * h) * (np.abs(np.abs(z[:, n:]) - limit) <= off[:, n:])], 1) if np.isfinite(limit) else 0
        size = np.concatenate([np.abs(dy) * np.abs(u) * STEEP, np.abs(dy * h)], 1)
        tol = tol + edge + size * (2.0 ** -19 + np.abs(np.concatenate([g, g], 1)) * 2.0 ** -21)
    else:
        s = slope(activation, z)
        dz = dy * s
        tol = np.abs(dy) * BEND[activation] * off_z
        if activation == "relu":
            tol = tol + np.abs(dy) * (np.abs(z) <= off_z)
        elif activation is not None:
            tol = tol + np.abs(dy) * STEEP * (2.0 ** -18 + np.minimum(np.abs(z) + np.abs(z) ** 3, 100.0) * 2.0 ** -20)
    rounded = tol + half * (np.abs(dz) + tol)
    if eps > 2.0 ** -9:  # (bf16's range is FP32's)
        rounded = rounded + 1e-37
    else:  # fp16 over a power of two that brings the largest to 2^13 or more: steps of 2^-24 of that
        rounded = rounded + 2.0 ** -24 * 2.0 ** -13 * (np.abs(dz).max() if dz.size else 0) * 2
    slack = np.abs(dz) + rounded
    out = {
        "x": (dz @ w, rounded @ np.abs(w) + sum_error(slack, w.T)),
        "w": (dz.T @ x, rounded.T @ np.abs(x) + sum_error(slack.T, x.T)),
        "bias": (dz.sum(0), (tol + (len(x) / 64 + 40) * 2.0 ** -24 * slack.sum(0, keepdims=True) / max(len(x), 1)).sum(0)),
    }
    return out, dz

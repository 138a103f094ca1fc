"""The dense linear layer: y = act(x W^T + bias) + residual in one call.

Outputs and scratch come from torch's allocator on the current stream, so calls on
several streams, and captured ones, do not share memory.  Failed checks raise
RuntimeError.
"""

from __future__ import annotations

import math

import torch

from ... import _native

_ACTIVATIONS = {None: 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4, "swiglu": 5}

_ops = None


def _lib():
    global _ops
    if _ops is None:
        _native.load_torch()
        _ops = torch.ops._vllm_mi355x
    return _ops


def dense_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                 activation: str | None = None, residual: torch.Tensor | None = None,
                 out_dtype: torch.dtype | None = None, clamp_limit: float | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
    """act(x W^T + bias) + residual, [..., n]: FP32 sums of exact products on the matrix
    cores, bias, activation and residual in FP32, one rounding to out_dtype (x's unless
    given).

    x [..., k] and weight [n, k] bf16 or fp16, of one type; x's leading axes one run of
    rows, unit inner strides; k up to 2^21, weight rows up to 2^24 and rows up to 2^26 (for
    gradients of x, weight or bias both up to 2^21, and 2^23 parts of 64 x 64 of x, of weight and
    of x W^T).  bias [n] (contiguous) and residual
    [..., n] (rows as x's) bf16, fp16 or fp32.  activation: None, "relu", "gelu" (of the
    error function), "gelu_tanh", "silu", or "swiglu": weight [2 n, k] and bias [2 n] hold the
    gate rows and then the up rows, and the result is SiLU(min(g, L)) clamp(u, -L, L), L the
    clamp_limit if one is given.  out: contiguous, of out_dtype, which it may be the residual
    itself; it carries no gradient.

    Differentiable once in x, weight, bias and residual, in reverse mode (a forward-mode tangent
    and torch.func's grad and vjp raise): x W^T + bias is kept in fp32, its gradient rounded to x's
    type (in fp16 over a power of two of the whole tensor) before the two products that follow.
    A backward pass computes the gradients that it is asked for; x is kept for the weight's alone,
    the weight for x's.  To capture a backward pass into a graph, let go of eager results of the
    same leaves first, as for any operator of torch."""
    if activation not in _ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}")
    if clamp_limit is not None and activation != "swiglu":
        raise ValueError("clamp_limit is of swiglu")
    ops = _lib()
    limit = math.inf if clamp_limit is None else float(clamp_limit)
    code = _ACTIVATIONS[activation]
    if out is None:
        return ops.dense_linear(x, weight, bias, code, residual, out_dtype or x.dtype, limit)
    if out_dtype is not None and out.dtype != out_dtype:
        raise RuntimeError("dense_linear: out must be of out_dtype")
    ops.dense_linear_out(x, weight, bias, code, residual, limit, out)
    return out

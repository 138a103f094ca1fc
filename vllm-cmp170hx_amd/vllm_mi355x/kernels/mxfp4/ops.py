"""MXFP4 operators: blocks of 32 elements along the last axis, E2M1 codes (two
a byte, the even element in the low nibble) under one E8M0 scale byte.

A packed tensor [..., k] is a pair of contiguous uint8 tensors: codes
[..., k / 2] and scales [..., k / 32].  k is a multiple of 32 (up to 2^32 in
products); every other size is free.  Outputs and scratch come from torch's
allocator on the current stream, so calls on several streams, and captured ones,
do not share memory (the fused MoE's workspace aside, which is the caller's).
Failed checks raise RuntimeError.
These are operators for inference: outputs carry no gradient.
"""

from __future__ import annotations

import math

import torch

from ... import _native

_ops = None


def _lib():
    global _ops
    if _ops is None:
        _native.load_torch()
        _ops = torch.ops._vllm_mi355x
    return _ops


def mxfp4_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of x [..., k] (bf16, fp16 or fp32, unit stride along k,
    the leading axes one run of rows).  A block's scale is the power of two two
    below its largest magnitude's; codes round to nearest, ties to even,
    saturating at 6 scales.  A block with a NaN or an infinity becomes NaN."""
    return _lib().mxfp4_quantize(x)


def mxfp4_dequantize(codes: torch.Tensor, scales: torch.Tensor,
                     out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values [..., k] of a packed pair, rounded once to out_dtype."""
    return _lib().mxfp4_dequantize(codes, scales, out_dtype)


def mxfp4_matmul(a: torch.Tensor, a_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
                 out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a [..., k] times the transpose of w [n, k], both packed: exact products,
    FP32 sums on the matrix cores, one rounding to out_dtype."""
    return _lib().mxfp4_matmul(a, a_scale, w, w_scale, out_dtype)


def mxfp4_linear(x: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
                 out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """x [..., k] (bf16, fp16 or fp32), quantized as mxfp4_quantize does, times
    the transpose of the packed w [n, k]; out_dtype: x's unless given."""
    return _lib().mxfp4_linear(x, w, w_scale, out_dtype)


def fused_mxfp4_moe(hidden_states: torch.Tensor, w1: torch.Tensor, w2: torch.Tensor,
                    w1_scale: torch.Tensor, w2_scale: torch.Tensor, topk_weights: torch.Tensor,
                    topk_ids: torch.Tensor, clamp_limit: float | None = None,
                    expert_map: torch.Tensor | None = None, workspace: dict | None = None,
                    output: torch.Tensor | None = None) -> torch.Tensor:
    """out [M, K] = sum over the top-k slots (slot order, FP32, one rounding) of
    router weight * w2_e(h), h = SiLU(min(g, L)) * clamp(u, -L, L) in FP32 and
    quantized to MXFP4, (g | u) = w1_e(x), x quantized to MXFP4.

    hidden_states [M, K] bf16 or fp16; w1 [E, 2 N, K / 2] (gate rows 0..N-1, up
    rows N..2N-1) and w2 [E, K, N / 2] codes with their scales; K and N
    multiples of 32 up to 65536, at most 1024 experts.  topk_weights / topk_ids [M, topk] (FP32 and int32, or
    other types of such values); expert_map: global id -> local expert or -1.  Slots routed outside the local experts add nothing.
    workspace: a dict that keeps the call's scratch; calls that share one must
    be on one stream.  (A captured call has scratch of its graph's own: a later
    call may replace the dict's by a larger one, the graph's has to stay.)
    output: contiguous, like hidden_states, which it may be."""
    ops = _lib()
    ids = topk_ids if topk_ids.dtype == torch.int32 else topk_ids.to(torch.int32)
    weights = topk_weights if topk_weights.dtype == torch.float32 else topk_weights.float()
    if expert_map is not None and expert_map.dtype != torch.int32:
        expert_map = expert_map.to(torch.int32)
    out = output if output is not None else torch.empty_like(
        hidden_states, memory_format=torch.contiguous_format)
    need = ops.mxfp4_moe_workspace(hidden_states, w1, w2, ids)
    if workspace is not None and hidden_states.is_cuda and torch.cuda.is_current_stream_capturing():
        workspace = None
    scratch = None if workspace is None else workspace.get("mxfp4")
    if scratch is None or scratch.numel() < need or scratch.device != hidden_states.device:
        scratch = torch.empty(need, dtype=torch.uint8, device=hidden_states.device)
        if workspace is not None:
            workspace["mxfp4"] = scratch
    ops.mxfp4_moe(hidden_states, w1, w2, w1_scale, w2_scale, weights.contiguous(), ids.contiguous(),
                  None if expert_map is None else expert_map.contiguous(),
                  math.inf if clamp_limit is None else float(clamp_limit), scratch, out)
    return out

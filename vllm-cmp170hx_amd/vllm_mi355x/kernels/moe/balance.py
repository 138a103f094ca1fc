"""A router's load: slots per expert, and the load-balance loss with its
gradient (no counterpart in the reference).

Both take what moe_route gives: logits [M, E] and topk_ids [M, topk] (int32, or
another type of such values), where padding rows hold -1.  Failed checks raise RuntimeError.
"""

from __future__ import annotations

import torch

from ... import _native
from .route import _SCORING


def moe_expert_counts(topk_ids: torch.Tensor, num_experts: int,
                      is_padding: torch.Tensor | None = None,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """Slots that chose each expert, int64 [num_experts]: ids outside [0,
    num_experts) and rows marked in is_padding (bool [M]) are not counted.
    With out, the counts are added to it (a running load)."""
    _native.load_torch()
    add = out is not None
    if out is None:
        out = torch.empty(num_experts, dtype=torch.int64, device=topk_ids.device)
    elif tuple(out.shape) != (num_experts,):
        raise RuntimeError("moe_expert_counts: out must be int64 [num_experts]")
    ids = topk_ids if topk_ids.dtype == torch.int32 else topk_ids.to(torch.int32)
    torch.ops._vllm_mi355x.moe_expert_counts(ids.contiguous(), is_padding, out, add)
    return out


def moe_balance_loss(logits: torch.Tensor, topk_ids: torch.Tensor, scoring: str = "softmax",
                     is_padding: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(loss, counts): loss = sum over experts of f_e P_e (FP32 scalar, 1 for even
    load), f_e = counts_e E / (n topk) over the n rows that is_padding does not
    mark, P_e the mean of the rows' probabilities: softmax of the logits, or
    (scoring "sigmoid") their sigmoids over the row's sum.  counts: int64 [E].

    Differentiable once in the logits (bf16, fp16 or fp32; rows in one stride, not
    overlapping), in reverse mode (a forward-mode tangent raises); the counts are
    constants.  A row whose logits are all -inf (with sigmoids: below -708.396, masks of
    the type's lowest value among them) adds nothing.  To capture a backward pass into a
    graph, let go of eager losses of the same leaves first, as for any operator of torch."""
    if scoring not in _SCORING:
        raise ValueError(f"unknown scoring {scoring!r}")
    _native.load_torch()
    ids = topk_ids if topk_ids.dtype == torch.int32 else topk_ids.to(torch.int32)
    return torch.ops._vllm_mi355x.moe_balance_loss(logits, ids.contiguous(), is_padding,
                                                   _SCORING[scoring])

"""Attention over packed sequences (no counterpart in the reference)."""

import math
from typing import Optional, Tuple, Union

import torch

from ._autograd import refuse_gradients, rows_in_place

__all__ = ["flash_attention_packed"]


def _forward(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    offsets: torch.Tensor,
    kv_offsets: Optional[torch.Tensor],
    softmax_scale: float,
    causal: bool,
    keep: bool,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    query, key, value = (rows_in_place(t) for t in (query, key, value))
    out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    lse = torch.empty(query.size(1), query.size(0), dtype=torch.float32, device=query.device) if keep else None
    torch.ops.tilefusion.flash_attention_packed(query, key, value, offsets, kv_offsets, softmax_scale, causal, out, lse)
    return out, lse


def flash_attention_packed(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    offsets: torch.Tensor,
    kv_offsets: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None,
    causal: bool = True,
    keep: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    refuse_gradients("flash_attention_packed", query, key, value)
    if query.dim() != 3:
        raise RuntimeError(f"flash_attention_packed: query must be [tokens, heads, D], got {list(query.shape)}")
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(query.size(-1))
    out, lse = _forward(query, key, value, offsets, kv_offsets, softmax_scale, causal, keep)
    return (out, lse) if keep else out

"""Attention over packed sequences, forward and backward (no counterpart in the reference)."""

import math
from typing import Any, Optional, Tuple, Union

import torch

from .. import _direct
from ._autograd import not_captured, records, refuse_transforms, rows_in_place

__all__ = ["flash_attention_packed", "flash_attention_packed_backward"]


def _scale(query: torch.Tensor, softmax_scale: Optional[float], op: str) -> float:
    if query.dim() != 3 or query.size(-1) == 0:
        raise RuntimeError(f"{op}: query must be [tokens, heads, D], got {list(query.shape)}")
    return 1.0 / math.sqrt(query.size(-1)) if softmax_scale is None else softmax_scale


def _within_reach(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor) -> Tuple[torch.Tensor, ...]:
    """query, key and value as they are where the kernels read them so, otherwise copies: rows in one piece, tokens less than 2^24 elements apart, and the
    heads of a group, which 32-bit offsets reach from one another, within 2^31 (those of a long text's [heads, tokens, D] may not be)."""
    query, key, value = (rows_in_place(t) for t in (query, key, value))
    query, key, value = (t.contiguous() if t.dim() == 3 and t.size(0) > 1 and t.stride(0) >= 2**24 else t for t in (query, key, value))
    if query.dim() == 3 and key.dim() == 3 and query.size(1) > key.size(1) > 0:
        group = query.size(1) // key.size(1)
        if 33 * query.stride(0) + group * query.stride(1) >= 2**31 - query.size(2):
            query = query.contiguous()
    return query, key, value


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
    query, key, value = _within_reach(query, key, value)
    out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    lse = torch.empty(query.size(1), query.size(0), dtype=torch.float32, device=query.device) if keep else None
    torch.ops.tilefusion.flash_attention_packed(query, key, value, offsets, kv_offsets, softmax_scale, causal, out, lse)
    return out, lse


def _backward(
    grad_out: torch.Tensor,
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    out: torch.Tensor,
    lse: torch.Tensor,
    offsets: torch.Tensor,
    kv_offsets: Optional[torch.Tensor],
    softmax_scale: float,
    causal: bool,
    of_query: bool,
    of_keys: bool,
) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor], Optional[torch.Tensor]]:
    """The gradients that are asked for, None in the place of the others."""
    query, key, value = _within_reach(query, key, value)
    grad_out, out = (rows_in_place(t.contiguous()) for t in (grad_out, out))
    grad_query = torch.empty(query.shape, dtype=query.dtype, device=query.device) if of_query else None
    grad_key, grad_value = (torch.empty(t.shape, dtype=t.dtype, device=t.device) if of_keys else None for t in (key, value))
    with torch.no_grad():
        torch.ops.tilefusion.flash_attention_packed_backward(
            grad_out, query, key, value, out, lse.contiguous(), offsets, kv_offsets, softmax_scale, causal, grad_query, grad_key, grad_value
        )
    return grad_query, grad_key, grad_value


class _FlashAttentionPacked(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, offsets: torch.Tensor, kv_offsets: Optional[torch.Tensor],
                softmax_scale: float, causal: bool) -> Tuple[torch.Tensor, ...]:
        out, lse = _forward(query, key, value, offsets, kv_offsets, softmax_scale, causal, True)
        ctx.save_for_backward(query, key, value, out, lse, offsets, kv_offsets)
        ctx.softmax_scale, ctx.causal = softmax_scale, causal
        ctx.mark_non_differentiable(lse)
        return out, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, grad_out: torch.Tensor, *_: Any) -> Tuple[Any, ...]:
        not_captured("flash_attention_packed")
        of_query, of_key, of_value = ctx.needs_input_grad[:3]
        grads = _backward(grad_out, *ctx.saved_tensors, ctx.softmax_scale, ctx.causal, of_query, of_key or of_value)
        return (*grads, None, None, None, None)


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
    """softmax(softmax_scale * Q @ K.T) @ V of every sequence and head, the sequences lying one behind the other.

    Args:
        query: [tokens, heads, D] fp16 or bf16, D 64 or 128; key, value: [kv_tokens, kv_heads, D], head h reads head h // (heads // kv_heads) of them.
            Slices of one projection and head-major tensors are read where they are; tokens 2^24 elements apart or more, and queries whose heads that
            share one of the keys reach 2^31 elements, are copied.
        offsets: [sequences + 1] int32, ascending: sequence b is tokens offsets[b] .. offsets[b + 1] - 1.
        kv_offsets: the same of the keys, where a sequence has keys from before (a prompt in pieces); None: as the queries.
        softmax_scale: 1 / sqrt(D) where it is None.
        causal: a sequence's last query sees all its keys, the one before all but the last, and so on.
        keep: also return lse [heads, tokens] fp32, the log-sum-exp of the scaled scores, for `flash_attention_packed_backward`.

    Returns out [tokens, heads, D], or (out, lse).  The device alone knows the lengths: a call can be captured and replayed with other offsets in the same
    tensors.  Rows that see no key (more queries than keys) and rows of no sequence (behind offsets[-1]) are zero, their lse -inf.  Scores, maxima
    and sums are fp32; the weights are rounded to the type for the product with V, in fp16 2^7 to 2^15 times as large.  Under autograd out carries the backward pass (once: no gradient of a
    gradient, no forward mode), and lse none; neither the call nor that pass is captured into a graph."""
    if not torch.compiler.is_compiling():
        direct = _direct.flash_attention_packed(query, key, value, offsets, kv_offsets, softmax_scale, causal, keep)   # (no gradient is asked for)
        if direct is not None:
            return direct if keep else direct[0]
    op = "flash_attention_packed"
    scale = _scale(query, softmax_scale, op)
    if records(op, query, key, value):
        out, lse = _FlashAttentionPacked.apply(query, key, value, offsets, kv_offsets, scale, causal)
    else:
        out, lse = _forward(query, key, value, offsets, kv_offsets, scale, causal, keep)
    return (out, lse) if keep else out


def flash_attention_packed_backward(
    grad_out: torch.Tensor,
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    out: torch.Tensor,
    lse: torch.Tensor,
    offsets: torch.Tensor,
    kv_offsets: Optional[torch.Tensor] = None,
    softmax_scale: Optional[float] = None,
    causal: bool = True,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients of query, key and value, from that of out [tokens, heads, D] and the out and lse that `flash_attention_packed` gave.

    exp(scores - lse) and the gradients of the scores are rounded to the type on the way, as operands of the products that follow (in fp16 times powers of
    two, so that the type's range is not theirs); sums, those over the heads of a group among them, are fp32.  The same bits every time.  Rows of no
    sequence, rows that see no key and keys that no row sees have zeros."""
    if not torch.compiler.is_compiling():
        direct = _direct.flash_attention_packed_backward(
            grad_out, query, key, value, out, lse, offsets, kv_offsets, softmax_scale, causal
        )
        if direct is not None:
            return direct
    op = "flash_attention_packed_backward"
    scale = _scale(query, softmax_scale, op)
    refuse_transforms(op, grad_out, query, key, value, out, lse)
    return _backward(grad_out, query, key, value, out, lse, offsets, kv_offsets, scale, causal, True, True)

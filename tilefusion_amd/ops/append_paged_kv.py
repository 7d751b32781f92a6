"""New tokens enter a paged cache, their positions rotated in on the way (no counterpart in the reference)."""

from typing import Optional, Tuple, Union

import torch

from .. import _direct
from ._autograd import refuse_gradients, rows_in_place

__all__ = ["append_paged_kv", "rotation_tables"]


def rotation_tables(
    positions: int, rotated: int, base: float = 10000.0, device: Union[str, torch.device] = "cuda"
) -> Tuple[torch.Tensor, torch.Tensor]:
    """cos and sin [positions, rotated / 2] fp32 of p * base ** (-2 i / rotated), the angles in 64 bits: made once for a model's longest text."""
    if positions < 0 or rotated <= 0 or rotated % 2 != 0:
        raise RuntimeError(f"rotation_tables: positions must not be negative and rotated positive and even, got {positions} and {rotated}")
    pair = torch.arange(0, rotated, 2, device=device, dtype=torch.float64)
    angle = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * base ** (-pair / rotated)
    return angle.cos().float(), angle.sin().float()


def append_paged_kv(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    offsets: Optional[torch.Tensor] = None,
    interleaved: bool = False,
    keep: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Rotates the queries and keys of new tokens by their positions and writes keys and values to their pages.

    Args:
        query: [tokens, heads, D] fp16 or bf16, D 64 or 128; key, value: [tokens, kv_heads, D].  Slices of one projection are read where they are.
        cos, sin: [positions, rotated / 2] fp32 (`rotation_tables`); the first `rotated` elements of a head are turned.
        key_cache, value_cache: [pages, page_size, kv_heads, D], written in place; any order of the first three dimensions in memory
            (a permuted [pages, kv_heads, page_size, D] is read fastest by `flash_decode_paged`), no rows on each other.
        page_table: [sequences, n] int32, the pages of each sequence in their order.
        lengths: [sequences] int32, the lengths with the new tokens.
        offsets: [sequences + 1] int32, ascending: sequence b's new tokens are offsets[b] .. offsets[b + 1] - 1, the last of them at position
            lengths[b] - 1.  None: token b is the one new token of sequence b.
        interleaved: pairs are neighbours (2 i, 2 i + 1); otherwise (i, i + rotated / 2).
        keep: also return the rotated keys, for the attention over the prompt itself (`flash_attention_packed`).

    Returns the rotated queries [tokens, heads, D], or (queries, keys).  The rotation is in fp32 and rounded once.  A token whose position has no
    page in the cache, or no row in the tables, leaves the cache as it is and its rotated rows are NaN; tokens of no sequence (behind
    offsets[-1], or of one that is shorter than its new tokens, as an idle slot of length 0) leave it as it is too, and their rows are zero.  Pages that
    new tokens go to belong to one sequence.  There is no gradient; the caches count as changed in place, so that a backward pass that has saved
    some of them raises."""
    if not torch.compiler.is_compiling():
        direct = _direct.append_paged_kv(
            query, key, value, cos, sin, key_cache, value_cache, page_table, lengths, offsets, interleaved, keep
        )
        if direct is not None:
            return direct if keep else direct[0]
    op = "append_paged_kv"
    refuse_gradients(op, query, key, value, cos, sin, key_cache, value_cache)
    if query.dim() != 3 or key.dim() != 3:
        raise RuntimeError(f"{op}: query must be [tokens, heads, D], key and value [tokens, kv_heads, D]")
    query, key, value = (rows_in_place(t) for t in (query, key, value))
    query_out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    key_out = torch.empty(key.shape, dtype=key.dtype, device=key.device) if keep else None
    torch.ops.tilefusion.append_paged_kv(
        query, key, value, cos.contiguous(), sin.contiguous(), key_cache, value_cache, page_table, lengths, offsets, interleaved, query_out, key_out
    )
    return (query_out, key_out) if keep else query_out

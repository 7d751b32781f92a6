"""Attention of one new token of every sequence over a paged cache (no counterpart in the reference)."""

import math
from typing import Optional

import torch

from .. import _direct
from ._autograd import refuse_gradients, rows_in_place

__all__ = ["flash_decode_paged"]


def flash_decode_paged(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    softmax_scale: Optional[float] = None,
) -> torch.Tensor:
    """out[b, h] = softmax(softmax_scale * query[b, h] @ K.T) @ V over the lengths[b] tokens of sequence b in the cache.

    Args:
        query: [sequences, heads, D] fp16 or bf16, D 64 or 128; head h reads head h // (heads // kv_heads) of the cache.
        key_cache, value_cache: [pages, page_size, kv_heads, D], page_size a multiple of 16; any order of the first three dimensions in memory,
            tokens less than 2^26 elements apart.
        page_table: [sequences, n] int32, the pages of each sequence in their order; entries beyond its length may hold anything.
        lengths: [sequences] int32, the new token included (`append_paged_kv` has put it there).
        softmax_scale: 1 / sqrt(D) where it is None.

    Returns [sequences, heads, D].  The cache is cut evenly over the chip whatever the lengths are, which only the device knows: a call can be
    captured and replayed with other lengths and tables in the same tensors.  A sequence of length 0 has rows of zeros, one that is
    longer than its row of the table, or names a page that the cache does not have within its length, NaN.  There is no gradient."""
    if not torch.compiler.is_compiling():
        direct = _direct.flash_decode_paged(query, key_cache, value_cache, page_table, lengths, softmax_scale)
        if direct is not None:
            return direct
    op = "flash_decode_paged"
    refuse_gradients(op, query, key_cache, value_cache)
    if query.dim() != 3 or query.size(-1) == 0:
        raise RuntimeError(f"{op}: query must be [sequences, heads, D], got {list(query.shape)}")
    if softmax_scale is None:
        softmax_scale = 1.0 / math.sqrt(query.size(-1))
    query = rows_in_place(query)
    out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
    torch.ops.tilefusion.flash_decode_paged(query, key_cache, value_cache, page_table, lengths, softmax_scale, out)
    return out

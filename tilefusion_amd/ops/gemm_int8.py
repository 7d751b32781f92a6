"""Products of 8-bit integers with scales, and the quantisation of rows (no counterpart in the reference)."""

from typing import Tuple

import torch

from .. import _direct

__all__ = ["gemm_int8", "quantize_rows"]


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows in 8 bits with a scale each: x [.., K] fp16 or bf16 -> q [.., K] int8, scale [..] fp32.

    scale = max|x| / 127 of a row (in fp32), q the whole number nearest to x / scale, the even one in the middle of two.
    A row of zeros has scale 0 and q 0; a row with an infinity or a NaN has scale NaN and q 0, so that every product of it is NaN.
    No gradient passes through a rounding: the results have none."""
    if not torch.compiler.is_compiling():
        direct = _direct.quantize_rows(x)
        if direct is not None:
            return direct
    if x.dim() < 1:
        raise RuntimeError("quantize_rows: x must have rows [.., K]")
    rows = x.detach().reshape(-1, x.size(-1)) if x.size(-1) > 0 else x.detach().reshape(0, 0)
    q = torch.empty(rows.shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(rows.size(0), dtype=torch.float32, device=x.device)
    torch.ops.tilefusion.quantize_rows(rows.contiguous(), q, scale)
    return q.reshape(x.shape), scale.reshape(x.shape[:-1])


def gemm_int8(
    tensor_a: torch.Tensor,
    tensor_b: torch.Tensor,
    scale_a: torch.Tensor,
    scale_b: torch.Tensor,
    tensor_c: torch.Tensor,
) -> None:
    """C[m, n] = scale_a[m] * scale_b[n] * sum_k A[m, k] * B[n, k], written into `tensor_c`.

    Args:
        tensor_a: [M, K] int8, row-major (the tokens; `quantize_rows` makes it).
        tensor_b: [N, K] int8 - the column-major K x N operand (the weight, a row for each output channel).
        scale_a: [M] fp32, one for each token.
        scale_b: [N] fp32, one for each output channel.
        tensor_c: [M, N] fp32, fp16 or bf16.

    The sum is exact (int32; K <= 131071), multiplied by scale_a, then by scale_b in fp32 and rounded once.  No gradient passes through.
    """
    if not torch.compiler.is_compiling() and _direct.gemm_int8(tensor_a, tensor_b, scale_a, scale_b, tensor_c):
        return
    torch.ops.tilefusion.gemm_int8(
        tensor_a.contiguous(), tensor_b.contiguous(), scale_a.contiguous(), scale_b.contiguous(), tensor_c
    )

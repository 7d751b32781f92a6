"""Core operations (counterpart of python/ops/__init__.py in the reference).

`__all__` lists the reference's operations and flash_decode; the others have no counterpart there:

    gemm_int8, quantize_rows                                  products of 8-bit integers with scales
    gated_ffn, gated_ffn_backward                             the gated feed-forward block
    linear_cross_entropy, linear_cross_entropy_backward       the cross entropy of a linear head
"""

from .flash_attention import FlashAttention, flash_attention
from .flash_decode import flash_decode
from .fused_two_gemms import fused_two_gemms
from .gated_ffn import gated_ffn, gated_ffn_backward  # noqa: F401
from .gemm import gemm
from .gemm_int8 import gemm_int8, quantize_rows  # noqa: F401
from .linear_cross_entropy import linear_cross_entropy, linear_cross_entropy_backward  # noqa: F401
from .scatter_nd import scatter_nd

__all__ = [
    "FlashAttention",
    "flash_attention",
    "flash_decode",
    "fused_two_gemms",
    "gemm",
    "scatter_nd",
]

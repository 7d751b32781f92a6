"""ctypes view of the C ABI in include/tilefusion_c.h (libtilefusion_hip.so).

The library is built in-tree by `make -C tilefusion_amd/csrc` (or __graft_entry__.build()).
There is no CPU fallback: loading fails loudly when the library is missing.
"""

import ctypes
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libtilefusion_hip.so")

TF_OK, TF_ERR_INVALID_ARG, TF_ERR_UNSUPPORTED, TF_ERR_LDS, TF_ERR_HIP = range(5)
TF_DTYPE_F32, TF_DTYPE_F16, TF_DTYPE_BF16 = range(3)
TF_ACT_SILU, TF_ACT_GELU, TF_ACT_GELU_TANH = range(3)

_vp, _i, _i64, _d, _sz = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_double, ctypes.c_size_t


class PagedCache(ctypes.Structure):
    """tf_paged_cache_t"""

    _fields_ = [("key", _vp), ("value", _vp), ("key_strides", _i64 * 3), ("value_strides", _i64 * 3), ("pages", _i64), ("page_size", _i64),
                ("kv_heads", _i64), ("D", _i64), ("page_table", _vp), ("table_width", _i64), ("table_stride", _i64), ("lengths", _vp),
                ("sequences", _i64), ("dtype", _i)]


class PackedAttention(ctypes.Structure):
    """tf_packed_attention_t"""

    _fields_ = [("query", _vp), ("key", _vp), ("value", _vp), ("query_strides", _i64 * 2), ("key_strides", _i64 * 2), ("value_strides", _i64 * 2),
                ("tokens", _i64), ("kv_tokens", _i64), ("sequences", _i64), ("heads", _i64), ("kv_heads", _i64), ("D", _i64), ("offsets", _vp),
                ("kv_offsets", _vp), ("softmax_scale", _d), ("causal", _i), ("dtype", _i)]


# name -> (restype, argtypes); every symbol include/tilefusion_c.h declares
SIGNATURES = {
    "tf_gemm_f16": (_i, [_vp, _vp, _vp, _i, _i64, _i64, _i64, _i, _i, _i, _i, _i, _vp]),
    "tf_fused_two_gemms_f16": (_i, [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i, _i, _i, _i, _vp]),
    "tf_flash_attention_fwd_f16": (_i, [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i, _i, _i, _i, _i, _d, _i, _vp]),
    "tf_gemm": (_i, [_vp, _vp, _vp, _i, _i, _i64, _i64, _i64, _i, _i, _i, _i, _i, _vp]),
    "tf_fused_two_gemms": (_i, [_vp, _vp, _vp, _vp, _i, _i64, _i64, _i64, _i64, _i64, _i, _i, _i, _i, _vp]),
    "tf_fused_two_gemms_workspace_bytes": (_sz, [_i, _i64, _i64, _i64, _i64, _i64]),
    "tf_fused_two_gemms_ws": (_i, [_vp, _vp, _vp, _vp, _i, _i64, _i64, _i64, _i64, _i64, _i, _i, _i, _i, _vp, _sz, _vp]),
    "tf_fused_two_gemms_narrow": (_i, [_vp, _vp, _vp, _vp, _i, _i64, _i64, _i64, _i64, _i64, _vp, _sz, _vp]),
    "tf_flash_attention_fwd": (_i, [_vp, _vp, _vp, _vp, _i, _i64, _i64, _i64, _i64, _i64, _i, _i, _i, _i, _i, _d, _i, _vp]),
    "tf_flash_attention_fwd_wide": (_i, [_vp, _vp, _vp, _vp, _i, _i64, _i64, _i64, _i64, _d, _i, _vp]),
    "tf_flash_attention_fwd_kt": (_i, [_vp, _vp, _vp, _vp, _i, _i64, _i64, _i64, _i64, _d, _i, _vp]),
    "tf_flash_decode_workspace_bytes": (_sz, [_i64, _i64, _i]),
    "tf_flash_decode_f16": (_i, [_vp, _vp, _vp, _vp, _vp, _sz, _i64, _i64, _i64, _i, _d, _vp]),
    "tf_flash_decode": (_i, [_vp, _vp, _vp, _vp, _i, _vp, _sz, _i64, _i64, _i64, _i, _d, _vp]),
    "tf_flash_decode_uncut": (_i, [_vp, _vp, _vp, _vp, _i, _i64, _i64, _i64, _i, _d, _vp]),
    "tf_flash_decode_static_max_partials": (_sz, []),
    "tf_flash_decode_static_prepare": (_i, []),
    "tf_flash_decode_static_f16": (_i, [_vp, _vp, _vp, _vp, _i64, _i64, _i64, _i, _d, _vp]),
    "tf_flash_attention_fwd_d8": (_i, [_vp, _vp, _vp, _vp, _i, _i64, _i64, _i64, _i64, _d, _i, _vp]),
    "tf_flash_attention_split_workspace": (_i64, [_i64, _i64, _i64, _i64]),
    "tf_flash_attention_fwd_split": (_i, [_vp, _vp, _vp, _vp, _i, _i64, _i64, _i64, _i64, _i, _d, _vp, _vp]),
    "tf_transpose_16bit": (_i, [_vp, _vp, _i64, _i64, _i64, _vp]),
    "tf_scatter_nd": (_i, [_vp, _vp, _vp, ctypes.POINTER(_i64), _i, _i64, _i, _i, _vp]),
    "tf_gemm_int8_workspace_bytes": (_sz, [_i64, _i64, _i64]),
    "tf_gemm_int8": (_i, [_vp, _vp, _vp, _vp, _vp, _i, _i64, _i64, _i64, _vp, _sz, _vp]),
    "tf_quantize_rows": (_i, [_vp, _vp, _vp, _i, _i64, _i64, _vp]),
    "tf_gated_ffn_workspace_bytes": (_sz, [_i64, _i64, _i64]),
    "tf_gated_ffn": (_i, [_vp] * 6 + [_i, _i, _i64, _i64, _i64, _vp, _sz, _vp]),
    "tf_gated_ffn_backward_workspace_bytes": (_sz, [_i64, _i64, _i64]),
    "tf_gated_ffn_backward": (_i, [_vp] * 9 + [_i, _i, _i64, _i64, _i64, _vp, _sz, _vp]),
    "tf_linear_cross_entropy_workspace_bytes": (_sz, [_i64, _i64, _i64]),
    "tf_linear_cross_entropy": (_i, [_vp] * 5 + [_i, _i64, _i64, _i64, _i64, _vp, _sz, _vp]),
    "tf_linear_cross_entropy_backward_workspace_bytes": (_sz, [_i64, _i64, _i64]),
    "tf_linear_cross_entropy_backward": (_i, [_vp] * 7 + [_i, _i64, _i64, _i64, _i64, _vp, _sz, _vp]),
    "tf_append_paged_kv": (_i, [ctypes.POINTER(PagedCache), _vp, _vp, _vp, ctypes.POINTER(_i64), _vp, _vp, _i64, _i64, _i, _vp, _i64, _i64, _vp, _vp, _vp]),
    "tf_flash_decode_paged_workspace_bytes": (_sz, [_i64] * 4),
    "tf_flash_decode_paged": (_i, [ctypes.POINTER(PagedCache), _vp, ctypes.POINTER(_i64), _vp, _i64, _d, _vp, _sz, _vp]),
    "tf_flash_attention_packed": (_i, [ctypes.POINTER(PackedAttention), _vp, _vp, _vp]),
    "tf_flash_attention_packed_backward_workspace_bytes": (_sz, [ctypes.POINTER(PackedAttention)]),
    "tf_flash_attention_packed_backward": (_i, [ctypes.POINTER(PackedAttention)] + [_vp] * 7 + [_sz, _vp]),
    "tf_product_kernel_index": (_i, [_i64, _i64, _i64, _i]),
    "tf_product_cols_plan": (_i, [_i64, _i64, _i64, ctypes.POINTER(_i)]),
    "tf_product_pair_plan": (_i, [_i64] * 6 + [ctypes.POINTER(_i)] * 2),
    "tf_linear_cross_entropy_backward_piece": (_i64, [_i64, _i64, _i64]),
    "tf_gemm_kernel_index": (_i, [_i64, _i64, _i64, _i]),
    "tf_flash_decode_plan": (_i, [_i64, _i64, _i64, _i, ctypes.POINTER(_i)]),
    "tf_flash_attention_rows": (_i, [_i64, _i64, _i64, _i64, _i]),
    "tf_flash_attention_pairs": (_i, [_i64, _i64, _i64, _i64, _i]),
    "tf_flash_attention_wide_rows": (_i, [_i64, _i64, _i]),
    "tf_flash_attention_packed_rows": (_i, [_i64] * 5),
    "tf_scatter_nd_plan": (_i, [_i64, _i64, _i64, _i, ctypes.POINTER(_i)]),
    "tf_fused_two_gemms_rows": (_i, [_i64, _i64, _i64, _i64, _i64, _sz]),
    "tf_jit_compile": (_i, [ctypes.c_char_p, ctypes.c_char_p, ctypes.POINTER(ctypes.c_char_p), _i,
                            ctypes.POINTER(ctypes.c_char_p), _i, ctypes.POINTER(_vp)]),
    "tf_jit_launch": (_i, [_vp] + [ctypes.c_uint] * 7 + [_vp, ctypes.POINTER(_vp)]),
    "tf_jit_clear_cache": (_i, []),
    "tf_jit_cache_dir": (ctypes.c_char_p, []),
    "tf_last_error": (ctypes.c_char_p, []),
    "tf_version": (ctypes.c_char_p, []),
}

_lib = None


def load():
    """Load libtilefusion_hip.so once and attach the argument types."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with `make -C tilefusion_amd/csrc` "
                "(there is no CPU fallback)")
        lib = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = res, args
        _lib = lib
    return _lib


def check(status, what):
    """Turn a non-zero status of the C ABI into a RuntimeError carrying tf_last_error()."""
    if status != TF_OK:
        msg = load().tf_last_error().decode("utf-8", "replace")
        raise RuntimeError(f"{what} failed (status {status}): {msg}")

"""Loader and ctypes signatures of ``librllm_kernels.so`` (the gfx950 C ABI).

Error model mirrors ``crates/rllm-kernels/src/cuda.rs:39-52``:
``CudaKernelError::{KernelError{code}, NotAvailable}`` become the exceptions
:class:`KernelError` (non-zero return code of an entry point) and
:class:`NotAvailable` (the native library is missing).  There is no CPU
fallback: every call goes through the HIP library or raises.
"""
from __future__ import annotations

import ctypes
import os

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(PKG_DIR, "librllm_kernels.so")
HEADER_PATH = os.path.join(os.path.dirname(PKG_DIR), "include", "rllm_kernels.h")

DTYPE_F16, DTYPE_BF16, DTYPE_FP8_E4M3, DTYPE_FP8_E5M2 = 0, 1, 2, 3
# FP8 rounding of the cache writes (RLLM_FP8_ROUND_* in include/rllm_kernels.h)
FP8_ROUND_TOWARD_ZERO, FP8_ROUND_NEAREST_EVEN = 0, 1


class KernelError(RuntimeError):
    """A native entry point returned a non-zero hipError_t code."""

    def __init__(self, code: int, what: str = ""):
        self.code = int(code)
        super().__init__(f"{what or 'kernel'} returned error code {self.code}")


class NotAvailable(RuntimeError):
    """The HIP library is not built / not loadable on this host."""


_lib = None

_P = ctypes.c_void_p
_I64 = ctypes.c_int64
_I32 = ctypes.c_int32
_F = ctypes.c_float
_U = ctypes.c_size_t  # uintptr_t stream

# name -> argtypes (restype int32 unless listed in _RESTYPE)
SIGNATURES = {
    "rllm_paged_attention_decode_f16": [_P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I64, _F, _U],
    "rllm_paged_attention_decode_f16_sync": [_P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I64, _F],
    "rllm_paged_attention_decode_fp8": [_P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I64, _F, _I32, _U],
    "rllm_paged_attention_decode_fp8_sync": [_P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I64, _F, _I32],
    "rllm_paged_attention_decode_bf16": [_P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I64, _F, _U],
    "rllm_paged_attention_decode_bf16_sync": [_P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I64, _F],
    "rllm_paged_attention_decode_ex": [_P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I64, _F,
                                       _I32, _I32, _F, _F, _I64, _P, _I64, _U],
    "rllm_paged_attention_decode_prefix_ex": [_P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I64, _F,
                                              _I32, _I32, _F, _F, _I64, _U],
    "rllm_paged_attention_mixed_ex": [_P, _P, _P, _P, _P, _I64, _I64, _I64, _P, _P, _P, _P, _I64, _I64, _P, _P,
                                      _I64, _I64, _I64, _I64, _F, _I32, _I32, _F, _F, _U],
    "rllm_paged_attention_decode_noalloc": [_P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I64, _F,
                                            _I32, _I32, _F, _F, _I64, _U],
    "rllm_paged_attention_decode_workspace_size": [_I64, _I64, _I64, _I64, _I64, _I64, _I64],
    "rllm_paged_attention_prefill_f16": [_P, _P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I64, _I64, _F, _U],
    "rllm_paged_attention_prefill_f16_sync": [_P, _P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I64, _I64, _F],
    "rllm_paged_attention_prefill_fp8": [_P, _P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I64, _I64, _F, _I32, _U],
    "rllm_paged_attention_prefill_fp8_sync": [_P, _P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I64, _I64, _F, _I32],
    "rllm_paged_attention_prefill_bf16": [_P, _P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I64, _I64, _F, _U],
    "rllm_paged_attention_prefill_bf16_sync": [_P, _P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I64, _I64, _F],
    "rllm_paged_attention_prefill_ex": [_P, _P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I64, _I64, _F,
                                        _I32, _I32, _F, _F, _U],
    "rllm_cache_write_f16": [_P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _U],
    "rllm_cache_write_f16_sync": [_P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64],
    "rllm_cache_write_bf16": [_P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _U],
    "rllm_cache_write_fp8": [_P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I32, _U],
    "rllm_cache_write_fp8_sync": [_P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I32],
    "rllm_cache_write_fp8_scaled": [_P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I32, _F, _F, _I32, _U],
    "rllm_cache_write_fp8_ex": [_P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I32, _F, _F, _I32, _I32, _U],
    "rllm_rope_cache_write": [_P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64,
                              _I64, _I64, _I32, _I32, _F, _F, _U],
    "rllm_rope_cache_write_ex": [_P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64,
                                 _I64, _I64, _I32, _I32, _F, _F, _I32, _U],
    "rllm_rope_tables": [_P, _P, _I64, _I64, _F],
    "rllm_cache_copy_blocks": [_P, _P, _I64, _P, _I64, _I64, _I64, _U],
    "rllm_cache_swap_out": [_P, _P, _I64, _P, _I64, _I64, _I64, _P, _I64, _P, _U],
    "rllm_cache_swap_in": [_P, _P, _I64, _P, _I64, _I64, _I64, _P, _I64, _P, _U],
    "rllm_fused_rmsnorm_f16": [_P, _P, _P, _I64, _I64, _F, _U],
    "rllm_fused_rmsnorm_f16_sync": [_P, _P, _P, _I64, _I64, _F],
    "rllm_fused_silu_mul_f16": [_P, _P, _P, _I64, _U],
    "rllm_fused_silu_mul_f16_sync": [_P, _P, _P, _I64],
    "rllm_rmsnorm_ex": [_P, _P, _P, _I64, _I64, _F, _I32, _U],
    "rllm_silu_mul_ex": [_P, _P, _P, _I64, _I32, _U],
    "rllm_mxfp4_page_bytes": [_I64, _I64],
    "rllm_cache_write_mxfp4": [_P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I32, _U],
    "rllm_cache_read_mxfp4": [_P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I32, _U],
    "rllm_rope_cache_write_mxfp4": [_P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64,
                                    _I64, _I64, _I32, _U],
    "rllm_paged_attention_decode_mxfp4": [_P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I64, _I64, _F,
                                          _I32, _P, _I64, _U],
    "rllm_paged_attention_decode_mxfp4_workspace_size": [_I64, _I64, _I64, _I64, _I64, _I64],
    "rllm_paged_attention_prefill_mxfp4": [_P, _P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I64, _I64, _I64,
                                           _F, _I32, _U],
    "rllm_key_bounds": [_P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I64, _I32, _U],
    "rllm_rope_cache_append": [_P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I64,
                               _I64, _I64, _I64, _I32, _I32, _F, _F, _I32, _U],
    "rllm_select_blocks": [_P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I64, _I64, _I64, _I64, _I64, _I64,
                           _I32, _I32, _P, _I64, _U],
    "rllm_select_blocks_workspace_size": [_I64, _I64, _I64],
    "rllm_paged_attention_sparse": [_P, _P, _P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _I64, _I64, _I64, _I64,
                                    _I64, _F, _I32, _I32, _F, _F, _U],
    "rllm_vector_add_f32": [_P, _P, _P, _I64, _U],
    "rllm_vector_add_f32_sync": [_P, _P, _P, _I64],
    "rllm_block_copy": [_P, _P, _I64, _U],
    "rllm_block_copy_sync": [_P, _P, _I64],
    "rllm_fused_rope_f16": [_P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _F, _U],
    "rllm_fused_rope_f16_sync": [_P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _F],
    "rllm_cache_block_copy": [_P, _P, _I64, _I64, _U],
    "rllm_cache_block_copy_sync": [_P, _P, _I64, _I64],
    "rllm_cache_zero": [_P, _I64, _U],
    "rllm_cache_zero_sync": [_P, _I64],
    "rllm_gpu_alloc": [ctypes.POINTER(ctypes.c_void_p), _I64],
    "rllm_gpu_free": [_P],
    "rllm_gpu_alloc_host": [ctypes.POINTER(ctypes.c_void_p), _I64],
    "rllm_gpu_free_host": [_P],
}
_RESTYPE = {"rllm_paged_attention_decode_workspace_size": _I64, "rllm_mxfp4_page_bytes": _I64,
            "rllm_paged_attention_decode_mxfp4_workspace_size": _I64, "rllm_select_blocks_workspace_size": _I64}


def lib() -> ctypes.CDLL:
    """The loaded native library; raises :class:`NotAvailable` if absent."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise NotAvailable(
            f"{LIB_PATH} is not built; run __graft_entry__.build() (hipcc --offload-arch=gfx950)")
    try:
        L = ctypes.CDLL(LIB_PATH)
    except OSError as e:  # pragma: no cover - depends on the host
        raise NotAvailable(f"cannot load {LIB_PATH}: {e}") from e
    for name, args in SIGNATURES.items():
        try:
            fn = getattr(L, name)
        except AttributeError:
            continue  # reported by tests/test_abi.py, which checks every exported name
        fn.argtypes = args
        fn.restype = _RESTYPE.get(name, _I32)
    _lib = L
    return L


def check(rc: int, what: str = "") -> None:
    """``check`` of attention.rs:417-420 / cache_ops.rs:107-110."""
    if rc != 0:
        raise KernelError(rc, what)


def call(name: str, *args) -> None:
    check(getattr(lib(), name)(*args), name)

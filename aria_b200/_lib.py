"""ctypes binding of libaria_q4.so (include/aria_q4.h).

There is deliberately no fallback: if the shared library is missing or the
current device is not a B200, every call raises.  Python is only the host-side
mirror of the reference's call surface; all arithmetic happens in the CUDA
kernels behind the C ABI.
"""
from __future__ import annotations

import ctypes
import importlib.metadata
import os
import sys

_PKG = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_PKG, "libaria_q4.so")

# status codes (aria_q4_status)
OK, EINVAL, EUNSUPPORTED, EALIGN, ECUDA, ENODEVICE, ESIZE = range(7)
LAYOUT_KN, LAYOUT_NK = 0, 1
FLAG_CONST_WEIGHTS = 1
FLAG_KERNEL_STREAM = 2
FLAG_KERNEL_REGISTER = 4
FLAG_KERNEL_TENSOR = 8
FLAG_EPILOGUE_GELU = 16
F32, F16, BF16 = 0, 1, 30


class PagedKVStruct(ctypes.Structure):
    """aria_paged_kv."""
    _fields_ = [("k_pages", ctypes.c_void_p), ("v_pages", ctypes.c_void_p), ("page_stride", ctypes.c_longlong),
                ("slot_stride", ctypes.c_longlong), ("head_stride", ctypes.c_longlong), ("num_pages", ctypes.c_int),
                ("page_size", ctypes.c_int), ("kv_heads", ctypes.c_int), ("head_dim", ctypes.c_int),
                ("dtype", ctypes.c_int), ("block_table", ctypes.c_void_p), ("table_stride", ctypes.c_int),
                ("max_pages", ctypes.c_int), ("lens", ctypes.c_void_p)]


class LogitRulesStruct(ctypes.Structure):
    """aria_logit_rules."""
    _fields_ = [("history", ctypes.c_void_p), ("history_row", ctypes.c_longlong), ("history_cap", ctypes.c_int),
                ("history_lens", ctypes.c_void_p), ("prompt_lens", ctypes.c_void_p), ("repetition", ctypes.c_void_p),
                ("frequency", ctypes.c_void_p), ("presence", ctypes.c_void_p), ("bias_tokens", ctypes.c_void_p),
                ("bias_values", ctypes.c_void_p), ("bias_row", ctypes.c_longlong), ("biases", ctypes.c_int),
                ("allowed", ctypes.c_void_p), ("allowed_row", ctypes.c_longlong)]


# every symbol include/aria_q4.h declares: (restype, argtypes)
_P = ctypes.c_void_p
_SZ = ctypes.c_size_t
_I = ctypes.c_int
_F = ctypes.c_float
_L = ctypes.c_longlong
SIGNATURES = {
    "aria_q4_0_packed_bytes": (_SZ, [_SZ]),
    "aria_q4_0_pack_f16": (_I, [_P, _SZ, _P, _P]),
    "aria_q4_0_pack_f32": (_I, [_P, _SZ, _P, _P]),
    "aria_q4_0_unpack_f32": (_I, [_P, _SZ, _P, _P]),
    "aria_q4_0_tiled_bytes": (_SZ, [_I, _I]),
    "aria_q4_0_repack": (_I, [_P, _I, _I, _I, _P, _SZ, _P]),
    "aria_q4_0_quantize_tiled": (_I, [_P, _I, _I, _I, _P, _SZ, _P]),
    "aria_q4_0_matmul": (_I, [_P, _I, _I, _I, _P, _I, _I, _P, _I, _I, _P, _F, _F, _P]),
    "aria_q4_0_matmul_ex": (_I, [_P, _I, _I, _I, _P, _I, _I, _P, _I, _I, _P, _F, _F, _I, _P]),
    "aria_q4_0_workspace_bytes": (_SZ, [_I, _I, _I]),
    "aria_q4_0_matmul_ws": (_I, [_P, _I, _I, _I, _P, _I, _I, _P, _I, _I, _P, _F, _F, _P, _SZ, _I, _P]),
    "aria_q4_0_kernel_choice": (_I, [_I, _I, _I, _I, _SZ, _I]),
    "aria_q4_0_matmul_static_ws": (_I, [_P, _I, _I, _I, _P, _I, _I, _P, _I, _I, _P, _F, _F, _I, _P]),
    "aria_q4_0_workspace_counter_bytes": (_SZ, []),
    "aria_q4_test_tensor_stall": (_I, [_P, _I, _I, _I, _P, _I, _I, _P, _I, _I, ctypes.c_uint, _P]),
    "aria_q4_0_matmul_ln": (_I, [_P, _I, _I, _I, _P, _I, _I, _P, _P, _F, _P, _I, _I, _P, _F, _F, _I, _P]),
    "aria_embed_f16": (_I, [_P, _P, _I, _I, _I, _P, _P, _I, _P, _P]),
    "aria_layernorm_f32": (_I, [_P, _I, _I, _P, _P, _F, _P, _I, _P]),
    "aria_attention_decode": (_I, [_P, _I, _I, _I, _P, _P, _I, _P, _P, _P]),
    "aria_flash_attn_fwd": (_I, [_P, _P, _P, _P, _P, _I, _I, _I, _F, _P]),
    "aria_attention_prefill": (_I, [_P, _I, _I, _I, _I, _P, _P, _P, _P, _I, _P]),
    "aria_paged_workspace_counter_bytes": (_SZ, []),
    "aria_attention_paged_workspace_bytes": (_SZ, [_P, _I, _I, _I]),
    "aria_attention_paged": (_I, [_P, _I, _I, _P, _L, _L, _P, _P, _L, _L, _F, _P, _L, _L, _P, _P, _P, _L, _P, _P, _P,
                                  _SZ, _P]),
    "aria_prompt_weights": (_I, [_P, _L, _L, _L, _P, _L, _L, _L, _I, _I, _I, _I, _I, _I, _P, _F, _I, _P, _L, _L, _P, _SZ,
                                 _P]),
    "aria_prompt_weights_workspace_bytes": (_SZ, [_I, _I, _I, _I, _I]),
    "aria_cache_evict_workspace_bytes": (_SZ, [_P, _I, _I]),
    "aria_cache_evict": (_I, [_P, _I, _P, _P, _P, _P, _L, _P, _I, _I, _I, _P, _P, _SZ, _P]),
    "aria_logits_workspace_bytes": (_SZ, [_I]),
    "aria_logits_adjust": (_I, [_P, _P, _I, _L, _I, _I, _P, _I, _L, _P, _P, _SZ, _P]),
    "aria_p2p_alloc": (_I, [_SZ, _P]),
    "aria_p2p_free": (_I, [_P]),
    "aria_p2p_ipc_handle": (_I, [_P, _P]),
    "aria_p2p_ipc_open": (_I, [_P, _P]),
    "aria_p2p_ipc_close": (_I, [_P]),
    "aria_p2p_allreduce_add": (_I, [_P, _P, _P, _I, _I, _P, _I, ctypes.c_uint, _P]),
    "aria_q4_strerror": (ctypes.c_char_p, [_I]),
    "aria_q4_last_cuda_error": (_I, []),
    "aria_q4_take_device_error": (_I, []),
    "aria_stream_capture_id": (_I, [_P, _P]),
    "aria_q4_abi_version": (_I, []),
}


class AriaQ4Error(RuntimeError):
    def __init__(self, fn: str, status: int, cuda_err: int = 0):
        msg = _lib().aria_q4_strerror(status).decode() if _LIB is not None else str(status)
        if status == ECUDA:
            msg += f" (cudaError {cuda_err})"
        super().__init__(f"{fn}: {msg}")
        self.status = status
        self.cuda_error = cuda_err


_LIB = None


def _lib() -> ctypes.CDLL:
    global _LIB
    if _LIB is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(f"{LIB_PATH} is missing: run `python -m aria_b200.build` (nvcc, sm_100a)")
        lib = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = res
            fn.argtypes = args
        _LIB = lib
    return _LIB


_FAST = None


def fastcall_key() -> str | None:
    """The Python and the torch that a build of aria_b200._fastcall is for, None without torch."""
    try:
        return f"{sys.implementation.cache_tag} torch {importlib.metadata.version('torch')}"
    except importlib.metadata.PackageNotFoundError:
        return None


class _LongWay:
    """In place of aria_b200._fastcall where it was not built, or not for this torch: every
    call goes the long way, through ctypes."""

    def __getattr__(self, name):
        return lambda *args: None


def fastcall():
    """The C++ binding of the serving operators, bound to the library's entry points."""
    global _FAST
    if _FAST is None:
        import torch  # noqa: F401  (loads what the module links against)
        try:
            from . import _fastcall
        except ImportError:
            _fastcall = None
        if _fastcall is None or _fastcall.key != fastcall_key():
            _FAST = _LongWay()
            return _FAST
        lib = _lib()
        _fastcall.bind(*(ctypes.cast(getattr(lib, f), ctypes.c_void_p).value for f in (
            "aria_attention_paged", "aria_prompt_weights", "aria_cache_evict", "aria_logits_adjust")), check)
        _FAST = _fastcall
    return _FAST


def lib() -> ctypes.CDLL:
    return _lib()


def check(fn: str, status: int) -> None:
    if status != OK:
        raise AriaQ4Error(fn, status, _lib().aria_q4_last_cuda_error())


def call(fn: str, *args) -> None:
    check(fn, getattr(_lib(), fn)(*args))

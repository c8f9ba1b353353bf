"""Loader for libgomlx_hip.so, the C ABI declared in include/gomlx_hip.h.

The library is the product: every op in this package runs through it.  There is
no CPU fallback — if the library is missing the import fails loudly.
"""
from __future__ import annotations

import ctypes
import os

_PKG_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
# GHIP_LIB_PATH selects another build of the same ABI (e.g. the sanitizer build
# of the host code, `make -C go-darwinml_amd/csrc asan`).
LIB_PATH = os.environ.get("GHIP_LIB_PATH") or os.path.join(_PKG_ROOT, "lib", "libgomlx_hip.so")
CSRC_DIR = os.path.join(_PKG_ROOT, "csrc")

# Dtype numbering of include/gomlx_hip.h (the reference's MPSGraphDType).
DT_BOOL, DT_INT8, DT_INT16, DT_INT32, DT_INT64 = 0, 1, 2, 3, 4
DT_FLOAT16, DT_BFLOAT16, DT_FLOAT32, DT_FLOAT64 = 5, 6, 7, 8
DT_UINT8, DT_UINT16, DT_UINT32, DT_UINT64 = 9, 10, 11, 12


class GHipError(ctypes.Structure):
    _fields_ = [("code", ctypes.c_int), ("message", ctypes.c_char_p)]


class BackendError(RuntimeError):
    """Raised when a C entry point returns a non-zero GHIP_ERR_* code."""

    def __init__(self, code: int, message: str):
        super().__init__(f"[code {code}] {message}")
        self.code = code


_i64 = ctypes.c_int64
_int = ctypes.c_int
_vp = ctypes.c_void_p
_f32 = ctypes.c_float
_errp = ctypes.POINTER(GHipError)
_byref = ctypes.byref

# The arrays of these two are spelled out: a structure of scalars is made in a third of the time.
class Rope(ctypes.Structure):
    """GHipRope."""
    _fields_ = ([("positions", _vp)] + [(f"position_stride{i}", _i64) for i in range(3)] + [("axes", _i64)]
                + [(f"section{i}", _i64) for i in range(4)] + [("freqs", _vp), ("rotary_dim", _i64), ("interleaved", _i64)])


class Kv4(ctypes.Structure):
    """GHipKv4."""
    _fields_ = ([("codes", _vp), ("scales", _vp)] + [(f"code_stride{i}", _i64) for i in range(3)]
                + [(f"scale_stride{i}", _i64) for i in range(3)])


_i64p = ctypes.POINTER(_i64)
_ropep = ctypes.POINTER(Rope)
_kv4p = ctypes.POINTER(Kv4)

# name -> argtypes (every entry point returns int except where noted).
SIGNATURES = {
    "ghip_softmax_rows": [_int, _vp, _vp, _i64, _i64, _int, _vp, _errp],
    "ghip_scale_mask_softmax_rows": [_int, _vp, _vp, _i64, _i64, _i64, _f32, _int, _vp, _vp, _errp],
    "ghip_rmsnorm_rows": [_int, _vp, _vp, _vp, _i64, _i64, _f32, _vp, _errp],
    "ghip_layernorm_rows": [_int, _vp, _vp, _vp, _vp, _i64, _i64, _f32, _vp, _errp],
    "ghip_gemm_batched": [_int, _int, _i64, _i64, _i64, _i64, _vp, _i64, _i64, _i64,
                          _vp, _i64, _i64, _i64, _vp, _i64, _i64, _i64, _vp, _errp],
    "ghip_gemm_grouped": [_int, _int, _int, _i64, _i64, _i64, _vp, _i64, _i64, ctypes.POINTER(_vp), _i64, _i64,
                          ctypes.POINTER(_vp), _i64, _vp, _errp],
    "ghip_gemm_batched_ws": [_int, _int, _i64, _i64, _i64, _i64, _vp, _i64, _i64, _i64,
                             _vp, _i64, _i64, _i64, _vp, _i64, _i64, _i64, _vp, _i64, _vp, _errp],
    "ghip_gemm_grouped_ws": [_int, _int, _int, _i64, _i64, _i64, _vp, _i64, _i64, ctypes.POINTER(_vp), _i64,
                             _i64, ctypes.POINTER(_vp), _i64, _vp, _i64, _vp, _errp],
    "ghip_gather_rows": [_vp, _i64, _i64, _vp, _i64, _vp, _vp, _errp],
    "ghip_argminmax": [_int, _vp, _i64, _i64, _i64, _int, _int, _vp, _vp, _errp],
    "ghip_iota": [_int, _vp, _i64, _i64, _i64, _vp, _errp],
    "ghip_device_name": [_int, ctypes.c_char_p, ctypes.c_size_t, _errp],
    "ghip_sdpa_fwd": [_int, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64,
                      ctypes.POINTER(_i64), ctypes.POINTER(_i64), ctypes.POINTER(_i64),
                      ctypes.POINTER(_i64), _f32, _int, _vp, _errp],
    "ghip_sdpa_fwd_masked": [_int, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64,
                             ctypes.POINTER(_i64), ctypes.POINTER(_i64), ctypes.POINTER(_i64),
                             ctypes.POINTER(_i64), _vp, _int, ctypes.POINTER(_i64), _f32, _int, _vp,
                             _errp],
    "ghip_sdpa_fwd_masked_ws": [_int, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _i64, _i64, _i64,
                                ctypes.POINTER(_i64), ctypes.POINTER(_i64), ctypes.POINTER(_i64),
                                ctypes.POINTER(_i64), _vp, _int, ctypes.POINTER(_i64), _f32, _int, _vp, _i64,
                                _vp, _errp],
    "ghip_scale_mask_softmax_rows_ex": [_int, _vp, _vp, _i64, _i64, _i64, _i64, _f32, _int, _vp, _int,
                                        ctypes.POINTER(_i64), _vp, _errp],
    "ghip_copy_strided": [_int, _vp, _vp, _int, ctypes.POINTER(_i64), ctypes.POINTER(_i64),
                          ctypes.POINTER(_i64), _vp, _errp],
    "ghip_softmax_cols": [_int, _vp, _vp, _i64, _i64, _i64, _int, _vp, _errp],
    "ghip_layernorm_cols": [_int, _vp, _vp, _vp, _vp, _i64, _i64, _i64, _f32, _vp, _errp],
    "ghip_sdpa_window_fwd": [_int] + [_vp] * 5 + [_i64] * 6 + [ctypes.POINTER(_i64)] * 4 + [_i64] * 3
                            + [_vp, _f32, _vp, _errp],
    "ghip_sdpa_window_bwd": [_int] + [_vp] * 9 + [_i64] * 6 + [ctypes.POINTER(_i64)] * 8 + [_i64] * 3
                            + [_vp, _f32, _vp, _i64, _vp, _errp],
    "ghip_kv_append": [_int] + [_vp] * 4 + [_i64] * 7 + [_vp, _i64, _vp, _vp] + [ctypes.POINTER(_i64)] * 4
                      + [_vp, _errp],
    "ghip_sdpa_paged": [_int] + [_vp] * 4 + [_i64] * 7 + [_vp, _i64, _vp] + [ctypes.POINTER(_i64)] * 4
                       + [_i64, _i64, _f32, _vp, _i64, _vp, _errp],
    "ghip_rope": [_int, _vp, _vp] + [_i64] * 4 + [_i64p, _i64p, _ropep, _int, _vp, _errp],
    "ghip_kv_append_rope": [_int] + [_vp] * 6 + [_i64] * 8 + [_vp, _i64, _vp, _vp] + [_i64p] * 6 + [_ropep, _vp, _errp],
    "ghip_kv4_append_rope": [_int] + [_vp] * 4 + [_kv4p] * 2 + [_i64] * 8 + [_vp, _i64, _vp, _vp] + [_i64p] * 4
                            + [_ropep, _vp, _errp],
    "ghip_kv4_read": [_int, _kv4p, _kv4p, _vp, _vp] + [_i64] * 7 + [_vp, _i64, _vp, _i64p, _i64p, _vp, _errp],
    "ghip_sdpa_paged_kv4": [_int, _vp, _kv4p, _kv4p, _vp] + [_i64] * 7 + [_vp, _i64, _vp, _i64p, _i64p, _i64, _i64, _f32,
                                                                          _vp, _i64, _vp, _errp],
    "ghip_token_logprobs": [_int, _vp, _i64, _vp] + [_i64] * 3 + [_f32] + [_vp] * 6 + [_i64, _vp, _errp],
    "ghip_token_logprobs_grad": [_int, _vp, _i64] + [_vp] * 5 + [_i64, _i64, _f32, _vp, _i64, _vp, _errp],
}

# name -> argtypes of the entry points that return int64_t.
SIGNATURES_I64 = {
    "ghip_sdpa_workspace_bytes": [_int, _i64, _i64, _i64, _i64, _i64, _i64, _int],
    "ghip_gemm_workspace_bytes": [_int, _int, _i64, _i64, _i64, _i64],
    "ghip_sdpa_window_bwd_workspace_bytes": [_int] + [_i64] * 9,
    "ghip_sdpa_paged_workspace_bytes": [_int] + [_i64] * 6,
    "ghip_sdpa_paged_kv4_workspace_bytes": [_i64] * 6,
    "ghip_token_logprobs_workspace_bytes": [_int] + [_i64] * 3,
}

_lib = None


def load():
    """Returns the loaded library (raises if it was never built)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise ImportError(
            f"gomlx_hip: {LIB_PATH} is missing; build it with "
            f"`make -C {CSRC_DIR}` (or __graft_entry__.build())")
    L = ctypes.CDLL(LIB_PATH)
    for name, argtypes in SIGNATURES.items():
        fn = getattr(L, name)
        fn.argtypes = argtypes
        fn.restype = ctypes.c_int
    for name, argtypes in SIGNATURES_I64.items():
        fn = getattr(L, name)
        fn.argtypes = argtypes
        fn.restype = ctypes.c_int64
    L.ghip_version.argtypes = []
    L.ghip_version.restype = ctypes.c_char_p
    L.ghip_error_clear.argtypes = [_errp]
    L.ghip_error_clear.restype = None
    _lib = L
    return L


def call(name: str, *args) -> None:
    """Calls entry point `name` with a fresh GHipError; raises BackendError on failure."""
    L = _lib or load()
    err = GHipError()
    rc = getattr(L, name)(*args, _byref(err))
    if rc != 0:
        msg = err.message.decode() if err.message else "(no message)"
        L.ghip_error_clear(_byref(err))
        raise BackendError(rc, msg)

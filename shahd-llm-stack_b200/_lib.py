"""ctypes binding of libshahd_b200.so (the C ABI declared in include/shahd_b200.h).

Loading fails loudly when the library is missing: there is no CPU path behind this package.
"""
from __future__ import annotations

import ctypes
import os

from . import build as _build

_i32 = ctypes.c_int32
_i64 = ctypes.c_int64
_u32 = ctypes.c_uint32
_vp = ctypes.c_void_p
_fp = ctypes.POINTER(ctypes.c_float)
_dp = ctypes.POINTER(ctypes.c_double)
_ip = ctypes.POINTER(ctypes.c_int32)
_up = ctypes.POINTER(ctypes.c_uint32)

SHAHD_OK = 0
SHAHD_EINVAL = -1
SHAHD_ENODEV = -2
SHAHD_ENOMEM = -3
SHAHD_ECUDA = -4
SHAHD_ESTATE = -5
SHAHD_ETIMEOUT = -6


class ShahdModelCfg(ctypes.Structure):
    _fields_ = [
        ("embed_dim", _i32), ("num_layers", _i32), ("num_heads", _i32), ("kv_heads", _i32), ("block_size", _i32),
        ("vocab_size", _i32), ("mlp_hidden", _i32), ("position_scheme", _i32), ("norm_kind", _i32),
        ("mlp_kind", _i32), ("weight_tying", _i32), ("reserved", _i32), ("layer_norm_eps", ctypes.c_double),
        ("rope_base", ctypes.c_double),
    ]


class ShahdSampling(ctypes.Structure):
    _fields_ = [("temperature", ctypes.c_double), ("top_k", _i32), ("reserved", _i32), ("top_p", ctypes.c_double)]


class ShahdSessionOpts(ctypes.Structure):
    _fields_ = [("max_seqs", _i32), ("kv_pages", _i32), ("device", _i32), ("flags", _i32)]


SHAHD_BF16 = 0
SHAHD_F16 = 1
SHAHD_F32 = 2


class ShahdRows(ctypes.Structure):
    """Rows of heads in device memory: value i of head h of row r at data[r * row_stride + h * head_stride + i]."""

    _fields_ = [("data", _vp), ("row_stride", _i64), ("head_stride", _i64)]


class ShahdKvCache(ctypes.Structure):
    """One layer of a paged K/V cache: pages [kv_heads][K|V][64][head_dim] of 16-bit values, a block table per sequence."""

    _fields_ = [("pool", _vp), ("page_stride", _i64), ("block_table", _vp), ("max_blocks", _i32), ("pages", _i32),
                ("kv_heads", _i32), ("head_dim", _i32)]


class ShahdRopeCfg(ctypes.Structure):
    _fields_ = [("head_dim", _i32), ("rotary_dim", _i32), ("layout", _i32), ("scaling", _i32), ("original_positions", _i32),
                ("reserved", _i32), ("base", ctypes.c_double), ("factor", ctypes.c_double), ("beta_fast", ctypes.c_double),
                ("beta_slow", ctypes.c_double), ("magnitude", ctypes.c_double)]


class ShahdRopeCall(ctypes.Structure):
    _fields_ = [("dtype", _i32), ("rows", _i32), ("num_heads", _i32), ("kv_heads", _i32), ("n", _i32), ("reserved", _i32),
                ("positions", _vp), ("offsets", _vp), ("q", ShahdRows), ("q_out", ShahdRows), ("k", ShahdRows),
                ("k_out", ShahdRows), ("v", ShahdRows), ("cache", ShahdKvCache)]


class ShahdPromptCall(ctypes.Structure):
    _fields_ = [("dtype", _i32), ("rows", _i32), ("n", _i32), ("num_heads", _i32), ("kv_heads", _i32), ("head_dim", _i32),
                ("scale", ctypes.c_double), ("offsets", _vp), ("q", ShahdRows), ("k", ShahdRows), ("v", ShahdRows),
                ("out", ShahdRows)]


class ShahdTreeCall(ctypes.Structure):
    _fields_ = [("dtype", _i32), ("rows", _i32), ("n", _i32), ("num_heads", _i32), ("max_nodes", _i32), ("reserved", _i32),
                ("scale", ctypes.c_double), ("offsets", _vp), ("lengths", _vp), ("masks", _vp), ("q", ShahdRows),
                ("k", ShahdRows), ("v", ShahdRows), ("out", ShahdRows), ("cache", ShahdKvCache), ("workspace", _vp),
                ("workspace_bytes", _i64)]


class ShahdVerifyCall(ctypes.Structure):
    _fields_ = [("dtype", _i32), ("rows", _i32), ("n", _i32), ("vocab", _i32), ("target", _vp), ("draft", _vp),
                ("target_stride", _i64), ("draft_stride", _i64), ("offsets", _vp), ("parents", _vp), ("tokens", _vp),
                ("uniforms", _vp), ("lengths", _vp), ("path", _vp), ("count", _vp), ("next_ids", _vp), ("commit", _vp),
                ("new_lengths", _vp)]


# name -> (restype, argtypes); every symbol include/shahd_b200.h declares
SIGNATURES = {
    "MatMulF64": (None, [_dp, _dp, _dp, _i32, _i32, _i32]),
    "MatMulNTF64": (None, [_dp, _dp, _dp, _i32, _i32, _i32, _i32]),
    "MatMulTNF64": (None, [_dp, _dp, _dp, _i32, _i32, _i32, _i32]),
    "MatMulF32": (None, [_fp, _fp, _fp, _i32, _i32, _i32]),
    "MatMulNTF32": (None, [_fp, _fp, _fp, _i32, _i32, _i32, _i32]),
    "MatMulTNF32": (None, [_fp, _fp, _fp, _i32, _i32, _i32, _i32]),
    "SetKernelThreads": (None, [ctypes.c_int]),
    "ShahdCpuSupportsAvx2Fma": (ctypes.c_int, []),
    "SetScalarKernels": (None, [ctypes.c_int]),
    "ShahdGpuAvailable": (ctypes.c_int, []),
    "ShahdLastError": (ctypes.c_char_p, []),
    "ShahdSetTensorCoreMinRows": (None, [ctypes.c_int]),
    "ShahdDeviceErrorFlag": (ctypes.c_int, []),
    "ShahdSetProgrammaticLaunch": (None, [ctypes.c_int]),
    "ShahdSetDecodeChains": (None, [ctypes.c_int]),
    "ShahdSetPersistentStep": (None, [ctypes.c_int]),
    "ShahdSetTensorCorePrefillAttention": (None, [ctypes.c_int]),
    "ShahdSetDecodeAttentionKernel": (None, [ctypes.c_int]),
    "ShahdSetFusedAttentionBlock": (None, [ctypes.c_int]),
    "ShahdSetPersistentPrefillProjections": (None, [ctypes.c_int]),
    "ShahdMatMulNTBF16Device": (ctypes.c_int, [_vp, _vp, _vp, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int, _vp]),
    "ShahdMatMulNTF32Device": (ctypes.c_int, [_vp, _vp, _vp, ctypes.c_int, ctypes.c_int, ctypes.c_int, ctypes.c_int, _vp]),
    "ShahdMatMulNTF32NoAlloc": (ctypes.c_int, [_fp, _fp, _fp, _i32, _i32, _i32, _i32]),
    "shahd_param_count": (_i64, [ctypes.POINTER(ShahdModelCfg)]),
    "shahd_init_params": (ctypes.c_int, [ctypes.POINTER(ShahdModelCfg), _u32, _fp, _i64]),
    "shahd_session_create": (ctypes.c_int, [ctypes.POINTER(ShahdModelCfg), _vp, _i32, _i64,
                                            ctypes.POINTER(ShahdSessionOpts), ctypes.POINTER(_vp)]),
    "shahd_session_destroy": (ctypes.c_int, [_vp]),
    "shahd_reset": (ctypes.c_int, [_vp, _ip, _i32]),
    "shahd_seq_length": (_i32, [_vp, _i32]),
    "shahd_prefill": (ctypes.c_int, [_vp, _ip, _ip, _ip, _i32]),
    "shahd_step": (ctypes.c_int, [_vp, _ip, _ip, _i32, _fp, _ip]),
    "shahd_generate": (ctypes.c_int, [_vp, _ip, _ip, _i32, _i32, ctypes.POINTER(ShahdSampling), _up, _ip]),
    "shahd_generate_device": (ctypes.c_int, [_vp, _vp, _ip, _i32, _i32, ctypes.POINTER(ShahdSampling), _vp, _vp, _vp]),
    "shahd_generate_logits": (ctypes.c_int, [_vp, _ip, _ip, _i32, _i32, _ip, _fp]),
    "shahd_sync": (ctypes.c_int, [_vp]),
    "shahd_verify": (ctypes.c_int, [_vp, _ip, _ip, _ip, _i32, _fp, _ip]),
    "shahd_truncate": (ctypes.c_int, [_vp, _ip, _ip, _i32]),
    "shahd_step_launches": (_i32, [_vp, _i32]),
    "shahd_kernel_launches": (_i64, [_vp]),
    "shahd_profile": (ctypes.c_int, [_vp, _i32]),
    "shahd_profile_read": (ctypes.c_int, [_vp, _i32, _dp, ctypes.POINTER(_i64), _dp]),
    "shahd_sample_logits": (ctypes.c_int, [_fp, _i32, _i32, ctypes.POINTER(ShahdSampling), _up, _ip]),
    "shahd_speculative_round": (ctypes.c_int, [_fp, _fp, _ip, _ip, _ip, _i32, _i32, _i32, ctypes.POINTER(ShahdSampling),
                                                _up, _ip, _ip, _ip]),
    "shahd_attention_create": (ctypes.c_int, [_i32, _i32, _i32, _i32, _i32, ctypes.c_double, _i32,
                                               ctypes.POINTER(_vp)]),
    "shahd_attention_destroy": (ctypes.c_int, [_vp]),
    "shahd_attention_length": (_i32, [_vp, _i32]),
    "shahd_attention_prefill": (ctypes.c_int, [_vp, _vp, _vp, _vp, _i32, _i32, _vp, _vp]),
    "shahd_attention_decode": (ctypes.c_int, [_vp, _vp, _vp, _vp, _i32, _vp, _vp]),
    "shahd_attention_cache": (ctypes.c_int, [_vp, ctypes.POINTER(ShahdKvCache)]),
    "shahd_attention_set_lengths": (ctypes.c_int, [_vp, _ip, _i32, _vp]),
    "shahd_rope_create": (ctypes.c_int, [ctypes.POINTER(ShahdRopeCfg), ctypes.POINTER(_vp)]),
    "shahd_rope_destroy": (ctypes.c_int, [_vp]),
    "shahd_rope_apply": (ctypes.c_int, [_vp, ctypes.POINTER(ShahdRopeCall), _vp]),
    "shahd_prompt_attention": (ctypes.c_int, [ctypes.POINTER(ShahdPromptCall), _vp]),
    "shahd_tree_attention_workspace": (_i64, [ctypes.POINTER(ShahdTreeCall)]),
    "shahd_tree_attention": (ctypes.c_int, [ctypes.POINTER(ShahdTreeCall), _vp]),
    "shahd_verify_tree": (ctypes.c_int, [ctypes.POINTER(ShahdVerifyCall), _vp]),
    "shahd_last_error": (ctypes.c_char_p, []),
}

_LIB: ctypes.CDLL | None = None


def load(build_if_missing: bool = True) -> ctypes.CDLL:
    """The process-lifetime handle of libshahd_b200.so (never closed, like GoFfiBackend.ts:36-42)."""
    global _LIB
    if _LIB is not None:
        return _LIB
    if not os.path.exists(_build.SO_PATH):
        if not build_if_missing:
            raise OSError(f"libshahd_b200.so not built at {_build.SO_PATH}")
        _build.build()
    lib = ctypes.CDLL(_build.SO_PATH)
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = res
        fn.argtypes = args
    _LIB = lib
    return lib


class ShahdError(RuntimeError):
    def __init__(self, code: int, message: str):
        super().__init__(message)
        self.code = code


def check(rc: int) -> None:
    if rc != SHAHD_OK:
        raise ShahdError(rc, load().shahd_last_error().decode(errors="replace"))


def last_error() -> str:
    return load().ShahdLastError().decode(errors="replace")

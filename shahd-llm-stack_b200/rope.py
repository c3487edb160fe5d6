"""Rotary positions on packed rows (ApplyRope, Brain/Ops/RotaryEmbedding.ts:63-75), with the layouts and frequency scalings
that the session's fused RoPE does not have, and the append of keys and values to a paged cache; with norms of the query and
key heads (NormRow, Brain/Sampling/CachedRowMath.ts:25-56, on heads) in the same pass where a model has them.

Buffers are device addresses (torch CUDA tensors work: their data_ptr()). Calls are asynchronous on `stream` (0: the
legacy default stream), keep nothing and can be captured into CUDA graphs.
"""
from __future__ import annotations

import ctypes

from . import _lib
from .attention import F32, KvCache, Rows

LAYOUTS = {"interleaved": 0, "half": 1}
NORMS = {"rms": 0, "layer": 1}
SCALINGS = {"none": 0, "linear": 1, "stretched": 2, "by_parts": 3}
_NO_ROWS = Rows()
_NO_CACHE = KvCache()


class HeadNorm:
    """Norms of the query and key heads before they are turned (Rope.apply's norm): "rms" x / sqrt(mean(x^2) + eps) * weight, or
    "layer" (x - mean) / sqrt(var + eps) * weight + bias over a head's values. Weights and biases: device addresses of [head_dim] values of
    weight_dtype, for all heads (0: 1 and 0)."""

    def __init__(self, kind: str = "rms", eps: float = 1e-6, q_weight: int = 0, k_weight: int = 0, q_bias: int = 0, k_bias: int = 0,
                 weight_dtype: int = F32):
        if kind not in NORMS:
            raise ValueError(f"HeadNorm: kind must be one of {list(NORMS)}, got {kind!r}")
        self.cfg = _lib.ShahdHeadNorm(NORMS[kind], weight_dtype, eps, q_weight, k_weight, q_bias, k_bias)


class Rope:
    """Pair i of a head's first rotary_dim values turns by position * base^(-2i / rotary_dim), scaled:
    "linear": all frequencies divided by factor; "stretched": base * factor^(r / (r - 2)) for base; "by_parts": pairs that
    make more than beta_fast turns in original_positions keep their frequency, pairs with fewer than beta_slow are divided
    by factor, a linear ramp between. layout: pairs (2i, 2i+1) "interleaved" or (i, i + rotary_dim / 2) "half".
    magnitude multiplies cos and sin."""

    def __init__(self, head_dim: int, rotary_dim: int | None = None, layout: str = "interleaved", base: float = 10000.0,
                 scaling: str = "none", factor: float = 1.0, original_positions: int = 0, beta_fast: float = 32.0,
                 beta_slow: float = 1.0, magnitude: float = 1.0):
        if layout not in LAYOUTS or scaling not in SCALINGS:
            raise ValueError(f"Rope: layout must be one of {list(LAYOUTS)} and scaling one of {list(SCALINGS)}, got "
                             f"{layout!r} and {scaling!r}")
        self.lib = _lib.load()
        self.head_dim, self.rotary_dim = head_dim, head_dim if rotary_dim is None else rotary_dim
        cfg = _lib.ShahdRopeCfg(head_dim, self.rotary_dim, LAYOUTS[layout], SCALINGS[scaling], original_positions, 0, base, factor,
                                beta_fast, beta_slow, magnitude)
        h = ctypes.c_void_p()
        _lib.check(self.lib.shahd_rope_create(ctypes.byref(cfg), ctypes.byref(h)))
        self.handle = h

    def close(self) -> None:
        if getattr(self, "handle", None):
            self.lib.shahd_rope_destroy(self.handle)
            self.handle = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def apply(self, dtype: int, rows: int, positions: int, q: Rows = _NO_ROWS, q_out: Rows = _NO_ROWS, num_heads: int = 0,
              k: Rows = _NO_ROWS, k_out: Rows = _NO_ROWS, v: Rows = _NO_ROWS, kv_heads: int = 0, cache: KvCache = _NO_CACHE,
              offsets: int = 0, n: int = 0, stream: int = 0, norm: HeadNorm | None = None) -> None:
        """Turns q [rows, num_heads, head_dim] into q_out and k [rows, kv_heads, head_dim] into k_out (both may be in
        place), and writes the turned k and v to `cache` at positions[row] of the row's sequence (offsets, int32 [n+1] on
        the device). Rows of negative position, and rows outside offsets[0] .. offsets[n]-1, are left as they are. With a norm
        the heads of q and k are normalised first, in the same pass."""
        call = _lib.ShahdRopeCall(dtype, rows, num_heads, kv_heads, n, 0, positions, offsets, q, q_out, k, k_out, v, cache)
        if norm is None:
            _lib.check(self.lib.shahd_rope_apply(self.handle, ctypes.byref(call), stream or None))
        else:
            _lib.check(self.lib.shahd_norm_rope_apply(self.handle, ctypes.byref(call), ctypes.byref(norm.cfg), stream or None))

"""Rotary positions on packed rows (ApplyRope, Brain/Ops/RotaryEmbedding.ts:63-75), with the layouts and frequency scalings
that the session's fused RoPE does not have, and the append of keys and values to a paged cache.

Buffers are device addresses (torch CUDA tensors work: their data_ptr()). Calls are asynchronous on `stream` (0: the
legacy default stream), keep nothing and can be captured into CUDA graphs.
"""
from __future__ import annotations

import ctypes

from . import _lib
from .attention import KvCache, Rows

LAYOUTS = {"interleaved": 0, "half": 1}
SCALINGS = {"none": 0, "linear": 1, "stretched": 2, "by_parts": 3}
_NO_ROWS = Rows()
_NO_CACHE = KvCache()


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
              offsets: int = 0, n: int = 0, stream: int = 0) -> None:
        """Turns q [rows, num_heads, head_dim] into q_out and k [rows, kv_heads, head_dim] into k_out (both may be in
        place), and writes the turned k and v to `cache` at positions[row] of the row's sequence (offsets, int32 [n+1] on
        the device). Rows of negative position, and rows outside offsets[0] .. offsets[n]-1, are left as they are."""
        call = _lib.ShahdRopeCall(dtype, rows, num_heads, kv_heads, n, 0, positions, offsets, q, q_out, k, k_out, v, cache)
        _lib.check(self.lib.shahd_rope_apply(self.handle, ctypes.byref(call), stream or None))

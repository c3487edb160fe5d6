"""FusedAttention as an operator (the attention core of MultiHeadAttention.Forward,
Brain/Nn/MultiHeadAttention.ts:46-74, with RoPE and CausalSoftmax, then AttendRow decode steps,
Brain/Sampling/CachedRowMath.ts:60-86) over the library's device-resident paged cache.

Q/K/V and outputs are fp32 device buffers passed by address (torch CUDA tensors work: their data_ptr()).
Calls are asynchronous on `stream` (0: the operator's own stream): the buffers must stay allocated until the
stream has reached the call, so pass torch's current stream when torch owns them.

Next to it, attention on the caller's own buffers: prompt_attention for prompts of different lengths packed into one
call, tree_attention for drafted token trees (or single new tokens) against a paged cache, such as FusedAttention's own
(FusedAttention.cache). They keep no state: calls on different streams or devices do not meet, and both can be
captured into CUDA graphs. A stream of 0 is the legacy default stream there.
A wait inside a kernel that gives up leaves rows undefined and is recorded: _lib.load().ShahdDeviceErrorFlag() is 0 as long
as none has.
"""
from __future__ import annotations

import ctypes

import numpy as np

from . import _lib

BF16, F16, F32 = _lib.SHAHD_BF16, _lib.SHAHD_F16, _lib.SHAHD_F32
Rows = _lib.ShahdRows
KvCache = _lib.ShahdKvCache
MAX_TREE_NODES = 64


class FusedAttention:
    """num_heads query heads over kv_heads kv heads, head_dim 32/64/128, `capacity` positions per sequence."""

    def __init__(self, max_seqs: int, num_heads: int, kv_heads: int, head_dim: int, capacity: int,
                 rope_base: float = 10000.0, device: int = 0):
        self.lib = _lib.load()
        self.max_seqs, self.num_heads, self.kv_heads, self.head_dim = max_seqs, num_heads, kv_heads, head_dim
        self.capacity = capacity
        h = ctypes.c_void_p()
        _lib.check(self.lib.shahd_attention_create(max_seqs, num_heads, kv_heads, head_dim, capacity, float(rope_base),
                                                   device, ctypes.byref(h)))
        self.handle = h

    def close(self) -> None:
        if self.handle:
            self.lib.shahd_attention_destroy(self.handle)
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

    def length(self, slot: int) -> int:
        return int(self.lib.shahd_attention_length(self.handle, slot))

    def prefill(self, q: int, k: int, v: int, n: int, T: int, out: int, stream: int = 0) -> None:
        """Sequences 0..n-1 restart at position 0; q [n, T, H, d], k/v [n, T, Hk, d], out [n, T, H, d]
        (device addresses, fp32)."""
        _lib.check(self.lib.shahd_attention_prefill(self.handle, q, k, v, n, T, out, stream or None))

    def decode(self, q: int, k: int, v: int, n: int, out: int, stream: int = 0) -> None:
        """One position per sequence 0..n-1: q [n, H, d], k/v [n, Hk, d] (before RoPE), out [n, H, d]."""
        _lib.check(self.lib.shahd_attention_decode(self.handle, q, k, v, n, out, stream or None))

    def cache(self) -> KvCache:
        """This operator's cache (bf16, one layer) as rope.apply and tree_attention take it; valid until close(). Keys appended
        to it must be turned as this operator turns its own (Rope(head_dim, base=rope_base)) if its decode steps are to read
        them; with rope_base 0 it turns nothing, and q and k are turned by any Rope before they get here."""
        out = KvCache()
        _lib.check(self.lib.shahd_attention_cache(self.handle, ctypes.byref(out)))
        return out

    def set_lengths(self, lengths, stream: int = 0) -> None:
        """Cached positions of sequences 0..len(lengths)-1, for rows that were appended through cache()."""
        a = np.ascontiguousarray(lengths, dtype=np.int32)
        _lib.check(self.lib.shahd_attention_set_lengths(self.handle, a.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)), a.size,
                                                        stream or None))


def prompt_attention(dtype: int, q: Rows, k: Rows, v: Rows, out: Rows, offsets: int, n: int, rows: int, num_heads: int,
                     kv_heads: int, head_dim: int, scale: float = 0.0, stream: int = 0) -> None:
    """Causal attention within each of n packed sequences: rows offsets[s] .. offsets[s+1]-1 (int32 on the device) of q and
    out [rows, num_heads, head_dim] and k, v [rows, kv_heads, head_dim], BF16 or F16. scale 0: 1/sqrt(head_dim)."""
    call = _lib.ShahdPromptCall(dtype, rows, n, num_heads, kv_heads, head_dim, scale, offsets, q, k, v, out)
    _lib.check(_lib.load().shahd_prompt_attention(ctypes.byref(call), stream or None))


def tree_attention_workspace(n: int, max_nodes: int, num_heads: int, cache: KvCache) -> int:
    """Bytes of device workspace that tree_attention needs for these sizes (0: none)."""
    call = _lib.ShahdTreeCall(n=n, max_nodes=max_nodes, num_heads=num_heads, cache=cache)
    size = int(_lib.load().shahd_tree_attention_workspace(ctypes.byref(call)))
    if size < 0:
        _lib.check(size)
    return size


def tree_attention(dtype: int, q: Rows, k: Rows, v: Rows, out: Rows, cache: KvCache, lengths: int, masks: int, offsets: int,
                   n: int, rows: int, max_nodes: int, num_heads: int, scale: float = 0.0, workspace: int = 0,
                   workspace_bytes: int = 0, stream: int = 0) -> None:
    """Attention of up to 64 new rows per sequence (a tree of drafted tokens; one row: a decode step) over the sequence's
    lengths[s] cached positions and over those of its own new rows whose bit its mask has (uint64 [rows], see
    tree_masks). q, out [rows, num_heads, head_dim]; k, v [rows, kv_heads, head_dim], not in the cache yet."""
    call = _lib.ShahdTreeCall(dtype, rows, n, num_heads, max_nodes, 0, scale, offsets, lengths, masks, q, k, v, out, cache,
                              workspace, workspace_bytes)
    _lib.check(_lib.load().shahd_tree_attention(ctypes.byref(call), stream or None))


def tree_masks(parents) -> np.ndarray:
    """The masks (uint64) of one sequence's tree for tree_attention: each node sees itself and its ancestors. parents[i] is
    node i's parent, below i; the root's (node 0) is not read."""
    if len(parents) > MAX_TREE_NODES:
        raise ValueError(f"tree_masks: at most {MAX_TREE_NODES} nodes per sequence, got {len(parents)}")
    masks: list[int] = []
    for i, p in enumerate(parents):
        if i and not 0 <= int(p) < i:
            raise ValueError(f"tree_masks: node {i} needs a parent in 0 .. {i - 1}, got {int(p)}")
        masks.append((masks[int(p)] if i else 0) | 1 << i)
    return np.array(masks, dtype=np.uint64)

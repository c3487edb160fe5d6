"""Pages shared between sequences: forking sequences of a paged cache (beams, several answers to one prompt, rows that were cut back or
have ended) and moving the held pages together. The block tables say all there is to know: a page is held when some sequence's
cached positions lie on it, and free otherwise.

Buffers are device addresses (torch CUDA tensors work: their data_ptr()). Calls are asynchronous on `stream` (0: the legacy default
stream), keep nothing and can be captured into CUDA graphs; a workspace belongs to one call at a time.
"""
from __future__ import annotations

import ctypes

from . import _lib

PagePool = _lib.ShahdPagePool


def pages_workspace(pages: int, new_n: int = 0) -> int:
    """Bytes of device workspace for pages_fork to new_n sequences, or for pages_compact (0 sequences)."""
    size = int(_lib.load().shahd_pages_workspace(pages, new_n))
    if size < 0:
        _lib.check(size)
    return size


def pages_fork(pool: PagePool, table: int, lengths: int, n: int, max_blocks: int, parents: int, keep: int, need: int, new_n: int,
               new_table: int, missing: int, workspace: int, workspace_bytes: int, stream: int = 0) -> None:
    """New sequence i keeps the first keep[i] positions of sequence parents[i] of `table` (int32 [n, max_blocks], cached positions
    lengths[n]) and gets pages for positions up to need[i]; a parent outside 0 .. n-1 makes it begin empty. Full pages are shared, a
    page that is partly filled is copied unless it can stay with one that goes on in it, fresh pages are the free ones in
    ascending order. new_table [new_n, max_blocks] must not overlap table; missing [new_n]: pages that were not to be had."""
    call = _lib.ShahdForkCall(pool, n, new_n, max_blocks, 0, table, lengths, parents, keep, need, new_table, missing, workspace, workspace_bytes)
    _lib.check(_lib.load().shahd_pages_fork(ctypes.byref(call), stream or None))


def pages_compact(pool: PagePool, table: int, lengths: int, n: int, max_blocks: int, new_table: int, used: int, workspace: int,
                  workspace_bytes: int, stream: int = 0) -> None:
    """Moves the held pages of a pool together at its front; new_table (which may be table) names them there, used [1] is their
    number."""
    call = _lib.ShahdCompactCall(pool, n, max_blocks, table, lengths, new_table, used, workspace, workspace_bytes)
    _lib.check(_lib.load().shahd_pages_compact(ctypes.byref(call), stream or None))

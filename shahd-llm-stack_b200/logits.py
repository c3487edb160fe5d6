"""Penalties for repeated tokens, biases and grammar masks on rows of logits that lie on the device, before sampling
(SampleFromLogits, Brain/Sampling/Sampler.ts:16-27, has none of them).

Buffers are device addresses (torch CUDA tensors work: their data_ptr()). Calls are asynchronous on `stream` (0: the legacy default
stream), keep nothing and can be captured into CUDA graphs.
"""
from __future__ import annotations

import ctypes

from . import _lib


def adjust_logits(dtype: int, logits: int, out: int, rows: int, vocab: int, n: int, sequences: int = 0, history: int = 0,
                  history_stride: int = 0, history_lengths: int = 0, prompt_lengths: int = 0, repetition: int = 0, presence: int = 0,
                  frequency: int = 0, bias_offsets: int = 0, bias_tokens: int = 0, bias_values: int = 0, bias_entries: int = 0,
                  masks: int = 0, mask_rows: int = 0, mask_count: int = 0, mask_stride: int | None = None,
                  logits_stride: int | None = None, out_stride: int | None = None, stream: int = 0) -> None:
    """Rows of logits [rows, vocab] into out (which may be logits; else no row of it shares memory with one of them). A row belongs to sequence sequences[row] (its own number
    without them). A token of that sequence's history [n, history_stride] (prompt first) is divided by repetition where its logit
    is positive, else multiplied; one that was generated c times loses c * frequency + presence; biases (token, value entries
    bias_offsets[s] .. bias_offsets[s+1]-1) are added; tokens whose bit the row's mask [mask_count, mask_stride words] lacks become
    -inf. int32 and float32 operands but for the logits."""
    words = (vocab + 31) // 32 if mask_stride is None and masks else mask_stride or 0
    call = _lib.ShahdLogitsCall(dtype, rows, n, vocab, logits, out, vocab if logits_stride is None else logits_stride,
                                vocab if out_stride is None else out_stride, sequences, history, history_stride, history_lengths,
                                prompt_lengths, repetition, presence, frequency, bias_offsets, bias_tokens, bias_values, bias_entries,
                                mask_count, masks, words, mask_rows)
    _lib.check(_lib.load().shahd_adjust_logits(ctypes.byref(call), stream or None))

"""shahd-llm-stack_b200: B200 (sm_100a) backend for the Shahd KV-cached decode path.

The product is libshahd_b200.so (C ABI in include/shahd_b200.h). This package builds it, loads it with
ctypes and mirrors the reference's host-side interface over it:
  backend.GpuBackend      — the ComputeBackend seam (MatMul / MatMulInto / MatMulNtAcc / MatMulNtInto / MatMulTnAcc)
  decode.Session          — device-resident model + paged KV cache, batched cached steps, on-device generate
  decode.CachedDecoder    — CachedDecoder over one session slot
  decode.cached_generate  — CachedGenerate
  attention.FusedAttention — the attention core (RoPE, causal prefill, AttendRow decode steps) as an operator
  attention.prompt_attention, attention.tree_attention — packed prompts, and drafted token trees over a paged cache
  attention.chunk_attention — the next rows of each sequence, parts of prompts and decode steps, over a paged cache
  rope.Rope, rope.HeadNorm — rotary positions on packed rows, norms of the heads before them, the append to a paged cache
  pages.pages_fork, pages.pages_compact — pages of a cache shared between sequences
  logits.adjust_logits    — penalties, biases and grammar masks before sampling
  speculative.verify_tree — SpeculativeSample's rule for drafted token trees, on the device
Import with importlib (the directory name has dashes): importlib.import_module("shahd-llm-stack_b200").
"""
from . import _lib, attention, backend, build, checkpoint, configs, decode, logits, pages, rope, sharding, speculative  # noqa: F401
from .attention import (  # noqa: F401
    BF16, F16, F32, FusedAttention, KvCache, Rows, chunk_attention, chunk_attention_workspace, prompt_attention, tree_attention,
    tree_attention_workspace, tree_masks)
from .backend import GpuBackend  # noqa: F401
from .decode import (  # noqa: F401
    GREEDY, CachedDecoder, ModelConfig, Sampling, Session, cached_generate, init_params, sample_from_logits)
from .logits import adjust_logits  # noqa: F401
from .pages import PagePool, pages_compact, pages_fork, pages_workspace  # noqa: F401
from .rope import HeadNorm, Rope  # noqa: F401
from .speculative import verify_tree  # noqa: F401


def load():
    """Load (building if needed) libshahd_b200.so; raises when it cannot be loaded."""
    return _lib.load()

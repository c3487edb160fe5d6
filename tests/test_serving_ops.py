"""The serving operators' argument checks and host logic, without a GPU: every refusal here comes before a device is asked for."""
import numpy as np
import pytest

from tests.conftest import has_gpu
from tests.helpers import pkg

ROWS = pkg.Rows(1 << 20, 128, 64)  # never followed: the calls are refused before
CACHE = pkg.KvCache(1 << 20, 2 * 2 * 64 * 64, 1 << 20, 4, 9, 2, 64)


def _refused(text, call, *args, **kwargs):
    with pytest.raises(pkg._lib.ShahdError, match=text) as e:
        call(*args, **kwargs)
    assert e.value.code == pkg._lib.SHAHD_EINVAL


def test_rope_configurations():
    for bad in (dict(head_dim=1), dict(head_dim=258), dict(rotary_dim=3), dict(rotary_dim=66), dict(rotary_dim=0)):
        _refused("rotary_dim", pkg.Rope, **{"head_dim": 64, **bad})
    for bad in (dict(base=1.0), dict(base=float("nan")), dict(magnitude=0.0), dict(magnitude=float("inf")), dict(scaling="linear", factor=0.5)):
        _refused("finite base", pkg.Rope, 64, **bad)
    _refused("rotary_dim >= 4", pkg.Rope, 64, 2, scaling="stretched", factor=2.0)
    _refused("original_positions", pkg.Rope, 64, scaling="by_parts", factor=2.0)
    _refused("original_positions", pkg.Rope, 64, scaling="by_parts", factor=2.0, original_positions=4096, beta_fast=1.0, beta_slow=1.0)
    with pytest.raises(ValueError, match="layout"):
        pkg.Rope(64, layout="both")
    with pkg.Rope(64, 32, "half", scaling="by_parts", factor=4.0, original_positions=4096) as rope:
        assert rope.rotary_dim == 32
    rope.close()


def test_rope_calls():
    with pkg.Rope(64) as rope:
        ok = dict(dtype=pkg.BF16, rows=4, positions=1 << 20, q=ROWS, q_out=ROWS, num_heads=2)
        _refused("dtype", rope.apply, **{**ok, "dtype": 7})
        _refused("rows >= 0", rope.apply, **{**ok, "rows": -1})
        _refused("num_heads or kv_heads", rope.apply, **{**ok, "num_heads": 0})
        _refused("n >= 1", rope.apply, **{**ok, "offsets": 1 << 20})
        _refused("k_out or a cache", rope.apply, **{**ok, "k": ROWS, "kv_heads": 2})
        _refused("a cache needs kv_heads", rope.apply, **ok, cache=CACHE, offsets=1 << 20, n=1)
        _refused("need n >= 1", rope.apply, **ok, k=ROWS, v=ROWS, kv_heads=2, cache=CACHE)
        _refused("the cache holds 2 kv heads", rope.apply, **{**ok, "q": pkg.Rows(1, 512, 64)}, k=ROWS, v=ROWS, kv_heads=4, cache=CACHE, offsets=1 << 20, n=1)
        _refused("page_stride", rope.apply, **ok, k=ROWS, v=ROWS, kv_heads=2, cache=pkg.KvCache(1 << 20, 100, 1 << 20, 4, 9, 2, 64), offsets=1 << 20, n=1)
        _refused("q needs row and head strides", rope.apply, **{**ok, "q": pkg.Rows(1 << 20, 128, 32)})
        _refused("q_out needs row and head strides", rope.apply, **{**ok, "q_out": pkg.Rows(1 << 20, -128, 64)})
        _refused("rows and heads of q_out share memory", rope.apply, **{**ok, "q_out": pkg.Rows(1 << 20, 64, 64)})
        _refused("too many rows", rope.apply, **{**ok, "rows": 2**30 + 1})
        _refused("too many sequences", rope.apply, **{**ok, "offsets": 1 << 20, "n": 2**30 + 1})


def test_prompt_calls():
    ok = dict(dtype=pkg.BF16, q=ROWS, k=ROWS, v=ROWS, out=ROWS, offsets=1 << 20, n=1, rows=4, num_heads=2, kv_heads=2, head_dim=64)
    call = pkg.prompt_attention
    _refused("dtype", call, **{**ok, "dtype": pkg.F32})
    _refused("head_dim 32, 64 or 128", call, **{**ok, "head_dim": 96})
    _refused("kv_heads dividing", call, **{**ok, "num_heads": 3})
    _refused("at most 8", call, **{**ok, "num_heads": 18})
    _refused("n, rows >= 0", call, **{**ok, "n": -1})
    _refused("scale", call, **{**ok, "scale": -1.0})
    _refused("scale", call, **{**ok, "scale": float("nan")})
    _refused("k needs strides that are multiples of 8", call, **{**ok, "k": pkg.Rows(1 << 20, 132, 64)})
    _refused("out needs row and head strides", call, **{**ok, "out": pkg.Rows(1 << 20, 128, 0)})
    _refused("too many rows", call, **{**ok, "n": 2**31 - 1, "rows": 2**30})
    _refused("too many rows", call, **{**ok, "rows": 2**30 + 1})
    _refused("too many rows and sequences", call, **{**ok, "n": 2**30 + 1, "num_heads": 1, "kv_heads": 1})
    _refused("share memory", call, **{**ok, "out": pkg.Rows(1 << 20, 64, 64)})
    _refused("share memory", call, **{**ok, "out": pkg.Rows(1 << 20, 64, 3 * 64)})
    if not has_gpu():
        with pytest.raises(pkg._lib.ShahdError) as e:
            call(**ok)
        assert e.value.code == pkg._lib.SHAHD_ENODEV


def test_tree_calls():
    ok = dict(dtype=pkg.F16, q=ROWS, k=ROWS, v=ROWS, out=ROWS, cache=CACHE, lengths=1 << 20, masks=1 << 20, offsets=1 << 20, n=1, rows=4, max_nodes=4, num_heads=2)
    call = pkg.tree_attention
    for nodes in (0, 65, -1):
        _refused("max_nodes in 1 .. 64", call, **{**ok, "max_nodes": nodes})
    _refused("pages and max_blocks", call, **{**ok, "cache": pkg.KvCache(1 << 20, 2 * 2 * 64 * 64, 1 << 20, 0, 9, 2, 64)})
    _refused("pages and max_blocks", call, **{**ok, "cache": pkg.KvCache(1 << 20, 2 * 2 * 64 * 64 + 4, 1 << 20, 4, 9, 2, 64)})
    _refused("dtype", call, **{**ok, "dtype": pkg.F32})
    _refused("rows >= 0", call, **{**ok, "rows": -4})
    _refused("too many rows", call, **{**ok, "rows": 2**30 + 1})
    _refused("share memory", call, **{**ok, "out": pkg.Rows(1 << 20, 64, 64)})
    _refused("v needs strides", call, **{**ok, "v": pkg.Rows(1 << 20, 132, 64)})
    big = pkg.KvCache(1 << 20, 2 * 2 * 64 * 64, 1 << 20, 512, 9, 2, 64)
    size = pkg.tree_attention_workspace(1, 4, 8, big)
    assert size > 0 and size % 32 == 0
    _refused("bytes of workspace", call, **{**ok, "cache": big, "num_heads": 8, "q": pkg.Rows(1 << 20, 512, 64), "out": pkg.Rows(1 << 20, 512, 64)})
    assert pkg.tree_attention_workspace(1000, 4, 8, big) > size  # long caches of 2000 tile pairs are still cut into ranges
    assert pkg.tree_attention_workspace(2000, 4, 8, big) == 0  # the pairs fill the device many times over: a block of threads each
    short = pkg.KvCache(1 << 20, 2 * 2 * 64 * 64, 1 << 20, 16, 9, 2, 64)
    assert pkg.tree_attention_workspace(1000, 4, 8, short) == 0
    _refused("at most 8", pkg.tree_attention_workspace, 1, 4, 64, big)


def test_verify_calls():
    at = 1 << 20
    ok = dict(dtype=pkg.F32, target=at, draft=at, vocab=10, tokens=at, parents=at, uniforms=at, offsets=at, n=1, rows=4, path=at, count=at, next_ids=at)
    call = pkg.verify_tree
    _refused("dtype", call, **{**ok, "dtype": 3})
    _refused("1 <= vocab", call, **{**ok, "vocab": 0})
    _refused("strides of at least vocab", call, **{**ok, "target_stride": 9})
    _refused("too many rows", call, **{**ok, "rows": 2**30 + 1})
    _refused("or sequences", call, **{**ok, "n": 2**30 + 1})
    _refused("need lengths", call, **{**ok, "commit": at})
    _refused("need lengths", call, **{**ok, "new_lengths": at})
    call(**{**ok, "n": 0})


def test_tree_masks():
    m = pkg.tree_masks([-1, 0, 0, 2, 1])
    assert m.dtype == np.uint64 and m.tolist() == [1, 3, 5, 13, 19]
    assert pkg.tree_masks([]).size == 0
    chain = pkg.tree_masks([-1] + list(range(63)))
    assert int(chain[63]) == 2**64 - 1
    with pytest.raises(ValueError, match="at most 64"):
        pkg.tree_masks([-1] + [0] * 64)
    for bad in ([-1, 1], [-1, -1], [-1, 0, 5]):
        with pytest.raises(ValueError, match="parent"):
            pkg.tree_masks(bad)

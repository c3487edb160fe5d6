"""Attention scores that are not finite, in prompts and trees: a row that sees a NaN or a score of +inf is NaN, a score of -inf
has weight 0 (a row that sees nothing else is NaN, one that sees nothing at all is 0), and rows that do not see the key keep their
results. Every column of a whole key block in turn, since columns take different ways through the exponentials."""
import math

import numpy as np
import pytest

from tests.helpers import pkg

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
from tests import serving_refs as R  # noqa: E402
from tests.test_gpu_serving_ops import (  # noqa: E402, F401
    BF16, F16, _cache_of, _gen, _held, _no_device_error, _normal, _offsets, _prompt, _random_masks, _tree)

KEYS = {32: 64, 64: 64, 128: 128}  # of a block


def _check_rows(got, q, k, v, seen, dtype):
    """got [t, H, d] against the definition in 64 bits, head by head. A key of score -inf has weight 0, as if it were not seen."""
    H, group = q.shape[1], q.shape[1] // k.shape[1]
    bad_rows = 0
    for h in range(H):
        x = torch.where(seen, q[:, h].double() @ k[:, h // group].double().T * q.shape[2] ** -0.5, -math.inf)
        nan = (x.isnan() | (x == math.inf)).any(1) | (seen.any(1) & (x == -math.inf).all(1))
        one = slice(h // group, h // group + 1)
        want, bound = R.attend(q[:, h:h + 1], torch.nan_to_num(k[:, one], 0.0, 0.0, 0.0), v[:, one], seen & x.isfinite(), q.shape[2] ** -0.5, dtype)
        assert bool(got[nan, h].isnan().all()), (h, torch.nonzero(nan & ~got[:, h].isnan().all(1)).flatten().tolist())
        off = (got[~nan, h].double() - want[~nan, 0]).abs()
        assert bool((off <= bound[~nan, 0].clamp(min=1e-30)).all()), h  # a NaN is not within it either
        bad_rows += int(nan.sum())
    return bad_rows


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf], ids=str)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_prompt_rows_that_see_a_score_that_is_not_finite(d, dtype, bad):
    keys = KEYS[d]
    # the bad key in every column of block 0; a sequence whose whole block 0 is bad; a sequence of a single, bad key
    lens = [keys + 72] * (keys + 1) + [1]
    off, g = _offsets(lens), _gen(61)
    q, k, v = (_normal(g, sum(lens), h, d, dtype=dtype) for h in (4, 2, 2))
    for c in range(keys):
        k[off[c] + c, 0, 0] = bad
    k[off[keys]:off[keys] + keys, 0, 0] = bad
    k[off[keys + 1], 0, 0] = bad
    out = _prompt(q, k, v, lens, dtype)
    spoiled = 0
    for s, t in enumerate(lens):
        b, e = off[s], off[s + 1]
        spoiled += _check_rows(out[b:e], q[b:e], k[b:e], v[b:e], torch.ones(t, t, device="cuda").tril().bool(), dtype)
    assert spoiled > 50 * keys


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf], ids=str)
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("H,Hk,d,nodes", [(4, 2, 32, 3), (4, 2, 64, 3), (4, 2, 128, 3), (8, 1, 64, 20), (8, 1, 128, 20)])
def test_tree_rows_that_see_a_score_that_is_not_finite(H, Hk, d, nodes, wide, dtype, bad):
    keys = KEYS[d]
    # the bad key in every column of the cache's block 0; a cache of bad keys only; a single, bad cached key; bad nodes, with and without a cache
    lengths = [keys + 40] * keys + [keys + 70, 1, 30, 0]
    if wide:
        lengths += [1500]  # over many ranges, the bad key in the middle
    n = len(lengths)
    counts = [nodes] * n
    g = _gen(62)
    q, k, v = (_normal(g, sum(counts), h, d, dtype=dtype) for h in (H, Hk, Hk))
    pool, table, cache = _cache_of(lengths, Hk, d, dtype, g)
    pool.normal_(generator=g)
    for s, at in [(c, [c]) for c in range(keys)] + [(keys, range(keys + 70)), (keys + 1, [0])] + ([(n - 1, [700])] if wide else []):
        for p in at:
            pool[table[s, p // 64], -1, 0, 0, p % 64, 0] = bad
    off = _offsets(counts)
    k[off[keys + 2], 0, 0], k[off[keys + 3] + 2, 0, 0] = bad, bad
    if wide:
        held = torch.cat([table, torch.full((n, 600 - table.shape[1]), -1, dtype=torch.int32, device="cuda")], 1)
        cache = pkg.KvCache(cache.pool, cache.page_stride, held.data_ptr(), 600, cache.pages, Hk, d)
    assert (pkg.tree_attention_workspace(n, nodes, H, cache) > 0) == wide
    masks = _random_masks(counts, 63)
    masks[off[keys + 3] + 1] = 0  # this row sees nothing at all
    out = _tree(q, k, v, cache, lengths, masks, counts, dtype)
    spoiled = 0
    for s, t in enumerate(counts):
        b, e, L = off[s], off[s + 1], lengths[s]
        cached = torch.stack([_held(pool, table, s, L, h) for h in range(Hk)], 2)
        bits = (masks[b:e, None] >> torch.arange(t, device="cuda")) & 1
        seen = torch.cat([torch.ones(t, L, dtype=torch.bool, device="cuda"), bits.bool()], 1)
        spoiled += _check_rows(out[b:e], q[b:e], torch.cat([cached[0], k[b:e]]), torch.cat([cached[1], v[b:e]]), seen, dtype)
    assert spoiled > keys
    assert bool((out[off[keys + 3] + 1] == 0).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("how", ["prompt", "pairs", "ranges"])
def test_large_scores_that_lie_close_to_each_other(how, d, dtype):
    """Scores of 2^27 (bf16) and 2^24 (fp16), exact in 32 bits, that grow along the keys by a few units in the last place, so that the
    maximum moves again and again, over blocks, tiles by turns and parts.

    The weights are right to 2^-13 although the product of a maximum with the scale is rounded by up to 1 and 1/8 in log2: an exponent
    of at most 150 is rounded once (2^-17), an exponential is good to 2.7e-6, and so is each of at most 40 changes of the maximum
    (2^-24 of a difference of offsets below 150, 2^-22 of its exponential)."""
    g, L = _gen(65), 290
    j = torch.arange(L, device="cuda")
    base, step = (2.0 ** 13, 16.0) if dtype == BF16 else (2.0 ** 12, 2.0)
    n = j // 5 + torch.randint(0, 3, (L,), generator=g, device="cuda") if dtype == BF16 else j + torch.randint(0, 8, (L,), generator=g, device="cuda")
    q, k, v = torch.zeros(L, 2, d, dtype=dtype, device="cuda"), torch.zeros(L, 1, d, dtype=dtype, device="cuda"), _normal(g, L, 1, d, dtype=dtype)
    q[:, 0, 0], q[:, 0, 1], k[:, 0, 0], k[:, 0, 1] = base, step, 2 * base if dtype == BF16 else base, n.to(dtype)
    q[:, 1] = -q[:, 0]
    scores = q[:, 0].double() @ k[:, 0].double().T
    assert torch.equal(scores.float().double(), scores) and torch.equal(scores[0], scores[0, 0] + step * (n - n[0]).double())
    scale = 0.125
    if how == "prompt":
        out, want, bound, rows = _prompt(q, k, v, [L], dtype, scale=scale), *_close(q, k, v, torch.ones(L, L, device="cuda").tril().bool(), scale, dtype), L
    else:
        rows = 70  # sequence s: the first 220 + s keys in the cache, the next one its own row
        pool, table, cache = _cache_of([L], 1, d, dtype, g)
        for p in range(L):
            pool[table[0, p // 64], -1, 0, 0, p % 64], pool[table[0, p // 64], -1, 0, 1, p % 64] = k[p, 0], v[p, 0]
        held = torch.full((rows, 1200 if how == "ranges" else table.shape[1]), -1, dtype=torch.int32, device="cuda")
        held[:, :table.shape[1]] = table
        cache = pkg.KvCache(cache.pool, cache.page_stride, held.data_ptr(), held.shape[1], cache.pages, 1, d)
        assert (pkg.tree_attention_workspace(rows, 1, 2, cache) > 0) == (how == "ranges")
        own = slice(220, 290)
        out = _tree(q[own], k[own], v[own], cache, list(range(220, 290)), torch.ones(rows, dtype=torch.int64, device="cuda"), [1] * rows, dtype, scale=scale)
        want, bound = _close(q[own], k, v, torch.ones(L, L, device="cuda").tril().bool()[own], scale, dtype)
    assert bool(((out.double() - want).abs() <= bound).all())


def _close(q, k, v, seen, scale, dtype):
    want, _ = R.attend(q, k, v, seen, scale, dtype)
    mass, _ = R.attend(q, k, v.abs(), seen, scale, dtype)
    u = R.HALF_STEP[dtype]
    # fp16 probabilities have a fixed step below 2^-14 of 2^7 times the largest, rounded offset included
    return want, u * want.abs() + mass * (u + 2.0 ** -12) + (2.0 ** -31 * v.abs().double().sum() + 2.0 ** -25 if dtype == F16 else 0.0)


@pytest.mark.parametrize("dtype,most", [(BF16, 2.0 ** 30), (F16, 2.0 ** 23)], ids=["bf16", "f16"])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_beyond_the_range_give_nan(dtype, most, sign):
    """Rows that see one key, of a score at the range's end (in log2) and just below it."""
    g = _gen(66)
    q, k, v = torch.zeros(2, 1, 64, dtype=dtype, device="cuda"), torch.zeros(2, 1, 64, dtype=dtype, device="cuda"), _normal(g, 2, 1, 64, dtype=dtype)
    q[:, 0, 3] = 2.0 ** 15
    k[0, 0, 3], k[1, 0, 3] = sign * most / 2 ** 15, sign * most / 2 ** 15 * (1 - 2.0 ** -7)
    out = _prompt(q, k, v, [1, 1], dtype, scale=1 / math.log2(math.e))
    assert bool(out[0].isnan().all()) and torch.equal(out[1], v[1])


@pytest.mark.parametrize("size", [2.0 ** 24, 2.0 ** 31, 2.0 ** 41, 2.0 ** 100])
@pytest.mark.parametrize("d", [64, 128])
def test_rows_that_leave_scores_beyond_the_range_are_right_or_nan(d, size):
    """A whole block of keys of scores far below the range, then ordinary ones: the weights of the first are 0."""
    g, L, keys = _gen(67), 3 * KEYS[d] + 5, KEYS[d]
    q, k, v = (_normal(g, L, h, d, dtype=BF16) for h in (2, 1, 1))
    q[:, :, 0], k[:, :, 0] = 0.0, 0.0
    q[:, :, 0], k[:keys, :, 0] = size ** 0.5 * 1.37, -(size ** 0.5) * (1 + torch.rand(keys, 1, generator=g, device="cuda"))
    out = _prompt(q, k, v, [L], BF16)
    seen = torch.ones(L, L, device="cuda").tril().bool()
    seen[keys:, :keys] = False
    want, bound = R.attend(q[keys:], k, v, seen[keys:], d ** -0.5, BF16)
    off = (out[keys:].double() - want).abs()
    assert bool((out[keys:].isnan() | (off <= bound)).all())
    if size <= 2.0 ** 24:
        assert bool(out.isfinite().all())

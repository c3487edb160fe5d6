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

"""Tree calls in the layout that each case is meant for, which the bytes of workspace tell: ranges of key blocks with more sequences
than a block has threads, so that the sums over sequences go round after round, and pairs of tiles on their own."""
import numpy as np
import pytest

from tests.helpers import pkg

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
from tests.test_gpu_serving_ops import (  # noqa: E402, F401
    BF16, CODE, F16, _cache_of, _check_tree, _gen, _ints, _no_device_error, _normal, _offsets, _random_masks, _rows, _tree)


def _wider(cache, table, blocks):
    held = torch.full((table.shape[0], blocks), -1, dtype=torch.int32, device="cuda")
    held[:, :table.shape[1]] = table
    return held, pkg.KvCache(cache.pool, cache.page_stride, held.data_ptr(), blocks, cache.pages, cache.kv_heads, cache.head_dim)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,heads,nodes,most,blocks", [
    (400, (4, 1, 64), 3, 500, 64), (400, (4, 1, 128), 3, 500, 64), (900, (8, 1, 128), 20, 300, 80), (650, (6, 2, 32), 2, 700, 100),
    (2300, (2, 1, 64), 2, 200, 64), (1150, (1, 1, 128), 1, 400, 64), (321, (8, 2, 64), 40, 300, 64), (385, (16, 2, 128), 17, 200, 64)], ids=str)
def test_ranges_with_more_sequences_than_threads(n, heads, nodes, most, blocks, dtype):
    H, Hk, d = heads
    rng = np.random.default_rng(n)
    lengths, counts = rng.integers(0, most, n), rng.integers(0, nodes + 1, n)
    lengths[rng.integers(0, n, n // 8)] = 0
    empty = rng.integers(0, n - 40)
    counts[empty:empty + 37] = 0  # a run of sequences without rows
    threads = 384 if d == 128 else 320
    ends = [s for s in (threads - 1, threads, 2 * threads - 1, 2 * threads, n - 1) if s < n]
    for s in ends:
        lengths[s], counts[s] = most, nodes
    lengths, counts = lengths.tolist(), counts.tolist()
    g = _gen(71)
    q, k, v = (_normal(g, sum(counts) + 2, h, d, dtype=dtype) for h in (H, Hk, Hk))
    pool, table, cache = _cache_of(lengths, Hk, d, dtype, g)
    pool.normal_(generator=g)
    held, cache = _wider(cache, table, blocks)
    assert pkg.tree_attention_workspace(n, nodes, H, cache) > 0
    masks = _random_masks(counts, 72)
    out = _tree(q, k, v, cache, lengths, masks, counts, dtype, max_nodes=nodes)
    _check_tree(q, k, v, pool, table, lengths, masks, counts, out, dtype, seqs=set(rng.integers(0, n, 12).tolist()) | set(rng.integers(threads, n, 24).tolist()) | set(ends))
    assert bool((out[sum(counts):] == 7.0).all())
    assert torch.equal(out, _tree(q, k, v, cache, lengths, masks, counts, dtype, max_nodes=nodes))


@pytest.mark.parametrize("n,heads,nodes,most,blocks,ranges", [
    (90, (8, 4, 128), 5, 700, None, False),   # the one tile of rows of two kv heads
    (80, (6, 2, 32), 64, 900, None, False),   # two tiles of rows
    (8, (32, 8, 128), 1, 2000, None, False),  # one tile by turns
    (1300, (2, 1, 64), 2, 300, None, False),
    (20, (32, 8, 128), 64, 6000, None, True),
    (5, (16, 2, 64), 33, 9000, None, True),
    (1, (16, 4, 64), 24, 2047, None, True),
    (72, (12, 4, 64), 26, 254, 512, False),   # a block of threads per pair in a table of long caches, too
    (256, (8, 2, 64), 1, 576, 64, True)], ids=str)
def test_layouts(n, heads, nodes, most, blocks, ranges):
    H, Hk, d = heads
    rng = np.random.default_rng(n)
    lengths, counts = rng.integers(0, most, n).tolist(), rng.integers(1, nodes + 1, n).tolist()
    lengths[0], counts[0] = most, nodes
    g = _gen(73)
    q, k, v = (_normal(g, sum(counts), h, d, dtype=BF16) for h in (H, Hk, Hk))
    pool, table, cache = _cache_of(lengths, Hk, d, BF16, g)
    pool.normal_(generator=g)
    if blocks:
        held, cache = _wider(cache, table, blocks)
    assert (pkg.tree_attention_workspace(n, nodes, H, cache) > 0) == ranges
    masks = _random_masks(counts, 74)
    out = _tree(q, k, v, cache, lengths, masks, counts, BF16, max_nodes=nodes)
    _check_tree(q, k, v, pool, table, lengths, masks, counts, out, BF16, seqs=set(rng.integers(0, n, 16).tolist()) | {0, n - 1})


def test_refusals_of_the_workspace():
    q = torch.zeros(4, 2, 64, dtype=BF16, device="cuda")
    table, pool = _ints([0] * 512), torch.zeros(8, 2, 2, 64, 64, dtype=BF16, device="cuda")
    cache = pkg.KvCache(pool.data_ptr(), pool.stride(0), table.data_ptr(), 512, 8, 2, 64)
    need = pkg.tree_attention_workspace(1, 4, 2, cache)
    assert need > 0
    off, mask, ws = _ints([0, 4]), torch.zeros(4, dtype=torch.int64, device="cuda"), torch.zeros(need + 32, dtype=torch.uint8, device="cuda")
    tree = dict(dtype=CODE[BF16], q=_rows(q), k=_rows(q), v=_rows(q), out=_rows(q), cache=cache, lengths=off.data_ptr(), masks=mask.data_ptr(), offsets=off.data_ptr(), n=1,
                rows=4, max_nodes=4, num_heads=2, workspace=ws.data_ptr(), workspace_bytes=need)
    for bad, text in ((dict(workspace_bytes=need - 1), "bytes of workspace"), (dict(workspace=0), "workspace is null"),
                      (dict(workspace=ws.data_ptr() + 16), "workspace must be aligned to 32"), (dict(workspace=torch.zeros(need, dtype=torch.uint8).data_ptr()), "workspace")):
        with pytest.raises(pkg._lib.ShahdError, match=text) as e:
            pkg.tree_attention(**{**tree, **bad})
        assert e.value.code == pkg._lib.SHAHD_EINVAL

"""The argument checks of the operators of a serving step over shared pages, without a GPU: every refusal here comes before a device is
asked for; and the rules of forking on a page by page restatement."""
import numpy as np
import pytest

from tests.conftest import has_gpu
from tests.helpers import pkg

torch = pytest.importorskip("torch")
from tests import step_refs as S  # noqa: E402

AT = 1 << 20  # never followed: the calls are refused before
ROWS = pkg.Rows(AT, 128, 64)
CACHE = pkg.KvCache(AT, 2 * 2 * 64 * 64, AT, 4, 9, 2, 64)
PAGE = 2 * 2 * 64 * 64


def _refused(text, call, *args, **kwargs):
    with pytest.raises(pkg._lib.ShahdError, match=text) as e:
        call(*args, **kwargs)
    assert e.value.code == pkg._lib.SHAHD_EINVAL


def _no_device(call, *args, **kwargs):
    if not has_gpu():
        with pytest.raises(pkg._lib.ShahdError) as e:
            call(*args, **kwargs)
        assert e.value.code == pkg._lib.SHAHD_ENODEV


def test_chunk_calls():
    call = pkg.chunk_attention
    size = pkg.chunk_attention_workspace(1, 4, 4, 2, CACHE)
    ok = dict(dtype=pkg.F16, q=ROWS, out=ROWS, cache=CACHE, lengths=AT, offsets=AT, n=1, rows=4, max_rows=4, num_heads=2, workspace=AT, workspace_bytes=size)
    assert size > 0 and size % 32 == 0
    _no_device(call, **ok)
    _refused("bytes of workspace", call, **{**ok, "workspace_bytes": size - 1})
    _refused("dtype", call, **{**ok, "dtype": pkg.F32})
    _refused("max_rows >= 1", call, **{**ok, "max_rows": 0})
    _refused("n, rows >= 0", call, **{**ok, "rows": -1})
    _refused("n, rows >= 0", call, **{**ok, "n": -1})
    _refused("at most 8", call, **{**ok, "num_heads": 18})
    _refused("head_dim 32, 64 or 128", call, **{**ok, "cache": pkg.KvCache(AT, 2 * 2 * 64 * 96, AT, 4, 9, 2, 96)})
    _refused("page_stride", call, **{**ok, "cache": pkg.KvCache(AT, PAGE + 4, AT, 4, 9, 2, 64)})
    _refused("scale", call, **{**ok, "scale": -1.0})
    _refused("scale", call, **{**ok, "scale": float("nan")})
    _refused("q needs strides that are multiples of 8", call, **{**ok, "q": pkg.Rows(AT, 132, 64)})
    _refused("out needs row and head strides", call, **{**ok, "out": pkg.Rows(AT, 128, 0)})
    _refused("share memory", call, **{**ok, "out": pkg.Rows(AT, 64, 64)})
    _refused("too many rows", call, **{**ok, "rows": 2**30 + 1})
    _refused("too many rows", call, **{**ok, "rows": 2**30, "n": 2**23, "max_rows": 2**30})
    _refused("too many rows or key blocks", pkg.chunk_attention_workspace, 100, 10**6, 10**6, 2, pkg.KvCache(AT, PAGE, AT, 1 << 24, 9, 2, 64))
    call(**{**ok, "n": 0})
    call(**{**ok, "rows": 0})
    # a block of threads for every pair of tiles where there are many, or enough over short caches: no workspace
    wide = lambda blocks: pkg.KvCache(AT, PAGE, AT, blocks, 9, 2, 64)  # noqa: E731
    assert pkg.chunk_attention_workspace(256, 256, 1, 8, wide(9)) == 0 and pkg.chunk_attention_workspace(256, 256, 1, 8, wide(900)) > 0
    assert pkg.chunk_attention_workspace(1000, 1000, 1, 8, wide(900)) == 0
    # a few pairs: clusters share them, ranges where that leaves too many steps
    assert 0 < pkg.chunk_attention_workspace(1, 64, 64, 8, wide(30)) != pkg.chunk_attention_workspace(1, 64, 64, 8, wide(3000))
    assert pkg.chunk_attention_workspace(0, 0, 1, 8, CACHE) >= 0


def test_head_norms():
    with pytest.raises(ValueError, match="kind"):
        pkg.HeadNorm("batch")
    ok = dict(dtype=pkg.BF16, rows=4, positions=AT, q=ROWS, q_out=ROWS, num_heads=2)
    with pkg.Rope(64) as rope:
        _no_device(rope.apply, **ok, norm=pkg.HeadNorm())
        for eps in (0.0, -1.0, float("nan"), float("inf"), 1e-50, 1e39):
            _refused("eps", rope.apply, **ok, norm=pkg.HeadNorm(eps=eps))
        _refused("weight_dtype", rope.apply, **ok, norm=pkg.HeadNorm(weight_dtype=5))
        _refused("biases", rope.apply, **ok, norm=pkg.HeadNorm("rms", q_bias=AT))
        bad = pkg.HeadNorm()
        bad.cfg.kind = 7
        _refused("unknown norm", rope.apply, **ok, norm=bad)
        # the checks of the calls without a norm
        norm = pkg.HeadNorm("layer", 1e-5, AT, AT, AT, AT)
        _refused("dtype", rope.apply, **{**ok, "dtype": 7}, norm=norm)
        _refused("num_heads or kv_heads", rope.apply, **{**ok, "num_heads": 0}, norm=norm)
        _refused("k_out or a cache", rope.apply, **ok, k=ROWS, kv_heads=2, norm=norm)
        _refused("need n >= 1", rope.apply, **ok, k=ROWS, v=ROWS, kv_heads=2, cache=CACHE, norm=norm)
        _refused("rows and heads of q_out share memory", rope.apply, **{**ok, "q_out": pkg.Rows(AT, 64, 64)}, norm=norm)
        rope.apply(**{**ok, "rows": 0}, norm=norm)


def test_logits_calls():
    call = pkg.adjust_logits
    ok = dict(dtype=pkg.F32, logits=AT, out=AT, rows=4, vocab=100, n=4)
    _no_device(call, **ok)
    _refused("dtype", call, **{**ok, "dtype": 3})
    for bad in (dict(rows=-1), dict(rows=2**20 + 1), dict(n=-1), dict(n=2**20 + 1), dict(vocab=0), dict(vocab=2**24 + 1)):
        _refused("rows and n in", call, **{**ok, **bad})
    _refused("a row for each", call, **{**ok, "n": 3})
    _refused("strides of at least vocab", call, **{**ok, "logits_stride": 99, "out_stride": 99})
    _refused("in place have one stride", call, **{**ok, "logits_stride": 101})
    penalties = dict(history=AT, history_stride=9, history_lengths=AT)
    _refused("history_lengths", call, **{**ok, **penalties, "history_lengths": 0})
    _refused("history_lengths", call, **{**ok, **penalties, "history_stride": -1})
    _refused("penalties with a history", call, **{**ok, "repetition": AT})
    _refused("penalties with a history", call, **{**ok, "prompt_lengths": AT})
    biases = dict(bias_offsets=AT, bias_tokens=AT, bias_values=AT, bias_entries=4)
    for bad in (dict(bias_offsets=0), dict(bias_tokens=0), dict(bias_values=0), dict(bias_entries=-1)):
        _refused("go together", call, **{**ok, **biases, **bad})
    _refused("masks need", call, **{**ok, "masks": AT, "mask_count": 2, "mask_stride": 3})
    _refused("masks need", call, **{**ok, "masks": AT, "mask_count": -2})
    _refused("masks need", call, **{**ok, "mask_rows": AT})
    call(**{**ok, "rows": 0})
    call(**{**ok, "n": 0, "sequences": AT})


def test_pages_calls():
    pool = pkg.PagePool(AT, PAGE, 0, 1, 9, 2, 64)
    size = pkg.pages_workspace(9, 4)
    ok = dict(pool=pool, table=AT, lengths=AT, n=3, max_blocks=5, parents=AT, keep=AT, need=AT, new_n=4, new_table=2 * AT, missing=AT, workspace=AT, workspace_bytes=size)
    call = pkg.pages_fork
    _no_device(call, **ok)
    _refused("bytes of workspace", call, **{**ok, "workspace_bytes": size - 1})
    _refused("overlap", call, **{**ok, "new_table": AT})
    _refused("overlap", call, **{**ok, "new_table": AT + 4 * 14})
    _refused("overlap", call, **{**ok, "new_table": AT - 4})
    for bad in (dict(n=-1), dict(n=2**20 + 1), dict(new_n=-1), dict(new_n=2**20 + 1), dict(max_blocks=0), dict(max_blocks=2**24 + 1), dict(n=2**20, max_blocks=2**11)):
        _refused("2\\^30 table entries", call, **{**ok, **bad})
    for pages in (0, 2**24 + 1):
        _refused("table entries", call, **{**ok, "pool": pkg.PagePool(AT, PAGE, 0, 1, pages, 2, 64)})
        _refused("table entries", pkg.pages_workspace, pages, 4)
    for bad in ((PAGE - 8, 0, 1, 9, 2, 64), (PAGE + 4, 0, 1, 9, 2, 64), (PAGE, 0, 0, 9, 2, 64), (PAGE, 0, 1, 9, 0, 64), (PAGE, 0, 1, 9, 2, 60), (PAGE, 0, 1, 9, 2, 264),
                (PAGE, PAGE, 2, 9, 2, 64), (PAGE, 8 * PAGE, 2, 9, 2, 64), (2 * PAGE - 8, PAGE, 2, 9, 2, 64), (2 * PAGE, PAGE + 4, 2, 9, 2, 64)):
        _refused("the pool needs", call, **{**ok, "pool": pkg.PagePool(AT, *bad)})
    for good in ((PAGE, 9 * PAGE, 2, 9, 2, 64), (2 * PAGE, PAGE, 2, 9, 2, 64)):
        _no_device(call, **{**ok, "pool": pkg.PagePool(AT, *good)})
    size = pkg.pages_workspace(9)
    ok = dict(pool=pool, table=AT, lengths=AT, n=3, max_blocks=5, new_table=AT, used=AT, workspace=AT, workspace_bytes=size)
    call = pkg.pages_compact
    _no_device(call, **ok)
    _refused("they may be one", call, **{**ok, "new_table": AT + 4})
    _refused("bytes of workspace", call, **{**ok, "workspace_bytes": 0})
    _refused("table entries", call, **{**ok, "n": -1})


def test_forked_tables_follow_their_rules():
    """On random tables: no page in which a sequence goes on is named by another; every position that is kept is where it was or copied."""
    rng = np.random.default_rng(3)
    for _ in range(60):
        pages, n, blocks, m = 60, int(rng.integers(1, 6)), 6, int(rng.integers(1, 9))
        lengths = rng.integers(0, 200, n)
        table = np.full((n, blocks), -1)
        free = rng.permutation(pages).tolist()
        for s in range(n):
            table[s, : -(-lengths[s] // 64)] = [free.pop() for _ in range(-(-lengths[s] // 64))]
        data = {}
        for s in range(n):
            for j in range(lengths[s]):
                data[int(table[s, j // 64]), j % 64] = (s, j)
        for _ in range(3):  # step after step
            parents = rng.integers(-1, n, m)
            keep = np.array([rng.integers(0, lengths[p] + 1) if p >= 0 and rng.random() < 0.4 else lengths[p] if p >= 0 else 0 for p in parents])
            need = keep + rng.integers(0, 3, m)
            new, missing, copies = S.fork(table, lengths, parents, keep, need, pages)
            if missing.any():
                break
            want = [[data[int(table[p, j // 64]), j % 64] for j in range(k)] for p, k in zip(parents, keep)]
            held = {int(p) for s in range(n) for p in table[s, : -(-lengths[s] // 64)]}
            assert not held & {b for _, b, _ in copies}
            for a, b, k in copies:
                for j in range(k):
                    data[b, j] = data[a, j]
            for i in range(m):
                for j in range(keep[i], need[i]):
                    data[int(new[i, j // 64]), j % 64] = ("new", i, j)
            for i in range(m):
                assert [data[int(new[i, j // 64]), j % 64] for j in range(keep[i])] == want[i]
                assert [data[int(new[i, j // 64]), j % 64] for j in range(keep[i], need[i])] == [("new", i, j) for j in range(keep[i], need[i])]
            table, lengths, n, m = new, need, len(parents), int(rng.integers(1, 9))

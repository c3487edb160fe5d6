"""The operators of a serving step over shared pages (shahd_pages_*, shahd_norm_rope_apply, shahd_chunk_attention,
shahd_adjust_logits) against plain restatements of their definitions, over sizes, layouts, masks and tables where they can go wrong."""
import math

import numpy as np
import pytest

from tests.helpers import pkg

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
from tests import serving_refs as R  # noqa: E402
from tests import step_refs as S  # noqa: E402
from tests.test_gpu_serving_ops import BF16, CODE, F16, F32, _cache_of, _gen, _held, _ints, _normal, _offsets, _rows, _stream, _within  # noqa: E402


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    torch.cuda.synchronize()
    assert pkg.load().ShahdDeviceErrorFlag() == 0


# ---- pages ---------------------------------------------------------------------------------------------------------


def _pool(pages, layers, kv, d, g, layer_major=False):
    shape = (layers, pages, kv, 2, 64, d) if layer_major else (pages, layers, kv, 2, 64, d)
    pool = torch.randint(-30000, 30000, shape, generator=g, device="cuda", dtype=torch.int16)
    view = pool.transpose(0, 1) if layer_major else pool
    return view, pkg.PagePool(pool.data_ptr(), view.stride(0), view.stride(1), layers, pages, kv, d)


def _fork(pool, table, lengths, parents, keep, need, stream=None):
    new_n, (n, blocks) = len(parents), table.shape
    new, missing = torch.full((max(new_n, 1), blocks), 77, dtype=torch.int32, device="cuda"), torch.full((max(new_n, 1),), 77, dtype=torch.int32, device="cuda")
    size = pkg.pages_workspace(pool.pages, new_n)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    t = [_ints(x) for x in (lengths, parents, keep, need)]
    dev = torch.as_tensor(table, dtype=torch.int32).cuda()
    pkg.pages_fork(pool, dev.data_ptr(), t[0].data_ptr(), n, blocks, t[1].data_ptr(), t[2].data_ptr(), t[3].data_ptr(), new_n, new.data_ptr(), missing.data_ptr(),
                   ws.data_ptr(), size, _stream())
    torch.cuda.synchronize()
    return new[:new_n], missing[:new_n]


def _check_fork(view, pool, table, lengths, parents, keep, need):
    before = view.clone()
    new, missing = _fork(pool, table, lengths, parents, keep, need)
    want, lost, copies = S.fork(np.asarray(table), lengths, parents, keep, need, pool.pages)
    assert np.array_equal(new.cpu().numpy(), want) and np.array_equal(missing.cpu().numpy(), lost)
    for a, b, k in copies:
        before[b, ..., :k, :] = before[a, ..., :k, :]
    assert torch.equal(view, before)
    return want, copies


def _tables(rng, n, blocks, pages, lengths, common=0):
    """Tables whose sequences share their first `common` blocks."""
    ids = rng.permutation(pages).tolist()
    table = np.full((n, blocks), -1, np.int64)
    shared = [ids.pop() for _ in range(common)]
    for s in range(n):
        k = -(-lengths[s] // 64)
        own = max(k - common, 0)
        table[s, :k] = (shared + [ids.pop() for _ in range(own)])[:k]
    return table


@pytest.mark.parametrize("seed", range(12))
def test_fork(seed):
    rng, g = np.random.default_rng(seed), _gen(seed)
    n, new_n, blocks = int(rng.integers(1, 12)), int(rng.integers(1, 40)), int(rng.integers(2, 9))
    lengths = [int(rng.integers(0, (blocks - 1) * 64 + 1)) for _ in range(n)]
    common = int(rng.integers(0, 3))
    view, pool = _pool(n * blocks + int(rng.integers(0, 60)), int(rng.integers(1, 4)), *[(2, 64), (1, 8), (3, 40), (4, 128)][seed % 4], g, seed % 2 == 1)
    table = _tables(rng, n, blocks, pool.pages, lengths, common)
    parents = [int(rng.integers(-1, n + 1)) for _ in range(new_n)]
    keep = [int(rng.integers(-3, 64 * blocks)) if rng.random() < 0.5 else lengths[p] if 0 <= p < n else 9 for p in parents]
    need = [max(k, 0) + int(rng.choice([0, 0, 1, 70])) for k in keep]
    _check_fork(view, pool, table, lengths, parents, keep, need)


def test_fork_who_keeps_a_partly_filled_page():
    g = _gen(1)
    view, pool = _pool(20, 2, 2, 64, g)
    table = np.full((2, 4), -1, np.int64)
    table[0, :3], table[1, :2] = [11, 4, 7], [11, 9]
    lengths = [150, 100]
    # all that name page 7 go on in it: the first keeps it
    want, copies = _check_fork(view, pool, table, lengths, [0, 0, 0], [150, 140, 129], [151, 141, 200])
    assert want[0, 2] == 7 and [c[:2] for c in copies] == [(7, 0), (7, 1)]
    # one of them only reads it: nobody may write there
    _, copies = _check_fork(view, pool, table, lengths, [0, 0, 0], [150, 150, 129], [151, 150, 200])
    assert [c[0] for c in copies] == [7, 7]
    # page 4 is full for one and partly filled for the other
    want, copies = _check_fork(view, pool, table, lengths, [0, 0], [150, 100], [151, 101])
    assert want[0, 2] == 7 and copies == [(4, 0, 36)]
    # a single one that is cut back
    want, copies = _check_fork(view, pool, table, lengths, [1], [70], [400])
    assert copies == [] and want[0].tolist() == [11, 9, 0, 1]
    # whole pages, nothing partly filled
    _, copies = _check_fork(view, pool, table, lengths, [0, 0], [128, 64], [192, 65])
    assert copies == []


def test_fork_when_pages_run_out_and_tables_name_none():
    g = _gen(2)
    view, pool = _pool(6, 1, 1, 32, g)
    table = np.array([[3, -1, 5, 900], [2, 2, -7, 2**31 - 1]])
    lengths = [256, 256]
    want, copies = _check_fork(view, pool, table, lengths, [0, 1, 5, -1], [190, 256, 3, 0], [256, 256, 100, 1])
    assert want[0].tolist()[:3] == [3, -1, 5]
    for lengths in ([10**9, -5], [0, 0], [2**31 - 1, 2**31 - 1]):
        _check_fork(view, pool, table, lengths, [0, 0, 1, 1, 0], [100, 100, 70, 300, 1], [2**31 - 1, 101, 257, 10**6, 64])


@pytest.mark.parametrize("n,new_n,blocks,pages,layers", [(1500, 2100, 9, 12000, 1), (3, 1, 300, 70000, 1), (40, 300, 30, 2000, 6)], ids=str)
def test_fork_large(n, new_n, blocks, pages, layers):
    rng, g = np.random.default_rng(n), _gen(n)
    view, pool = _pool(pages, layers, 1, 8, g)
    lengths = [int(x) for x in rng.integers(0, min(64 * blocks, 64 * pages // (2 * n)), n)]
    table = _tables(rng, n, blocks, pages, lengths)
    parents = rng.integers(0, n, new_n).tolist()
    keep = [lengths[p] for p in parents]
    _check_fork(view, pool, table, lengths, parents, keep, [k + 1 for k in keep])


@pytest.mark.parametrize("pages", [32767, 32768, 32769])
def test_fork_and_compact_around_the_sizes_that_one_kernel_sees_to(pages):
    """Tables of 32768 entries over as many pages, one less and one more."""
    rng, g = np.random.default_rng(pages), _gen(17)
    n, blocks = 64, 512
    lengths = [int(rng.integers(0, blocks * 64 + 1)) for _ in range(n)]
    view, pool = _pool(pages, 1, 1, 8, g)
    table = rng.permutation(pages)[: (pages // 64) * 64].reshape(64, -1)
    table = np.concatenate([table, np.full((n, blocks - table.shape[1]), -1)], 1) if table.shape[1] < blocks else table
    parents, keep = rng.integers(0, n, n), rng.integers(0, blocks * 64 + 1, n)
    _check_fork(view, pool, table, lengths, parents.tolist(), keep.tolist(), (keep + rng.integers(0, 300, n)).tolist())
    _compact(view, pool, table, lengths)


def test_fork_from_no_sequences_and_to_none():
    g = _gen(3)
    view, pool = _pool(5, 1, 1, 64, g)
    new, missing = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    size = pkg.pages_workspace(5, 2)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    p, k, m = _ints([0, -1]), _ints([5, 0]), _ints([65, 64])
    pkg.pages_fork(pool, 0, 0, 0, 3, p.data_ptr(), k.data_ptr(), m.data_ptr(), 2, new.data_ptr(), missing.data_ptr(), ws.data_ptr(), size, _stream())
    assert new.tolist() == [[0, 1, -1], [2, -1, -1]] and missing.tolist() == [0, 0]
    pkg.pages_fork(pool, 0, 0, 0, 3, 0, 0, 0, 0, 0, 0, ws.data_ptr(), size, _stream())


def _compact(view, pool, table, lengths, in_place=False):
    before = view.clone()
    n, blocks = table.shape
    dev, ln = torch.as_tensor(table, dtype=torch.int32).cuda(), _ints(lengths)
    new, used = dev if in_place else torch.full_like(dev, 77), _ints([77])
    size = pkg.pages_workspace(pool.pages)
    ws = torch.full((size,), 255, dtype=torch.uint8, device="cuda")
    pkg.pages_compact(pool, dev.data_ptr(), ln.data_ptr(), n, blocks, new.data_ptr(), used.data_ptr(), ws.data_ptr(), size, _stream())
    want, held, moves = S.compact(np.asarray(table), lengths, pool.pages)
    assert used.item() == held and np.array_equal(new.cpu().numpy(), want)
    after = before.clone()
    for a, b in moves:
        after[b] = before[a]
    assert torch.equal(view, after)
    return want


@pytest.mark.parametrize("seed", range(10))
def test_compact(seed):
    rng, g = np.random.default_rng(100 + seed), _gen(seed)
    n, blocks = int(rng.integers(1, 30)), int(rng.integers(1, 9))
    lengths = [int(rng.integers(0, blocks * 64 + 1)) for _ in range(n)]
    view, pool = _pool(n * blocks + int(rng.integers(0, 200)), int(rng.integers(1, 4)), *[(2, 64), (1, 8), (3, 40), (4, 128)][seed % 4], g, seed % 2 == 1)
    table = _tables(rng, n, blocks, pool.pages, lengths, int(rng.integers(0, 3)))
    if seed == 3:
        table[0, 0], table[-1, -1] = 10**6, -9
    new = _compact(view, pool, table, lengths, in_place=seed % 3 == 0)
    assert np.array_equal(_compact(view, pool, new, lengths), new)  # what lies together stays


def test_compact_edges():
    g = _gen(5)
    view, pool = _pool(65, 1, 1, 64, g)
    _compact(view, pool, np.array([[64]]), [64])                       # the last page to the first place
    _compact(view, pool, np.array([[64, 0]]), [0])                     # nothing held
    _compact(view, pool, np.arange(65)[None, ::-1].copy(), [65 * 64])  # all held
    _compact(view, pool, np.array([[33, 33, 33], [33, 5, 64]]), [192, 192])
    big, pool = _pool(70001, 1, 1, 8, g)
    ids = np.random.default_rng(1).permutation(70001)[:40000].reshape(100, 400)
    _compact(big, pool, ids, [400 * 64 - 5] * 100)


def test_fork_and_compact_beyond_32_bits():
    """Pages whose bytes lie beyond 2^32 in the pool."""
    pages, layers, kv, d = 2100, 8, 8, 128
    pool_t = torch.zeros(pages, layers, kv, 2, 64, d, dtype=torch.int16, device="cuda")  # 4.4 GB
    pool = pkg.PagePool(pool_t.data_ptr(), pool_t.stride(0), pool_t.stride(1), layers, pages, kv, d)
    table = np.array([[2099, 2098]])
    pool_t[2098] = torch.randint(1, 99, pool_t[0].shape, device="cuda", dtype=torch.int16)
    pool_t[2099] = 5
    new, missing = _fork(pool, table, [100], [0, 0], [100, 100], [101, 101])
    assert new.tolist() == [[2099, 2098], [2099, 0]] and torch.equal(pool_t[0, :, :, :, :36], pool_t[2098, :, :, :, :36])
    assert int(pool_t[0, :, :, :, 36:].abs().max()) == 0
    dev, used = torch.tensor([[2099, 2098]], dtype=torch.int32, device="cuda"), _ints([0])
    size = pkg.pages_workspace(pages)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    ln = _ints([100])
    pkg.pages_compact(pool, dev.data_ptr(), ln.data_ptr(), 1, 2, dev.data_ptr(), used.data_ptr(), ws.data_ptr(), size, _stream())
    assert dev.tolist() == [[1, 0]] and used.item() == 2 and torch.equal(pool_t[0], pool_t[2098]) and torch.equal(pool_t[1], pool_t[2099])


# ---- norms of heads ------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("heads,kv,d,r", [(4, 4, 64, 64), (16, 4, 128, 64), (3, 1, 128, 128), (2, 2, 32, 32), (5, 1, 80, 24), (2, 1, 6, 2), (1, 1, 256, 256),
                                          (33, 9, 64, 6), (4, 2, 128, 54), (7, 2, 8, 2), (3, 1, 16, 16), (2, 1, 250, 250)])
def test_norm_rope(dtype, kind, layout, heads, kv, d, r):
    g, N = _gen(1), 45
    cdt = BF16 if dtype == F32 else dtype
    pool, table, cache = _cache_of([N], kv, d, cdt, g) if d % 8 == 0 else (None, None, None)
    q, k, v = (3 * _normal(g, N, h, d) + 0.5 for h in (heads, kv, kv))
    q[3], k[4] = 0.0, 1e-4 * k[4]  # heads that eps decides
    q, k, v = (x.to(dtype) for x in (q, k, v))
    w = [(1 + 0.3 * _normal(g, d)) for _ in range(2)] + [0.2 * _normal(g, d) for _ in range(2)]
    wt = [F32, BF16, F16][(heads + d) % 3]
    w = [x.to(wt) for x in w]
    pos = torch.randperm(N, generator=g, device="cuda").int()
    pos[2] = -1
    norm = pkg.HeadNorm(kind, 1e-5, w[0].data_ptr(), w[1].data_ptr(), *([w[2].data_ptr(), w[3].data_ptr()] if kind == "layer" else []), weight_dtype=CODE[wt])
    q_out, k_out = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    off = _ints([0, N])
    more = dict(v=_rows(v), cache=cache, offsets=off.data_ptr(), n=1) if cache else {}
    with pkg.Rope(d, r, layout, magnitude=1.25) as rope:
        rope.apply(CODE[dtype], N, pos.data_ptr(), q=_rows(q), q_out=_rows(q_out), num_heads=heads, k=_rows(k), k_out=_rows(k_out), kv_heads=kv, norm=norm,
                   stream=_stream(), **more)
    keep = pos >= 0
    freq = R.frequencies(r)
    for x, y, i in ((q, q_out, 0), (k, k_out, 1)):
        want, bound = S.norm_rope(x, pos, freq, layout, 1.25, kind, 1e-5, w[i], w[2 + i] if kind == "layer" else None, dtype)
        _within(y[keep], want[keep], bound[keep])
        assert bool((y[2] == 7.0).all())
        if i == 1 and cache:
            want, bound = S.norm_rope(x, pos, freq, layout, 1.25, kind, 1e-5, w[1], w[3] if kind == "layer" else None, cdt)
            for h in range(kv):
                held_k, held_v = _held(pool, table, 0, N, h)
                at = pos[keep].long()
                _within(held_k[at], want[keep][:, h], bound[keep][:, h])
                assert torch.equal(held_v[at], v[keep][:, h].to(cdt))


@pytest.mark.parametrize("shift", [0, 1])
@pytest.mark.parametrize("layout,r", [("interleaved", 64), ("half", 64), ("half", 26)])
def test_norm_rope_in_place_strided_unaligned_and_without_weights(shift, layout, r):
    """A fused [N, H + 2 Hk, d] buffer in place, aligned and one element off; no weights; more rows than warps run at once."""
    g, N, H, Hk, d = _gen(3), 5000, 6, 2, 64
    flat = _normal(g, N * (H + 2 * Hk) * d + 8, dtype=BF16)
    qkv = flat[shift:shift + N * (H + 2 * Hk) * d].view(N, H + 2 * Hk, d)
    before, old = flat.clone(), qkv.clone()
    pos = torch.arange(N, dtype=torch.int32, device="cuda")
    q, k = _rows(qkv[:, :H]), _rows(qkv[:, H:H + Hk])
    with pkg.Rope(d, r, layout) as rope:
        rope.apply(pkg.BF16, N, pos.data_ptr(), q=q, q_out=q, num_heads=H, k=k, k_out=k, kv_heads=Hk, stream=_stream(), norm=pkg.HeadNorm("rms", 1e-6))
    want, bound = S.norm_rope(old[:, :H + Hk], pos, R.frequencies(r), layout, 1.0, "rms", 1e-6, None, None, BF16)
    _within(qkv[:, :H + Hk], want, bound)
    assert torch.equal(qkv[:, H + Hk:], old[:, H + Hk:]) and torch.equal(flat[:shift], before[:shift])
    assert torch.equal(flat[shift + qkv.numel():], before[shift + qkv.numel():])


def test_norm_rope_of_one_operand_and_values_that_are_not_finite():
    g = _gen(4)
    k = _normal(g, 9, 3, 64)
    k[1, 0, 5], k[2, 1, 60], k[3, 2, 0] = math.nan, math.inf, 1e30
    out = torch.full_like(k, 7.0)
    w = _normal(g, 64)
    pos, off = torch.arange(9, dtype=torch.int32, device="cuda"), _ints([1, 8])
    with pkg.Rope(64, 64, "half") as rope:
        rope.apply(pkg.F32, 9, pos.data_ptr(), k=_rows(k), k_out=_rows(out), kv_heads=3, offsets=off.data_ptr(), n=1, norm=pkg.HeadNorm("rms", 1e-6, k_weight=w.data_ptr()),
                   stream=_stream())
    want, bound = S.norm_rope(k, pos, R.frequencies(64), "half", 1.0, "rms", 1e-6, w, None, F32)
    fine = torch.ones(9, 3, dtype=torch.bool, device="cuda")
    fine[1, 0] = fine[2, 1] = fine[3, 2] = False
    fine[0] = fine[8] = False
    _within(out[fine], want[fine], bound[fine])
    assert bool((out[0] == 7.0).all()) and bool((out[8] == 7.0).all()) and bool(out[1, 0].isnan().all())


# ---- logits --------------------------------------------------------------------------------------------------------


def _bits(allowed):
    """[m, V] truth values as words."""
    m, V = allowed.shape
    full = np.zeros((m, -(-V // 32) * 32), np.uint8)
    full[:, :V] = allowed
    return torch.tensor(np.packbits(full, axis=1, bitorder="little").view(np.int32), device="cuda")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("V,rows,n,held,shift,stride", [(1, 1, 1, 1, 0, 0), (7, 5, 2, 9, 1, 0), (33, 4, 4, 0, 0, 3), (4096, 3, 2, 500, 0, 0), (8191, 2, 1, 3000, 3, 0),
                                                        (8193, 2, 2, 10, 0, 7), (50257, 6, 3, 9000, 0, 0), (40000, 300, 7, 100, 0, 8)], ids=str)
@pytest.mark.parametrize("what", ["all", "penalties", "biases", "masks", "in place"])
def test_adjust_logits(dtype, V, rows, n, held, shift, stride, what):
    rng, g = np.random.default_rng(V + rows), _gen(V)
    wide = V + stride
    flat = (4 * _normal(g, rows * wide + 8)).to(dtype)
    logits = flat[shift:shift + rows * wide].view(rows, wide)
    logits[0, V // 2] = -math.inf
    outs = flat if what == "in place" else torch.full_like(flat, 7.0)
    place = shift if what != "penalties" else 2  # results that begin elsewhere in a 16-byte piece
    out = outs[place:place + rows * wide].view(rows, wide)
    source, behind = logits.clone(), out.clone()
    history = rng.integers(-2, V + 2, (n, max(held, 1)))
    history[:, ::3] = rng.integers(0, max(V // 50, 1), history[:, ::3].shape)
    lens, prompt = rng.integers(0, held + 1, n), rng.integers(-1, held + 2, n)
    lens[0] = held
    if n > 1:
        lens[1] = [10**9, -3][rows % 2]
    rep, pres, freq = (torch.tensor(rng.uniform(a, b, n), dtype=F32, device="cuda") for a, b in ((0.7, 1.5), (-1, 1), (-0.5, 0.5)))
    seqs = rng.integers(0, n, rows)
    if rows > 2:
        seqs[1], seqs[2] = -1, n
    counts = rng.integers(0, 6, n)
    bo = np.concatenate([[0], np.cumsum(counts)])
    bt, bv = rng.integers(-1, V + 1, max(bo[-1], 1)), rng.uniform(-9, 9, max(bo[-1], 1)).astype(np.float32)
    bt[1::2] = bt[::2][: len(bt[1::2])]  # tokens that are there twice
    allowed = rng.random((3, V)) < 0.5
    mrow = rng.integers(-1, 4, rows)
    dev = dict(history=_ints(history.ravel()), lens=_ints(lens), prompt=_ints(prompt), seqs=_ints(seqs), bo=_ints(bo), bt=_ints(bt), bv=torch.tensor(bv, device="cuda"),
               masks=_bits(allowed), mrow=_ints(mrow))
    more = {}
    everything = what in ("all", "in place")
    if everything or what == "penalties":
        more.update(history=dev["history"].data_ptr(), history_stride=history.shape[1] if held else 0, history_lengths=dev["lens"].data_ptr(),
                    prompt_lengths=dev["prompt"].data_ptr(), repetition=rep.data_ptr(), presence=pres.data_ptr(), frequency=freq.data_ptr())
    if everything or what == "biases":
        more.update(bias_offsets=dev["bo"].data_ptr(), bias_tokens=dev["bt"].data_ptr(), bias_values=dev["bv"].data_ptr(), bias_entries=int(bo[-1]))
    if everything or what == "masks":
        more.update(masks=dev["masks"].data_ptr(), mask_rows=dev["mrow"].data_ptr(), mask_count=3)
    pkg.adjust_logits(CODE[dtype], logits.data_ptr(), out.data_ptr(), rows, V, n, sequences=dev["seqs"].data_ptr(), logits_stride=wide, out_stride=wide, stream=_stream(),
                      **more)
    torch.cuda.synchronize()
    for i in list(range(min(rows, 6))) + [rows - 1]:
        s = int(seqs[i])
        if not 0 <= s < n:
            assert torch.equal(out[i].nan_to_num(), behind[i].nan_to_num())
            continue
        h = history[s, : min(max(lens[s], 0), held)].tolist() if "history" in more else []
        want, bound = S.adjust(source[i, :V].double(), h, int(prompt[s]), rep[s].double(), pres[s].double(), freq[s].double(),
                               list(zip(bt[bo[s]:bo[s + 1]].tolist(), bv[bo[s]:bo[s + 1]].tolist())) if "bias_tokens" in more else [],
                               torch.tensor(allowed[mrow[i]], device="cuda") if "masks" in more and 0 <= mrow[i] < 3 else None, dtype)
        gone = want == -math.inf
        assert torch.equal(out[i, :V] == -math.inf, gone)
        _within(out[i, :V][~gone], want[~gone], bound[~gone])
        assert torch.equal(out[i, V:], behind[i, V:])
    assert torch.equal(outs[:place], torch.full_like(outs[:place], 7.0) if what != "in place" else outs[:place])


def test_adjust_logits_plain_rows_and_counts():
    """Without a history, biases and masks a row passes as it is; many repetitions of few tokens count as many."""
    g = _gen(6)
    x = _normal(g, 3, 700, dtype=BF16)
    x[0, 3], x[1, 4] = math.nan, math.inf
    out = torch.zeros_like(x)
    pkg.adjust_logits(pkg.BF16, x.data_ptr(), out.data_ptr(), 3, 700, 3, stream=_stream())
    assert torch.equal(out.nan_to_num(5.0), x.nan_to_num(5.0))
    x = torch.zeros(1, 700, device="cuda")
    history = _ints([5] * 70000 + [6] * 30000)
    held, freq = _ints([100000]), torch.ones(1, device="cuda")
    pkg.adjust_logits(pkg.F32, x.data_ptr(), x.data_ptr(), 1, 700, 1, history=history.data_ptr(), history_stride=100000, history_lengths=held.data_ptr(),
                      frequency=freq.data_ptr(), stream=_stream())
    assert x[0, 5] == -70000 and x[0, 6] == -30000 and int((x != 0).sum()) == 2


# ---- chunks over the cache -----------------------------------------------------------------------------------------

HEADS = [(4, 4, 32), (4, 4, 64), (16, 4, 64), (8, 1, 64), (12, 4, 64), (10, 2, 32), (4, 2, 128), (7, 1, 128), (6, 1, 64), (1, 1, 128)]


def _chunk(q, cache, lengths, rows, dtype, max_rows=None, scale=0.0, out=None):
    out = torch.full(q.shape, 7.0, dtype=dtype, device="cuda") if out is None else out
    top = max(max(rows), 1) if max_rows is None else max_rows
    N, H = q.shape[:2]
    size = pkg.chunk_attention_workspace(len(rows), N, top, H, cache)
    ws = torch.full((max(size, 16),), 255, dtype=torch.uint8, device="cuda")
    off, ln = _ints(_offsets(rows)), _ints(lengths)
    pkg.chunk_attention(CODE[dtype], _rows(q), _rows(out), cache, ln.data_ptr(), off.data_ptr(), len(rows), N, top, H, scale, ws.data_ptr(), size, _stream())
    torch.cuda.synchronize()
    return out


def _check_chunk(q, pool, table, lengths, rows, out, dtype, scale=0.0, seqs=None, most=None):
    """most: positions that the table has place for. Entries that name no page hold nothing."""
    off, (pages, _, Hk), most = _offsets(rows), pool.shape[:3], most or 1 << 30
    for s, t in enumerate(rows):
        if t == 0 or (seqs is not None and s not in seqs):
            continue
        b, L = off[s], min(max(lengths[s], 0), most)
        total = min(L + t, most)
        held = torch.stack([_held(pool, table.clamp(0, pages - 1), s, total, h) for h in range(Hk)], 2)  # [2, total, Hk, d]
        at = torch.arange(total, device="cuda")
        name = table[s, at // 64]
        there = (name >= 0) & (name < pages)
        kk, vv = (torch.where(there[:, None, None], x, 0.0) for x in held)
        for c in range(0, t, 1024):
            e = min(c + 1024, t)
            seen = there & (at <= L + torch.arange(c, e, device="cuda")[:, None])
            want, bound = R.attend(q[b + c:b + e], kk, vv, seen, scale or q.shape[2] ** -0.5, dtype)
            _within(out[b + c:b + e], want, bound)


def _chunk_case(g, lengths, rows, heads, dtype, behind=2, spread=2):
    H, Hk, d = heads
    q = _normal(g, sum(rows) + behind, H, d, dtype=dtype)
    total = [max(a, 0) + b for a, b in zip(lengths, rows)]
    pool, table, cache = _cache_of(total, Hk, d, dtype, g, spread=spread, fill=math.nan)
    for s, n in enumerate(total):  # what lies behind a sequence, in its last page too, is never used
        for b in range(-(-n // 64)):
            k = min(64, n - 64 * b)
            pool[table[s, b], -1, :, :, :k] = torch.randn(Hk, 2, k, d, generator=g, device="cuda").to(dtype)
    return q, pool, table, cache


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("lengths,rows", [
    ([0, 1, 63, 64, 65, 127, 128, 129], [1, 1, 1, 1, 1, 1, 1, 1]),
    ([0, 0, 700, 5, 130], [3, 1, 17, 0, 64]),
    ([1500], [300]), ([0], [1]), ([0], [700]), ([4000], [1]), ([63], [129]), ([100, 900, 0, 64], [1, 260, 513, 1]), ([2000, 3], [33, 65]),
], ids=str)
def test_chunk_attention(dtype, heads, lengths, rows):
    q, pool, table, cache = _chunk_case(_gen(11), lengths, rows, heads, dtype)
    out = _chunk(q, cache, lengths, rows, dtype)
    _check_chunk(q, pool, table, lengths, rows, out, dtype)
    assert bool((out[sum(rows):] == 7.0).all())


@pytest.mark.parametrize("n,heads,most_rows,most", [(90, (8, 4, 128), 5, 700), (330, (4, 1, 64), 3, 500), (40, (6, 2, 32), 300, 900), (6, (32, 8, 128), 200, 6000),
                                                    (1300, (2, 1, 64), 2, 300), (5, (16, 2, 64), 700, 9000), (700, (4, 2, 64), 40, 100)], ids=str)
def test_chunk_attention_many_sequences(n, heads, most_rows, most):
    """Ranges cut across pairs, heads and sequences, empty ones among them, more sequences than threads; repeated bit for bit."""
    rng = np.random.default_rng(n)
    lengths, rows = rng.integers(0, most, n).tolist(), rng.integers(0, most_rows + 1, n).tolist()
    rows[0], rows[-1] = 0, most_rows
    q, pool, table, cache = _chunk_case(_gen(n), lengths, rows, heads, BF16, spread=1)
    out = _chunk(q, cache, lengths, rows, BF16)
    _check_chunk(q, pool, table, lengths, rows, out, BF16, seqs=set(rng.integers(0, n, 25).tolist()) | {n - 1})
    assert bool((out[sum(rows):] == 7.0).all())
    assert torch.equal(out, _chunk(q, cache, lengths, rows, BF16))
    # the layout of the work may be another where longer chunks are allowed for
    _check_chunk(q, pool, table, lengths, rows, _chunk(q, cache, lengths, rows, BF16, max_rows=5000), BF16, seqs=set(rng.integers(0, n, 9).tolist()))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("lengths,rows", [
    ([0, 1, 63, 64, 65, 127, 128, 129], [1, 1, 1, 1, 1, 1, 1, 1]), ([0, 0, 700, 5, 130], [3, 1, 17, 0, 64]), ([100, 900, 0, 64], [1, 260, 513, 1]),
    ([0], [1]), ([0, 300, 0], [0, 2, 0]), ([5000], [3]), ([3000, 17, 2000], [1, 1, 130]),
], ids=str)
def test_chunk_attention_short_lengths_in_a_long_table(dtype, heads, lengths, rows):
    """Room for 2000 pages a sequence: the work goes in ranges, which cut pairs where they like."""
    q, pool, table, cache = _chunk_case(_gen(17), lengths, rows, heads, dtype)
    wide = torch.cat([table, torch.full((len(rows), 2000 - table.shape[1]), 2**31 - 1, dtype=torch.int32, device="cuda")], 1)
    cache = pkg.KvCache(cache.pool, cache.page_stride, wide.data_ptr(), 2000, cache.pages, heads[1], heads[2])
    out = _chunk(q, cache, lengths, rows, dtype)
    _check_chunk(q, pool, table, lengths, rows, out, dtype)
    assert bool((out[sum(rows):] == 7.0).all())
    assert torch.equal(out, _chunk(q, cache, lengths, rows, dtype))


@pytest.mark.parametrize("heads", [(4, 4, 64), (10, 2, 32), (16, 4, 128), (7, 1, 128), (6, 2, 64)], ids=str)
@pytest.mark.parametrize("blocks", [None, 2000])
def test_chunk_attention_ranges_over_many_pairs(heads, blocks):
    """Rows that make several pairs a sequence, of which the last has one tile or two: whole tables and wide ones."""
    rng = np.random.default_rng(heads[0])
    rows = [1, 700, 33, 0, 512, 2, 190, 65, 1, 1, 300]
    lengths = rng.integers(0, 2500, len(rows)).tolist()
    q, pool, table, cache = _chunk_case(_gen(18), lengths, rows, heads, BF16, spread=1)
    if blocks:
        table = torch.cat([table, torch.full((len(rows), blocks - table.shape[1]), -1, dtype=torch.int32, device="cuda")], 1)
        cache = pkg.KvCache(cache.pool, cache.page_stride, table.data_ptr(), blocks, cache.pages, heads[1], heads[2])
    _check_chunk(q, pool, table, lengths, rows, _chunk(q, cache, lengths, rows, BF16), BF16)


@pytest.mark.parametrize("heads", [(4, 4, 64), (16, 4, 128), (10, 2, 32)], ids=str)
def test_chunk_attention_pages_that_are_not_there(heads):
    g, lengths, rows = _gen(21), [300, 0, 64, 500], [70, 40, 1, 200]
    q, pool, table, cache = _chunk_case(g, lengths, rows, heads, F16)
    table[0, 1], table[0, 4] = -1, pool.shape[0]     # holes
    table[1, 0] = 2**31 - 1                          # nothing at all: rows of 0
    table[2, 0] = -5                                 # its only page but the row's own
    table[3, :4] = -1
    out = _chunk(q, cache, lengths, rows, F16)
    _check_chunk(q, pool, table, lengths, rows, out, F16)
    assert bool((out[70:110] == 0).all())


@pytest.mark.parametrize("heads", [(4, 2, 64), (2, 2, 128)], ids=str)
def test_chunk_attention_lengths_past_the_table_and_rows_past_the_most(heads):
    g, H, Hk, d = _gen(22), *heads
    blocks, rows, lengths = 5, [200, 9, 150, 3], [200, 10**9, -7, 2**31 - 1]
    pool = _normal(g, 22, 1, Hk, 2, 64, d, dtype=BF16)
    table = torch.randperm(20, generator=g, device="cuda").int().view(4, 5)
    cache = pkg.KvCache(pool.data_ptr(), pool.stride(0), table.data_ptr(), blocks, 22, Hk, d)
    q = _normal(g, sum(rows), H, d, dtype=BF16)
    out = _chunk(q, cache, lengths, rows, BF16)
    _check_chunk(q, pool, table, lengths, rows, out, BF16, most=320)
    short = _chunk(q, cache, lengths, rows, BF16, max_rows=100)
    keep = torch.cat([torch.arange(t, device="cuda") < 100 for t in rows])
    assert bool((short[~keep] == 7.0).all())
    _check_chunk(q[keep], pool, table, lengths, [100, 9, 100, 3], short[keep], BF16, most=320)


def test_chunk_attention_strides_scale_and_growing_scores():
    g, H, Hk, d, rows, lengths = _gen(23), 6, 2, 64, [130, 1, 70], [500, 90, 0]
    _, pool, table, cache = _chunk_case(g, lengths, rows, (H, Hk, d), F16)
    wide = _normal(g, sum(rows), H + 4, d + 8, dtype=F16)
    q = wide[:, 2:2 + H, :d]
    pool[:, :, :, 0] *= 1 + torch.arange(64, device="cuda").half()[:, None] / 8  # maxima that keep moving
    buffer = torch.full((H, sum(rows), d + 16), 7.0, dtype=F16, device="cuda")  # heads outside rows
    out = buffer[:, :, :d].transpose(0, 1)
    _chunk(q, cache, lengths, rows, F16, scale=0.3, out=out)
    _check_chunk(q, pool, table, lengths, rows, out, F16, scale=0.3)
    assert bool((buffer[:, :, d:] == 7.0).all())


def test_chunk_attention_keeps_sequences_apart():
    """A sequence whose values are not finite spoils no other, nor do rows of q that belong to none."""
    g, rows, lengths = _gen(24), [40, 60, 1, 90], [100, 30, 70, 0]
    q, pool, table, cache = _chunk_case(g, lengths, rows, (4, 2, 64), BF16)
    q[sum(rows):] = math.nan
    for bad in (math.nan, math.inf, -math.inf):
        pool[table[1, :2].long()] = bad
        out = _chunk(q, cache, lengths, rows, BF16)
        _check_chunk(q, pool, table, lengths, rows, out, BF16, seqs={0, 2, 3})


def test_chunk_attention_scores_that_are_not_finite():
    """A key of -inf scores has weight 0, a row that sees no other is NaN, and so is one that sees +inf or NaN; earlier rows are not."""
    g, H, d, L, T = _gen(25), 2, 64, 100, 90
    q, pool, table, cache = _chunk_case(g, [L], [T], (H, H, d), BF16)
    q[:, :, 0] = 1.0
    place = lambda j: pool[table[0, j // 64], -1, :, 0, j % 64, 0]  # noqa: E731
    place(130).fill_(math.inf)
    place(20).fill_(-math.inf)
    out = _chunk(q, cache, [L], [T], BF16)
    assert bool(out[:T][30:].isnan().all()) and bool(out[:30].isfinite().all())
    place(130).fill_(0.0)
    kept, pool0 = table.clone(), pool.clone()
    out = _chunk(q, cache, [L], [T], BF16)
    pool0[table[0, 0], -1, :, 0, 20, 0] = -3e4  # far below all others: the same weights
    want = _chunk(q, pkg.KvCache(pool0[:, -1].data_ptr(), pool0.stride(0), kept.data_ptr(), cache.max_blocks, cache.pages, H, d), [L], [T], BF16)
    assert torch.equal(out[:T], want[:T])
    pool[:, -1, :, 0, :, 0] = -math.inf
    assert bool(_chunk(q, cache, [L], [T], BF16)[:T].isnan().all())


def test_chunk_attention_in_a_pool_beyond_32_bits():
    g, Hk, d, pages = _gen(26), 8, 128, 40000
    pool = torch.zeros(pages, 1, Hk, 2, 64, d, dtype=BF16, device="cuda")  # 10.5 GB
    table = torch.tensor([[39999, 20000, 39998, 7]], dtype=torch.int32, device="cuda")
    pool[table[0].long()] = torch.randn(4, 1, Hk, 2, 64, d, generator=g, device="cuda").to(BF16)
    cache = pkg.KvCache(pool.data_ptr(), pool.stride(0), table.data_ptr(), 4, pages, Hk, d)
    q = _normal(g, 60, 16, d, dtype=BF16)
    _check_chunk(q, pool, table, [180], [60], _chunk(q, cache, [180], [60], BF16), BF16)


def test_chunk_attention_of_one_row_is_a_decode_step():
    """The same rows through tree_attention, whose own key lies beside the cache."""
    g, n, H, Hk, d = _gen(27), 40, 8, 2, 64
    lengths = np.random.default_rng(1).integers(0, 600, n).tolist()
    q, pool, table, cache = _chunk_case(g, lengths, [1] * n, (H, Hk, d), BF16, behind=0)
    out = _chunk(q, cache, lengths, [1] * n, BF16)
    own = [torch.stack([pool[table[s, x // 64], -1, :, i, x % 64] for s, x in enumerate(lengths)]) for i in (0, 1)]
    other = torch.empty_like(out)
    off, ln, masks = _ints(range(n + 1)), _ints(lengths), torch.ones(n, dtype=torch.int64, device="cuda")
    size = pkg.tree_attention_workspace(n, 1, H, cache)
    ws = torch.empty(max(size, 32), dtype=torch.uint8, device="cuda")
    pkg.tree_attention(pkg.BF16, _rows(q), _rows(own[0]), _rows(own[1]), _rows(other), cache, ln.data_ptr(), masks.data_ptr(), off.data_ptr(), n, n, 1, H,
                       workspace=ws.data_ptr(), workspace_bytes=size, stream=_stream())
    assert float((out.float() - other.float()).abs().max()) <= 4 * 2.0 ** -8 * float(out.float().abs().max())


@pytest.mark.parametrize("blocks", [9, 3000])
def test_chunk_attention_offsets_and_lengths_that_make_no_sense(blocks):
    """Nothing outside the buffers is read or written, whatever the offsets and lengths on the device are; a later call is not harmed."""
    g, n, H, Hk, d, N = _gen(28), 40, 4, 2, 64, 300
    q = _normal(g, N, H, d, dtype=BF16)
    pool = _normal(g, 30, 1, Hk, 2, 64, d, dtype=BF16)
    table = torch.randint(-5, 35, (n, blocks), generator=g, device="cuda", dtype=torch.int32)
    cache = pkg.KvCache(pool.data_ptr(), pool.stride(0), table.data_ptr(), blocks, 30, Hk, d)
    size = pkg.chunk_attention_workspace(n, N, N, H, cache)
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    guard = torch.full((N + 64, H, d), 7.0, dtype=BF16, device="cuda")
    out = guard[32:32 + N]
    for seed in range(6):
        rng = np.random.default_rng(seed)
        off = _ints(rng.integers(-2**31, 2**31, n + 1) if seed % 3 == 0 else rng.integers(-10, N + 10, n + 1) if seed % 3 == 1 else [0, N] * (n // 2) + [0])
        ln = _ints(rng.integers(-2**31, 2**31, n) if seed % 2 else rng.integers(0, 64 * blocks, n))
        pkg.chunk_attention(pkg.BF16, _rows(q), _rows(out), cache, ln.data_ptr(), off.data_ptr(), n, N, N, H, workspace=ws.data_ptr(), workspace_bytes=size, stream=_stream())
        torch.cuda.synchronize()
        assert bool((guard[:32] == 7.0).all()) and bool((guard[32 + N:] == 7.0).all())
    off, ln = _ints([0, 100] + [100] * (n - 1)), _ints([60] * n)
    table.clamp_(0, 29)
    pkg.chunk_attention(pkg.BF16, _rows(q), _rows(out), cache, ln.data_ptr(), off.data_ptr(), n, N, N, H, workspace=ws.data_ptr(), workspace_bytes=size, stream=_stream())
    torch.cuda.synchronize()
    _check_chunk(q, pool, table, [60] * n, [100] + [0] * (n - 1), out, BF16)


def test_adjust_logits_long_histories_with_many_biases():
    """Histories and lists of biases beyond what 16-bit cells hold; a slice whose tokens are on no list, there are too many of them."""
    g, V, held = _gen(29), 5000, 40000
    rng = np.random.default_rng(29)
    history = rng.integers(0, V, (2, held))
    history[1, :30000] = 17
    bt, bv = rng.integers(-5, V + 5, 70000), rng.normal(size=70000).astype(np.float32)
    bo = [0, 60000, 70000]
    x = _normal(g, 6, V, dtype=F16)
    out, seqs = torch.empty_like(x), [0, 0, 1, 1, 1, 0]
    lens, prompt = [held, held - 7], [100, 30001]
    dev = [_ints(history.ravel()), _ints(lens), _ints(prompt), _ints(seqs), _ints(bo), _ints(bt), torch.tensor(bv, device="cuda")]
    rep, pres, freq = (torch.tensor(v, device="cuda") for v in ([1.2, 0.9], [0.3, -0.2], [0.01, 0.5]))
    pkg.adjust_logits(pkg.F16, x.data_ptr(), out.data_ptr(), 6, V, 2, sequences=dev[3].data_ptr(), history=dev[0].data_ptr(), history_stride=held,
                      history_lengths=dev[1].data_ptr(), prompt_lengths=dev[2].data_ptr(), repetition=rep.data_ptr(), presence=pres.data_ptr(), frequency=freq.data_ptr(),
                      bias_offsets=dev[4].data_ptr(), bias_tokens=dev[5].data_ptr(), bias_values=dev[6].data_ptr(), bias_entries=70000, stream=_stream())
    for i, s in enumerate(seqs):
        want, bound = S.adjust(x[i].double(), history[s, : lens[s]].tolist(), prompt[s], rep[s].double(), pres[s].double(), freq[s].double(),
                               list(zip(bt[bo[s]:bo[s + 1]].tolist(), bv[bo[s]:bo[s + 1]].tolist())), None, F16)
        _within(out[i], want, bound)
    # the same without biases, in 16-bit cells and as many tokens as a slice has
    short = _ints(np.stack([rng.permutation(V), rng.permutation(V)]).ravel())
    ln = _ints([V, V])
    pkg.adjust_logits(pkg.F16, x.data_ptr(), out.data_ptr(), 6, V, 2, sequences=dev[3].data_ptr(), history=short.data_ptr(), history_stride=V, history_lengths=ln.data_ptr(),
                      presence=pres.data_ptr(), stream=_stream())
    for i, s in enumerate(seqs):
        want, bound = S.adjust(x[i].double(), list(range(V)), 0, torch.ones((), device="cuda").double(), pres[s].double(), torch.zeros((), device="cuda").double(), [], None,
                               F16)
        _within(out[i], want, bound)


@pytest.mark.parametrize("held", [5000, 17000])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_adjust_logits_many_rows_of_a_sequence_that_has_most_tokens(held, dtype):
    """Rows that go four together, sequences that end inside such a group, histories with nearly every token, in 16-bit and 32-bit cells."""
    g, V, rows, n = _gen(31), 5000, 1200, 290
    rng = np.random.default_rng(held)
    history = np.stack([rng.permutation(held) % V for _ in range(n)])
    seqs = np.arange(rows) * n // rows
    seqs[5], seqs[6] = -1, 9
    lens, prompt = rng.integers(held - 9, held + 1, n), rng.integers(0, held, n)
    bt, bv = rng.integers(0, V, 3 * n), rng.normal(size=3 * n).astype(np.float32)
    x = _normal(g, rows, V, dtype=dtype)
    out = torch.empty_like(x)
    rep, pres, freq = (torch.tensor(rng.uniform(a, b, n), dtype=F32, device="cuda") for a, b in ((0.7, 1.5), (-1, 1), (-0.5, 0.5)))
    dev = [_ints(history.ravel()), _ints(lens), _ints(prompt), _ints(seqs), _ints(3 * np.arange(n + 1)), _ints(bt), torch.tensor(bv, device="cuda")]
    pkg.adjust_logits(CODE[dtype], x.data_ptr(), out.data_ptr(), rows, V, n, sequences=dev[3].data_ptr(), history=dev[0].data_ptr(), history_stride=held,
                      history_lengths=dev[1].data_ptr(), prompt_lengths=dev[2].data_ptr(), repetition=rep.data_ptr(), presence=pres.data_ptr(), frequency=freq.data_ptr(),
                      bias_offsets=dev[4].data_ptr(), bias_tokens=dev[5].data_ptr(), bias_values=dev[6].data_ptr(), bias_entries=3 * n, stream=_stream())
    for i in [0, 1, 2, 3, 4, 6, 7, 8, 601, 1198, 1199]:
        s = int(seqs[i])
        want, bound = S.adjust(x[i].double(), history[s, : lens[s]].tolist(), int(prompt[s]), rep[s].double(), pres[s].double(), freq[s].double(),
                               list(zip(bt[3 * s:3 * s + 3].tolist(), bv[3 * s:3 * s + 3].tolist())), None, dtype)
        _within(out[i], want, bound)


def test_adjust_logits_rows_beyond_32_bits():
    """Rows, and histories, whose places pass 2^31 elements."""
    g, V, apart = _gen(37), 1000, (1 << 31) + 40
    x, h = torch.empty(2 * apart + V, dtype=BF16, device="cuda"), torch.empty((1 << 30) - 1 + 64, dtype=torch.int32, device="cuda")
    rows = x.as_strided((3, V), (apart, 1))
    rows.copy_(_normal(g, 3, V))
    before, hold = rows.clone(), (1 << 30) - 1
    h[:64], h[hold:] = 5, 9
    held, seqs, pres = _ints([64, 64]), _ints([1, 0, 1]), torch.ones(2, device="cuda")
    pkg.adjust_logits(pkg.BF16, x.data_ptr(), x.data_ptr(), 3, V, 2, sequences=seqs.data_ptr(), history=h.data_ptr(), history_stride=hold, history_lengths=held.data_ptr(),
                      frequency=pres.data_ptr(), logits_stride=apart, out_stride=apart, stream=_stream())
    want = before.clone()
    for i, t in enumerate((9, 5, 9)):
        want[i, t] = (before[i, t].float() - 64).to(BF16)  # the same two roundings: to 32 bits, to the type
    assert torch.equal(rows, want)


def test_operators_with_nothing_to_do():
    """Sequences without rows, rows without sequences, vocabularies of one token."""
    q = torch.full((4, 2, 64), 7.0, dtype=BF16, device="cuda")
    pool, table = torch.zeros(2, 1, 2, 2, 64, 64, dtype=BF16, device="cuda"), _ints([0, 1])
    cache = pkg.KvCache(pool.data_ptr(), pool.stride(0), table.data_ptr(), 1, 2, 2, 64)
    size = pkg.chunk_attention_workspace(2, 4, 3, 2, cache)
    ws, off, ln = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda"), _ints([0, 0, 0]), _ints([5, 0])
    pkg.chunk_attention(pkg.BF16, _rows(q), _rows(q), cache, ln.data_ptr(), off.data_ptr(), 2, 4, 3, 2, workspace=ws.data_ptr(), workspace_bytes=size, stream=_stream())
    assert bool((q == 7.0).all())
    x, seqs, held = torch.ones(3, 1, device="cuda"), _ints([0, -1, 5]), _ints([3])
    history, pres = _ints([0, 0, 9]), torch.ones(1, device="cuda")
    pkg.adjust_logits(pkg.F32, x.data_ptr(), x.data_ptr(), 3, 1, 1, sequences=seqs.data_ptr(), history=history.data_ptr(), history_stride=3, history_lengths=held.data_ptr(),
                      presence=pres.data_ptr(), stream=_stream())
    assert x.tolist() == [[0.0], [1.0], [1.0]]

"""The serving operators on caller-owned buffers (shahd_rope_*, shahd_prompt_attention, shahd_tree_attention,
shahd_verify_tree) against 64-bit restatements of their definitions, over head layouts, lengths, strides, masks and page tables
where they can go wrong, and one serving step made of all of them."""
import math

import numpy as np
import pytest

from tests.helpers import pkg

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
from tests import serving_refs as R  # noqa: E402

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
CODE = {BF16: pkg.BF16, F16: pkg.F16, F32: pkg.F32}
HEADS = [(4, 4, 32), (4, 4, 64), (16, 4, 64), (8, 1, 64), (12, 4, 64), (10, 2, 32), (4, 2, 128), (7, 1, 128), (6, 1, 64), (1, 1, 128)]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _rows(t):
    return pkg.Rows(t.data_ptr(), t.stride(0), t.stride(1))


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _ints(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def _offsets(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(int)


def _within(got, want, bound):
    off = (got.double() - want).abs()
    assert bool(torch.isfinite(got.float()).all())
    worst = float((off / bound.clamp(min=1e-30)).max()) if off.numel() else 0.0
    assert worst <= 1.0, worst


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    torch.cuda.synchronize()
    assert pkg.load().ShahdDeviceErrorFlag() == 0


# ---- rotary positions ----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("heads,kv,d,r", [(4, 4, 64, 64), (16, 4, 128, 64), (3, 1, 128, 128), (2, 2, 32, 32), (5, 1, 80, 24), (2, 1, 6, 2),
                                          (1, 1, 256, 256)])
def test_rope_turns_queries_and_keys(dtype, layout, heads, kv, d, r):
    g, N = _gen(1), 37
    q, k = _normal(g, N, heads, d, dtype=dtype), _normal(g, N, kv, d, dtype=dtype)
    pos = torch.randint(0, 1 << 20, (N,), generator=g, device="cuda", dtype=torch.int32)
    pos[:3] = _ints([0, 1, -1])
    q_out, k_out = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    with pkg.Rope(d, r, layout) as rope:
        rope.apply(CODE[dtype], N, pos.data_ptr(), q=_rows(q), q_out=_rows(q_out), num_heads=heads, k=_rows(k), k_out=_rows(k_out), kv_heads=kv,
                   stream=_stream())
    freq = R.frequencies(r)
    for x, y in ((q, q_out), (k, k_out)):
        want, off = R.rotate(x, pos, freq, layout)
        keep = pos >= 0
        _within(y[keep], want[keep], off[keep] + R.HALF_STEP[dtype] * want[keep].abs() + 1e-7)
        assert bool((y[2] == 7.0).all())  # a negative position leaves its row


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("heads,kv,d,r", [(4, 2, 128, 54), (33, 9, 64, 6), (5, 5, 32, 30), (2, 1, 128, 126), (41, 3, 24, 10), (3, 1, 256, 250),
                                          (7, 2, 8, 2), (6, 2, 64, 40)])
def test_rope_rotary_parts_of_any_even_size(dtype, layout, heads, kv, d, r):
    """In place and into the cache; what lies behind the rotated part passes as it is, whatever it holds."""
    g, N = _gen(11), 67
    cdt = BF16 if dtype == F32 else dtype
    pool, table, cache = _cache_of([N], kv, d, cdt, g)
    q, k, v = (_normal(g, N, h, d, dtype=dtype) for h in (heads, kv, kv))
    if r < d:
        q[5, :, r:], k[6, :, d - 1], v[7, :, 0] = math.inf, math.nan, -math.inf
    old_q, old_k = q.clone(), k.clone()
    pos = torch.randperm(N, generator=g, device="cuda").int()
    with pkg.Rope(d, r, layout) as rope:
        rope.apply(CODE[dtype], N, pos.data_ptr(), q=_rows(q), q_out=_rows(q), num_heads=heads, k=_rows(k), k_out=_rows(k), kv_heads=kv, v=_rows(v),
                   cache=cache, offsets=_ints([0, N]).data_ptr(), n=1, stream=_stream())
    freq = R.frequencies(r)
    for old, new in ((old_q, q), (old_k, k)):
        want, off = R.rotate(old, pos, freq, layout)
        _within(new[..., :r], want[..., :r], (off + R.HALF_STEP[dtype] * want.abs() + 1e-7)[..., :r])
        assert torch.equal(new[..., r:].nan_to_num(9.0), old[..., r:].nan_to_num(9.0))
    for h in range(kv):
        held_k, held_v = _held(pool, table, 0, N, h)
        at = pos.long()
        assert torch.equal(held_v[at].nan_to_num(9.0), v[:, h].to(cdt).nan_to_num(9.0))
        if dtype != F32:  # one rounding for both
            assert torch.equal(held_k[at].nan_to_num(9.0), k[:, h].nan_to_num(9.0))
        else:
            want, off = R.rotate(old_k, pos, freq, layout)
            _within(held_k[at][:, :r], want[:, h, :r], (off + R.HALF_STEP[cdt] * want.abs() * 1.01 + 1e-7)[:, h, :r])


@pytest.mark.parametrize("scaling,factor", [("linear", 4.0), ("stretched", 8.0), ("by_parts", 16.0)])
def test_rope_scalings_far_positions_and_single_operands(scaling, factor):
    g, N, d, r = _gen(2), 9, 128, 96
    k = _normal(g, N, 3, d)
    pos = _ints([0, 5, 4095, 4096, 65535, 131071, 1 << 20, (1 << 24) + 1, 2**31 - 1])
    out = torch.empty_like(k)
    rope = pkg.Rope(d, r, "half", 500000.0, scaling, factor, 8192, 32.0, 1.0, 1.25)
    rope.apply(pkg.F32, N, pos.data_ptr(), k=_rows(k), k_out=_rows(out), kv_heads=3, stream=_stream())
    want, off = R.rotate(k, pos, R.frequencies(r, 500000.0, scaling, factor, 8192), "half", 1.25)
    # a 64-bit turn of 2^31 radians per step 1 is itself off by 2^31 2^-52 / 2 pi
    _within(out, want, off + 2.0 ** -24 * want.abs() + 2.0 ** 31 * 2.0 ** -50 * 4)
    only = torch.empty_like(k)
    rope.apply(pkg.F32, N, pos.data_ptr(), q=_rows(k), q_out=_rows(only), num_heads=3, stream=_stream())
    assert torch.equal(only, out)


@pytest.mark.parametrize("shift", [0, 1])
def test_rope_in_place_strided_and_unaligned(shift):
    """A fused [N, H + 2 Hk, d] buffer turned in place, aligned and one element off (the piece and the pair path)."""
    g, N, H, Hk, d = _gen(3), 130, 6, 2, 64
    flat = _normal(g, N * (H + 2 * Hk) * d + 8, dtype=BF16)
    qkv = flat[shift:shift + N * (H + 2 * Hk) * d].view(N, H + 2 * Hk, d)
    before = flat.clone()
    old = qkv.clone()
    pos = torch.arange(N, dtype=torch.int32, device="cuda") * 3
    q, k = _rows(qkv[:, :H]), _rows(qkv[:, H:H + Hk])
    with pkg.Rope(d, 32, "half") as rope:
        rope.apply(pkg.BF16, N, pos.data_ptr(), q=q, q_out=q, num_heads=H, k=k, k_out=k, kv_heads=Hk, stream=_stream())
    want, off = R.rotate(old[:, :H + Hk], pos, R.frequencies(32), "half")
    _within(qkv[:, :H + Hk], want, off + 2.0 ** -8 * want.abs() + 1e-7)
    assert torch.equal(qkv[:, :H + Hk, 32:], old[:, :H + Hk, 32:]) and torch.equal(qkv[:, H + Hk:], old[:, H + Hk:])
    assert torch.equal(flat[:shift], before[:shift]) and torch.equal(flat[shift + qkv.numel():], before[shift + qkv.numel():])


def _cache_of(lens, Hk, d, dtype, g, pages_more=3, spread=1, fill=0.0):
    """(pool [pages, spread, Hk, 2, 64, d], table, view of layer spread-1): pages in an order of chance."""
    blocks = max(1, max((-(-int(x) // 64) for x in lens), default=1))
    need = [-(-int(x) // 64) for x in lens]
    pages = sum(need) + pages_more
    pool = torch.full((pages, spread, Hk, 2, 64, d), fill, dtype=dtype, device="cuda")
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    table = np.full((max(len(lens), 1), blocks), -1, np.int32)
    for i, b in enumerate(need):
        table[i, :b] = [order.pop() for _ in range(b)]
    table = torch.tensor(table, device="cuda")
    layer = pool[:, spread - 1]
    return pool, table, pkg.KvCache(layer.data_ptr(), pool.stride(0), table.data_ptr(), blocks, pages, Hk, d)


def _held(pool, table, s, length, h):
    """The cached K and V rows [length, d] of kv head h of sequence s."""
    if length == 0:
        return pool[0, -1, h, :, :0]
    at = torch.arange(length, device="cuda")
    page = table[s, at // 64].long()
    return pool[page, -1, h, :, at % 64].transpose(0, 1)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("layout,r,aligned", [("interleaved", 64, True), ("half", 64, True), ("half", 16, True), ("interleaved", 26, True), ("half", 64, False)])
def test_rope_appends_to_the_cache(dtype, layout, r, aligned):
    g, Hk, H, d = _gen(4), 2, 4, 64
    lens, start = [3, 0, 70, 1, 129], [0, 5, 61, 63, 200]
    off = _offsets(lens)
    N = off[-1] + 2  # two rows behind the last sequence
    cdt = BF16 if dtype == F32 else dtype
    pool, table, cache = _cache_of([a + b for a, b in zip(start, lens)], Hk, d, cdt, g, spread=2, fill=3.0)
    table[3, 1] = 10 ** 6  # position 64 of sequence 3 would be there: it has none
    q = _normal(g, N, H, d, dtype=dtype)
    wide = _normal(g, N * 2 * Hk * d + 1, dtype=dtype)
    kv = wide[0 if aligned else 1:][:N * 2 * Hk * d].view(N, 2 * Hk, d)
    k, v = kv[:, :Hk], kv[:, Hk:]
    seq = np.repeat(np.arange(len(lens)), lens)
    pos = _ints([start[s] + i - off[s] for i, s in enumerate(seq)] + [9, 9])
    pos[off[2] + 5] = -1        # not committed
    pos[off[4] + 1] = 64 * table.shape[1]  # beyond the table: turned, not written
    q_out, k_out = torch.full_like(q, 7.0), torch.full((N, Hk, d), 7.0, dtype=dtype, device="cuda")
    before = pool.clone()
    offsets = _ints(off)
    with pkg.Rope(d, r, layout) as rope:
        rope.apply(CODE[dtype], N, pos.data_ptr(), q=_rows(q), q_out=_rows(q_out), num_heads=H, k=_rows(k), k_out=_rows(k_out), v=_rows(v), kv_heads=Hk,
                   cache=cache, offsets=offsets.data_ptr(), n=len(lens), stream=_stream())
    kw, ko = R.rotate(k, pos, R.frequencies(r), layout)
    want, bound = before.double(), torch.zeros_like(before, dtype=torch.float64)
    done = torch.zeros(N, dtype=torch.bool)
    for i, s in enumerate(seq):
        p = int(pos[i])
        done[i] = p >= 0
        if p < 0 or p >= 64 * table.shape[1]:
            continue
        page = int(table[s, p // 64])
        want[page, -1, :, 0, p % 64] = kw[i]
        bound[page, -1, :, 0, p % 64] = ko[i] + R.HALF_STEP[cdt] * kw[i].abs() + 1e-7
        want[page, -1, :, 1, p % 64] = v[i].to(cdt).double()
    off_by = (pool.double() - want).abs()
    assert bool((off_by <= bound).all())  # pages, layers and positions of nobody stay as they were, to the bit
    done = done.cuda()
    _within(k_out[done], kw[done], ko[done] + R.HALF_STEP[dtype] * kw[done].abs() + 1e-7)
    assert bool((k_out[~done] == 7.0).all()) and bool((q_out[~done] == 7.0).all()) and bool((q_out[done] != 7.0).any())


# ---- packed prompts ------------------------------------------------------------------------------------------------


def _prompt(q, k, v, lens, dtype, scale=0.0, out=None, rows=None):
    H, d, Hk = q.shape[1], q.shape[2], k.shape[1]
    out = torch.full(q.shape, 7.0, dtype=dtype, device="cuda") if out is None else out
    off = _ints(_offsets(lens))
    pkg.prompt_attention(CODE[dtype], _rows(q), _rows(k), _rows(v), _rows(out), off.data_ptr(), len(lens), q.shape[0] if rows is None else rows, H, Hk, d,
                         scale, _stream())
    torch.cuda.synchronize()
    return out


def _check_prompt(q, k, v, out, lens, dtype, scale=0.0, skip=()):
    off = _offsets(lens)
    for s, t in enumerate(lens):
        if t == 0 or s in skip:
            continue
        b, e = off[s], off[s + 1]
        seen = torch.ones(t, t, device="cuda").tril().bool()
        want, bound = R.attend(q[b:e], k[b:e], v[b:e], seen, scale or q.shape[2] ** -0.5, dtype)
        _within(out[b:e], want, bound)


LENS = [[1], [0, 5, 0], [128], [127, 129, 1, 0], [16, 15, 17, 64, 65], [300, 33, 641], [1025]]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("lens", LENS, ids=str)
def test_prompt_attention(dtype, heads, lens):
    H, Hk, d = heads
    g, N = _gen(5), sum(lens) + 3
    q, k, v = (_normal(g, N, h, d, dtype=dtype) for h in (H, Hk, Hk))
    out = _prompt(q, k, v, lens, dtype)
    _check_prompt(q, k, v, out, lens, dtype)
    assert bool((out[sum(lens):] == 7.0).all())  # rows behind the last sequence


@pytest.mark.parametrize("n", [70, 1100])
def test_prompt_attention_many_sequences(n):
    rng = np.random.default_rng(n)
    lens = rng.integers(0, 40, n).tolist()
    lens[n // 2] = 700
    g = _gen(6)
    q, k, v = (_normal(g, sum(lens), h, 64, dtype=BF16) for h in (8, 2, 2))
    out = _prompt(q, k, v, lens, BF16)
    some = set(rng.integers(0, n, 40).tolist()) | {0, n // 2, n - 1}
    _check_prompt(q, k, v, out, lens, BF16, skip=[s for s in range(n) if s not in some])
    assert torch.equal(out, _prompt(q, k, v, lens, BF16))  # run to run


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prompt_attention_growing_scores(dtype):
    """Scores that grow along the keys, so the running maximum moves by far more than the lazy step, and shrink again."""
    g, lens = _gen(7), [900, 411]
    q, k, v = (_normal(g, sum(lens), h, 64, dtype=dtype) for h in (4, 2, 2))
    ramp = torch.linspace(0, 12, 900, device="cuda")
    k = (k * torch.cat([ramp, ramp.flip(0)[:411]])[:, None, None]).to(dtype)
    out = _prompt(q, k, v, lens, dtype, scale=1.0)
    _check_prompt(q, k, v, out, lens, dtype, scale=1.0)


@pytest.mark.parametrize("order", ["fused", "heads first", "one head"])
def test_prompt_attention_strides(order):
    g, lens, d = _gen(8), [200, 77], 64
    N = sum(lens)
    if order == "fused":
        qkv = _normal(g, N, 8 + 2 * 2, d, dtype=BF16)
        q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
        out = torch.full((N, 10, d + 8), 7.0, dtype=BF16, device="cuda")[:, 1:9, 8:]
    elif order == "heads first":
        q, k, v, out = (_normal(g, h, N, d, dtype=BF16).transpose(0, 1) for h in (8, 2, 2, 8))
    else:
        q, k, v, out = (_normal(g, N, 3, d, dtype=BF16)[:, 1:2] for _ in range(4))
    _prompt(q, k, v, lens, BF16, out=out)
    _check_prompt(q, k, v, out, lens, BF16)
    if order == "fused":
        whole = out._base
        assert bool((whole[:, 0] == 7.0).all()) and bool((whole[:, 9] == 7.0).all()) and bool((whole[:, 1:9, :8] == 7.0).all())


def test_prompt_attention_keeps_sequences_apart():
    """NaN and infinities in a neighbour, and behind the last sequence, reach no row of the others."""
    g, lens = _gen(9), [70, 50, 200, 9]
    off = _offsets(lens)
    q, k, v = (_normal(g, sum(lens) + 40, h, 64, dtype=BF16) for h in (4, 4, 4))
    for bad in (math.nan, math.inf, -math.inf):
        for x in (q, k, v):
            x[off[1]:off[2]] = bad
            x[off[4]:] = bad
        out = _prompt(q, k, v, lens, BF16)
        _check_prompt(q, k, v, out, lens, BF16, skip=(1,))


# ---- trees over the cache ------------------------------------------------------------------------------------------


def _tree(q, k, v, cache, lengths, masks, nodes, dtype, max_nodes=None, scale=0.0, out=None):
    H = q.shape[1]
    out = torch.full(q.shape, 7.0, dtype=dtype, device="cuda") if out is None else out
    top = max(max(nodes), 1) if max_nodes is None else max_nodes
    size = pkg.tree_attention_workspace(len(nodes), top, H, cache)
    ws = torch.full((max(size, 16),), 255, dtype=torch.uint8, device="cuda")
    off, ln = _ints(_offsets(nodes)), _ints(lengths)
    pkg.tree_attention(CODE[dtype], _rows(q), _rows(k), _rows(v), _rows(out), cache, ln.data_ptr(), masks.data_ptr(), off.data_ptr(), len(nodes), q.shape[0], top, H,
                       scale, ws.data_ptr(), size, _stream())
    torch.cuda.synchronize()
    return out


def _check_tree(q, k, v, pool, table, lengths, masks, nodes, out, dtype, scale=0.0, gone=None, seqs=None):
    off, Hk = _offsets(nodes), k.shape[1]
    for s, t in enumerate(nodes):
        if t == 0 or (seqs is not None and s not in seqs):
            continue
        b, e, L = off[s], off[s + 1], lengths[s]
        held = torch.stack([_held(pool, table.clamp(0, pool.shape[0] - 1), s, L, h) for h in range(Hk)], 2)  # [2, L, Hk, d]
        kk, vv = torch.cat([held[0], k[b:e]]), torch.cat([held[1], v[b:e]])
        there = torch.ones(L, dtype=torch.bool, device="cuda")
        if gone is not None and L:
            there = (table[s, torch.arange(L, device="cuda") // 64] >= 0) & (table[s, torch.arange(L, device="cuda") // 64] < pool.shape[0])
        bits = (masks[b:e, None] >> torch.arange(t, device="cuda")) & 1
        seen = torch.cat([there.expand(t, L), bits.bool()], 1)
        want, bound = R.attend(q[b:e], kk, vv, seen, scale or q.shape[2] ** -0.5, dtype)
        _within(out[b:e], want, bound)


def _random_masks(nodes, seed, empty=True):
    rng = np.random.default_rng(seed)
    out = []
    for t in nodes:
        parents = [-1] + [int(rng.integers(max(0, i - 4), i)) for i in range(1, t)]
        m = pkg.tree_masks(parents[:t])
        if empty and t > 2:
            m[1], m[2] = 0, np.uint64(1 << (t - 1))  # sees no node; sees a later node only
        out.append(m)
    return torch.tensor(np.concatenate(out).view(np.int64) if out else np.zeros(0, np.int64), device="cuda")


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("lengths,nodes", [
    ([0, 1, 63, 64, 65, 127, 128, 129], [1, 1, 1, 1, 1, 1, 1, 1]),
    ([0, 0, 700, 5, 130], [3, 1, 17, 0, 64]),
    ([1500], [24]), ([2049], [64]), ([0], [1]), ([0], [64]), ([4000], [1]),
], ids=str)
def test_tree_attention(dtype, heads, lengths, nodes):
    H, Hk, d = heads
    g, N = _gen(11), sum(nodes) + 2
    q, k, v = (_normal(g, N, h, d, dtype=dtype) for h in (H, Hk, Hk))
    pool, table, cache = _cache_of(lengths, Hk, d, dtype, g, spread=2)
    pool.normal_(generator=g)
    masks = _random_masks(nodes, 3)
    out = _tree(q, k, v, cache, lengths, masks, nodes, dtype)
    _check_tree(q, k, v, pool, table, lengths, masks, nodes, out, dtype)
    assert bool((out[sum(nodes):] == 7.0).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("lengths,nodes", [
    ([0, 1, 63, 64, 65, 127, 128, 129], [1, 1, 1, 1, 1, 1, 1, 1]),
    ([0, 0, 700, 5, 130], [3, 1, 17, 0, 64]), ([0, 300, 0], [0, 2, 0]), ([0], [1]), ([0], [64]),
], ids=str)
def test_tree_attention_short_lengths_in_a_long_cache(dtype, heads, lengths, nodes):
    """Room for 600 pages a sequence: the work goes in ranges. Unused pages and table entries hold what must not be read."""
    H, Hk, d = heads
    g, N = _gen(17), sum(nodes) + 2
    q, k, v = (_normal(g, N, h, d, dtype=dtype) for h in (H, Hk, Hk))
    pool, table, cache = _cache_of(lengths, Hk, d, dtype, g, fill=math.nan)
    for s, L in enumerate(lengths):
        for b in range(-(-L // 64)):
            pool[table[s, b], -1, :, :, : min(64, L - 64 * b)] = torch.randn(Hk, 2, min(64, L - 64 * b), d, generator=g, device="cuda").to(dtype)
    wide = torch.cat([table, torch.full((len(nodes), 600 - table.shape[1]), 2**31 - 1, dtype=torch.int32, device="cuda")], 1)
    cache = pkg.KvCache(cache.pool, cache.page_stride, wide.data_ptr(), 600, cache.pages, Hk, d)
    assert pkg.tree_attention_workspace(len(nodes), max(nodes), H, cache) > 0
    masks = _random_masks(nodes, 9)
    out = _tree(q, k, v, cache, lengths, masks, nodes, dtype)
    _check_tree(q, k, v, pool, table, lengths, masks, nodes, out, dtype)
    assert bool((out[sum(nodes):] == 7.0).all())


@pytest.mark.parametrize("nodes", [1, 7, 40])
def test_tree_attention_many_sequences(nodes):
    """Grids of several waves, ragged lengths, nodes fewer than max_nodes."""
    rng = np.random.default_rng(nodes)
    n = 150
    lengths, counts = rng.integers(0, 900, n).tolist(), rng.integers(0, nodes + 1, n).tolist()
    g = _gen(12)
    q, k, v = (_normal(g, max(sum(counts), 1), h, 64, dtype=BF16) for h in (8, 2, 2))
    pool, table, cache = _cache_of(lengths, 2, 64, BF16, g)
    pool.normal_(generator=g)
    masks = _random_masks(counts, 4)
    out = _tree(q, k, v, cache, lengths, masks, counts, BF16, max_nodes=nodes)
    _check_tree(q, k, v, pool, table, lengths, masks, counts, out, BF16, seqs=set(rng.integers(0, n, 30).tolist()))
    assert torch.equal(out, _tree(q, k, v, cache, lengths, masks, counts, BF16, max_nodes=nodes))


@pytest.mark.parametrize("n,heads,nodes,most", [(90, (8, 4, 128), 5, 700), (330, (4, 1, 64), 3, 500), (80, (6, 2, 32), 64, 900), (20, (32, 8, 128), 64, 6000),
                                                (1300, (2, 1, 64), 2, 300), (5, (16, 2, 64), 33, 9000)], ids=str)
def test_tree_attention_layouts_of_the_work(n, heads, nodes, most):
    """Pairs of heads, pairs of row tiles and ranges cut across sequences, empty ones among them, more sequences than threads."""
    H, Hk, d = heads
    rng = np.random.default_rng(n)
    lengths, counts = rng.integers(0, most, n).tolist(), rng.integers(0, nodes + 1, n).tolist()
    lengths[0], counts[n // 2], counts[-1] = most, nodes, 0
    g = _gen(16)
    q, k, v = (_normal(g, max(sum(counts), 1), h, d, dtype=F16) for h in (H, Hk, Hk))
    pool, table, cache = _cache_of(lengths, Hk, d, F16, g)
    pool.normal_(generator=g)
    masks = _random_masks(counts, 8)
    out = _tree(q, k, v, cache, lengths, masks, counts, F16, max_nodes=nodes)
    _check_tree(q, k, v, pool, table, lengths, masks, counts, out, F16, seqs=set(rng.integers(0, n, 16).tolist()) | {0, n // 2})
    assert torch.equal(out, _tree(q, k, v, cache, lengths, masks, counts, F16, max_nodes=nodes))


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("n", [1, 40])
def test_tree_attention_reads_nothing_behind_the_lengths(bad, n):
    lengths = ([333, 64, 1, 130, 0] * 8)[:n]
    nodes = ([5, 2, 9, 33, 3] * 8)[:n]
    g = _gen(13)
    q, k, v = (_normal(g, sum(nodes) + 64, h, 64, dtype=BF16) for h in (4, 2, 2))
    for x in (q, k, v):
        x[sum(nodes):] = bad
    pool, table, cache = _cache_of(lengths, 2, 64, BF16, g, fill=bad)
    for s, L in enumerate(lengths):
        for p in range(L):
            if p % 64 == 0:
                pool[table[s, p // 64], -1, :, :, : min(64, L - p)] = _normal(g, 2, 2, min(64, L - p), 64, dtype=BF16)
    masks = _random_masks(nodes, 5)
    out = _tree(q, k, v, cache, lengths, masks, nodes, BF16)
    _check_tree(q, k, v, pool, table, lengths, masks, nodes, out, BF16)


def test_tree_attention_pages_that_are_not_there():
    lengths, nodes = [500, 300, 128], [4, 1, 3]
    g = _gen(14)
    q, k, v = (_normal(g, sum(nodes), h, 128, dtype=BF16) for h in (8, 2, 2))
    pool, table, cache = _cache_of(lengths, 2, 128, BF16, g)
    pool.normal_(generator=g)
    table[0, 0], table[0, 3], table[1, 4], table[2, 0], table[2, 1] = -1, 10 ** 6, 2 ** 31 - 1, -5, pool.shape[0]
    masks = _random_masks(nodes, 6)
    masks[-1] = 0  # and this row sees no node either: nothing at all
    out = _tree(q, k, v, cache, lengths, masks, nodes, BF16)
    _check_tree(q, k, v, pool, table, lengths, masks, nodes, out, BF16, gone=True)
    assert bool((out[-1] == 0).all())
    # lengths beyond the table, and negative ones, are cut
    again = _tree(q, k, v, cache, [10 ** 9, -3, 64 * table.shape[1]], masks, nodes, BF16)
    _check_tree(q, k, v, pool, table, [64 * table.shape[1], 0, 64 * table.shape[1]], masks, nodes, again, BF16, gone=True)


def test_tree_attention_and_append_in_a_pool_beyond_32_bits():
    """A pool of more than 2^31 elements whose last pages are in use."""
    Hk, d, pages, L = 8, 128, 20000, 200
    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip("needs 8 GB")
    g = _gen(15)
    pool = torch.empty(pages, 1, Hk, 2, 64, d, dtype=BF16, device="cuda")
    assert pool.numel() > 2 ** 31
    table = _ints([pages - 1, pages - 3, pages - 2, pages - 4]).view(1, 4)
    cache = pkg.KvCache(pool.data_ptr(), pool.stride(0), table.data_ptr(), 4, pages, Hk, d)
    k, v = _normal(g, L, Hk, d, dtype=BF16), _normal(g, L, Hk, d, dtype=BF16)
    pos, off = torch.arange(L, dtype=torch.int32, device="cuda"), _ints([0, L])
    with pkg.Rope(d, d, "half") as rope:
        rope.apply(pkg.BF16, L, pos.data_ptr(), k=_rows(k), v=_rows(v), kv_heads=Hk, cache=cache, offsets=off.data_ptr(), n=1, stream=_stream())
    kw, _ = R.rotate(k, pos, R.frequencies(d), "half")
    held = torch.stack([_held(pool, table, 0, L, h) for h in range(Hk)], 2)
    _within(held[0], kw, 2.0 ** -8 * kw.abs() + 1e-5)
    assert torch.equal(held[1], v)
    q, k1, v1 = (_normal(g, 3, h, d, dtype=BF16) for h in (32, Hk, Hk))
    masks = _random_masks([3], 7)
    out = _tree(q, k1, v1, cache, [L], masks, [3], BF16)
    _check_tree(q, k1, v1, pool, table, [L], masks, [3], out, BF16)


# ---- verification --------------------------------------------------------------------------------------------------


def _verify_case(nodes, V, dtype, seed, branch=3, sharp=2.5, near=1.0):
    g, rng = _gen(seed), np.random.default_rng(seed)
    N = sum(nodes)
    logits = _normal(g, N, V) * sharp
    target = torch.softmax(logits, 1).to(dtype)
    draft = torch.softmax(logits + _normal(g, N, V) * near, 1).to(dtype)
    parents = np.concatenate([[-1] + [int(rng.integers(max(0, i - branch), i)) for i in range(1, t)] for t in nodes if t]).astype(np.int32)
    off = _offsets(nodes)
    tokens = np.zeros(N, np.int32)
    rows = draft.float().cpu().numpy().astype(np.float64)
    for s, t in enumerate(nodes):
        for i in range(1, t):
            p = rows[off[s] + parents[off[s] + i]]
            tokens[off[s] + i] = min(V - 1, int(np.searchsorted(np.cumsum(p), rng.random() * p.sum())))
    return target, draft, tokens, parents, rng.random(N).astype(np.float32)


def _verify(target, draft, tokens, parents, uniforms, nodes, lengths=None, vocab=None):
    n, N = len(nodes), sum(nodes)
    path, commit = (torch.full((N + 2,), 77, dtype=torch.int32, device="cuda") for _ in range(2))
    count, following, new = (torch.full((n,), 77, dtype=torch.int32, device="cuda") for _ in range(3))
    off, tk, pr, un = _ints(_offsets(nodes)), _ints(tokens), _ints(parents), torch.tensor(uniforms, device="cuda")
    ln = _ints(lengths) if lengths is not None else None
    more = {} if ln is None else dict(lengths=ln.data_ptr(), commit=commit.data_ptr(), new_lengths=new.data_ptr())
    pkg.verify_tree(CODE[target.dtype], target.data_ptr(), draft.data_ptr(), target.shape[1] if vocab is None else vocab, tk.data_ptr(), pr.data_ptr(), un.data_ptr(),
                    off.data_ptr(), n, N, path.data_ptr(), count.data_ptr(), following.data_ptr(), target_stride=target.stride(0), draft_stride=draft.stride(0),
                    stream=_stream(), **more)
    torch.cuda.synchronize()
    assert path[N:].tolist() == [77, 77] and commit[N:].tolist() == [77, 77]
    return [x.cpu().numpy() for x in (path[:N], count, following, commit[:N], new)]


def _check_verify(target, draft, tokens, parents, uniforms, nodes, got, lengths=None, vocab=None):
    off = _offsets(nodes)
    tn, dn = target.float().cpu().numpy().astype(np.float64), draft.float().cpu().numpy().astype(np.float64)
    total = 0
    for s, t in enumerate(nodes):
        b, e = off[s], off[s + 1]
        L = 0 if lengths is None else lengths[s]
        if t == 0:
            assert got[1][s] == 0 and got[2][s] == -1 and (lengths is None or got[4][s] == L)
            continue
        taken, following = R.verify(tn[b:e, :vocab], dn[b:e, :vocab], tokens[b:e], parents[b:e], uniforms[b:e].astype(np.float64))
        total += len(taken) - 1
        assert got[0][b:e].tolist() == taken + [-1] * (t - len(taken)), s
        assert (got[1][s], got[2][s]) == (len(taken) - 1, following), s
        if lengths is not None:
            commit = [-1] * t
            for depth, i in enumerate(taken):
                commit[i] = L + depth
            assert got[3][b:e].tolist() == commit and got[4][s] == L + len(taken)
    return total


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("nodes,V", [([1], 7), ([2, 0, 9], 1), ([8], 4096), ([9, 24, 1, 0, 16] * 3, 1001), ([12] * 5, 32768), ([5, 3], 50257), ([30] * 300, 300)],
                         ids=lambda x: str(x)[:24])
def test_verify_tree(dtype, nodes, V):
    case = _verify_case(nodes, V, dtype, 21)
    lengths = [100 * s for s in range(len(nodes))]
    got = _verify(*case, nodes, lengths)
    _check_verify(*case, nodes, got, lengths)
    bare = _verify(*case, nodes)
    assert all(np.array_equal(a, b) for a, b in zip(got[:3], bare[:3]))


@pytest.mark.parametrize("near", [0.0, 0.3, 6.0])
def test_verify_tree_chains_and_wide_trees(near):
    """Drafts equal to, near and far from the target: all taken, some, hardly any; wide trees refuse many siblings."""
    taken = 0
    for branch, nodes in ((1, [40] * 4), (64, [40] * 4), (2, [700, 520])):
        case = _verify_case(nodes, 513, F32, 22, branch=branch, near=near)
        if branch == 64:
            case[3][1:40] = 0  # all under the root
        got = _verify(*case, nodes)
        taken += _check_verify(*case, nodes, got)
    if near == 0.0:
        assert taken >= 40  # p = q: every candidate is taken


def test_verify_tree_edges():
    V, nodes = 64, [4]
    one = lambda i: torch.nn.functional.one_hot(torch.tensor(i), V).float()  # noqa: E731
    flat = torch.full((V,), 1.0 / V)
    tokens, parents = np.array([0, 5, 6, 7], np.int32), np.array([-1, 0, 1, 2], np.int32)

    def walk(t, d, u, tk=tokens, pr=parents):
        t, d = (torch.stack(x).cuda() for x in (t, d))
        u = np.array(u, np.float32)
        got = _verify(t, d, tk, pr, u, [len(tk)])
        _check_verify(t, d, tk, pr, u, [len(tk)], got)
        return got

    # the target surely takes 5, 6, 7, then 9; u = 0 and the largest u below 1
    for u in (0.0, float(np.nextafter(np.float32(1), np.float32(0)))):
        got = walk([one(5), one(6), one(7), one(9)], [flat] * 4, [u] * 4)
        assert got[0].tolist() == [0, 1, 2, 3] and got[2][0] == 9
    # the target gives the candidate nothing: refused even at u = 0, the draw avoids it
    assert walk([one(9)] * 4, [flat] * 4, [0.0] * 4)[2][0] == 9
    # q = 0 at the candidate: taken when p > 0
    assert walk([flat] * 4, [one(1)] * 4, [0.5] * 4)[1][0] == 3
    # p = q and refused is impossible (u < 1); a row without mass draws 0; NaN, negative and infinite u
    assert walk([torch.zeros(V)] * 4, [flat] * 4, [0.5] * 4)[2][0] == 0
    spoiled = flat.clone()
    spoiled[3], spoiled[4] = math.nan, -1.0
    walk([spoiled] * 4, [flat] * 4, [0.99, 0.99, 0.99, 0.99])
    # tokens outside the vocabulary and parents that are not below are passed over
    walk([flat] * 4, [flat] * 4, [0.3] * 4, np.array([0, -1, 64, 2**31 - 1], np.int32))
    walk([flat] * 4, [flat] * 4, [0.3] * 4, tokens, np.array([0, 1, 3, -7], np.int32))


@pytest.mark.parametrize("V", [64, 50257])
@pytest.mark.parametrize("refused", [0, 1, 2])
def test_verify_tree_rows_with_an_infinite_value_draw_token_0(V, refused):
    target = torch.full((1 + refused, V), 1.0 / V)
    target[0, 33], target[0, 5], target[0, 6] = math.inf, 0.0, 0.0
    draft = torch.full((1 + refused, V), 1.0 / V)
    for u in (0.0, 0.5):
        got = _verify(target.cuda(), draft.cuda(), np.array([0, 5, 6][: 1 + refused], np.int32), np.array([-1, 0, 0][: 1 + refused], np.int32),
                      np.full(1 + refused, u, np.float32), [1 + refused])
        assert got[1][0] == 0 and got[2][0] == 0


def test_verify_tree_follows_the_distribution():
    """Over many independent sequences, the first token after the root is distributed as the target's row, whatever the draft."""
    V, n = 8, 40000
    g = _gen(23)
    p, q = torch.softmax(_normal(g, 1, V) * 1.5, 1), torch.softmax(_normal(g, 1, V) * 1.5, 1)
    target, draft = p.repeat(3 * n, 1), q.repeat(3 * n, 1)
    tokens = torch.multinomial(q[0], 3 * n, replacement=True, generator=g).cpu().numpy().astype(np.int32)
    parents = np.tile(np.array([-1, 0, 0], np.int32), n)
    uniforms = torch.rand(3 * n, generator=g, device="cuda").cpu().numpy()
    got = _verify(target, draft, tokens, parents, uniforms, [3] * n)
    path = got[0].reshape(n, 3)
    first = np.where(path[:, 1] > 0, tokens.reshape(n, 3)[np.arange(n), np.maximum(path[:, 1], 0)], got[2])
    share = np.bincount(first, minlength=V) / n
    # 5 standard deviations of each share
    want = p[0].double().cpu().numpy()
    assert np.all(np.abs(share - want) <= 5 * np.sqrt(want * (1 - want) / n) + 1e-9)


def test_verify_tree_strided_rows():
    nodes = [6, 6]
    target, draft, tokens, parents, u = _verify_case(nodes, 1000, F32, 24)
    wide_t, wide_d = torch.ones(12, 1003, device="cuda"), torch.ones(12, 1010, device="cuda")
    wide_t[:, 1:1001], wide_d[:, 2:1002] = target, draft
    t, d = wide_t[:, 1:1001], wide_d[:, 2:1002]  # unlike alignment, more values between the rows
    got = _verify(t, d, tokens, parents, u, nodes, vocab=1000)
    _check_verify(t, d, tokens, parents, u, nodes, got)


# ---- together ------------------------------------------------------------------------------------------------------


def test_serving_step_over_the_fused_attention_cache():
    """Prompts of different lengths into a FusedAttention operator's cache, a verify pass over drafted trees, the accepted rows
    committed, and FusedAttention.decode going on from there; every attention row against 64 bits on the host's own copy."""
    H, Hk, d, V = 8, 2, 64, 500
    lens, nodes = [130, 1, 64, 300], [9, 1, 24, 5]
    n, g = len(lens), _gen(31)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side), pkg.FusedAttention(n, H, Hk, d, 400, 10000.0) as op, pkg.Rope(d) as rope:
        st = _stream()
        cache = op.cache()
        assert (cache.kv_heads, cache.head_dim, cache.max_blocks) == (Hk, d, 7)
        N = sum(lens)
        q, k, v = (_normal(g, N, h, d, dtype=BF16) for h in (H, Hk, Hk))
        off = _ints(_offsets(lens))
        pos = _ints([i for t in lens for i in range(t)])
        qr, kr, out = torch.empty_like(q), torch.empty_like(k), torch.empty_like(q)
        rope.apply(pkg.BF16, N, pos.data_ptr(), q=_rows(q), q_out=_rows(qr), num_heads=H, k=_rows(k), k_out=_rows(kr), v=_rows(v), kv_heads=Hk, cache=cache,
                   offsets=off.data_ptr(), n=n, stream=st)
        pkg.prompt_attention(pkg.BF16, _rows(qr), _rows(kr), _rows(v), _rows(out), off.data_ptr(), n, N, H, Hk, d, stream=st)
        side.synchronize()
        _check_prompt(qr, kr, v, out, lens, BF16)
        # drafted trees
        M = sum(nodes)
        target, draft, tokens, parents, u = _verify_case(nodes, V, F32, 32)
        noff = _offsets(nodes)
        depth = np.zeros(M, np.int32)
        for s, t in enumerate(nodes):
            for i in range(1, t):
                depth[noff[s] + i] = depth[noff[s] + parents[noff[s] + i]] + 1
        masks = torch.tensor(np.concatenate([pkg.tree_masks(parents[noff[s]:noff[s + 1]]) for s in range(n)]).view(np.int64), device="cuda")
        q1, k1, v1 = (_normal(g, M, h, d, dtype=BF16) for h in (H, Hk, Hk))
        toff, ln = _ints(noff), _ints(lens)
        tpos = _ints(np.repeat(lens, nodes) + depth)
        q1r, k1r, o1 = torch.empty_like(q1), torch.empty_like(k1), torch.empty_like(q1)
        rope.apply(pkg.BF16, M, tpos.data_ptr(), q=_rows(q1), q_out=_rows(q1r), num_heads=H, k=_rows(k1), k_out=_rows(k1r), kv_heads=Hk, stream=st)
        size = pkg.tree_attention_workspace(n, 24, H, cache)
        ws = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
        pkg.tree_attention(pkg.BF16, _rows(q1r), _rows(k1r), _rows(v1), _rows(o1), cache, ln.data_ptr(), masks.data_ptr(), toff.data_ptr(), n, M, 24, H,
                           workspace=ws.data_ptr(), workspace_bytes=size, stream=st)
        path, commit = (torch.empty(M, dtype=torch.int32, device="cuda") for _ in range(2))
        count, following, new = (torch.empty(n, dtype=torch.int32, device="cuda") for _ in range(3))
        tk, pr, un = _ints(tokens), _ints(parents), torch.tensor(u, device="cuda")
        pkg.verify_tree(pkg.F32, target.data_ptr(), draft.data_ptr(), V, tk.data_ptr(), pr.data_ptr(), un.data_ptr(), toff.data_ptr(), n, M, path.data_ptr(),
                        count.data_ptr(), following.data_ptr(), lengths=ln.data_ptr(), commit=commit.data_ptr(), new_lengths=new.data_ptr(), stream=st)
        rope.apply(pkg.BF16, M, commit.data_ptr(), k=_rows(k1), v=_rows(v1), kv_heads=Hk, cache=cache, offsets=toff.data_ptr(), n=n, stream=st)
        side.synchronize()
        got = [x.cpu().numpy() for x in (path, count, following, commit, new)]
        _check_verify(target, draft, tokens, parents, u, nodes, got, lens)
        history = []  # per sequence: the turned keys and the values, as committed
        for s, t in enumerate(nodes):
            b, e = noff[s], noff[s + 1]
            c0, c1 = _offsets(lens)[s], _offsets(lens)[s + 1]
            bits = (masks[b:e, None] >> torch.arange(t, device="cuda")) & 1
            seen = torch.cat([torch.ones(t, lens[s], dtype=torch.bool, device="cuda"), bits.bool()], 1)
            want, bound = R.attend(q1r[b:e], torch.cat([kr[c0:c1], k1r[b:e]]), torch.cat([v[c0:c1], v1[b:e]]), seen, d ** -0.5, BF16)
            _within(o1[b:e], want, bound)
            took = [b + i for i in got[0][b:e] if i >= 0]
            history.append((torch.cat([kr[c0:c1], k1r[took]]), torch.cat([v[c0:c1], v1[took]])))
        # the operator's own decode step goes on from the committed rows
        op.set_lengths(got[4], st)
        q2, k2, v2 = (_normal(g, n, h, d) for h in (H, Hk, Hk))
        o2 = torch.empty_like(q2)
        op.decode(q2.data_ptr(), k2.data_ptr(), v2.data_ptr(), n, o2.data_ptr(), st)
        side.synchronize()
        p2 = torch.tensor(got[4], device="cuda")
        q2w, _ = R.rotate(q2, p2, R.frequencies(d), "interleaved")
        k2w, _ = R.rotate(k2, p2, R.frequencies(d), "interleaved")
        for s in range(n):
            kk, vv = torch.cat([history[s][0], k2w[s:s + 1].to(BF16)]), torch.cat([history[s][1], v2[s:s + 1].to(BF16)])
            want, _ = R.attend(q2w[s:s + 1], kk, vv, torch.ones(1, len(kk), dtype=torch.bool, device="cuda"), d ** -0.5, BF16)
            assert op.length(s) == got[4][s] + 1
            # the operator's own bar: 2e-2 of the output's range (tests/test_gpu_fused_attention.py)
            assert float((o2[s].double() - want[0]).abs().max()) < 2e-2 * float(want.max() - want.min())


def test_captured_step_follows_its_inputs():
    """Rope with append, tree attention (in parts) and verification in one captured graph, replayed on other inputs and lengths;
    a second graph with a workspace of its own runs between the first one's replays."""
    H, Hk, d, V, T = 8, 2, 64, 700, 6
    g = _gen(41)
    lengths = [500, 20]
    pool, table, cache = _cache_of([640, 640], Hk, d, BF16, g)
    pool.normal_(generator=g)
    wide = torch.cat([table, torch.full((2, 90), -1, dtype=torch.int32, device="cuda")], 1)  # room for long caches: the work goes in parts
    cache = pkg.KvCache(cache.pool, cache.page_stride, wide.data_ptr(), 100, cache.pages, Hk, d)
    n, M = 2, 2 * T
    off = _ints([0, T, 2 * T])
    size = pkg.tree_attention_workspace(n, T, H, cache)
    assert size > 0
    parents = np.tile(np.array([-1, 0, 0, 1, 3, 2], np.int32), 2)
    masks = torch.tensor(np.tile(pkg.tree_masks(parents[:T]), 2).view(np.int64), device="cuda")
    pr = _ints(parents)

    def buffers():
        b = dict(ws=torch.empty(size, dtype=torch.uint8, device="cuda"), ln=_ints(lengths), pos=_ints([0] * M), tk=_ints([0] * M), un=torch.zeros(M, device="cuda"),
                 target=torch.zeros(M, V, device="cuda"), draft=torch.zeros(M, V, device="cuda"))
        for name, h in (("q", H), ("k", Hk), ("v", Hk), ("qr", H), ("kr", Hk), ("out", H)):
            b[name] = torch.zeros(M, h, d, dtype=BF16, device="cuda")
        for name, m in (("path", M), ("commit", M), ("count", n), ("next", n), ("new", n)):
            b[name] = torch.zeros(m, dtype=torch.int32, device="cuda")
        return b

    rope = pkg.Rope(d)

    def step(b):
        st = _stream()
        rope.apply(pkg.BF16, M, b["pos"].data_ptr(), q=_rows(b["q"]), q_out=_rows(b["qr"]), num_heads=H, k=_rows(b["k"]), k_out=_rows(b["kr"]), kv_heads=Hk, stream=st)
        pkg.tree_attention(pkg.BF16, _rows(b["qr"]), _rows(b["kr"]), _rows(b["v"]), _rows(b["out"]), cache, b["ln"].data_ptr(), masks.data_ptr(), off.data_ptr(), n, M, T,
                           H, workspace=b["ws"].data_ptr(), workspace_bytes=size, stream=st)
        pkg.verify_tree(pkg.F32, b["target"].data_ptr(), b["draft"].data_ptr(), V, b["tk"].data_ptr(), pr.data_ptr(), b["un"].data_ptr(), off.data_ptr(), n, M,
                        b["path"].data_ptr(), b["count"].data_ptr(), b["next"].data_ptr(), lengths=b["ln"].data_ptr(), commit=b["commit"].data_ptr(),
                        new_lengths=b["new"].data_ptr(), stream=st)

    graphs = []
    for _ in range(2):
        b = buffers()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step(b)
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(b)
        graphs.append((graph, b))
    for r in range(3):
        now = [[500, 20], [63, 640], [0, 129]][r]
        cases = []
        for i, (graph, b) in enumerate(graphs):
            for name in ("q", "k", "v"):
                b[name].normal_(generator=g)
            case = _verify_case([T, T], V, F32, 50 + 2 * r + i)
            b["target"].copy_(case[0]), b["draft"].copy_(case[1]), b["tk"].copy_(_ints(case[2])), b["un"].copy_(torch.tensor(case[4], device="cuda"))
            b["ln"].copy_(_ints(now)), b["pos"].copy_(_ints(np.repeat(now, T) + np.tile([0, 1, 1, 2, 3, 2], 2)))
            cases.append((case[0], case[1], case[2], parents, case[4]))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for (graph, _), s in zip(graphs, streams):  # both at the same time
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (graph, b), case in zip(graphs, cases):
            qw, qo = R.rotate(b["q"], b["pos"], R.frequencies(d), "interleaved")
            _within(b["qr"], qw, qo + 2.0 ** -8 * qw.abs() + 1e-7)
            _check_tree(b["qr"], b["kr"], b["v"], pool, table, now, masks, [T, T], b["out"], BF16)
            got = [b[x].cpu().numpy() for x in ("path", "count", "next", "commit", "new")]
            _check_verify(*case, [T, T], got, now)


def test_calls_on_two_streams_at_once():
    g, lens = _gen(42), [300, 200]
    sets = [[_normal(g, 500, h, 64, dtype=BF16) for h in (8, 2, 2)] for _ in range(2)]
    alone = [_prompt(*x, lens, BF16) for x in sets]
    off = _ints(_offsets(lens))
    outs = [torch.empty_like(a) for a in alone]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for (q, k, v), o, s in zip(sets, outs, streams):
            pkg.prompt_attention(pkg.BF16, _rows(q), _rows(k), _rows(v), _rows(o), off.data_ptr(), 2, 500, 8, 2, 64, stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(alone, outs))


def test_operators_run_where_their_buffers_are():
    """Buffers on another device than the current one: the call runs there and leaves the current device as it was."""
    if torch.cuda.device_count() < 2:
        pytest.skip("needs 2 GPUs")
    g = torch.Generator(device="cuda:1").manual_seed(1)
    q, k, v = (torch.randn(90, h, 64, generator=g, device="cuda:1").to(BF16) for h in (4, 2, 2))
    out, off = torch.empty_like(q), torch.tensor([0, 90], dtype=torch.int32, device="cuda:1")
    torch.cuda.synchronize(1)
    with torch.cuda.device(0):
        pkg.prompt_attention(pkg.BF16, _rows(q), _rows(k), _rows(v), _rows(out), off.data_ptr(), 1, 90, 4, 2, 64, stream=torch.cuda.current_stream(1).cuda_stream)
        assert torch.cuda.current_device() == 0
    torch.cuda.synchronize(1)
    want, bound = R.attend(q, k, v, torch.ones(90, 90, device="cuda:1").tril().bool(), 0.125, BF16)
    _within(out, want, bound)


def test_refusals_on_a_device():
    q = torch.zeros(4, 2, 64, dtype=BF16, device="cuda")
    off, host = _ints([0, 4]), torch.zeros(4, 2, 64, dtype=BF16)
    ok = dict(dtype=pkg.BF16, q=_rows(q), k=_rows(q), v=_rows(q), out=_rows(q), offsets=off.data_ptr(), n=1, rows=4, num_heads=2, kv_heads=2, head_dim=64)
    for bad, text in ((dict(k=_rows(host)), "k is not a device address"), (dict(offsets=0), "offsets is null"),
                      (dict(v=pkg.Rows(q.data_ptr() + 2, 128, 64)), "v must be aligned to 16"), (dict(offsets=16), "offsets is not a device address")):
        with pytest.raises(pkg._lib.ShahdError, match=text):
            pkg.prompt_attention(**{**ok, **bad})
    table, pool = _ints([0] * 8), torch.zeros(8, 2, 2, 64, 64, dtype=BF16, device="cuda")
    cache = pkg.KvCache(pool.data_ptr(), pool.stride(0), table.data_ptr(), 8, 8, 2, 64)
    need = pkg.tree_attention_workspace(1, 4, 2, cache)
    mask = torch.zeros(4, dtype=torch.int64, device="cuda")
    tree = dict(dtype=pkg.BF16, q=_rows(q), k=_rows(q), v=_rows(q), out=_rows(q), cache=cache, lengths=off.data_ptr(), masks=mask.data_ptr(), offsets=off.data_ptr(), n=1,
                rows=4, max_nodes=4, num_heads=2, workspace=pool.data_ptr(), workspace_bytes=need)
    if need:
        with pytest.raises(pkg._lib.ShahdError, match="bytes of workspace"):
            pkg.tree_attention(**{**tree, "workspace_bytes": need - 1})
        with pytest.raises(pkg._lib.ShahdError, match="workspace is null"):
            pkg.tree_attention(**{**tree, "workspace": 0})
    with pytest.raises(pkg._lib.ShahdError, match="masks must be aligned to 8"):
        pkg.tree_attention(**{**tree, "masks": mask.data_ptr() + 4})
    with pkg.Rope(64) as rope, pytest.raises(pkg._lib.ShahdError, match="positions is null"):
        rope.apply(pkg.BF16, 4, 0, k=_rows(q), k_out=_rows(q), kv_heads=2)
    with pytest.raises(pkg._lib.ShahdError, match="uniforms is null"):
        pkg.verify_tree(pkg.BF16, q.data_ptr(), q.data_ptr(), 64, off.data_ptr(), off.data_ptr(), 0, off.data_ptr(), 1, 4, off.data_ptr(), off.data_ptr(), off.data_ptr())
    with pkg.FusedAttention(2, 4, 2, 64, 16) as op:
        with pytest.raises(pkg._lib.ShahdError, match="not in 0 .. 16"):
            op.set_lengths([3, 17])
        with pytest.raises(pkg._lib.ShahdError, match="1 <= n <= 2"):
            op.set_lengths([1, 1, 1])
        op.set_lengths([16, 0])
        assert (op.length(0), op.length(1)) == (16, 0)
    # empty calls launch nothing and succeed
    pkg.prompt_attention(**{**ok, "n": 0}), pkg.prompt_attention(**{**ok, "rows": 0})
    pkg.tree_attention(**{**tree, "rows": 0})
    assert bool((q == 0).all())

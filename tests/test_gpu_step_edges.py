"""The operators of a serving step over shared pages at the ends of their ranges: values, layouts and buffers that the other tests do not reach."""
import math

import numpy as np
import pytest

from tests.helpers import pkg

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
from tests import serving_refs as R  # noqa: E402
from tests import step_refs as S  # noqa: E402
from tests.test_gpu_serving_ops import BF16, CODE, F16, F32, _cache_of, _gen, _held, _ints, _normal, _offsets, _rows, _stream, _within  # noqa: E402
from tests.test_gpu_step_ops import _check_chunk, _check_fork, _chunk, _chunk_case, _pool  # noqa: E402


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    torch.cuda.synchronize()
    assert pkg.load().ShahdDeviceErrorFlag() == 0


# ---- logits --------------------------------------------------------------------------------------------------------

REPETITIONS = [1.3, 0.7, 3.0, 1e-30, 1e-39, 2.0**-149, 1.7e38, 3.4e38]  # below 2^-128 and above 2^126 a reciprocal leaves the range


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("each", [1, 80], ids=["rows on their own", "rows of a sequence together"])
def test_repetition_is_one_division_or_one_product(dtype, each):
    """Where nothing else is asked for, a known token's logit is the 32-bit quotient or product, bit for bit."""
    g, V, n = _gen(41), 4000, len(REPETITIONS)
    x = (_normal(g, n * each, V) * 3).to(dtype)
    x[:, 0], x[:, 2] = 2.0**-24, -(2.0**-24)  # quotients by small numbers stay finite in 32 bits
    history, held, seqs = _ints(list(range(0, V, 2)) * n), _ints([V // 2] * n), _ints(np.arange(n * each) // each)
    rep = torch.tensor(REPETITIONS, dtype=F32)
    out, dev = torch.empty_like(x), rep.cuda()
    pkg.adjust_logits(CODE[dtype], x.data_ptr(), out.data_ptr(), n * each, V, n, sequences=seqs.data_ptr(), history=history.data_ptr(), history_stride=V // 2,
                      history_lengths=held.data_ptr(), repetition=dev.data_ptr(), stream=_stream())
    wide = x.float().cpu()
    r = rep.repeat_interleave(each)[:, None]
    want = torch.where(wide > 0, wide / r, wide * r)
    want[:, 1::2] = wide[:, 1::2]
    assert bool(want[:, ::2].isfinite().any(1).all())
    assert torch.equal(out.cpu(), want.to(dtype))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shift,stride", [(0, 0), (1, 0), (3, 5), (0, 8)])
@pytest.mark.parametrize("mode", ["in place", "another buffer", "two halves"])
def test_logits_leave_what_lies_around_their_rows(dtype, shift, stride, mode):
    """The values in front of the first row, between rows and behind the last one's stride."""
    g, V, rows = _gen(43), 4099, 7
    wide = (2 * V if mode == "two halves" else V) + stride
    flat = (4 * _normal(g, shift + rows * wide + 64)).to(dtype)
    other = flat if mode != "another buffer" else torch.full_like(flat, 7.0)
    at = shift + (V if mode == "two halves" else 0)  # of the results
    before, source = other.clone(), flat.clone()
    history, held, pres = _ints(range(0, V, 3)), _ints([V // 3]), torch.full((1,), 2.0, device="cuda")
    seqs, size = _ints([0] * 3 + [-1] + [0] * 3), flat.element_size()
    pkg.adjust_logits(CODE[dtype], flat.data_ptr() + shift * size, other.data_ptr() + at * size, rows, V, 1, sequences=seqs.data_ptr(), history=history.data_ptr(),
                      history_stride=V // 3, history_lengths=held.data_ptr(), presence=pres.data_ptr(), logits_stride=wide, out_stride=wide, stream=_stream())
    want = before.clone()
    for i in (0, 1, 2, 4, 5, 6):
        row = source[shift + i * wide:shift + i * wide + V].clone()
        row[: 3 * (V // 3) : 3] = (row[: 3 * (V // 3) : 3].float() - 2).to(dtype)
        want[at + i * wide:at + i * wide + V] = row
    assert torch.equal(other, want)
    if mode == "another buffer":
        assert torch.equal(flat, source)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("V,rows,n", [(131072, 3, 3), (151936, 64, 16), (262144, 2, 2), (262147, 40, 10)], ids=str)
@pytest.mark.parametrize("held", [700, 32768])
def test_logits_of_large_vocabularies(dtype, V, rows, n, held):
    """Rows of many slices, on their own and in groups, histories in 16-bit and 32-bit cells."""
    rng, g = np.random.default_rng(V + held), _gen(V)
    x = (4 * _normal(g, rows, V)).to(dtype)
    history = rng.integers(0, V, (n, held))
    history[:, ::5] = rng.integers(0, 40, history[:, ::5].shape)
    history[:, 1::50] = V - 1
    prompt, seqs = rng.integers(0, held, n), np.sort(rng.integers(0, n, rows))
    bt, bv = rng.integers(0, V, 4 * n), rng.normal(size=4 * n).astype(np.float32)
    allowed = rng.random((2, V)) < 0.7
    full = np.zeros((2, -(-V // 32) * 32), np.uint8)
    full[:, :V] = allowed
    mrow = rng.integers(-1, 2, rows)
    rep, pres, freq = (torch.tensor(rng.uniform(a, b, n), dtype=F32, device="cuda") for a, b in ((0.7, 1.5), (-1, 1), (-0.5, 0.5)))
    dev = [_ints(history.ravel()), _ints([held] * n), _ints(prompt), _ints(seqs), _ints(4 * np.arange(n + 1)), _ints(bt), torch.tensor(bv, device="cuda"),
           torch.tensor(np.packbits(full, axis=1, bitorder="little").view(np.int32), device="cuda"), _ints(mrow)]
    out = torch.empty_like(x)
    pkg.adjust_logits(CODE[dtype], x.data_ptr(), out.data_ptr(), rows, V, n, sequences=dev[3].data_ptr(), history=dev[0].data_ptr(), history_stride=held,
                      history_lengths=dev[1].data_ptr(), prompt_lengths=dev[2].data_ptr(), repetition=rep.data_ptr(), presence=pres.data_ptr(), frequency=freq.data_ptr(),
                      bias_offsets=dev[4].data_ptr(), bias_tokens=dev[5].data_ptr(), bias_values=dev[6].data_ptr(), bias_entries=4 * n, masks=dev[7].data_ptr(), mask_count=2,
                      mask_rows=dev[8].data_ptr(), stream=_stream())
    for i in sorted({0, 1, rows // 2, rows - 1}):
        s = int(seqs[i])
        want, bound = S.adjust(x[i].double(), history[s].tolist(), int(prompt[s]), rep[s].double(), pres[s].double(), freq[s].double(),
                               list(zip(bt[4 * s:4 * s + 4].tolist(), bv[4 * s:4 * s + 4].tolist())),
                               torch.tensor(allowed[mrow[i]], device="cuda") if mrow[i] >= 0 else None, dtype)
        gone = want == -math.inf
        assert torch.equal(out[i] == -math.inf, gone)
        _within(out[i][~gone], want[~gone], bound[~gone])


# ---- norms of heads ------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("layout,d,r", [("interleaved", 64, 64), ("half", 64, 32), ("half", 64, 26), ("interleaved", 32, 6), ("half", 80, 24)])
@pytest.mark.parametrize("place", [False, True], ids=["", "in place"])
def test_norms_of_warps_that_walk_over_rows_that_are_passed_over(dtype, kind, layout, d, r, place):
    """More rows than warps run at once, so that each goes from row to row with the next one's values on their way: rows of negative
    position, rows in front of the first sequence and behind the last, whose values are not finite, and empty sequences among them."""
    g, N, H, Hk = _gen(d + r), 9000, 3, 2
    cdt = BF16 if dtype == F32 else dtype
    lens = [1700, 0, 3000, 1, 2500, 900]
    first, total = 31, sum(lens)
    offsets = [first + int(x) for x in _offsets(lens)]
    pool, table, cache = _cache_of(lens, Hk, d, cdt, g)
    q, k, v = ((2 * _normal(g, N, h, d) + 0.25).to(dtype) for h in (H, Hk, Hk))
    pos = torch.full((N,), 5, dtype=torch.int32, device="cuda")
    for s, n in enumerate(lens):
        pos[offsets[s]:offsets[s + 1]] = torch.randperm(n, generator=g, device="cuda").int()
    pos[torch.rand(N, generator=g, device="cuda") < 0.3] = -1
    pos[first + 100:first + 5000:2368] = -1  # the second row of some warps, and rows that follow each other on one
    pos[first + 200:first + 203] = -7
    keep = pos >= 0
    keep[:first] = keep[first + total:] = False
    for x in (q, k, v):
        x[~keep] = math.nan
    w = [1 + 0.3 * _normal(g, d) for _ in range(2)] + [0.2 * _normal(g, d) for _ in range(2)]
    norm = pkg.HeadNorm(kind, 1e-5, w[0].data_ptr(), w[1].data_ptr(), *([w[2].data_ptr(), w[3].data_ptr()] if kind == "layer" else []))
    old_q, old_k, before = q.clone(), k.clone(), pool.clone()
    q_out, k_out = (q, k) if place else (torch.full_like(q, 7.0), torch.full_like(k, 7.0))
    with pkg.Rope(d, r, layout) as rope:
        rope.apply(CODE[dtype], N, pos.data_ptr(), q=_rows(q), q_out=_rows(q_out), num_heads=H, k=_rows(k), k_out=_rows(k_out), kv_heads=Hk, v=_rows(v), cache=cache,
                   offsets=_ints(offsets).data_ptr(), n=len(lens), norm=norm, stream=_stream())
    freq = R.frequencies(r)
    for x, y, i in ((old_q, q_out, 0), (old_k, k_out, 1)):
        want, bound = S.norm_rope(x[keep], pos[keep], freq, layout, 1.0, kind, 1e-5, w[i], w[2 + i] if kind == "layer" else None, dtype)
        _within(y[keep], want, bound)
        assert bool(y[~keep].isnan().all() if place else (y[~keep] == 7.0).all())
    want, bound = S.norm_rope(old_k[keep], pos[keep], freq, layout, 1.0, kind, 1e-5, w[1], w[3] if kind == "layer" else None, cdt)
    full, off = torch.zeros(N, Hk, d, dtype=torch.float64, device="cuda"), torch.zeros(N, Hk, d, dtype=torch.float64, device="cuda")
    full[keep], off[keep] = want, bound
    held_rows = torch.zeros(pool.shape[0], 64, dtype=torch.bool, device="cuda")
    for s, n in enumerate(lens):
        rows = torch.arange(offsets[s], offsets[s + 1], device="cuda")
        rows = rows[keep[rows]]
        at = pos[rows].long()
        held_rows[table[s, at // 64].long(), at % 64] = True
        for h in range(Hk):
            held_k, held_v = _held(pool, table, s, n, h)
            _within(held_k[at], full[rows, h], off[rows, h])
            assert torch.equal(held_v[at], v[rows, h].to(cdt))
    apart = (pool.view(torch.int16) != before.view(torch.int16)).any(-1).any(2).any(2).any(1)  # [pages, 64]
    assert not bool((apart & ~held_rows).any())


# ---- chunks over the cache -----------------------------------------------------------------------------------------


@pytest.mark.parametrize("heads,n,most_rows", [((32, 8, 128), 16, 1500), ((16, 16, 128), 16, 1100), ((32, 8, 64), 16, 1500), ((16, 16, 64), 26, 1300), ((32, 8, 32), 16, 1500),
                                               ((64, 8, 64), 14, 900), ((32, 8, 128), 140, 200), ((28, 4, 64), 150, 300)], ids=str)
@pytest.mark.parametrize("blocks", [None, 400], ids=["", "head after head"])
def test_chunks_of_many_pairs_of_tiles(heads, n, most_rows, blocks):
    """A block of threads for every pair of tiles: sequences of many pairs, last pairs of one tile and of two, pages that are not there, an empty sequence;
    head after head where the table has room for more than the L2 cache holds; repeated bit for bit."""
    H, Hk, d = heads
    rng, G = np.random.default_rng(H + d + n), H // Hk
    span, slots = 2 * (128 // G), 148 * (1 if d == 128 else 2)
    rows, lengths = rng.integers(1, most_rows + 1, n).tolist(), rng.integers(0, 300, n).tolist()
    rows[1], rows[2], rows[3], rows[-1] = 0, most_rows, span + 1, 3 * span // 2
    lengths[2], lengths[4] = 0, 299
    dtype = BF16 if Hk == 8 else F16
    q, pool, table, cache = _chunk_case(_gen(n + d), lengths, rows, heads, dtype, spread=1)
    table[2, 1], table[n - 1, 0], table[5, 0] = -1, pool.shape[0], -9
    width = table.shape[1]
    if blocks:
        table = torch.cat([table, torch.full((n, blocks - width), -1, dtype=torch.int32, device="cuda")], 1)
        cache = pkg.KvCache(cache.pool, cache.page_stride, table.data_ptr(), blocks, cache.pages, Hk, d)
        assert n * blocks * 64 * Hk * 2 * d * 2 > 126e6
    assert min((sum(rows) + 2) // span + n, n * -(-most_rows // span)) * Hk >= 4 * slots  # as many pairs as this layout begins at
    assert pkg.chunk_attention_workspace(n, sum(rows) + 2, most_rows, H, cache) == 0
    out = _chunk(q, cache, lengths, rows, dtype)
    _check_chunk(q, pool, table, lengths, rows, out, dtype, seqs={0, 2, 3, 4, 5, 6, n - 1})
    assert bool((out[sum(rows):] == 7.0).all())
    assert torch.equal(out, _chunk(q, cache, lengths, rows, dtype))


# ---- pages ---------------------------------------------------------------------------------------------------------


def test_room_that_a_fork_gave_is_free_again_unless_the_lengths_cover_it():
    view, pool = _pool(12, 2, 1, 64, _gen(44))
    table, missing_room = np.full((1, 6), -1, np.int64), [64, 64]
    table[0, 0] = 5
    room, _ = _check_fork(view, pool, table, [64], [0, 0], missing_room, [200, 300])
    assert room.tolist() == [[5, 0, 1, 2, -1, -1], [5, 3, 4, 6, 7, -1]]
    # by their cached positions alone the pages beyond are free, although the table names them
    again, _ = _check_fork(view, pool, room, [64, 64], [1, 0], [64, 64], [128, 128])
    assert again.tolist() == [[5, 0, -1, -1, -1, -1], [5, 1, -1, -1, -1, -1]]
    # by lengths that cover the room they are held, and go with those that keep them
    kept, _ = _check_fork(view, pool, room, [200, 300], [1, 0], [300, 200], [300, 384])
    assert kept.tolist() == [[5, 3, 4, 6, 7, -1], [5, 0, 1, 2, 8, 9]]

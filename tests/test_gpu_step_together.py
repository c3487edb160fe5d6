"""The operators of a serving step over shared pages together, as a server runs them: forked conversations, further parts of prompts
and decode steps in one call, adjusted logits; on a FusedAttention operator's cache; captured, on two streams, on another device."""
import numpy as np
import pytest

from tests.helpers import pkg

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
from tests import serving_refs as R  # noqa: E402
from tests import step_refs as S  # noqa: E402
from tests.test_gpu_serving_ops import BF16, F16, F32, _gen, _ints, _normal, _offsets, _rows, _stream, _within  # noqa: E402


@pytest.fixture(autouse=True)
def _no_device_error():
    yield
    torch.cuda.synchronize()
    assert pkg.load().ShahdDeviceErrorFlag() == 0


class Server:
    """A pool of `layers` layers and what a step of it takes; `history` keeps each sequence's keys and values per layer beside it."""

    def __init__(self, layers, pages, blocks, H, Hk, d, seed):
        self.g = _gen(seed)
        self.layers, self.pages, self.blocks, self.H, self.Hk, self.d = layers, pages, blocks, H, Hk, d
        self.memory = torch.full((pages, layers, Hk, 2, 64, d), float("nan"), dtype=BF16, device="cuda")
        self.pool = pkg.PagePool(self.memory.data_ptr(), self.memory.stride(0), self.memory.stride(1), layers, pages, Hk, d)
        self.table, self.lengths, self.n = torch.zeros(0, blocks, dtype=torch.int32, device="cuda"), [], 0
        self.history = []  # per sequence and layer: keys, values [length, Hk, d]
        self.norm_w = [1 + 0.2 * _normal(self.g, d) for _ in range(2)]
        self.norm = pkg.HeadNorm("rms", 1e-6, self.norm_w[0].data_ptr(), self.norm_w[1].data_ptr())
        self.rope = pkg.Rope(d, layout="half")

    def fork(self, parents, keep, need):
        new_n = len(parents)
        new, missing = torch.empty(new_n, self.blocks, dtype=torch.int32, device="cuda"), torch.empty(new_n, dtype=torch.int32, device="cuda")
        size = pkg.pages_workspace(self.pages, new_n)
        ws = torch.empty(size, dtype=torch.uint8, device="cuda")
        old, p, k, m = _ints(self.lengths), _ints(parents), _ints(keep), _ints(need)
        table = self.table
        pkg.pages_fork(self.pool, table.data_ptr() if self.n else 0, old.data_ptr() if self.n else 0, self.n, self.blocks, p.data_ptr(), k.data_ptr(), m.data_ptr(), new_n,
                       new.data_ptr(), missing.data_ptr(), ws.data_ptr(), size, _stream())
        assert missing.tolist() == [0] * new_n
        self.history = [[(kk[:c], vv[:c]) for kk, vv in self.history[q]] if 0 <= q < self.n
                        else [(torch.zeros(0, self.Hk, self.d, dtype=BF16, device="cuda"),) * 2 for _ in range(self.layers)] for q, c in zip(parents, keep)]
        self.table, self.lengths, self.n = new, list(keep), new_n

    def compact(self, need):
        """need: positions that have pages, those for what comes among them."""
        size = pkg.pages_workspace(self.pages)
        ws, used, ln = torch.empty(size, dtype=torch.uint8, device="cuda"), _ints([0]), _ints(need)
        pkg.pages_compact(self.pool, self.table.data_ptr(), ln.data_ptr(), self.n, self.blocks, self.table.data_ptr(), used.data_ptr(), ws.data_ptr(), size, _stream())
        assert int(self.table.max()) < used.item()

    def step(self, rows):
        """rows[s] new rows of each sequence through every layer; each layer's attention is checked."""
        n, N, off, ln = self.n, sum(rows), _ints(_offsets(rows)), _ints(self.lengths)
        pos = _ints([x + i for x, t in zip(self.lengths, rows) for i in range(t)])
        for layer in range(self.layers):
            view = self.memory[:, layer]
            cache = pkg.KvCache(view.data_ptr(), self.memory.stride(0), self.table.data_ptr(), self.blocks, self.pages, self.Hk, self.d)
            q, k, v = (_normal(self.g, N, h, self.d, dtype=BF16) for h in (self.H, self.Hk, self.Hk))
            qr, out = torch.empty_like(q), torch.empty_like(q)
            self.rope.apply(pkg.BF16, N, pos.data_ptr(), q=_rows(q), q_out=_rows(qr), num_heads=self.H, k=_rows(k), kv_heads=self.Hk, v=_rows(v), cache=cache,
                            offsets=off.data_ptr(), n=n, norm=self.norm, stream=_stream())
            size = pkg.chunk_attention_workspace(n, N, max(rows), self.H, cache)
            ws = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
            pkg.chunk_attention(pkg.BF16, _rows(qr), _rows(out), cache, ln.data_ptr(), off.data_ptr(), n, N, max(rows), self.H, workspace=ws.data_ptr(),
                                workspace_bytes=size, stream=_stream())
            torch.cuda.current_stream().synchronize()
            freq = R.frequencies(self.d)
            want_q, bound_q = S.norm_rope(q, pos, freq, "half", 1.0, "rms", 1e-6, self.norm_w[0], None, BF16)
            _within(qr, want_q, bound_q)
            at = 0
            for s, t in enumerate(rows):
                if t == 0:
                    continue
                name = self.table[s, torch.arange(self.lengths[s] + t, device="cuda") // 64].long()
                assert bool((name >= 0).all())
                held = view[name, :, :, torch.arange(self.lengths[s] + t, device="cuda") % 64]  # [positions, Hk, 2, d]
                kk, vv = held[:, :, 0], held[:, :, 1]
                before = self.history[s][layer]
                L = self.lengths[s]
                assert torch.equal(kk[:L], before[0]) and torch.equal(vv[:L], before[1])  # nobody has written over what it keeps
                assert torch.equal(vv[L:], v[at:at + t])
                want_k, bound_k = S.norm_rope(k[at:at + t], pos[at:at + t], freq, "half", 1.0, "rms", 1e-6, self.norm_w[1], None, BF16)
                _within(kk[L:], want_k, bound_k)
                seen = torch.arange(L + t, device="cuda") <= L + torch.arange(t, device="cuda")[:, None]
                want, bound = R.attend(qr[at:at + t], kk, vv, seen, self.d ** -0.5, BF16)
                _within(out[at:at + t], want, bound)
                self.history[s][layer] = (kk, vv)
                at += t
        self.lengths = [x + t for x, t in zip(self.lengths, rows)]


@pytest.mark.parametrize("H,Hk,d", [(8, 2, 64), (4, 4, 32), (8, 1, 128)])
def test_conversations_that_fork_grow_and_end(H, Hk, d):
    s = Server(2, 60, 12, H, Hk, d, 1)
    s.fork([-1, -1], [0, 0], [150, 90])
    s.step([150, 90])                                          # two prompts
    s.fork([0, 0, 1, 0], [150, 150, 90, 150], [151, 180, 300, 151])
    s.step([1, 30, 210, 1])                                    # answers of the first, a further part of the second
    s.fork([0, 1, 1, 2], [151, 180, 64, 300], [152, 181, 65, 301])
    s.step([1, 1, 1, 1])
    s.fork([3, 0], [290, 152], [291, 280])                     # two have ended, one is cut back
    s.compact([291, 280])
    s.step([1, 128])
    s.fork([1, 1, -1], [280, 280, 0], [281, 281, 700])
    s.compact(s.lengths)                                       # pages for what comes are let go
    s.fork([0, 1, 2], [280, 280, 0], [281, 281, 700])          # and come again
    s.step([1, 1, 700])


def test_a_step_on_the_fused_attention_cache():
    """Prompts by the operator itself, a further part of each through chunk_attention, and its own decode steps from there."""
    H, Hk, d, n, T = 8, 2, 64, 3, 100
    g, more = _gen(2), [70, 1, 129]
    with pkg.FusedAttention(n, H, Hk, d, 400, 10000.0) as op, pkg.Rope(d) as rope:
        st = _stream()
        q, k, v = (_normal(g, n, T, h, d) for h in (H, Hk, Hk))
        out = torch.empty_like(q)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            st = _stream()
            op.prefill(q.data_ptr(), k.data_ptr(), v.data_ptr(), n, T, out.data_ptr(), st)
            cache, N = op.cache(), sum(more)
            q1, k1, v1 = (_normal(g, N, h, d, dtype=BF16) for h in (H, Hk, Hk))
            off, ln, pos = _ints(_offsets(more)), _ints([T] * n), _ints([T + i for t in more for i in range(t)])
            qr, o1 = torch.empty_like(q1), torch.empty_like(q1)
            rope.apply(pkg.BF16, N, pos.data_ptr(), q=_rows(q1), q_out=_rows(qr), num_heads=H, k=_rows(k1), v=_rows(v1), kv_heads=Hk, cache=cache, offsets=off.data_ptr(),
                       n=n, stream=st)
            size = pkg.chunk_attention_workspace(n, N, 129, H, cache)
            ws = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
            pkg.chunk_attention(pkg.BF16, _rows(qr), _rows(o1), cache, ln.data_ptr(), off.data_ptr(), n, N, 129, H, workspace=ws.data_ptr(), workspace_bytes=size, stream=st)
            lengths = [T + t for t in more]
            op.set_lengths(lengths, st)
            q2, k2, v2 = (_normal(g, n, h, d) for h in (H, Hk, Hk))
            o2 = torch.empty_like(q2)
            op.decode(q2.data_ptr(), k2.data_ptr(), v2.data_ptr(), n, o2.data_ptr(), st)
            side.synchronize()
        freq, at = R.frequencies(d), _offsets(more)
        for s in range(n):
            first, _ = R.rotate(k[s], torch.arange(T, device="cuda"), freq, "interleaved")
            p1 = torch.arange(T, T + more[s], device="cuda")
            second, _ = R.rotate(k1[at[s]:at[s + 1]], p1, freq, "interleaved")
            kk, vv = torch.cat([first.to(BF16), second.to(BF16)]), torch.cat([v[s].to(BF16), v1[at[s]:at[s + 1]]])
            seen = torch.arange(len(kk), device="cuda") <= p1[:, None]
            want, bound = R.attend(qr[at[s]:at[s + 1]], kk, vv, seen, d ** -0.5, BF16)
            # keys that lie within an error of a border are rounded the other way: a step of 2^-8 of a key's value more in the scores
            apart = 2.0 ** -7 * d ** -0.5 * float((qr[at[s]:at[s + 1]].double().abs().amax(0) * kk.double().abs().amax()).sum(-1).max())
            _within(o1[at[s]:at[s + 1]], want, bound + 1e-4 * apart * vv.double().abs().max())
            p2 = torch.tensor([lengths[s]], device="cuda")
            q2w, k2w = (R.rotate(x[s:s + 1], p2, freq, "interleaved")[0] for x in (q2, k2))
            want, _ = R.attend(q2w, torch.cat([kk, k2w.to(BF16)]), torch.cat([vv, v2[s:s + 1].to(BF16)]), torch.ones(1, len(kk) + 1, dtype=torch.bool, device="cuda"),
                               d ** -0.5, BF16)
            # the operator's own bar: 2e-2 of the output's range (tests/test_gpu_fused_attention.py)
            assert float((o2[s].double() - want[0]).abs().max()) < 2e-2 * float(want.max() - want.min())


class Step:
    """Fork, norm + rope + append, chunk attention and logits on buffers of its own, as one call."""

    def __init__(self, seed, n=3, H=8, Hk=2, d=64, V=900, wide=None, device="cuda"):
        self.n, self.H, self.Hk, self.d, self.V, self.pages, self.blocks = n, H, Hk, d, V, 8 * n + 26, wide or 8
        dev = dict(device=device)
        self.g = torch.Generator(device=device).manual_seed(seed)
        ints = lambda x: torch.tensor(x, dtype=torch.int32, **dev)  # noqa: E731
        self.memory = torch.zeros(self.pages, 1, Hk, 2, 64, d, dtype=F16, **dev)
        self.pool = pkg.PagePool(self.memory.data_ptr(), self.memory.stride(0), 0, 1, self.pages, Hk, d)
        self.table = torch.full((n, self.blocks), -1, dtype=torch.int32, **dev)
        self.table[:, :6] = torch.randperm(self.pages, generator=self.g, **dev).int()[: n * 6].view(n, 6)
        self.new = torch.empty_like(self.table)
        self.lengths, self.parents, self.keep, self.need = (ints([0] * n) for _ in range(4))
        self.missing = ints([0] * n)
        self.rows, self.offsets = [2] * n, ints(_offsets([2] * n))
        N = 2 * n
        self.pos = ints([0] * N)
        self.q, self.k, self.v = (torch.zeros(N, h, d, dtype=F16, **dev) for h in (H, Hk, Hk))
        self.qr, self.out = torch.empty_like(self.q), torch.empty_like(self.q)
        self.logits, self.seqs = torch.zeros(N, V, **dev), ints(np.repeat(np.arange(n), 2))
        self.adjusted = torch.empty_like(self.logits)
        self.hist, self.held = torch.zeros(n, 40, dtype=torch.int32, **dev), ints([0] * n)
        self.rep, self.pres = torch.ones(n, **dev), torch.zeros(n, **dev)
        self.cache = pkg.KvCache(self.memory.data_ptr(), self.memory.stride(0), self.new.data_ptr(), self.blocks, self.pages, Hk, d)
        self.fork_bytes, self.chunk_bytes = pkg.pages_workspace(self.pages, n), pkg.chunk_attention_workspace(n, N, 2, H, self.cache)
        self.ws = [torch.empty(max(x, 1), dtype=torch.uint8, **dev) for x in (self.fork_bytes, self.chunk_bytes)]
        self.norm, self.rope = pkg.HeadNorm("layer", 1e-5), pkg.Rope(d)

    def new_inputs(self):
        for x in (self.q, self.k, self.v, self.logits, self.memory):
            x.normal_(generator=self.g)
        draw = lambda top, n: torch.randint(0, top, (n,), generator=self.g, device=self.q.device, dtype=torch.int32)  # noqa: E731
        self.lengths.copy_(draw(380, self.n)), self.parents.copy_(draw(self.n, self.n))
        self.keep.copy_(self.lengths[self.parents.long()]), self.need.copy_(self.keep + 2)
        self.pos.copy_(torch.stack([self.keep, self.keep + 1], 1).view(-1))
        self.hist.copy_(draw(self.V, 40 * self.n).view(self.n, 40)), self.held.copy_(draw(41, self.n))
        self.rep.copy_(1 + torch.rand(self.n, generator=self.g, device=self.q.device)), self.pres.copy_(torch.rand(self.n, generator=self.g, device=self.q.device))
        self.before = self.memory.clone()

    def run(self, stream):
        N = 2 * self.n
        pkg.pages_fork(self.pool, self.table.data_ptr(), self.lengths.data_ptr(), self.n, self.blocks, self.parents.data_ptr(), self.keep.data_ptr(), self.need.data_ptr(),
                       self.n, self.new.data_ptr(), self.missing.data_ptr(), self.ws[0].data_ptr(), self.fork_bytes, stream)
        self.rope.apply(pkg.F16, N, self.pos.data_ptr(), q=_rows(self.q), q_out=_rows(self.qr), num_heads=self.H, k=_rows(self.k), v=_rows(self.v), kv_heads=self.Hk,
                        cache=self.cache, offsets=self.offsets.data_ptr(), n=self.n, norm=self.norm, stream=stream)
        pkg.chunk_attention(pkg.F16, _rows(self.qr), _rows(self.out), self.cache, self.keep.data_ptr(), self.offsets.data_ptr(), self.n, N, 2, self.H,
                            workspace=self.ws[1].data_ptr(), workspace_bytes=self.chunk_bytes, stream=stream)
        pkg.adjust_logits(pkg.F32, self.logits.data_ptr(), self.adjusted.data_ptr(), N, self.V, self.n, sequences=self.seqs.data_ptr(), history=self.hist.data_ptr(),
                          history_stride=40, history_lengths=self.held.data_ptr(), repetition=self.rep.data_ptr(), presence=self.pres.data_ptr(), stream=stream)

    def check(self):
        lengths, parents, keep, need = (x.tolist() for x in (self.lengths, self.parents, self.keep, self.need))
        want, lost, copies = S.fork(self.table.cpu().numpy(), lengths, parents, keep, need, self.pages)
        assert np.array_equal(self.new.cpu().numpy(), want) and not self.missing.any()
        wq, bq = S.norm_rope(self.q, self.pos, R.frequencies(self.d), "interleaved", 1.0, "layer", 1e-5, None, None, F16)
        _within(self.qr, wq, bq)
        for a, b, k in copies:
            self.before[b, ..., :k, :] = self.before[a, ..., :k, :]
        for s in range(self.n):
            at = torch.arange(keep[s] + 2, device=self.q.device)
            held = self.memory[self.new[s, at // 64].long(), 0, :, :, at % 64]
            assert torch.equal(held[: keep[s]], self.before[self.new[s, at // 64].long(), 0, :, :, at % 64][: keep[s]])
            seen = at <= keep[s] + torch.arange(2, device=self.q.device)[:, None]
            w, b = R.attend(self.qr[2 * s:2 * s + 2], held[:, :, 0], held[:, :, 1], seen, self.d ** -0.5, F16)
            _within(self.out[2 * s:2 * s + 2], w, b)
            for i in (2 * s, 2 * s + 1):
                w, b = S.adjust(self.logits[i].double(), self.hist[s, : self.held[s]].tolist(), 0, self.rep[s].double(), self.pres[s].double(),
                                torch.zeros((), dtype=torch.float64, device=self.q.device), [], None, F32)
                _within(self.adjusted[i], w, b)


@pytest.mark.parametrize("wide", [None, 2000])
def test_captured_step_follows_its_inputs(wide):
    """Two captured steps with workspaces of their own, replayed side by side on new inputs."""
    steps = [Step(5, wide=wide), Step(6, n=9, wide=wide) if wide else Step(6, n=5)]
    graphs = []
    for s in steps:
        s.new_inputs()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            s.run(_stream())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            s.run(_stream())
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(3):
        for s in steps:
            s.new_inputs()
        torch.cuda.synchronize()
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for s in steps:
            s.check()


def test_steps_on_two_streams_at_once():
    steps = [Step(7), Step(8, n=6)]
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(4):
        for s in steps:
            s.new_inputs()
        torch.cuda.synchronize()
        for _ in range(3):  # the same inputs again: the same results
            for stream, s in zip(streams, steps):
                s.run(stream.cuda_stream)
        torch.cuda.synchronize()
        for s in steps:
            s.check()


def test_steps_run_where_their_buffers_are():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs 2 GPUs")
    s = Step(9, device="cuda:1")
    s.new_inputs()
    torch.cuda.synchronize(1)
    with torch.cuda.device(0):
        s.run(torch.cuda.current_stream(1).cuda_stream)
        assert torch.cuda.current_device() == 0
    torch.cuda.synchronize(1)
    with torch.cuda.device(1):
        s.check()


def test_refusals_on_a_device():
    x, i = torch.zeros(4, 2, 64, dtype=BF16, device="cuda"), _ints([0] * 64)
    host = torch.zeros(4, 2, 64, dtype=BF16)
    pool = torch.zeros(8, 2, 2, 64, 64, dtype=BF16, device="cuda")
    cache = pkg.KvCache(pool.data_ptr(), pool.stride(0), i.data_ptr(), 8, 8, 2, 64)
    size = pkg.chunk_attention_workspace(1, 4, 4, 2, cache)
    chunk = dict(dtype=pkg.BF16, q=_rows(x), out=_rows(x), cache=cache, lengths=i.data_ptr(), offsets=i.data_ptr(), n=1, rows=4, max_rows=4, num_heads=2,
                 workspace=pool.data_ptr(), workspace_bytes=size)
    for bad, text in ((dict(q=_rows(host)), "q is not a device address"), (dict(offsets=0), "offsets is null"), (dict(lengths=i.data_ptr() + 2), "lengths must be aligned"),
                      (dict(out=pkg.Rows(x.data_ptr() + 2, 128, 64)), "out must be aligned to 16"), (dict(workspace=0), "workspace is null"),
                      (dict(cache=pkg.KvCache(pool.data_ptr(), pool.stride(0), 16, 8, 8, 2, 64)), "block_table is not a device address")):
        with pytest.raises(pkg._lib.ShahdError, match=text):
            pkg.chunk_attention(**{**chunk, **bad})
    with pkg.Rope(64) as rope:
        ok = dict(dtype=pkg.BF16, rows=4, positions=i.data_ptr(), q=_rows(x), q_out=_rows(x), num_heads=2)
        with pytest.raises(pkg._lib.ShahdError, match="q_weight is not a device address"):
            rope.apply(**ok, norm=pkg.HeadNorm(q_weight=host.data_ptr()))
        with pytest.raises(pkg._lib.ShahdError, match="positions is null"):
            rope.apply(**{**ok, "positions": 0}, norm=pkg.HeadNorm())
    logits = torch.zeros(4, 100, device="cuda")
    ok = dict(dtype=pkg.F32, logits=logits.data_ptr(), out=logits.data_ptr(), rows=4, vocab=100, n=4)
    for bad, text in ((dict(logits=host.data_ptr(), out=host.data_ptr()), "logits is not a device address"), (dict(out=0), "out is null"),
                      (dict(sequences=i.data_ptr() + 1), "sequences must be aligned"), (dict(masks=16, mask_count=1), "masks is not a device address")):
        with pytest.raises(pkg._lib.ShahdError, match=text):
            pkg.adjust_logits(**{**ok, **bad})
    pages = pkg.PagePool(pool.data_ptr(), pool.stride(0), 0, 1, 8, 2, 64)
    size = pkg.pages_workspace(8, 2)
    other = _ints([0] * 64)
    fork = dict(pool=pages, table=i.data_ptr(), lengths=i.data_ptr(), n=1, max_blocks=8, parents=i.data_ptr(), keep=i.data_ptr(), need=i.data_ptr(), new_n=2,
                new_table=other.data_ptr(), missing=other.data_ptr() + 128, workspace=x.data_ptr(), workspace_bytes=size)
    for bad, text in ((dict(parents=0), "parents is null"), (dict(workspace=x.data_ptr() + 8), "workspace must be aligned to 16"), (dict(keep=16), "keep is not a device")):
        with pytest.raises(pkg._lib.ShahdError, match=text):
            pkg.pages_fork(**{**fork, **bad})
    compact = dict(pool=pages, table=i.data_ptr(), lengths=i.data_ptr(), n=1, max_blocks=8, new_table=i.data_ptr(), used=0, workspace=x.data_ptr(), workspace_bytes=size)
    with pytest.raises(pkg._lib.ShahdError, match="used is null"):
        pkg.pages_compact(**compact)

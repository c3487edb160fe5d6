"""Measured cases of the operators of a serving step over shared pages: forking and compacting the pages of a cache, norms of the
query and key heads with the rotary positions and the append, attention of chunks of new tokens over the cache, and penalties,
biases and grammar masks on the logits.

`run` computes an operator from elementary torch operations (32 bits, 64 where positions need them), or, with `own` set, calls
the framework's kernels. `exact` restates the definitions in 64 bits, sequence by sequence."""
import importlib
import math
import random

import numpy as np
import torch

own = False

PAGE = 64  # positions of a cache page
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---- cases ---------------------------------------------------------------------------------------------------------


def listed():
    return [
        # one user's next message in a conversation, Phase2Modern-style shape: latency
        _chunk("chunk one user", "bf16", 1, 1, 96, 96, 1700, 1700, 16, 4, 64),
        # a server's mixed step: most sequences add one token, some a part of their prompt
        _chunk("chunk mixed step", "bf16", 48, 6, 200, 512, 0, 1500, 16, 4, 64),
        # parts of long documents over what is cached of them, wide heads
        _chunk("chunk long documents", "f16", 4, 4, 1500, 2048, 10000, 24000, 32, 8, 128),
        # one decode step of 64 sequences of the Phase2Modern-style shape: latency
        _norm("norm step", "bf16", 64, 1, 1, 16, 4, 64, 64, "interleaved", "rms"),
        # prompts in 32 bits, appended to the bf16 cache; means taken off, with biases
        _norm("norm prompts f32", "f32", 16, 700, 1024, 16, 4, 64, 64, "half", "layer"),
        # long contexts, wide heads
        _norm("norm long context", "f16", 8, 6000, 8192, 32, 8, 128, 128, "half", "rms"),
        # a step of the MicroChat batch: penalties for what the conversations hold
        _logits("logits step", "f32", 64, 64, 4096, 511, 0, False),
        # a step over the Phase2Modern-style vocabulary with biases, and grammars for some rows
        _logits("logits batch", "f32", 256, 256, 32768, 2047, 100, True),
        # drafted rows of 16-bit logits, several for a sequence, a large odd vocabulary
        _logits("logits drafted rows", "bf16", 128, 512, 50257, 8000, 20, True),
        # beam search: 8 requests of 4 beams choose their parents, MicroChat shape
        _pages("pages beams", "fork", 32, 32, 4, 511, 1, 6, 4, 64),
        # 8 answers for each of 16 prompts, Phase2Modern-style shape (a page of all layers is 1 MiB)
        _pages("pages samples", "fork", 16, 128, 8, 1500, 512, 16, 4, 64),
        # a pool of one layer at the FusedAttention shape, half of it free after requests have ended
        _pages("pages compact", "compact", 256, 256, 1, 575, 2100, 1, 2, 64),
    ]


def draw(rng):
    kind = rng.choice(("chunk", "norm", "logits", "pages"))
    spread = rng.randrange(1 << 20)
    heads = rng.choice(((4, 4, 32), (4, 4, 64), (16, 4, 64), (8, 2, 64), (8, 1, 64), (12, 4, 64), (4, 2, 128), (16, 4, 128), (32, 8, 128)))
    if kind == "chunk":
        n, length, rows = _log(rng, 1, 256), _log(rng, 1, 24000), _log(rng, 1, 4000)
        length = max(1, min(length, 80_000_000 // (n * heads[1] * heads[2])))
        rows = max(1, min(rows, int(2e9 / (n * heads[0] * (length + 2000))), 40_000_000 // (n * heads[0] * heads[2])))
        return _chunk(None, rng.choice(("bf16", "f16")), n, rng.randint(1, n), max(1, rows // 3), rows, rng.choice((0, length // 2)), length, *heads, spread)
    if kind == "norm":
        n, most = _log(rng, 1, 256), _log(rng, 1, 4096)
        most = max(1, min(most, 50000 // n, 1_400_000 // (n * heads[0])))
        r = rng.choice((heads[2], heads[2] // 2, 2 * rng.randrange(1, heads[2] // 2)))
        return _norm(None, rng.choice(("bf16", "f16", "f32")), n, max(1, most // 3), most, *heads, r, rng.choice(("interleaved", "half")),
                     rng.choice(("rms", "layer")), spread)
    if kind == "logits":
        rows, vocab, held = _log(rng, 1, 400), _log(rng, 300, 32000), _log(rng, 1, 8000)
        return _logits(None, rng.choice(("f32", "bf16", "f16")), rng.randint(1, rows), rows, vocab, held, rng.choice((0, _log(rng, 1, 200))), rng.random() < 0.5,
                       spread)
    n, most = _log(rng, 1, 200), _log(rng, 1, 1500)
    layers, (_, kv_heads, dim) = rng.choice((1, 2, 6)), heads
    pages = max(1, 24_000_000 // (layers * kv_heads * dim * 128))  # that 48 MB hold
    if rng.random() < 0.4:
        n = min(n, pages)
        most = min(most, pages // n * PAGE)
        return _pages(None, "compact", n, n, 1, most, rng.randint(0, pages), layers, kv_heads, dim, spread)
    group, n = rng.randint(1, 8), min(n, 2 * pages)
    if rng.random() < 0.5:
        return _pages(None, "fork", n, n, group, most, rng.choice((0, 1, 100)), layers, kv_heads, dim, spread)
    n = max(1, n // group)
    return _pages(None, "fork", n, n * group, group, most, rng.choice((0, 1, 100)), layers, kv_heads, dim, spread)


def _log(rng, least, most):
    return int(round(math.exp(rng.uniform(math.log(least), math.log(most)))))


def _case(name, **values):
    return values if name is None else {"name": name, **values}


def _chunk(name, dtype, seqs, long, least, most, least_len, most_len, heads, kv_heads, dim, spread=1):
    """`long` of the sequences have least .. most new rows, the others one."""
    return _case(name, op="chunk", dtype=dtype, seqs=seqs, long=long, least=least, most=most, least_len=least_len, most_len=most_len, heads=heads, kv_heads=kv_heads,
                 dim=dim, spread=spread)


def _norm(name, dtype, seqs, least, most, heads, kv_heads, dim, rotary, layout, norm, spread=1):
    return _case(name, op="norm", dtype=dtype, seqs=seqs, least=least, most=most, heads=heads, kv_heads=kv_heads, dim=dim, rotary=rotary, layout=layout, norm=norm,
                 spread=spread)


def _logits(name, dtype, seqs, rows, vocab, held, biases, masked, spread=1):
    return _case(name, op="logits", dtype=dtype, seqs=seqs, rows=rows, vocab=vocab, held=held, biases=biases, masked=masked, spread=spread)


def _pages(name, what, seqs, new, group, most, room, layers, kv_heads, dim, spread=1):
    """room: positions that a forked sequence is to have pages for beyond those it keeps; for compact, pages that nobody holds."""
    return _case(name, op=what, dtype="bf16", seqs=seqs, new=new, group=group, most=most, room=room, layers=layers, kv_heads=kv_heads, dim=dim, spread=spread)


def _rows(case):
    """New rows of each sequence, and the positions cached before them."""
    r = random.Random(case["spread"])
    n = case["seqs"]
    if case["op"] == "chunk":
        many = set(r.sample(range(n), case["long"]))
        rows = [r.randint(case["least"], case["most"]) if i in many else 1 for i in range(n)]
        rows[min(many)] = case["most"]
        return rows, [r.randint(case["least_len"], case["most_len"]) for _ in range(n)]
    rows = [r.randint(case["least"], case["most"]) for _ in range(n)]
    rows[r.randrange(n)] = case["most"]
    return rows, [r.randint(0, 511) for _ in range(n)]


def _family(case):
    """Cached positions of the sequences; and for forks each new one's parent, what it keeps and what it is to have room for."""
    r = random.Random(case["spread"])
    lengths = [r.randint(1, case["most"]) for _ in range(case["seqs"])]
    lengths[0] = case["most"]
    if case["op"] == "compact":
        return lengths, [], [], []
    g = case["group"]
    if case["new"] == case["seqs"]:  # beams: a parent of the same group
        for i in range(case["seqs"]):
            lengths[i] = lengths[i // g * g]
        parents = [min(i // g * g + r.randrange(g), case["seqs"] - 1) for i in range(case["new"])]
    else:
        parents = [i // g for i in range(case["new"])]
    keep = [lengths[p] for p in parents]
    return lengths, parents, keep, [k + case["room"] for k in keep]


def _copied(case):
    """Rows of a page (of 64) that a fork copies, over all its new sequences."""
    _, parents, keep, room = _family(case)
    return sum(k % PAGE for i, (p, k, m) in enumerate(zip(parents, keep, room)) if m > k and p in parents[:i])


def work(case):
    size = TYPES[case["dtype"]].itemsize
    if case["op"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        held = case["seqs"] * (case["held"] * 3 // 4 * 4 + case["biases"] * 8)
        return {"bytes": 2 * rows * vocab * size + held + (rows * vocab // 16 if case["masked"] else 0), "flops": 4 * rows * vocab}
    line = 2 * case["kv_heads"] * case["dim"] * size  # a position's K and V of one layer
    if case["op"] == "fork":
        lengths, parents, keep, room = _family(case)
        return {"bytes": 2 * _copied(case) * line * case["layers"] + 4 * sum(-(-x // PAGE) for x in lengths + room), "flops": 0}
    if case["op"] == "compact":
        used = sum(-(-x // PAGE) for x in _family(case)[0])
        moved = used * case["room"] / (used + case["room"])  # held pages behind the first `used`
        return {"bytes": 2 * moved * PAGE * line * case["layers"] + 8 * used, "flops": 0}
    rows, cached = _rows(case)
    n, H, Hk, d = sum(rows), case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "norm":
        return {"bytes": n * ((2 * H + 2 * Hk) * d * size + 2 * Hk * d * 2 + 4), "flops": n * (H + Hk) * (4 * d + 3 * case["rotary"])}
    return {"bytes": 2 * n * H * d * size + sum(t + c for t, c in zip(rows, cached)) * line,
            "flops": sum(4 * d * H * (t * c + t * (t + 1) // 2) for t, c in zip(rows, cached))}


# ---- inputs --------------------------------------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = random.Random(seed)
    s = dict(case, dtype=TYPES[case["dtype"]])
    if case["op"] == "logits":
        return _prepare_logits(s, g)
    if case["op"] in ("fork", "compact"):
        return _prepare_pages(s, case, g, r)
    rows, cached = _rows(case)
    s["rows"], s["n"] = sum(rows), len(rows)
    starts = np.concatenate([[0], np.cumsum(rows)])
    s["offsets"] = _ints(starts)
    seq = np.repeat(np.arange(len(rows)), rows)
    s["seq"], s["within"] = (torch.tensor(x, device="cuda") for x in (seq, np.arange(sum(rows)) - starts[seq]))
    s["longest"] = max(rows)
    s["lengths"] = _ints(cached)
    s["q"] = _normal(g, s["rows"], s["heads"], s["dim"], dtype=s["dtype"])
    s["out"] = torch.empty_like(s["q"])
    _cache(s, g, r, [a + b for a, b in zip(cached, rows)], torch.bfloat16 if s["dtype"] == torch.float32 else s["dtype"])
    if case["op"] == "norm":
        s["k"], s["v"] = (_normal(g, s["rows"], s["kv_heads"], s["dim"], dtype=s["dtype"]) for _ in range(2))
        s["q"] *= 4.0  # heads of several magnitudes, as projections give them
        s["positions"] = (s["lengths"][s["seq"]] + s["within"]).to(torch.int32)
        s["weights"] = [1 + 0.2 * _normal(g, s["dim"]) for _ in range(2)] + [0.1 * _normal(g, s["dim"]) for _ in range(2)]
    if own:
        _own_state(s)
    return s


def _ints(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _table(r, positions, blocks, more):
    """Pages in an order of chance, `more` of them nobody's, and the tables that name them: (table, pages)."""
    count = sum(-(-p // PAGE) for p in positions) + more
    ids = list(range(count))
    r.shuffle(ids)
    table = np.full((len(positions), blocks), -1, dtype=np.int32)
    for i, p in enumerate(positions):
        k = -(-p // PAGE)
        table[i, :k] = ids[:k]
        del ids[:k]
    return _ints(table), count


def _cache(s, g, r, positions, dtype):
    s["blocks"] = max(1, -(-max(positions) // PAGE))
    s["table"], s["pages"] = _table(r, positions, s["blocks"], 3)
    s["pool"] = torch.empty(s["pages"], s["kv_heads"], 2, PAGE, s["dim"], dtype=dtype, device="cuda").normal_(generator=g)


def _prepare_pages(s, case, g, r):
    lengths, parents, keep, room = _family(case)
    s["n"], s["blocks"] = len(lengths), max(-(-x // PAGE) for x in lengths + room)
    fresh = sum(-(-m // PAGE) - k // PAGE for k, m in zip(keep, room)) if parents else case["room"]
    s["table"], s["pages"] = _table(r, lengths, s["blocks"], fresh + 2 if parents else fresh)
    if parents and s["new"] == s["n"]:  # beams of a request share what they had in common
        leader, b = torch.arange(s["n"], device="cuda") // s["group"] * s["group"], torch.arange(s["blocks"], device="cuda")
        s["table"] = torch.where(b < (_ints(lengths) // PAGE)[:, None], s["table"][leader], s["table"])
    s["pool"] = torch.empty(s["pages"], s["layers"], s["kv_heads"], 2, PAGE, s["dim"], dtype=s["dtype"], device="cuda").normal_(generator=g)
    s["lengths"], s["parents"], s["keep"], s["need"] = (_ints(np.array(x, dtype=np.int32)) for x in (lengths, parents, keep, room))
    s["new_table"] = torch.empty(max(s["new"], 1), s["blocks"], dtype=torch.int32, device="cuda")
    s["missing"], s["used"] = (torch.empty(k, dtype=torch.int32, device="cuda") for k in (max(s["new"], 1), 1))
    if own:
        _own_state(s)
    return s


def _prepare_logits(s, g):
    n, rows, vocab, held = s["seqs"], s["rows"], s["vocab"], s["held"]
    s["logits"] = (_normal(g, rows, vocab) * 3).to(s["dtype"])
    s["out"] = torch.empty_like(s["logits"])
    u = torch.rand(n, held, generator=g, device="cuda")
    s["history"] = (u ** 3 * vocab).to(torch.int32).clamp_(max=vocab - 1)  # some tokens come again and again
    s["held_lengths"] = torch.randint(held // 2, held + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
    s["prompt_lengths"] = (s["held_lengths"] * torch.rand(n, generator=g, device="cuda")).to(torch.int32)
    s["repetition"] = 1 + 0.3 * torch.rand(n, generator=g, device="cuda")
    s["presence"], s["frequency"] = (torch.rand(n, generator=g, device="cuda") for _ in range(2))
    s["sequences"] = _ints(np.arange(rows) * n // rows)
    s["entries"] = n * min(s["biases"], vocab)
    if s["entries"]:
        each = s["entries"] // n
        s["bias_offsets"] = _ints(np.arange(n + 1) * each)
        first = torch.rand(n, 1, generator=g, device="cuda")
        # every token of a list once: places that lie a fixed step apart
        s["bias_tokens"] = ((first * vocab).long() + torch.arange(each, device="cuda") * (vocab // each)).remainder(vocab).to(torch.int32).reshape(-1)
        s["bias_values"] = _normal(g, s["entries"]) * 4
    if s["masked"]:
        words = -(-vocab // 32)
        s["grammars"] = max(1, rows // 2)
        s["masks"] = torch.randint(-(1 << 31), 1 << 31, (s["grammars"], words), generator=g, device="cuda", dtype=torch.int32)
        s["mask_rows"] = torch.where(torch.arange(rows, device="cuda") % 4 == 3, -1, torch.arange(rows, device="cuda") % s["grammars"]).to(torch.int32)
    return s


def _own_state(s):
    """What a program keeps beside its tensors."""
    pkg = _pkg()
    if s["op"] in ("fork", "compact"):
        s["pages_of"] = pkg.PagePool(s["pool"].data_ptr(), s["pool"].stride(0), s["pool"].stride(1), s["layers"], s["pages"], s["kv_heads"], s["dim"])
        size = pkg.pages_workspace(s["pages"], s["new"])
    else:
        s["cache"] = pkg.KvCache(s["pool"].data_ptr(), s["pool"].stride(0), s["table"].data_ptr(), s["blocks"], s["pages"], s["kv_heads"], s["dim"])
        size = pkg.chunk_attention_workspace(s["n"], s["rows"], s["longest"], s["heads"], s["cache"]) if s["op"] == "chunk" else 0
    if s["op"] == "norm":
        s["plan"] = pkg.Rope(s["dim"], s["rotary"], s["layout"])
        w = [x.data_ptr() for x in s["weights"]]
        s["head_norm"] = pkg.HeadNorm(s["norm"], 1e-6, w[0], w[1], *(w[2:] if s["norm"] == "layer" else ()))
    s["workspace"] = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")


# ---- one pass ------------------------------------------------------------------------------------------------------


def _pkg():
    return importlib.import_module("shahd-llm-stack_b200")


def run(s):
    if own:
        calls = {"chunk": _own_chunk, "norm": _own_norm, "logits": _own_logits, "fork": _own_fork, "compact": _own_compact}
        return calls[s["op"]](s, _pkg(), torch.cuda.current_stream().cuda_stream)
    return {"chunk": _plain_chunk, "norm": _plain_norm, "logits": _plain_logits, "fork": _plain_fork, "compact": _plain_compact}[s["op"]](s)


def _type(s, pkg):
    return {torch.bfloat16: pkg.BF16, torch.float16: pkg.F16, torch.float32: pkg.F32}[s["dtype"]]


def _of(t, pkg):
    return pkg.Rows(t.data_ptr(), t.stride(0), t.stride(1))


def _own_chunk(s, pkg, stream):
    pkg.chunk_attention(_type(s, pkg), _of(s["q"], pkg), _of(s["out"], pkg), s["cache"], s["lengths"].data_ptr(), s["offsets"].data_ptr(), s["n"], s["rows"],
                        s["longest"], s["heads"], workspace=s["workspace"].data_ptr(), workspace_bytes=s["workspace"].numel(), stream=stream)
    return s["out"]


def _own_norm(s, pkg, stream):
    s["plan"].apply(_type(s, pkg), s["rows"], s["positions"].data_ptr(), q=_of(s["q"], pkg), q_out=_of(s["out"], pkg), num_heads=s["heads"], k=_of(s["k"], pkg),
                    kv_heads=s["kv_heads"], v=_of(s["v"], pkg), cache=s["cache"], offsets=s["offsets"].data_ptr(), n=s["n"], norm=s["head_norm"], stream=stream)
    return s["out"], s["pool"]


def _own_logits(s, pkg, stream):
    more = {}
    if s["entries"]:
        more = dict(bias_offsets=s["bias_offsets"].data_ptr(), bias_tokens=s["bias_tokens"].data_ptr(), bias_values=s["bias_values"].data_ptr(),
                    bias_entries=s["entries"])
    if s["masked"]:
        more.update(masks=s["masks"].data_ptr(), mask_rows=s["mask_rows"].data_ptr(), mask_count=s["grammars"])
    pkg.adjust_logits(_type(s, pkg), s["logits"].data_ptr(), s["out"].data_ptr(), s["rows"], s["vocab"], s["seqs"], sequences=s["sequences"].data_ptr(),
                      history=s["history"].data_ptr(), history_stride=s["held"], history_lengths=s["held_lengths"].data_ptr(),
                      prompt_lengths=s["prompt_lengths"].data_ptr(), repetition=s["repetition"].data_ptr(), presence=s["presence"].data_ptr(),
                      frequency=s["frequency"].data_ptr(), stream=stream, **more)
    return s["out"]


def _own_fork(s, pkg, stream):
    pkg.pages_fork(s["pages_of"], s["table"].data_ptr(), s["lengths"].data_ptr(), s["n"], s["blocks"], s["parents"].data_ptr(), s["keep"].data_ptr(),
                   s["need"].data_ptr(), s["new"], s["new_table"].data_ptr(), s["missing"].data_ptr(), s["workspace"].data_ptr(), s["workspace"].numel(), stream)
    return s["new_table"], s["missing"], s["pool"]


def _own_compact(s, pkg, stream):
    pkg.pages_compact(s["pages_of"], s["table"].data_ptr(), s["lengths"].data_ptr(), s["n"], s["blocks"], s["new_table"].data_ptr(), s["used"].data_ptr(),
                      s["workspace"].data_ptr(), s["workspace"].numel(), stream)
    return s["new_table"], s["used"], s["pool"]


def _plain_chunk(s):
    n, t, m, H, Hk, d = s["n"], s["longest"], s["blocks"] * PAGE, s["heads"], s["kv_heads"], s["dim"]
    held = s["pool"][s["table"].long().clamp(min=0)].float()  # [n, blocks, hk, 2, 64, d]
    k, v = (held[:, :, :, i].transpose(1, 2).reshape(n, Hk, m, d) for i in (0, 1))
    at = s["offsets"][:-1].long()[:, None] + torch.arange(t, device="cuda")  # places past a sequence's end hold some row
    q = s["q"].float()[torch.clamp(at, max=s["rows"] - 1)].transpose(1, 2)
    scores = (q.reshape(n, Hk, H // Hk * t, d) @ k.transpose(2, 3)).mul_(d ** -0.5).reshape(n, Hk, H // Hk, t, m)
    seen = torch.arange(m, device="cuda") <= (s["lengths"][:, None] + torch.arange(t, device="cuda"))[..., None]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    p = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    out = (p.reshape(n, Hk, -1, m) @ v).reshape(n, Hk, H // Hk, t, d) / p.sum(-1, keepdim=True)
    return out.reshape(n, H, t, d)[s["seq"], :, s["within"]].to(s["dtype"])


def _plain_norm(s):
    r, half = s["rotary"], s["rotary"] // 2
    freq = 10000.0 ** (-2 * torch.arange(half, device="cuda", dtype=torch.float64) / r)
    angle = s["positions"].double()[:, None] * freq
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(x, weight, bias):
        x = x.float()
        if s["norm"] == "layer":
            x = x - x.mean(-1, keepdim=True)
        y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight
        if s["norm"] == "layer":
            y = y + bias
        a, b = (y[..., 0:r:2], y[..., 1:r:2]) if s["layout"] == "interleaved" else (y[..., :half], y[..., half:r])
        c, e = a * cos - b * sin, a * sin + b * cos
        a.copy_(c)
        b.copy_(e)
        return y

    q, k = turned(s["q"], s["weights"][0], s["weights"][2]).to(s["dtype"]), turned(s["k"], s["weights"][1], s["weights"][3])
    at = s["positions"].long()
    page = s["table"][s["seq"], at // PAGE].long()
    s["pool"][page, :, 0, at % PAGE] = k.to(s["pool"].dtype)
    s["pool"][page, :, 1, at % PAGE] = s["v"].to(s["pool"].dtype)
    return q, s["pool"]


def _plain_logits(s):
    n, vocab = s["seqs"], s["vocab"]
    at, history = torch.arange(s["held"], device="cuda"), s["history"].long()
    there, said = at < s["held_lengths"][:, None], at >= s["prompt_lengths"][:, None]
    count, known = torch.zeros(n, vocab, device="cuda"), torch.zeros(n, vocab, device="cuda")
    count.scatter_add_(1, history, (there & said).float())
    known.scatter_add_(1, history, there.float())
    row = s["sequences"].long()
    x, count = s["logits"].float(), count[row]
    rep = s["repetition"][row, None]
    x = torch.where(known[row] > 0, torch.where(x > 0, x / rep, x * rep), x)
    x = x - (count * s["frequency"][row, None] + (count > 0) * s["presence"][row, None])
    if s["entries"]:
        bias = torch.zeros(n, vocab, device="cuda")
        bias.scatter_(1, s["bias_tokens"].long().reshape(n, -1), s["bias_values"].reshape(n, -1))
        x = x + bias[row]
    if s["masked"]:
        v = torch.arange(vocab, device="cuda")
        allowed = (s["masks"][s["mask_rows"].long().clamp(min=0)][:, v >> 5] >> (v & 31)) & 1
        x = torch.where((allowed > 0) | (s["mask_rows"] < 0)[:, None], x, -math.inf)
    return x.to(s["dtype"])


def _held(s):
    """Which pages the sequences' cached positions lie on; one place more for what names none."""
    b = torch.arange(s["blocks"], device="cuda")
    named = torch.where(b < ((s["lengths"] + PAGE - 1) // PAGE)[:, None], s["table"].long(), s["pages"])
    held = torch.zeros(s["pages"] + 1, dtype=torch.bool, device="cuda")
    held[named.reshape(-1)] = True
    return held[: s["pages"]], named


def _in_order(flags):
    """The places of the set flags, in order, in a list as long as `flags`, and how many there are."""
    rank = flags.cumsum(0)
    order = torch.full((len(flags) + 1,), -1, dtype=torch.int64, device="cuda")
    order[torch.where(flags, rank - 1, len(flags))] = torch.arange(len(flags), device="cuda")
    return order[:-1], rank[-1]


def _plain_fork(s):
    held, _ = _held(s)
    free, count = _in_order(~held)
    b, one = torch.arange(s["blocks"], device="cuda"), torch.arange(s["new"], device="cuda")
    full, kept = s["keep"] // PAGE, (s["keep"] + PAGE - 1) // PAGE
    source = s["table"][s["parents"].long()].long()
    writes = (s["keep"] % PAGE > 0) & (s["need"] > s["keep"])  # into a page that is partly filled
    last = source[one, full.long().clamp(max=s["blocks"] - 1)]
    # a page that every new row which names it would write into stays with the first of them
    named = (b < kept[:, None]) & ~((b == full[:, None]) & writes[:, None])
    read = torch.zeros(s["pages"] + 1, dtype=torch.bool, device="cuda")
    read[torch.where(named, source, s["pages"]).reshape(-1)] = True
    first = torch.full((s["pages"] + 1,), s["new"], dtype=torch.int64, device="cuda")
    first.scatter_reduce_(0, torch.where(writes, last, s["pages"]), one, "amin")
    copies = writes & (read[last] | (first[last] != one))
    upto = torch.maximum((s["need"] + PAGE - 1) // PAGE, kept)
    wants = copies + upto - kept
    start = wants.cumsum(0) - wants
    place = torch.where(copies[:, None] & (b == full[:, None]), start[:, None], start[:, None] + copies[:, None] + b - kept[:, None])
    page = torch.where(place < count, free[place.clamp(0, s["pages"] - 1)], -1)
    new = torch.where(b < (kept - copies.int())[:, None], source, torch.where(b < upto[:, None], page, -1))
    missing = wants - (count - start).clamp(min=0).minimum(wants)
    to = new[one, full.long().clamp(max=s["blocks"] - 1)]
    some = (copies & (to >= 0)).nonzero()[:, 0]
    line = torch.arange(PAGE, device="cuda") < (s["keep"] % PAGE)[some, None]
    s["pool"][to[some]] = torch.where(line[:, None, None, None, :, None], s["pool"][last[some]], s["pool"][to[some]])
    return new.to(torch.int32), missing.to(torch.int32), s["pool"]


def _plain_compact(s):
    held, named = _held(s)
    used = held.sum()
    front = torch.arange(s["pages"], device="cuda") < used
    holes, _ = _in_order(front & ~held)
    behind, _ = _in_order(~front & held)
    to = torch.arange(s["pages"] + 1, device="cuda")
    to[-1] = -1
    moved = (behind >= 0).nonzero()[:, 0]
    to[behind[moved]] = holes[moved]
    s["pool"][holes[moved]] = s["pool"][behind[moved]]
    return to[named].to(torch.int32), used.reshape(1).to(torch.int32), s["pool"]


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------


def exact(case, seed):
    if work(case)["flops"] > 3e12:
        return None
    s = prepare(case, seed)
    return {"chunk": _exact_chunk, "norm": _exact_norm, "logits": _exact_logits, "fork": _exact_fork, "compact": _exact_compact}[case["op"]](s)


def _exact_chunk(s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    bounds, lengths, group = s["offsets"].tolist(), s["lengths"].tolist(), s["heads"] // s["kv_heads"]
    for i in range(s["n"]):
        b, e = bounds[i], bounds[i + 1]
        total = lengths[i] + e - b
        for h in range(s["kv_heads"]):
            pages = s["pool"][s["table"][i, : -(-total // PAGE)].long(), h].double()
            k, v = (pages[:, j].reshape(-1, s["dim"])[:total] for j in (0, 1))
            for c in range(b, e, 512):  # some rows at a time
                rows = torch.arange(c, min(c + 512, e), device="cuda")
                x = torch.einsum("rgd,md->grm", s["q"][rows, h * group:(h + 1) * group].double(), k) / math.sqrt(s["dim"])
                later = torch.arange(total, device="cuda") > lengths[i] + (rows - b)[:, None]
                out[rows, h * group:(h + 1) * group] = torch.einsum("grm,md->rgd", torch.softmax(x.masked_fill(later, -math.inf), -1), v)
    return out


def _exact_norm(s):
    r = s["rotary"]
    waves = torch.tensor([10000.0 ** (-2.0 * i / r) for i in range(r // 2)], dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.ones(s["rows"], r // 2, dtype=torch.float64, device="cuda"), s["positions"].double()[:, None] * waves)[:, None]

    def turned(x, weight, bias):
        x = x.double()
        if s["norm"] == "layer":
            x = torch.nn.functional.layer_norm(x, x.shape[-1:], weight.double(), bias.double(), 1e-6)
        else:
            x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * weight.double()
        pairs = x[..., :r].unflatten(-1, (r // 2, 2) if s["layout"] == "interleaved" else (2, r // 2))
        z = torch.view_as_complex(pairs.contiguous() if s["layout"] == "interleaved" else pairs.transpose(-1, -2).contiguous()) * turn
        z = torch.view_as_real(z)
        z = z.flatten(-2) if s["layout"] == "interleaved" else z.transpose(-1, -2).flatten(-2)
        return torch.cat([z, x[..., r:]], -1)

    pool = s["pool"].double()
    seq, at = s["seq"], s["positions"].long()
    where = s["table"][seq, at // PAGE].long(), at % PAGE
    for j, x in ((0, turned(s["k"], s["weights"][1], s["weights"][3])), (1, s["v"].double())):
        pool[where[0], :, j, where[1]] = x
    return turned(s["q"], s["weights"][0], s["weights"][2]), pool


def _exact_logits(s):
    out = s["logits"].double()
    history, held, prompt, row = (s[x].tolist() for x in ("history", "held_lengths", "prompt_lengths", "sequences"))
    vocab = s["vocab"]
    for i in range(s["seqs"]):
        known = torch.bincount(torch.tensor(history[i][: held[i]], dtype=torch.int64), minlength=vocab).to("cuda") > 0
        count = torch.bincount(torch.tensor(history[i][min(prompt[i], held[i]): held[i]], dtype=torch.int64), minlength=vocab).to("cuda").double()
        at = [j for j, x in enumerate(row) if x == i]
        x, rep = out[at], s["repetition"][i].double()
        x = torch.where(known, torch.where(x > 0, x / rep, x * rep), x) - count * s["frequency"][i].double() - (count > 0) * s["presence"][i].double()
        if s["entries"]:
            b, e = s["bias_offsets"][i], s["bias_offsets"][i + 1]
            x[:, s["bias_tokens"][b:e].long()] += s["bias_values"][b:e].double()
        out[at] = x
    if s["masked"]:
        bits = np.unpackbits(s["masks"].cpu().numpy().view(np.uint8), axis=1, bitorder="little")[:, :vocab]
        allowed = torch.tensor(bits, device="cuda").bool()
        for j, m in enumerate(s["mask_rows"].tolist()):
            if m >= 0:
                out[j, ~allowed[m]] = -math.inf
    return out


def _exact_fork(s):
    table, lengths, parents, keep, need = (s[x].tolist() for x in ("table", "lengths", "parents", "keep", "need"))
    held = {p for row, n in zip(table, lengths) for p in row[: -(-n // PAGE)]}
    free = [p for p in range(s["pages"]) if p not in held]
    writers, readers = {}, set()
    for i, (p, k, m) in enumerate(zip(parents, keep, need)):
        readers |= set(table[p][: k // PAGE])
        if k % PAGE:
            if m > k:
                writers.setdefault(table[p][k // PAGE], []).append(i)
            else:
                readers.add(table[p][k // PAGE])
    new, missing, pool = [], [], s["pool"].clone()
    for i, (p, k, m) in enumerate(zip(parents, keep, need)):
        row, lost = table[p][: -(-k // PAGE)], 0
        if k % PAGE and m > k:
            page = row[-1]
            if page in readers or writers[page][0] != i:
                row[-1] = free.pop(0) if free else -1
                lost += row[-1] < 0
                if row[-1] >= 0:
                    pool[row[-1], ..., : k % PAGE, :] = pool[page, ..., : k % PAGE, :]
        while len(row) * PAGE < m:
            row.append(free.pop(0) if free else -1)
            lost += row[-1] < 0
        new.append(row + [-1] * (s["blocks"] - len(row)))
        missing.append(lost)
    return torch.tensor(new, dtype=torch.int32), torch.tensor(missing, dtype=torch.int32), pool


def _exact_compact(s):
    table, lengths = s["table"].tolist(), s["lengths"].tolist()
    held = sorted({p for row, n in zip(table, lengths) for p in row[: -(-n // PAGE)]})
    holes = iter(sorted(set(range(len(held))) - set(held)))
    pool, to = s["pool"].clone(), {}
    for p in held:
        to[p] = p if p < len(held) else next(holes)
        if to[p] != p:
            pool[to[p]] = s["pool"][p]
    new = [[to[p] for p in row[: -(-n // PAGE)]] + [-1] * (s["blocks"] - -(-n // PAGE)) for row, n in zip(table, lengths)]
    return torch.tensor(new, dtype=torch.int32), torch.tensor([len(held)], dtype=torch.int32), pool

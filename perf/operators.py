"""Measured cases of the serving operators: rotary positions with the append to a paged cache, causal attention over
packed prompts, attention of drafted token trees over the cache, and the verification of those trees.

`run` computes an operator from elementary torch operations (32 bits, 64 where positions or sums need them), or, with
`own` set, calls the framework's kernels. `exact` restates the definitions in 64 bits, sequence by sequence."""
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
        # one decode step of 64 sequences of the MicroChat shape: latency
        _rope("rope step", "bf16", 64, 1, 1, 4, 4, 64, 64, "interleaved", "none", 1.0, 511, True),
        # prompts of the Phase2Modern-style shape in 32 bits, appended to the bf16 cache
        _rope("rope prompts f32", "f32", 16, 700, 1024, 16, 4, 64, 64, "half", "linear", 4.0, 0, True),
        # long contexts, the first half of each head rotated, frequencies scaled by parts
        _rope("rope long context", "f16", 8, 6000, 8192, 32, 8, 128, 64, "half", "by_parts", 8.0, 60000, False),
        # short ragged chat prompts of the MicroChat shape: latency
        _prompt("prompts short", "bf16", 64, 1, 128, 4, 4, 64),
        # prompts of the Phase2Modern-style shape up to its whole context
        _prompt("prompts 2048", "bf16", 16, 300, 2048, 16, 4, 64),
        # few long documents, wide heads
        _prompt("prompts 8192", "f16", 2, 7000, 8192, 16, 2, 128),
        # one new token for each of 256 sequences at the FusedAttention shape
        _tree("tree single tokens", "bf16", 256, 1, 1, 400, 576, 8, 2, 64),
        # one user, a tree of 24 drafted tokens, Phase2Modern-style
        _tree("tree one user", "bf16", 1, 24, 24, 1900, 2047, 16, 4, 64),
        # a full batch with long caches and large trees, wide heads
        _tree("tree long caches", "f16", 16, 33, 64, 20000, 32768, 32, 8, 128),
        # one user, a chain of seven drafted tokens over the MicroChat vocabulary
        _verify("verify one user", "f32", 1, 8, 8, 1, 4096),
        # a batch of trees over the Phase2Modern-style vocabulary
        _verify("verify batch", "f32", 64, 9, 24, 3, 32768),
        # the same from 16-bit probabilities, a large odd vocabulary
        _verify("verify batch bf16", "bf16", 128, 5, 16, 4, 50257),
    ]


def draw(rng):
    kind = rng.choice(("rope", "prompt", "tree", "verify"))
    spread = rng.randrange(1 << 20)
    heads = rng.choice(((4, 4, 32), (4, 4, 64), (16, 4, 64), (8, 2, 64), (8, 1, 64), (12, 4, 64), (4, 2, 128), (16, 4, 128), (32, 8, 128)))
    if kind == "rope":
        n, most = _log(rng, 1, 256), _log(rng, 1, 4096)
        most = max(1, min(most, 60000 // n, 4_000_000 // (n * heads[0])))
        r = rng.choice((heads[2], heads[2] // 2, 2 * rng.randrange(1, heads[2] // 2)))
        scaling = rng.choice(("none", "linear", "stretched", "by_parts")) if r > 2 else "linear"
        return _rope(None, rng.choice(("bf16", "f16", "f32")), n, max(1, most // 3), most, *heads, r, rng.choice(("interleaved", "half")), scaling,
                     rng.choice((1.5, 4.0, 8.0)), _log(rng, 1, 100000), rng.random() < 0.5, spread)
    if kind == "prompt":
        n, most = _log(rng, 1, 64), _log(rng, 1, 8000)
        most = max(1, min(most, int(math.sqrt(8000 * 8000 * 16 / (n * heads[0])))))
        return _prompt(None, rng.choice(("bf16", "f16")), n, rng.choice((0, most // 2)), most, *heads, spread)
    if kind == "tree":
        n, length, nodes = _log(rng, 1, 256), _log(rng, 1, 32768), rng.choice((1, _log(rng, 1, 64)))
        length = max(1, min(length, 16 * 20000 * 8 * 128 // (n * heads[1] * heads[2]), 16 * 20000 * 32 * 33 // (n * heads[0] * nodes)))
        return _tree(None, rng.choice(("bf16", "f16")), n, max(1, nodes // 2), nodes, rng.choice((0, length // 2)), length, *heads, spread)
    n, nodes, vocab = _log(rng, 1, 128), _log(rng, 1, 24), _log(rng, 300, 50000)
    return _verify(None, rng.choice(("f32", "bf16", "f16")), n, max(1, nodes // 2), nodes, rng.randrange(1, 5), vocab, spread)


def _log(rng, least, most):
    return int(round(math.exp(rng.uniform(math.log(least), math.log(most)))))


def _case(name, **values):
    return values if name is None else {"name": name, **values}


def _rope(name, dtype, seqs, least, most, heads, kv_heads, dim, rotary, layout, scaling, factor, start, append, spread=1):
    return _case(name, op="rope", dtype=dtype, seqs=seqs, least=least, most=most, heads=heads, kv_heads=kv_heads, dim=dim, rotary=rotary, layout=layout,
                 scaling=scaling, factor=factor, start=start, append=append, spread=spread)


def _prompt(name, dtype, seqs, least, most, heads, kv_heads, dim, spread=1):
    return _case(name, op="prompt", dtype=dtype, seqs=seqs, least=least, most=most, heads=heads, kv_heads=kv_heads, dim=dim, spread=spread)


def _tree(name, dtype, seqs, least, most, least_len, most_len, heads, kv_heads, dim, spread=1):
    return _case(name, op="tree", dtype=dtype, seqs=seqs, least=least, most=most, least_len=least_len, most_len=most_len, heads=heads, kv_heads=kv_heads, dim=dim,
                 spread=spread)


def _verify(name, dtype, seqs, least, most, branch, vocab, spread=1):
    return _case(name, op="verify", dtype=dtype, seqs=seqs, least=least, most=most, branch=branch, vocab=vocab, spread=spread)


def _rows(case):
    """Rows of each sequence (tokens, nodes) and, for trees, its cached length."""
    r = random.Random(case["spread"])
    rows = [r.randint(case["least"], case["most"]) for _ in range(case["seqs"])]
    rows[r.randrange(len(rows))] = case["most"]
    return rows, [r.randint(case["least_len"], case["most_len"]) for _ in rows] if case["op"] == "tree" else None


def work(case):
    rows, cached = _rows(case)
    n = sum(rows)
    if case["op"] == "verify":  # the last node's rows of the target and the draft, and the tree
        size = TYPES[case["dtype"]].itemsize
        return {"bytes": case["seqs"] * 2 * case["vocab"] * size + 20 * n, "flops": case["seqs"] * 3 * case["vocab"]}
    H, Hk, d, size = case["heads"], case["kv_heads"], case["dim"], TYPES[case["dtype"]].itemsize
    if case["op"] == "rope":
        written = n * H * d * size + (n * 2 * Hk * d * 2 if case["append"] else n * Hk * d * size)
        return {"bytes": n * (H + (2 if case["append"] else 1) * Hk) * d * size + written + 4 * n, "flops": n * (H + Hk) * case["rotary"] * 3}
    moved = n * (2 * H + 2 * Hk) * d * size
    if case["op"] == "prompt":
        return {"bytes": moved, "flops": sum(2 * d * H * t * (t + 1) for t in rows)}
    return {"bytes": moved + sum(cached) * Hk * 2 * d * size, "flops": sum(4 * d * H * t * (c + 1) for t, c in zip(rows, cached))}


# ---- inputs --------------------------------------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = random.Random(seed)
    rows, cached = _rows(case)
    s = dict(case, dtype=TYPES[case["dtype"]], rows=sum(rows), n=len(rows))
    starts = np.concatenate([[0], np.cumsum(rows)])
    s["offsets"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    seq = np.repeat(np.arange(len(rows)), rows)
    within = np.arange(sum(rows)) - starts[seq]
    s["seq"], s["within"] = (torch.tensor(x, device="cuda") for x in (seq, within))
    s["longest"] = max(rows)
    return {"rope": _prepare_rope, "prompt": _prepare_prompt, "tree": _prepare_tree, "verify": _prepare_verify}[case["op"]](s, g, r, rows, cached)


def _normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def _cache(s, g, r, positions, dtype):
    """A cache of one layer that holds `positions` of each sequence: pages in an order of chance, some of them nobody's."""
    s["blocks"] = max(1, -(-max(positions) // PAGE))
    count = sum(-(-p // PAGE) for p in positions) + 3
    ids = list(range(count))
    r.shuffle(ids)
    table = np.zeros((s["n"], s["blocks"]), dtype=np.int32)
    for i, p in enumerate(positions):
        k = -(-p // PAGE)
        table[i, :k] = ids[:k]
        del ids[:k]
    s["table"] = torch.tensor(table, device="cuda")
    s["pages"] = count
    s["pool"] = torch.empty(count, s["kv_heads"], 2, PAGE, s["dim"], dtype=dtype, device="cuda").normal_(generator=g)
    if own:
        s["cache"] = _pkg().KvCache(s["pool"].data_ptr(), s["pool"].stride(0), s["table"].data_ptr(), s["blocks"], count, s["kv_heads"], s["dim"])


def _prepare_rope(s, g, r, rows, _):
    d, t = s["dim"], s["dtype"]
    s["q"], s["k"], s["v"] = (_normal(g, s["rows"], h, d, dtype=t) for h in (s["heads"], s["kv_heads"], s["kv_heads"]))
    chance = random.Random(s["spread"] + 1)  # where a case's sequences stand, and so its cache's size, goes by the case
    start = torch.tensor([chance.randint(0, min(s["start"], 2048) if s["append"] else s["start"]) for _ in rows], device="cuda")
    s["positions"] = (start[s["seq"]] + s["within"]).to(torch.int32)
    s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
    if s["append"]:
        _cache(s, g, r, [int(a) + b for a, b in zip(start.tolist(), rows)], torch.bfloat16 if t == torch.float32 else t)
    s["magnitude"] = 0.1 * math.log(s["factor"]) + 1 if s["scaling"] == "by_parts" else 1.0
    if own:
        s["plan"] = _pkg().Rope(d, s["rotary"], s["layout"], 10000.0, s["scaling"], s["factor"], 4096, 32.0, 1.0, s["magnitude"])
    return s


def _prepare_prompt(s, g, r, rows, _):
    s["q"], s["k"], s["v"] = (_normal(g, s["rows"], h, s["dim"], dtype=s["dtype"]) for h in (s["heads"], s["kv_heads"], s["kv_heads"]))
    s["out"] = torch.empty_like(s["q"])
    return s


def _tree_of(r, nodes, branch):
    """Parents of a drafted tree: each node but the root hangs under one of the last `branch` nodes before it."""
    return [-1] + [r.randrange(max(0, i - branch), i) for i in range(1, nodes)] if nodes else []


def _prepare_tree(s, g, r, rows, cached):
    _prepare_prompt(s, g, r, rows, cached)
    _cache(s, g, r, cached, s["dtype"])
    s["lengths"] = torch.tensor(cached, dtype=torch.int32, device="cuda")
    masks = []
    for t in rows:
        seen = []
        for i, p in enumerate(_tree_of(r, t, 4)):
            seen.append((seen[p] if i else 0) | 1 << i)
        masks += seen
    s["masks"] = torch.tensor(np.array(masks, dtype=np.uint64).view(np.int64), device="cuda")
    if own:
        size = _pkg().tree_attention_workspace(s["n"], s["longest"], s["heads"], s["cache"])
        s["workspace"] = torch.empty(max(size, 1), dtype=torch.uint8, device="cuda")
    return s


def _prepare_verify(s, g, r, rows, _):
    parents = [p for t in rows for p in _tree_of(r, t, s["branch"])]
    s["parents"] = torch.tensor(parents, dtype=torch.int32, device="cuda")
    logits = _normal(g, s["rows"], s["vocab"]) * 2.5
    s["target"] = torch.softmax(logits, 1).to(s["dtype"])
    logits += _normal(g, s["rows"], s["vocab"])  # the draft model is near the target
    draft = torch.softmax(logits, 1)
    s["draft"] = draft.to(s["dtype"])
    above = torch.clamp(s["parents"].long(), min=0) + s["offsets"][s["seq"]]
    point = torch.rand(s["rows"], 1, generator=g, device="cuda")
    total = torch.cumsum(draft, 1)
    # each node's token is drawn from its parent's draft row
    s["tokens"] = torch.searchsorted(total[above].contiguous(), point).clamp_(max=s["vocab"] - 1).to(torch.int32).reshape(-1)
    s["uniforms"] = torch.rand(s["rows"], generator=g, device="cuda")
    s["lengths"] = torch.randint(0, 2000, (s["n"],), generator=g, device="cuda", dtype=torch.int32)
    s["path"], s["commit"] = (torch.empty(s["rows"], dtype=torch.int32, device="cuda") for _ in range(2))
    s["count"], s["next"], s["new_lengths"] = (torch.empty(s["n"], dtype=torch.int32, device="cuda") for _ in range(3))
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------


def _pkg():
    return importlib.import_module("shahd-llm-stack_b200")


def run(s):
    if own:
        return {"rope": _own_rope, "prompt": _own_prompt, "tree": _own_tree, "verify": _own_verify}[s["op"]](s, _pkg(), torch.cuda.current_stream().cuda_stream)
    return {"rope": _plain_rope, "prompt": _plain_prompt, "tree": _plain_tree, "verify": _plain_verify}[s["op"]](s)


def _type(s, pkg):
    return {torch.bfloat16: pkg.BF16, torch.float16: pkg.F16, torch.float32: pkg.F32}[s["dtype"]]


def _of(t, pkg):
    return pkg.Rows(t.data_ptr(), t.stride(0), t.stride(1))


def _own_rope(s, pkg, stream):
    more = dict(v=_of(s["v"], pkg), cache=s["cache"], offsets=s["offsets"].data_ptr(), n=s["n"]) if s["append"] else dict(k_out=_of(s["k_out"], pkg))
    s["plan"].apply(_type(s, pkg), s["rows"], s["positions"].data_ptr(), q=_of(s["q"], pkg), q_out=_of(s["q_out"], pkg), num_heads=s["heads"], k=_of(s["k"], pkg),
                    kv_heads=s["kv_heads"], stream=stream, **more)
    return s["q_out"], s["pool"] if s["append"] else s["k_out"]


def _own_prompt(s, pkg, stream):
    pkg.prompt_attention(_type(s, pkg), _of(s["q"], pkg), _of(s["k"], pkg), _of(s["v"], pkg), _of(s["out"], pkg), s["offsets"].data_ptr(), s["n"], s["rows"],
                         s["heads"], s["kv_heads"], s["dim"], stream=stream)
    return s["out"]


def _own_tree(s, pkg, stream):
    pkg.tree_attention(_type(s, pkg), _of(s["q"], pkg), _of(s["k"], pkg), _of(s["v"], pkg), _of(s["out"], pkg), s["cache"], s["lengths"].data_ptr(),
                       s["masks"].data_ptr(), s["offsets"].data_ptr(), s["n"], s["rows"], s["longest"], s["heads"], workspace=s["workspace"].data_ptr(),
                       workspace_bytes=s["workspace"].numel(), stream=stream)
    return s["out"]


def _own_verify(s, pkg, stream):
    pkg.verify_tree(_type(s, pkg), s["target"].data_ptr(), s["draft"].data_ptr(), s["vocab"], s["tokens"].data_ptr(), s["parents"].data_ptr(),
                    s["uniforms"].data_ptr(), s["offsets"].data_ptr(), s["n"], s["rows"], s["path"].data_ptr(), s["count"].data_ptr(), s["next"].data_ptr(),
                    lengths=s["lengths"].data_ptr(), commit=s["commit"].data_ptr(), new_lengths=s["new_lengths"].data_ptr(), stream=stream)
    return s["path"], s["count"], s["next"], s["commit"], s["new_lengths"]


def _frequencies(s):
    r, f = s["rotary"], s["factor"]
    i = torch.arange(r // 2, device="cuda", dtype=torch.float64)
    base = 10000.0 * f ** (r / (r - 2)) if s["scaling"] == "stretched" else 10000.0
    freq = base ** (-2 * i / r)
    if s["scaling"] == "linear":
        freq = freq / f
    if s["scaling"] == "by_parts":  # pairs that turn often keep their frequency, those that turn seldom are divided
        low, high = (r * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(10000.0)) for turns in (32.0, 1.0))
        low, high = max(math.floor(low), 0), min(math.ceil(high), r - 1)
        part = torch.clamp((i - low) / max(high - low, 0.001), 0, 1)
        freq = freq * (1 - part) + freq / f * part
    return freq


def _plain_rope(s):
    r, half = s["rotary"], s["rotary"] // 2
    angle = s["positions"].double()[:, None] * _frequencies(s)
    cos, sin = ((x * s["magnitude"]).float()[:, None] for x in (angle.cos(), angle.sin()))

    def rotated(x):
        y = x.float().clone()
        a, b = (y[..., 0:r:2], y[..., 1:r:2]) if s["layout"] == "interleaved" else (y[..., :half], y[..., half:r])
        c, e = a * cos - b * sin, a * sin + b * cos
        a.copy_(c)
        b.copy_(e)
        return y

    q, k = rotated(s["q"]).to(s["dtype"]), rotated(s["k"])
    if not s["append"]:
        return q, k.to(s["dtype"])
    at = s["positions"].long()
    page = s["table"][s["seq"], at // PAGE].long()
    s["pool"][page, :, 0, at % PAGE] = k.to(s["pool"].dtype)
    s["pool"][page, :, 1, at % PAGE] = s["v"].to(s["pool"].dtype)
    return q, s["pool"]


def _padded(s, x):
    """Packed rows [N, h, d] as [n, h, longest, d]: places past a sequence's end hold some row."""
    at = s["offsets"][:-1].long()[:, None] + torch.arange(s["longest"], device="cuda")
    return x.float()[torch.clamp(at, max=max(s["rows"] - 1, 0))].transpose(1, 2)


def _attend(s, q, k, v, seen):
    """softmax(q k / sqrt(d)) v over [n, h, t, d] and [n, hk, m, d] where `seen` [n, t, m]; the packed rows of the answer."""
    n, H, t, d = q.shape
    Hk = k.shape[1]
    scores = q.reshape(n, Hk, H // Hk * t, d) @ k.transpose(2, 3) * d ** -0.5
    scores = scores.reshape(n, Hk, H // Hk, t, -1).masked_fill_(~seen[:, None, None], -math.inf)
    scores -= torch.clamp(scores.amax(-1, keepdim=True), min=-3e38)
    p = scores.exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.reshape(n, Hk, -1, p.shape[-1]) @ v).reshape(n, Hk, H // Hk, t, d) / torch.where(total > 0, total, 1.0)
    return out.reshape(n, H, t, d)[s["seq"], :, s["within"]].to(s["dtype"])


def _plain_prompt(s):
    at = torch.arange(s["longest"], device="cuda")
    return _attend(s, _padded(s, s["q"]), _padded(s, s["k"]), _padded(s, s["v"]), (at[:, None] >= at).expand(s["n"], -1, -1))


def _plain_tree(s):
    n, t, m = s["n"], s["longest"], s["blocks"] * PAGE
    held = s["pool"][s["table"].long()].float()  # [n, blocks, hk, 2, 64, d]
    k, v = (held[:, :, :, i].transpose(1, 2).reshape(n, s["kv_heads"], m, s["dim"]) for i in (0, 1))
    k, v = torch.cat([k, _padded(s, s["k"])], 2), torch.cat([v, _padded(s, s["v"])], 2)
    node = torch.arange(t, device="cuda")
    bits = torch.zeros(n, t, dtype=torch.int64, device="cuda")
    bits[s["seq"], s["within"]] = s["masks"]
    cached = torch.arange(m, device="cuda") < s["lengths"][:, None]
    seen = torch.cat([cached[:, None].expand(n, t, m), (bits[:, :, None] >> node & 1).bool()], 2)
    return _attend(s, _padded(s, s["q"]), k, v, seen)


def _plain_verify(s):
    n, first = s["n"], s["offsets"][:-1].long()
    size = s["offsets"].diff().long()
    one = torch.arange(n, device="cuda")
    cur, depth = (torch.zeros(n, dtype=torch.int64, device="cuda") for _ in range(2))
    a, z = torch.zeros(n, dtype=torch.float64, device="cuda"), torch.ones(n, dtype=torch.float64, device="cuda")
    path = torch.full((n, s["longest"]), -1, dtype=torch.int32, device="cuda")
    commit = torch.full((s["rows"],), -1, dtype=torch.int32, device="cuda")
    path[:, 0] = 0
    commit[first] = s["lengths"]
    last = s["rows"] - 1
    for i in range(1, s["longest"]):  # a node's fate hangs on those before it
        at = torch.clamp(first + i, max=last)
        asked = (i < size) & (s["parents"][at].long() == cur)
        token = s["tokens"][at].long()
        p, q = (s[x][first + cur].double() for x in ("target", "draft"))
        took = asked & (s["uniforms"][at].double() * q[one, token] * z < torch.clamp(p[one, token] - a * q[one, token], min=0))
        lost = asked & ~took
        a = torch.where(lost, a + z, a)
        z = torch.where(lost, torch.clamp(p - a[:, None] * q, min=0).sum(1), z)
        a, z = torch.where(took, 0.0, a), torch.where(took, 1.0, z)
        depth += took
        cur = torch.where(took, i, cur)
        path.scatter_(1, depth[:, None], cur[:, None].to(torch.int32))
        commit[at] = torch.where(took, s["lengths"] + depth, commit[at]).to(torch.int32)
    p, q = (s[x][first + cur].double() for x in ("target", "draft"))
    left = torch.clamp(p - a[:, None] * q, min=0)
    left = torch.where((z > 0)[:, None], left, p)
    sums = left.cumsum(1)
    reached = (sums >= s["uniforms"][first].double()[:, None] * sums[:, -1:]) & (left > 0)
    token = reached.to(torch.int8).argmax(1).to(torch.int32)
    path = torch.where(torch.arange(s["longest"], device="cuda") <= depth[:, None], path, -1)[s["seq"], s["within"]]
    return path, depth.to(torch.int32), token, commit, (s["lengths"] + depth + 1).to(torch.int32)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    bounds = s["offsets"].tolist()
    if case["op"] == "rope":
        return _exact_rope(s)
    if case["op"] == "verify":
        return _exact_verify(s, bounds)
    if work(case)["flops"] > 3e12:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group = s["heads"] // s["kv_heads"]
    for i in range(s["n"]):
        b, e = bounds[i], bounds[i + 1]
        held = int(s["lengths"][i]) if case["op"] == "tree" else 0
        for h in range(s["kv_heads"]):
            k, v = s["k"][b:e, h].double(), s["v"][b:e, h].double()
            if held:
                pages = s["pool"][s["table"][i, : -(-held // PAGE)].long(), h].double()
                k, v = (torch.cat([pages[:, j].reshape(-1, s["dim"])[:held], x]) for j, x in ((0, k), (1, v)))
            for c in range(b, e, 1024):  # some rows at a time
                rows = torch.arange(c, min(c + 1024, e), device="cuda")
                if case["op"] == "tree":
                    seen = (s["masks"][rows, None] >> torch.arange(e - b, device="cuda")) % 2 != 0
                    seen = torch.cat([torch.ones(len(rows), held, dtype=torch.bool, device="cuda"), seen], 1)
                else:
                    seen = torch.arange(b, e, device="cuda") <= rows[:, None]
                x = torch.einsum("rgd,md->grm", s["q"][rows, h * group:(h + 1) * group].double(), k) / math.sqrt(s["dim"])
                x = torch.softmax(x.masked_fill(~seen, -math.inf), -1)
                out[rows, h * group:(h + 1) * group] = torch.einsum("grm,md->rgd", x, v)
    return out


def _exact_rope(s):
    r, factor = s["rotary"], s["factor"]
    waves = []
    for i in range(r // 2):
        f = 10000.0 ** (-2.0 * i / r)
        if s["scaling"] == "linear":
            f /= factor
        elif s["scaling"] == "stretched":
            f /= factor ** (2.0 * i / (r - 2))
        elif s["scaling"] == "by_parts":
            ends = [r / 2 * math.log(4096 / (2 * math.pi * turns), 10000.0) for turns in (32.0, 1.0)]
            ends = max(math.floor(ends[0]), 0), min(math.ceil(ends[1]), r - 1)
            slow = min(1.0, max(0.0, (i - ends[0]) / max(ends[1] - ends[0], 0.001)))
            f -= f * slow * (1 - 1 / factor)
        waves.append(f)
    angle = s["positions"].double()[:, None] * torch.tensor(waves, dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.full_like(angle, s["magnitude"]), angle)[:, None]

    def rotated(x):
        x = x.double()
        pairs = x[..., :r].unflatten(-1, (r // 2, 2) if s["layout"] == "interleaved" else (2, r // 2))
        z = torch.view_as_complex(pairs.contiguous() if s["layout"] == "interleaved" else pairs.transpose(-1, -2).contiguous()) * turn
        z = torch.view_as_real(z)
        z = z.flatten(-2) if s["layout"] == "interleaved" else z.transpose(-1, -2).flatten(-2)
        return torch.cat([z, x[..., r:]], -1)

    q, k = rotated(s["q"]), rotated(s["k"])
    if not s["append"]:
        return q, k
    pool = s["pool"].double()
    at = s["positions"].long()
    where = s["table"][s["seq"], at // PAGE].long(), at % PAGE
    for i, x in ((0, k), (1, s["v"].double())):
        pool[where[0], :, i, where[1]] = x
    return q, pool


def _exact_verify(s, bounds):
    tokens, parents, u, lengths = (s[x].cpu().numpy() for x in ("tokens", "parents", "uniforms", "lengths"))
    path, commit = np.full(s["rows"], -1), np.full(s["rows"], -1)
    count, following = np.zeros(s["n"], dtype=np.int64), np.zeros(s["n"], dtype=np.int64)
    for i in range(s["n"]):
        b = bounds[i]
        cur, took = 0, [0]
        p, q = (s[x][b].double().cpu().numpy() for x in ("target", "draft"))
        a, z = 0.0, 1.0
        for j in range(1, bounds[i + 1] - b):
            if parents[b + j] != cur:
                continue
            t = tokens[b + j]
            if float(u[b + j]) * q[t] * z < max(0.0, p[t] - a * q[t]):
                cur, a, z = j, 0.0, 1.0
                took.append(j)
                p, q = (s[x][b + j].double().cpu().numpy() for x in ("target", "draft"))
            else:
                a += z
                z = float(np.maximum(p - a * q, 0).sum())
        left = np.maximum(p - a * q, 0) if z > 0 else p
        sums = np.cumsum(left)
        following[i] = int(np.argmax((sums >= float(u[b]) * sums[-1]) & (left > 0)))
        path[b:b + len(took)] = took
        commit[b + np.array(took)] = lengths[i] + np.arange(len(took))
        count[i] = len(took) - 1
    return tuple(torch.tensor(x, dtype=torch.int32) for x in (path, count, following, commit, lengths + count + 1))

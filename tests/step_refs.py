"""Restatements of the operators of a serving step over shared pages, with the error bounds that the tests hold the kernels to."""
import math

import numpy as np
import torch

from tests import serving_refs as R

PAGE = 64


def normalise(x, kind, eps, weight, bias):
    """x [rows, heads, d] in 64 bits with its heads normalised, and how far a kernel's 32-bit values may be off.

    A sum of squares: at most 16 steps in a lane and 5 over lanes, all terms positive, so 21 half steps h = 2^-24 of itself; its mean, eps and
    the root add 4, half of which (a root) the scale keeps: below 13 h. Two products: 15 h of |x scale w|; the last step, with
    the bias, h of the result. A mean of d values is off by at most 22 h mean|x|, a difference to it by that and h of its own: all of
    them move the variance by less than 2 (that over sigma) of it."""
    h = 2.0 ** -24
    x = x.double()
    w = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if weight is None else weight.double()
    b = torch.zeros_like(w) if bias is None else bias.double()
    if kind == "layer":
        mu = x.mean(-1, keepdim=True)
        apart = x - mu
        moved = 22 * h * x.abs().mean(-1, keepdim=True) + h * apart.abs()
    else:
        apart, moved = x, torch.zeros_like(x)
    scale = 1 / (apart.square().mean(-1, keepdim=True) + eps).sqrt()
    y = apart * scale * w + b
    share = moved.square().mean(-1, keepdim=True).sqrt() * scale  # of the scale, through the variance
    off = (apart * scale * w).abs() * (15 * h + share) + moved * scale * w.abs() + h * y.abs()
    return y, off * 1.01


def norm_rope(x, positions, freq, layout, magnitude, kind, eps, weight, bias, dtype):
    """Normalised and turned, with the bound for a result of `dtype`."""
    y, off = normalise(x, kind, eps, weight, bias)
    turned, more = R.rotate(y, positions, freq, layout, magnitude)
    r = 2 * len(freq)
    a, b = (off[..., 0:r:2], off[..., 1:r:2]) if layout == "interleaved" else (off[..., : r // 2], off[..., r // 2 : r])
    both = (a + b) * abs(magnitude)
    spread = off.clone()
    if layout == "interleaved":
        spread[..., 0:r:2] = spread[..., 1:r:2] = both
    else:
        spread[..., : r // 2] = spread[..., r // 2 : r] = both
    return turned, (spread + more) * 1.01 + R.HALF_STEP[dtype] * turned.abs() + 1e-7


def adjust(logits, history, prompt, rep, pres, freq, biases, allowed, dtype):
    """One row (float64 [V]) of sequence data; `history` the tokens that count, the first `prompt` of them the prompt's; `biases` a
    list of (token, value), of which a token's last counts; `allowed` [V] bool or None. The row and its bound: each of the four
    32-bit steps is off by half a step of what it gives, the result by half a step of its type."""
    V, h = logits.shape[0], 2.0 ** -24
    known, count = torch.zeros(V, dtype=torch.bool), torch.zeros(V, dtype=torch.float64)
    for i, t in enumerate(history):
        if 0 <= t < V:
            known[t] = True
            count[t] += i >= prompt
    known, count = known.to(logits.device), count.to(logits.device)
    x = torch.where(known, torch.where(logits > 0, logits / rep, logits * rep), logits)
    off = h * x.abs() * known
    fine = count * freq + pres * (count > 0)
    y = x - fine
    off = off + h * fine.abs() + h * y.abs() * (count > 0)
    add = torch.zeros(V, dtype=torch.float64)
    for t, v in biases:
        if 0 <= t < V:
            add[t] = v
    z = y + add.to(y.device)
    off = off + h * z.abs() * (add != 0).to(y.device)
    if allowed is not None:
        z = torch.where(allowed, z, -math.inf)
    return z, torch.nan_to_num((off * 1.01 + R.HALF_STEP[dtype] * z.abs()), posinf=0.0) + 1e-7


def fork(table, lengths, parents, keep, need, pages):
    """(new table, missing, copies (from, to, positions)) by the rules of shahd_pages_fork, one thing after another."""
    n, blocks = table.shape
    held = set()
    cut = [min(max(int(x), 0), blocks * PAGE) for x in lengths]
    for s in range(n):
        held |= {int(p) for p in table[s, : -(-cut[s] // PAGE)] if 0 <= p < pages}
    free = [p for p in range(pages) if p not in held][::-1]
    plan, writers, readers = [], {}, set()
    for i in range(len(parents)):
        q = int(parents[i])
        there = 0 <= q < n
        k = min(max(int(keep[i]), 0), cut[q]) if there else 0
        m = max(int(need[i]), k)
        row = [int(x) for x in table[q, : -(-k // PAGE)]] if there else []
        writes = k % PAGE != 0 and m > k
        plan.append((k, m, row, writes))
        for b, p in enumerate(row):
            if 0 <= p < pages:
                if writes and b == len(row) - 1:
                    writers.setdefault(p, []).append(i)
                else:
                    readers.add(p)
    new, missing, copies = np.full((len(parents), blocks), -1, np.int64), [], []
    for i, (k, m, row, writes) in enumerate(plan):
        lost = 0

        def fresh():
            nonlocal lost
            if free:
                return free.pop()
            lost += 1
            return -1

        if writes and 0 <= row[-1] < pages and (row[-1] in readers or writers[row[-1]][0] != i):
            was, row[-1] = row[-1], fresh()
            if row[-1] >= 0:
                copies.append((was, row[-1], k % PAGE))
        while len(row) < min(-(-m // PAGE), blocks):
            row.append(fresh())
        lost += max(-(-m // PAGE) - blocks, 0)
        new[i, : len(row)] = row
        missing.append(lost)
    return new, np.array(missing), copies


def compact(table, lengths, pages):
    """(new table, held pages, moves (from, to))."""
    n, blocks = table.shape
    there = [[int(p) for p in table[s, : -(-min(max(int(lengths[s]), 0), blocks * PAGE) // PAGE)]] for s in range(n)]
    held = sorted({p for row in there for p in row if 0 <= p < pages})
    taken = set(held)
    holes = iter([p for p in range(len(held)) if p not in taken])
    to = {p: p if p < len(held) else next(holes) for p in held}
    new = np.full((n, blocks), -1, np.int64)
    for s, row in enumerate(there):
        new[s, : len(row)] = [to.get(p, -1) for p in row]
    return new, len(held), [(p, q) for p, q in to.items() if p != q]

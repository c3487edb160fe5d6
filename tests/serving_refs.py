"""64-bit restatements of the serving operators, sequence by sequence (torch, any device), with the error bounds that the
tests hold the kernels to."""
import math

import numpy as np
import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def attend(q, k, v, seen, scale, dtype):
    """q [t, H, d], k, v [m, Hk, d], seen [t, m] -> the rows [t, H, d] in 64 bits and how far a kernel's may be off.

    Rounding the result costs half a step u of its own value. Rounding each probability costs at most u of it, so u sum p |v|. A
    score is a 32-bit sum of d exact products: off by at most (d + 2) 2^-23 sum |q k| scale (units that truncate), and a
    probability by twice that. The sum over m keys in 32 bits costs at most (m + 8) 2^-23 sum p |v|, the exponential and the
    division some 2^-20. fp16 probabilities below 2^-14 of 2^7 times the largest have a fixed step: 2^-25 / 2^7 each."""
    t, H, d = q.shape
    group = H // k.shape[1]
    out, bound = torch.zeros(t, H, d, dtype=torch.float64, device=q.device), torch.zeros(t, H, d, dtype=torch.float64, device=q.device)
    u = HALF_STEP[dtype]
    q, k, v = q.double(), k.double(), v.double()
    any_seen = seen.any(1)
    for h in range(H):
        kk, vv = k[:, h // group], v[:, h // group]
        x = torch.where(seen, q[:, h] @ kk.T * scale, -math.inf)
        p = torch.softmax(torch.where(any_seen[:, None], x, 0.0), 1) * any_seen[:, None]
        mass = p @ vv.abs()
        off = (d + 2) * 2.0 ** -23 * scale * torch.where(seen, q[:, h].abs() @ kk.abs().T, 0.0).amax(1, keepdim=True)
        out[:, h] = p @ vv
        bound[:, h] = u * out[:, h].abs() + mass * (u + 2 * off + (k.shape[0] + 8) * 2.0 ** -23 + 2.0 ** -20) * 1.01
        if dtype == torch.float16:
            bound[:, h] += 2.0 ** -32 * (vv.abs() * 1.0).sum(0) + 2.0 ** -25
    return out, bound


def frequencies(rotary, base=10000.0, scaling="none", factor=1.0, original=0, beta_fast=32.0, beta_slow=1.0):
    f = []
    if scaling == "stretched":
        base = base * factor ** (rotary / (rotary - 2))
    for i in range(rotary // 2):
        w = base ** (-2.0 * i / rotary)
        if scaling == "linear":
            w /= factor
        if scaling == "by_parts":
            low, high = (rotary * math.log(original / (n * 2 * math.pi)) / (2 * math.log(base)) for n in (beta_fast, beta_slow))
            low, high = max(math.floor(low), 0), min(math.ceil(high), rotary - 1)
            slow = min(1.0, max(0.0, (i - low) / max(high - low, 0.001)))
            w = w * (1 - slow) + w / factor * slow
        f.append(w)
    return np.array(f)


def rotate(x, positions, freq, layout, magnitude=1.0):
    """x [rows, heads, d] turned, in 64 bits, and how far a kernel's may be off before rounding: the turn's fraction is rounded
    to 32 bits (2^-26 of a turn, 2 pi 2^-26 in the angle), sincospi is good to 2^-22, the magnitude, two products and a sum
    take four more half steps: below 5e-7 (|a| + |b|) magnitude in all."""
    r = 2 * len(freq)
    x = x.double()
    angle = positions.double()[:, None] * torch.tensor(freq, dtype=torch.float64, device=x.device)
    cos, sin = (angle.cos() * magnitude)[:, None], (angle.sin() * magnitude)[:, None]
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if layout == "interleaved" else (x[..., : r // 2], x[..., r // 2 : r])
    y, off = x.clone(), torch.zeros_like(x)
    at = (slice(0, r, 2), slice(1, r, 2)) if layout == "interleaved" else (slice(0, r // 2), slice(r // 2, r))
    y[..., at[0]], y[..., at[1]] = a * cos - b * sin, a * sin + b * cos
    off[..., at[0]] = off[..., at[1]] = 5e-7 * abs(magnitude) * (a.abs() + b.abs())
    return y, off


def verify(target, draft, tokens, parents, uniforms):
    """One sequence's walk (numpy float64 rows [T, V]): taken nodes (the root first) and the token drawn after them."""
    cur, taken, w, z = 0, [0], 0.0, 1.0
    V = target.shape[1]
    clean = lambda row: np.where(row > 0, row, 0.0)  # noqa: E731
    for i in range(1, len(tokens)):
        if not 0 <= parents[i] < i or parents[i] != cur or not 0 <= tokens[i] < V:
            continue
        p, q = clean(target[cur]), clean(draft[cur])
        if uniforms[i] * q[tokens[i]] * z < max(0.0, p[tokens[i]] - w * q[tokens[i]]):
            cur, w, z = i, 0.0, 1.0
            taken.append(i)
        elif z > 0:
            w += z
            z = math.fsum(np.maximum(p - w * q, 0.0))
    p, q = clean(target[cur]), clean(draft[cur])
    left = np.maximum(p - w * q, 0.0) if z > 0 else p
    sums = np.cumsum(left)
    hit = (sums >= uniforms[0] * sums[-1]) & (left > 0)
    return taken, int(np.argmax(hit)) if hit.any() else 0

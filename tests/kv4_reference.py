"""Plain 64-bit restatements of the operators around the 4-bit cache, and bounds of what the kernels may be off by."""
import math

import numpy as np
import torch

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}     # half a step, relative
# and half a step of the subnormal numbers: fp16 outputs below 2^-14 lie 2^-24 apart, whatever their size
SUBNORMAL = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


def quantize(x, group):
    """[..., D] -> codes, steps, offsets in 64 bits."""
    y = x.double().unflatten(-1, (-1, group))
    lo, hi = y.amin(-1), y.amax(-1)
    step = ((hi - lo) / 15).to(x.dtype).double()
    bad = ~torch.isfinite(y).all(-1)
    step = torch.where(bad, 0.0, step)
    lo = torch.where(bad, math.nan, lo)
    safe = torch.where(step > 0, step, 1.0)[..., None]
    # 64 bits do not hold every difference either (0.25 + 2^-126 does not fit): its rounding error decides where it would sit on a border
    off = lo[..., None]
    d = y - off
    err = (y - (d + off)) + (((d + off) - d) - off)
    code = (d / safe).round()
    up, down = (d - (code + 0.5) * safe) + err, (d - (code - 0.5) * safe) + err
    odd = code % 2 == 1
    code = code + ((up > 0) | ((up == 0) & odd)).double() - ((down < 0) | ((down == 0) & odd)).double()
    code = torch.where(step[..., None] > 0, code, 0.0).nan_to_num(0.0).clamp(0, 15)
    return code.flatten(-2), step, lo


def held(x, group):
    """What the cache holds for x, in 64 bits."""
    code, step, lo = quantize(x, group)
    return (lo[..., None] + step[..., None] * code.unflatten(-1, (-1, group))).flatten(-2)


def cell_bytes(d, group):
    return 16 * (d + 8 * d // group)


def write_row(cache, slot, k, v, group, page_size):
    """Enters one token [kv_heads, D] into a numpy uint8 cache, byte by byte as the format says."""
    heads, d = k.shape
    page, place = divmod(slot, page_size)
    cell, r = divmod(place, 16)
    base = cell * cell_bytes(d, group)
    blocks = max(1, d // 128)
    kper, vper = min(4, d // 32), min(2, d // 64)
    for side, x in enumerate((k, v)):
        code, step, lo = quantize(x, group)
        code = code.to(torch.int64).numpy()
        pairs = torch.stack((step.to(x.dtype), lo.to(x.dtype)), -1).contiguous().view(torch.uint8).reshape(heads, d // group, 4).numpy()
        for h in range(heads):
            for e in range(0, d, 4):
                word = sum(int(code[h, e + j]) << (4 * j) for j in range(4))
                b, in_block = (e // 128, e % 128) if blocks > 1 or d == 128 else (0, e)
                if side == 0:
                    w, rest = divmod(in_block, 32)
                    at = ((((b * 16 + r) * 4 + rest // 8) * kper + w) * 2 + rest % 8 // 4) * 2
                else:
                    w, rest = divmod(in_block, 64)
                    half, rest = divmod(rest, 32)
                    at = 8 * d + ((((((b * 2 + r // 8) * 8 + rest // 4) * 4 + r % 8 // 2) * vper + w) * 2 + half) * 2 + r % 2) * 2
                cache[page, h, base + at] = word & 255
                cache[page, h, base + at + 1] = word >> 8
            for g in range(d // group):
                at = base + 16 * d + side * 64 * (d // group) + (r * (d // group) + g) * 4
                cache[page, h, at:at + 4] = pairs[h, g]


def rotary(x, positions, frequencies, interleaved, factor):
    r = 2 * len(frequencies)
    angle = positions.double().view(-1, 1, 1) * frequencies
    c, s = angle.cos(), angle.sin()
    y = x.double().clone()
    a, b = (x[..., :r:2].double(), x[..., 1:r:2].double()) if interleaved else (x[..., :r // 2].double(), x[..., r // 2:r].double())
    first, second = (a * c - b * s) * factor, (b * c + a * s) * factor
    if interleaved:
        y[..., :r:2], y[..., 1:r:2] = first, second
    else:
        y[..., :r // 2], y[..., r // 2:r] = first, second
    return y


def attention(q, k, v, length, scale, window, group, dense=False):
    """One request: q [n, heads, D], k, v [length, kv_heads, D] as given to append.  Returns out, bound of its error, lse, bound of a score's rounding
    (64 bits).

    The bound counts, per output: half a step of the output's type; half an fp16 step (2^-11) of every product weight * step, times
    |code - 8|; 2^-10 for what bounded scores do to the weights (2^-20 of the sum of |q| |k| per score, twice) and for sums in 32 bits;
    weights that become subnormal, 2^-28 of the largest each.
    dense: for many queries keys and values are rounded to fp16 on the way, middle and result (2^-11 each): a score is then off by 2^-10 of the
    sum of |q| (|k| + |middle|), a weight by twice that relative to the others, and the values count for 2^-10 more."""
    n, heads, d = q.shape
    kv_heads = k.shape[1]
    ratio = heads // kv_heads
    out = torch.zeros(n, heads, d, dtype=torch.float64)
    bound = torch.zeros_like(out)
    lse = torch.full((n, heads), -math.inf, dtype=torch.float64)
    score_bound = torch.zeros((), dtype=torch.float64)
    if n == 0 or length == 0:
        return out, bound, lse, score_bound
    pos = torch.arange(length - n, length)[:, None]
    tok = torch.arange(length)
    seen = tok <= pos
    if window:
        seen &= tok > pos - window
    kd = held(k[:length], group)
    _, kstep, klo = quantize(k[:length], group)
    code, step, lo = quantize(v[:length], group)
    vd = held(v[:length], group)
    away = (step[..., None] * (code.unflatten(-1, (-1, group)) - 8).abs()).flatten(-2)
    whole = away + (lo + 8 * step).abs().repeat_interleave(group, -1)
    for h in range(heads):
        g = h // ratio
        s = q[:, h].double() @ kd[:, g].T * scale
        mag = (q[:, h].double().abs() @ kd[:, g].abs().T * scale)
        s = torch.where(seen, s, -math.inf)
        rows = seen.any(-1)
        p = torch.zeros_like(s)
        p[rows] = s[rows].softmax(-1)
        lse[rows, h] = s[rows].logsumexp(-1)
        pv = torch.where(seen[..., None], p[..., None] * vd[None, :, g], 0.0) if p.numel() * d <= 1 << 26 else None
        out[:, h] = pv.sum(1) if pv is not None else p @ vd[:, g]
        worst = torch.where(seen, mag, 0.0).nan_to_num(0.0).amax(-1, keepdim=True)
        a, w = p @ away[:, g].nan_to_num(0.0), p @ whole[:, g].nan_to_num(0.0)
        bound[:, h] = HALF[q.dtype] * (out[:, h].abs() + w * 2.0 ** -9) + 2.0 ** -11 * a + (2.0 ** -10 * 2.0 ** -4 + 2.0 ** -19 * worst) * w + \
            length * 2.0 ** -28 * whole[:, g].nan_to_num(0.0).amax(0) + SUBNORMAL[q.dtype]
        if dense:
            middle = klo + 8 * kstep
            size = kd.abs() + middle.abs().repeat_interleave(group, -1)
            off = torch.where(seen, 2.0 ** -10 * q[:, h].double().abs() @ size[:, g].T * scale, 0.0).nan_to_num(0.0).amax(-1, keepdim=True)
            score_bound = torch.maximum(score_bound, off.max())
            bound[:, h] += (2.0 ** -10 + torch.expm1(2 * off)) * w + 2.0 ** -11 * w
    return out, bound, lse, score_bound


def pages_of(lengths, page_size, extra, seed):
    """A block table of pages in any order, and the number of pages."""
    used = [-(-n // page_size) for n in lengths]
    pages = sum(used) + extra
    order = np.random.RandomState(seed).permutation(pages)
    table = np.zeros((len(lengths), max(used + [1])), dtype=np.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    return torch.from_numpy(table), pages

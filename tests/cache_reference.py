"""Plain reference of the paged 8-bit cache, on the CPU: append in FP32 as the definition says (its results are exact), attention in
64 bits row by row, with the error that the kernel's arithmetic may make computed beside each output."""
import math

import numpy as np
import torch

LOW, HIGH = -100, 120
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def exponent_of(scale):
    """Exponent of a stored scale as the library reads it: the float's exponent field, clamped."""
    return min(max(((int(np.float32(scale).view(np.uint32)) >> 23) & 255) - 127, LOW), HIGH)


def exponent_for(most):
    """Smallest e with most <= 448 * 2^e, clamped."""
    if not most > 0:
        return LOW
    e = math.floor(math.log2(most)) - 9
    while most > 448.0 * 2.0 ** e:
        e += 1
    return min(max(e, LOW), HIGH)


def to_e4m3(x):
    """float32 array within 448 to e4m3 bytes, infinities and NaN as NaN."""
    x = np.where(np.isfinite(x), x, np.float32(np.nan)).astype(np.float32)
    return torch.from_numpy(np.ascontiguousarray(x)).to(torch.float8_e4m3fn).view(torch.uint8).numpy()


def from_e4m3(b):
    return torch.from_numpy(np.ascontiguousarray(b)).view(torch.float8_e4m3fn).to(torch.float64).numpy()


def rotate(x, cos, sin):
    """x [heads][D], cos and sin [D], all float32; products rounded before the sum."""
    h = x.shape[-1] // 2
    lo, hi = x[..., :h], x[..., h:]
    with np.errstate(invalid="ignore", over="ignore"):
        return np.concatenate([lo * cos[:h] - hi * sin[:h], hi * cos[h:] + lo * sin[h:]], -1).astype(np.float32)


class Pages:
    """Host copy of a cache with both halves as [page][head][slot][D] bytes."""

    def __init__(self, keys, values, scales):
        k, v = keys.cpu().view(torch.uint8).numpy(), values.cpu().view(torch.uint8).numpy()
        pages, heads, blocks, _, width = k.shape
        self.size, self.heads, self.width, self.pages = 16 * blocks, heads, width, pages
        self.k = k.reshape(pages, heads, self.size, width).copy()
        self.v = np.ascontiguousarray(v.transpose(0, 1, 2, 4, 3)).reshape(pages, heads, self.size, width).copy()
        self.scales = scales.cpu().numpy().copy()


def spans(starts, lengths, tokens):
    """(b, first row, count, position of the first row) of every sequence."""
    for b in range(len(lengths)):
        low, high = (min(max(int(s), 0), tokens) for s in (starts[b], starts[b + 1]))
        count = max(0, high - low)
        yield b, low, count, max(int(lengths[b]), 0) - count


def append(pages, k, v, table, starts, lengths, q=None, cos=None, sin=None, out_q=None):
    """Appends to ``pages`` in place; returns the rotated queries on top of ``out_q`` (float32, unrounded)."""
    k, v = k.float().numpy(), v.float().numpy()
    size, tokens = pages.size, k.shape[0]
    limit = table.shape[1] * size
    if cos is not None:
        cos, sin = cos.numpy(), sin.numpy()
        limit = min(limit, cos.shape[0])
    rotated = None if q is None else out_q.float().numpy().copy()
    for b, row, count, first in spans(starts, lengths, tokens):
        held = {}
        for i in range(count):
            at = first + i
            if 0 <= at < limit:
                held.setdefault(at // size, []).append((at % size, row + i, at))
                if q is not None:
                    rotated[row + i] = rotate(q[row + i].float().numpy(), cos[at], sin[at])
        for column, new in held.items():
            page = int(table[b, column])
            if not 0 <= page < pages.pages:
                continue
            slots, rows = [s for s, _, _ in new], [r for _, r, _ in new]
            turned = np.stack([k[r] if cos is None else rotate(k[r], cos[at], sin[at]) for _, r, at in new])
            for which, cells, x in ((0, pages.k, turned), (1, pages.v, v[rows])):
                for h in range(pages.heads):
                    y = x[:, h]
                    finite = np.abs(y[np.isfinite(y)])
                    e, before = exponent_for(float(finite.max(initial=0.0))), exponent_of(pages.scales[page, h, which])
                    if slots[0] > 0:
                        e = max(e, before)
                        if e > before:
                            kept = cells[page, h, :slots[0]]
                            cells[page, h, :slots[0]] = to_e4m3((from_e4m3(kept) * 2.0 ** (before - e)).astype(np.float32))
                    pages.scales[page, h, which] = 2.0 ** e
                    with np.errstate(invalid="ignore"):
                        cells[page, h, slots] = to_e4m3((y.astype(np.float64) * 2.0 ** -e).astype(np.float32))
    return rotated


def attention(pages, q, table, starts, lengths, causal=True, radius=-1, max_keys=0):
    """float64 output, lse and the error that the kernel may make in each, for the rows of the sequences; rows of none are NaN.

    The bounds count the roundings. Scores: q in one (16-bit types, exact) or two fp16 terms (2^-22 of each value), products summed
    in FP32 (a step of 2^-24 for each of the D terms, doubled for the matrix core's own order and rounding), and the exponent's
    argument, rounded to 2^-24 of its size twice. Weights: half a step of fp16 (2^-11) or of two terms (2^-22); those 2^-21 and more below
    the largest (weight times V scale) are off by at most half of fp16's smallest step instead, 2^-32 of the largest. exp2 and the
    sums: 2^-23 each and 2^-24 for every key. The output: half a step of its type."""
    size, heads, width = pages.size, pages.heads, pages.width
    tokens, query_heads, _ = q.shape
    group = query_heads // heads
    two = q.dtype == torch.float32
    rows = q.double().numpy()
    out = np.full((tokens, query_heads, width), np.nan)
    tol = np.zeros((tokens, query_heads, width))
    lse, lse_tol = np.full((tokens, query_heads, 2), np.nan), np.zeros((tokens, query_heads, 2))
    weight_step = 2.0 ** -22 if two else 2.0 ** -11
    exponents = np.clip(((pages.scales.view(np.uint32) >> 23) & 255).astype(int) - 127, LOW, HIGH)
    most = table.shape[1] * size
    if max_keys:
        most = min(most, max_keys)
    for b, row, count, first in spans(starts, lengths, tokens):
        length = min(max(int(lengths[b]), 0), most)
        place = np.arange(length)
        ids = np.asarray(table[b], dtype=np.int64)[place // size] if length else np.zeros(0, np.int64)
        real = (ids >= 0) & (ids < pages.pages)
        safe = np.where(real, ids, 0)
        for h in range(heads):
            ek, ev = exponents[safe, h, 0], exponents[safe, h, 1]
            k8, v8 = from_e4m3(pages.k[safe, h, place % size]), from_e4m3(pages.v[safe, h, place % size])
            k, v = k8 * np.exp2(ek.astype(float))[:, None], v8 * np.exp2(ev.astype(float))[:, None]
            for i in range(count):
                at = first + i
                sees = real.copy()
                if causal:
                    sees &= place <= at
                if radius >= 0:
                    sees &= np.abs(place - at) <= radius
                for n in range(h * group, (h + 1) * group):
                    r = row + i
                    if not sees.any():
                        out[r, n], lse[r, n] = 0.0, (-math.inf, 0.0)
                        continue
                    x = rows[r, n]
                    with np.errstate(all="ignore"):
                        s = k[sees] @ x / math.sqrt(width)
                        size_of_s = np.abs(k[sees]) @ np.abs(x) / math.sqrt(width)
                        m = s.max()
                        p = np.exp(s - m)
                        l = p.sum()
                        out[r, n], lse[r, n] = p @ v[sees] / l, (m, l)
                        off = size_of_s.max() * (2 * width * 2.0 ** -24 + (2.0 ** -22 if two else 0.0))
                        off += 2 * 2.0 ** -24 * (1.5 * np.abs(s).max() + np.abs(ev[sees]).max() + 32)
                        keys = sees.sum()
                        share = p @ np.abs(v[sees]) / l
                        small = 2.0 ** -32 * (p * np.exp2(ev[sees].astype(float))).max() * np.abs(v8[sees]).sum(0) / l
                        sums = keys * 2.0 ** -24 + 8 * 2.0 ** -23
                        tol[r, n] = HALF_STEP[q.dtype] * np.abs(out[r, n]) + share * (weight_step + 2 * off + 2 * sums) + small
                        if q.dtype == torch.float16:
                            tol[r, n] += 2.0 ** -25
                        lse_tol[r, n] = off + 2.0 ** -22 * abs(m), l * (2 * off + sums)
    return out, lse, tol, lse_tol

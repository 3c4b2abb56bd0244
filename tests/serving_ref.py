"""The 8-bit decoder layer's operators from their definitions, in 64 bits (numpy; slow and plain)."""
import math

import numpy as np
import torch


def f64(t):
    return t.detach().cpu().double().numpy()


def half_step(dtype):
    """A rounding to ``dtype`` is off by at most this, relative to the value."""
    return torch.finfo(dtype).eps / 2


def smallest_half_step(dtype):
    """... and by at most this where the value is too small for a full mantissa."""
    return float(torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2)


def to_integers(x, scale):
    """x / scale to the nearest integers, ties to even; zeros where there is no finite scale."""
    if not np.isfinite(scale) or scale == 0:
        return np.zeros_like(x)
    return np.clip(np.rint(x / np.float64(scale)), -127, 127)


def quantize_rows(x):
    x = f64(x)
    scales = np.array([np.float32(np.abs(r).max() / 127) for r in x], dtype=np.float32)
    return np.stack([to_integers(r, s) for r, s in zip(x, scales)]).astype(np.int8), scales


def matmul_scaled(a, sa, b, sb, bias):
    """(result, what a 32-bit evaluation of it may be off by)."""
    p = (f64(a) @ f64(b).T) * f64(sa)[:, None] * f64(sb)[None, :]
    add = np.zeros(b.shape[0]) if bias is None else f64(bias)
    # the integer's conversion, two products and one sum, each rounded to 24 bits
    return p + add, 4 * 2.0 ** -24 * (np.abs(p) + np.abs(add)) + 4 * 2.0 ** -149


def rotate(x, cos, sin, interleaved):
    """x [heads, d] at one position, in 64 bits."""
    half = len(cos)
    y = x.copy()
    one, two = (np.arange(half) * 2, np.arange(half) * 2 + 1) if interleaved else (np.arange(half), np.arange(half) + half)
    y[:, one] = x[:, one] * cos - x[:, two] * sin
    y[:, two] = x[:, two] * cos + x[:, one] * sin
    return y


def append(data, scales, starts, lengths, table, k, v, cos, sin, interleaved):
    """The cache after the call (copies), everything as numpy arrays; k and v [tokens, heads, d] in 64 bits."""
    data, scales = data.copy(), scales.copy()
    page = data.shape[3]
    for b, length in enumerate(lengths):
        first, fresh = starts[b], starts[b + 1] - starts[b]
        old = length - fresh
        for lo in range(old // page * page, length, page):
            if fresh == 0:
                break
            slot, begin, end = table[b][lo // page], max(lo, old), min(lo + page, length)
            for side, x in enumerate((k, v)):
                rows = x[first + begin - old:first + end - old]
                if side == 0 and cos is not None:
                    rows = np.stack([rotate(r, cos[begin + i], sin[begin + i], interleaved) for i, r in enumerate(rows)])
                for h in range(data.shape[2]):
                    with np.errstate(invalid="ignore"):
                        now = np.float32(np.abs(rows[:, h]).max() / 127)
                    was = scales[side, slot, h] if begin > lo else np.float32(0)
                    kept = data[side, slot, h, :begin - lo]
                    if np.isfinite(now) and now > was and was > 0:
                        kept[:] = np.rint(kept.astype(np.float64) * np.float64(was) / np.float64(now)).astype(np.int8)
                    if np.isfinite(now):
                        now = max(now, was)
                    scales[side, slot, h] = now
                    data[side, slot, h, begin - lo:end - lo] = to_integers(rows[:, h], now).astype(np.int8)
    return data, scales


def attend(data, scales, starts, lengths, table, q, scale, causal, window, softcap, dtype):
    """(result, bound): NaN rows of the result are those that no sequence has.  The bound follows a kernel that multiplies exact f16
    or bf16 queries and 8-bit keys into 32-bit sums, holds softmax statistics in 32 bits, rounds the weights to f16 and the
    result to ``dtype``."""
    tokens, heads, d = q.shape
    page, group = data.shape[3], heads // data.shape[2]
    out, bound = np.full(q.shape, np.nan), np.zeros(q.shape)
    for b, length in enumerate(lengths):
        first, fresh = starts[b], starts[b + 1] - starts[b]
        if fresh == 0:
            continue
        at = np.arange(length)
        slot, row = np.array(table[b], dtype=np.int64)[at // page], at % page
        for h in range(heads):
            k = data[0, slot, h // group, row].astype(np.float64) * scales[0, slot, h // group][:, None].astype(np.float64)
            v = data[1, slot, h // group, row].astype(np.float64) * scales[1, slot, h // group][:, None].astype(np.float64)
            for i in range(fresh):
                position = length - fresh + i
                lo = max(0, position - window + 1) if window > 0 else 0
                hi = position + 1 if causal else length
                x = q[first + i, h]
                if lo >= hi:
                    out[first + i, h] = 0
                    continue
                s = k[lo:hi] @ x * scale
                # d + 6 roundings, of the sum, the two scales' products and their own, each against the sum of magnitudes; keys
                # may be summed as integers plus 128 (up to 255) with 128 times the sum of the query taken off again
                unsigned = 256 * scales[0, slot[lo:hi], h // group].astype(np.float64)[:, None]
                off = ((d + 6) * 2.0 ** -24 * abs(scale) * ((np.abs(k[lo:hi]) + unsigned) @ np.abs(x))).max()
                if softcap > 0:
                    s = softcap * np.tanh(s / softcap)  # its slope is at most 1
                    off += 16 * 2.0 ** -24 * softcap
                off += 4 * 2.0 ** -24 * np.abs(s).max()  # exponents in powers of two
                p = np.exp(s - s.max())
                p /= p.sum()
                o, most = p @ v[lo:hi], p @ np.abs(v[lo:hi])
                out[first + i, h] = o
                # weights: twice the scores' error (numerator and sum), twice f16's half step (the sum may be over the rounded weights:
                # with w (1 + e) for w, |e| <= u, the result moves by |sum w e (v - o)| / sum w (1 + e) <= 2 u / (1 - u) sum w |v|), the
                # exponential's and the sums' roundings
                error = most * (2 * off + 2 * 2.0 ** -11 + 2.0 ** -20 + (hi - lo) * 2.0 ** -23)
                # f16 has steps of 2^-24 at its lower end.  Weights are held as p * scale / r * 2^n, r at most twice the largest
                # scale of the sequence's pages (rows of one call are weighed together, whatever the mask leaves to each), and n at least 7 (more would leave no room for a maximum that grows by up to 2^8 before it is
                # taken up), so half a step is 2^-25 * 2^-7 * 2 * scale = 2^-31 * scale for each integer; sums of p are at least 1
                integers = np.abs(data[1, slot[lo:hi], h // group, row[lo:hi]].astype(np.float64)).sum(axis=0)
                error += 2.0 ** -31 * np.abs(scales[1, slot, h // group]).max() * integers
                bound[first + i, h] = error + half_step(dtype) * (np.abs(o) + error) + smallest_half_step(dtype)
    return out, bound


def attend_capped(data, scales, starts, lengths, table, q, scale, softcap, dtype, missing=()):
    """As ``attend`` with a causal mask; without the tokens of the pages (sequence, index in its table) that are ``missing``.  The bound is
    for caps of any size, 0 for none: a capped score is off by 16 units of 2^-24 of itself.  (Just above
    a half of the cap it is cap (1 - q), q = 2 / (e^(2 z) + 1) = 0.54: e to 2^-22 and four roundings of its argument of 1, so the
    denominator to 5.9 + 1 units, the quotient to another 4; 10.9 * 0.54 / 0.46 + 1 = 13.7.  Below, a quotient of sums of positive terms: 9.)"""
    tokens, heads, d = q.shape
    page, group = data.shape[3], heads // data.shape[2]
    out, bound = np.full(q.shape, np.nan), np.zeros(q.shape)
    for b, length in enumerate(lengths):
        first, fresh = starts[b], starts[b + 1] - starts[b]
        at = np.array([j for j in range(length) if (b, j // page) not in missing], dtype=np.int64)
        slot, row = np.array(table[b], dtype=np.int64)[at // page], at % page
        for h in range(heads):
            of = scales[:, slot, h // group].astype(np.float64)[..., None]
            k, v = (data[side, slot, h // group, row].astype(np.float64) * of[side] for side in (0, 1))
            for i in range(fresh):
                hi = int((at <= length - fresh + i).sum())
                x = q[first + i, h]
                if hi == 0:
                    out[first + i, h] = 0
                    continue
                s = k[:hi] @ x * scale
                off = ((d + 6) * 2.0 ** -24 * abs(scale) * ((np.abs(k[:hi]) + 256 * of[0, :hi]) @ np.abs(x))).max()
                if softcap > 0:
                    s = softcap * np.tanh(s / softcap)
                off += (16 + 4) * 2.0 ** -24 * np.abs(s).max()
                if softcap > 0:
                    off = min(off, 2 * softcap)  # both lie within the cap
                p = np.exp(s - s.max())
                p /= p.sum()
                o, most = p @ v[:hi], p @ np.abs(v[:hi])
                out[first + i, h] = o
                error = most * (2 * off + 2 * 2.0 ** -11 + 2.0 ** -20 + hi * 2.0 ** -23)
                error += 2.0 ** -31 * of[1].max() * np.abs(v[:hi] / of[1, :hi]).sum(axis=0)
                bound[first + i, h] = error + half_step(dtype) * (np.abs(o) + error) + smallest_half_step(dtype)
    return out, bound

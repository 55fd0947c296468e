"""Plain 64-bit forms of the operators over several sequences (include/hp_hip.h, "Several sequences at once").

Written from their definitions, with numpy loops over sequences, heads and positions; inputs are the values that the
device buffers hold.  Each returns float64 (not rounded to the output type), and, where a bound needs it, what the
rounding errors of an f32 evaluation scale with.
"""
from __future__ import annotations

import math

import numpy as np


def rms(x, weight, eps):
    x = np.asarray(x, np.float64)
    y = x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps)
    return y if weight is None else y * np.asarray(weight, np.float64)


def rotate(x, position, dims, base, factors):
    """Rows [head][D] of one token at `position`."""
    y = np.array(x, np.float64)
    for u in range(dims // 2):
        a = position * base ** (-2.0 * u / dims)
        if factors is not None:
            a /= float(factors[u])
        c, s = math.cos(a), math.sin(a)
        p, q = x[:, u].copy(), x[:, u + dims // 2].copy()
        y[:, u] = p * c - q * s
        y[:, u + dims // 2] = p * s + q * c
    return y


def places(lengths, offsets, tokens, page_size, width):
    """(row, sequence, position) of every row that belongs to a sequence and has a place in its table."""
    out = []
    for s, n in enumerate(lengths):
        begin, end = (s, s + 1) if offsets is None else (offsets[s], offsets[s + 1])
        for t in range(begin, min(end, tokens)):
            p = int(n) - (end - t)
            if 0 <= p < width * page_size:
                out.append((t, s, p))
    return out


def append(q, k, v, lengths, offsets, pages, page_size, page_count, *, q_norm=None, k_norm=None, norm_values=False,
           eps=1e-6, rope_dims=0, base=10000.0, factors=None):
    """Per placed row: (row, q [Hq][D], k, v [Hkv][D], page or -1, slot)."""
    got = []
    for t, s, p in places(lengths, offsets, len(k), page_size, pages.shape[1]):
        qt = None if q is None else (rms(q[t], q_norm, eps) if q_norm is not None else np.asarray(q[t], np.float64))
        kt = rms(k[t], k_norm, eps) if k_norm is not None else np.asarray(k[t], np.float64)
        vt = k[t] if v is None else v[t]
        vt = rms(vt, None, eps) if norm_values else np.asarray(vt, np.float64)
        qt = None if qt is None else rotate(qt, p, rope_dims, base, factors)
        kt = rotate(kt, p, rope_dims, base, factors)
        page = int(pages[s, p // page_size])
        got.append((t, qt, kt, vt, page if 0 <= page < page_count else -1, p % page_size))
    return got


def attend(q, k, v, scale):
    """One query row q [D] over k, v [n][D]: (out [D], sum p |v| [D], largest sum |q k| of a score)."""
    if len(k) == 0:
        z = np.zeros(v.shape[-1])
        return z, z, 0.0
    with np.errstate(all="ignore"):
        e = k @ q * scale
        p = np.exp(e - e.max())
        p /= p.sum()
        # (a weight of exactly 0 makes a NaN of an infinite value)
        return p @ v, p @ np.abs(v), float((np.abs(k) @ np.abs(q)).max() * scale)


def paged_attention(q, keys, values, lengths, pages, page_size, page_count, window, scale):
    """q [S][Hq][D] over pools [page][Hkv][slot][D] (as values): out, sum p |v|, score sizes and key counts per (s, h)."""
    S, H, D = q.shape
    group = H // keys.shape[1]
    out, mass = np.zeros((S, H, D)), np.zeros((S, H, D))
    size, count = np.zeros((S, H)), np.zeros((S, H), np.int64)
    for s in range(S):
        end = min(max(int(lengths[s]), 0), pages.shape[1] * page_size)
        at = np.arange(max(0, end - window) if window else 0, end)
        page = pages[s, at // page_size]
        at, page = at[(page >= 0) & (page < page_count)], page[(page >= 0) & (page < page_count)]
        for h in range(H):
            k, v = keys[page, h // group, at % page_size], values[page, h // group, at % page_size]
            out[s, h], mass[s, h], size[s, h] = attend(np.asarray(q[s, h], np.float64), np.asarray(k, np.float64),
                                                       np.asarray(v, np.float64), scale)
            count[s, h] = len(at)
    return out, mass, size, count


def packed_attention(q, k, v, offsets, window, scale, only=None):
    """Rows of every sequence (or those in `only`): {row: (out [Hq][D], sum p |v|, score size [Hq], keys)}."""
    group = q.shape[1] // k.shape[1]
    got = {}
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    for begin, end in zip(offsets[:-1], offsets[1:]):
        for t in range(begin, end):
            if only is not None and t not in only:
                continue
            first = max(begin, t - window + 1) if window else begin
            rows = [attend(q[t, h], k[first:t + 1, h // group], v[first:t + 1, h // group], scale)
                    for h in range(q.shape[1])]
            got[t] = (np.stack([r[0] for r in rows]), np.stack([r[1] for r in rows]), np.array([r[2] for r in rows]),
                      t + 1 - first)
    return got


def logit_rules(logits, history=None, lengths=None, prompts=None, repetition=None, frequency=None, presence=None,
                bias_ids=None, bias_values=None, bias_counts=None, allowed=None):
    """The rules in f32, step by step as they are defined: [rows][n] f32, to the bit."""
    out = np.array(logits, np.float32)
    rows, n = out.shape
    f32 = np.float32
    with np.errstate(all="ignore"):
        for i in range(rows):
            if history is not None:
                told = [int(t) for t in history[i, :max(0, min(int(lengths[i]), history.shape[1]))]]
                start = 0 if prompts is None else max(0, int(prompts[i]))
                for t in {t for t in told if 0 <= t < n}:
                    x = out[i, t]
                    r = f32(1.0) if repetition is None else f32(repetition[i])
                    x = f32(x / r) if x > 0 else f32(x * r)
                    c = sum(1 for u in told[start:] if u == t)
                    x = f32(x - f32((f32(0.0) if frequency is None else f32(frequency[i])) * f32(c)))
                    if c:
                        x = f32(x - (f32(0.0) if presence is None else f32(presence[i])))
                    out[i, t] = x
            if bias_ids is not None:
                last = {}
                for t, b in zip(bias_ids[i][:max(0, int(bias_counts[i]))], bias_values[i]):
                    last[int(t)] = f32(b)
                for t, b in last.items():
                    if 0 <= t < n:
                        out[i, t] = f32(out[i, t] + b)
            if allowed is not None:
                bits = (np.asarray(allowed[i], np.uint32)[np.arange(n) // 32] >> (np.arange(n) % 32).astype(np.uint32)) & 1
                out[i, bits == 0] = -np.inf
    return out

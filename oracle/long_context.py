"""Plain forms of the operators of long contexts (include/hp_hip.h, "Long contexts"): page plans, pages of 8 bits with a
scale for each block and KV head, key bounds, block selection and attention over blocks.

Written from their definitions, with loops over sequences, blocks and heads, in whole numbers or 64 bits.
"""
from __future__ import annotations

import math

import numpy as np

from .serving import attend

MOST = {"i8": 127.0, "e4m3": 448.0}
BF16_MOST = 3.3895313892515355e38
F32_MOST = float(np.finfo(np.float32).max)


def plan(pages, lengths, new, keep, free, free_count, page_size, page_count, rows):
    """The arrays after a step, each as the header says; `pages` and `free` are not changed."""
    pages, free = pages.copy(), free.copy()
    S, W = pages.shape
    named = lambda e: 0 <= e < page_count  # noqa: E731
    stack = list(free[:max(0, min(int(free_count), page_count))])
    old = [max(0, int(n)) for n in lengths]
    for s in range(S):
        k = 0 if keep is None else int(keep[s])
        if k < 0:
            old[s] = 0
        for i in range(W if k < 0 else min(W, k // page_size)):
            if named(pages[s, i]) and len(stack) < page_count:
                stack.append(pages[s, i])
            pages[s, i] = -1
    full = list(stack)
    fresh = [int(o > 0) for o in old] if new is None else [max(0, int(n)) for n in new]
    missing, after, offsets = np.zeros(S, np.int64), np.zeros(S, np.int64), np.concatenate([[0], np.cumsum(fresh)])
    for s in range(S):
        after[s] = old[s] + fresh[s]
        for i in range(-(-old[s] // page_size), min(W, -(-int(after[s]) // page_size))):
            if not named(pages[s, i]):
                entry = stack.pop() if stack else -1
                pages[s, i] = entry if named(entry) else -1
        if fresh[s]:  # the pages that the new tokens lie in
            missing[s] = sum(i >= W or not named(pages[s, i]) for i in range(old[s] // page_size, -(-int(after[s]) // page_size)))
    free[:len(full)] = full
    maps = np.full((3, rows), -1, np.int64)
    for s in range(S):
        for t in range(fresh[s]):
            row, p = (s if new is None else int(offsets[s]) + t), old[s] + t
            if row < rows:
                page = int(pages[s, p // page_size]) if p // page_size < W else -1
                maps[:, row] = s, p, page * page_size + p % page_size if named(page) else -1
    return dict(pages=pages, lengths=after, free=free, free_count=len(stack), missing=missing, offsets=offsets,
                sequences=maps[0], positions=maps[1], slots=maps[2])


def block_scale(kind, most):
    """The scale of a block whose largest magnitude is `most`."""
    if most > 0:
        s = most / 127.0 if kind == "i8" else 2.0 ** math.ceil(math.log2(most / 448.0))
    else:
        s = 0.0
    return min(max(s, 2.0 ** -100), 2.0 ** 100)


def grown_scale(kind, old, most):
    """The scale of a block that was begun with the scale `old`."""
    if not most > old * MOST[kind]:
        return old
    return min(max(block_scale(kind, most), 1.25 * old if kind == "i8" else 0.0), 2.0 ** 100)


def outward(x, up):
    """f32 values in bf16's steps, rounded up or down; a NaN becomes the largest or smallest finite number."""
    x = np.where(np.isnan(x), BF16_MOST if up else -BF16_MOST, np.clip(x, -BF16_MOST, BF16_MOST)).astype(np.float32)
    bits = x.view(np.uint32) & np.uint32(0xffff0000)  # toward zero
    cut = bits.view(np.float32)
    short = cut < x if up else cut > x
    return np.where(short, (bits + np.uint32(0x10000)).view(np.float32), cut)


def bounds(keys, lengths, pages, page_size, page_count, block, touched):
    """keys [page][kv][slot][D] f32: {(page, block of the page): (least [kv][D], largest)} of the touched (s, block)s."""
    got = {}
    for s, b in touched:
        first = b * block
        page = int(pages[s, first // page_size])
        if not 0 <= page < page_count:
            continue
        end = min(int(lengths[s]), first + block)
        x = keys[page, :, first % page_size:first % page_size + end - first]
        odd = np.isnan(x).any(1)
        with np.errstate(all="ignore"):
            lo, hi = np.where(odd, np.nan, np.nanmin(x, 1)), np.where(odd, np.nan, np.nanmax(x, 1))
        got[page, first % page_size // block] = outward(lo, False), outward(hi, True)
    return got


def select(q, bound, lengths, pages, page_size, page_count, block, budget, first, last):
    """q [S][Hq][D], bound [page][kv][block][2][D]: the chosen blocks of every (sequence, KV head)."""
    S, H, D = q.shape
    kv, per = bound.shape[1], page_size // block
    q = np.clip(np.where(np.isnan(q), 0.0, q), -F32_MOST, F32_MOST)
    got = []
    for s in range(S):
        n = min(-(-max(0, int(lengths[s])) // block), pages.shape[1] * per)
        for h in range(kv):
            scores = []
            for b in range(n):
                page = int(pages[s, b // per])
                if not 0 <= page < page_count:
                    continue
                lo, hi = bound[page, h, b % per].astype(np.float64)
                rows = q[s, h * (H // kv):(h + 1) * (H // kv)]
                score = max(math.fsum(np.maximum(r * lo, r * hi)) for r in rows)
                scores.append((-math.inf if b < first or b >= n - last else -score, b))
            got.append(sorted(b for _, b in sorted(scores)[:budget]))
    return got


def block_attention(q, keys, values, lengths, pages, page_size, page_count, window, scale, lists=None, block=16):
    """q [S][Hq][D] over pools [page][kv][slot][D] of values; `lists` (one a (sequence, KV head)): their blocks only.
    out, sum p |v|, score sizes and key counts per (s, h)."""
    S, H, D = q.shape
    group = H // keys.shape[1]
    out, mass = np.zeros((S, H, D)), np.zeros((S, H, D))
    size, count = np.zeros((S, H)), np.zeros((S, H), np.int64)
    for s in range(S):
        end = min(max(int(lengths[s]), 0), pages.shape[1] * page_size)
        for h in range(H):
            if lists is None:
                at = np.arange(max(0, end - window) if window else 0, end)
            else:
                mine = [int(b) for b in lists[s * keys.shape[1] + h // group] if 0 <= int(b) * block < end]
                at = np.concatenate([np.arange(b * block, min(end, b * block + block)) for b in mine] + [np.zeros(0, int)]).astype(int)
            page = pages[s, at // page_size]
            at, page = at[(page >= 0) & (page < page_count)], page[(page >= 0) & (page < page_count)]
            k, v = keys[page, h // group, at % page_size], values[page, h // group, at % page_size]
            out[s, h], mass[s, h], size[s, h] = attend(np.asarray(q[s, h], np.float64), np.asarray(k, np.float64),
                                                       np.asarray(v, np.float64), scale)
            count[s, h] = len(at)
    return out, mass, size, count

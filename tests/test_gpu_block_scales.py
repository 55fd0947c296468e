"""Attention over pages whose blocks' value scales lie far apart, where each block's own share of the result can be told
from the others'.

Bounds.  A weight times its block's scale goes to f16 in two parts, at 2^9 to 2^12 for a row's largest W: what the parts
miss is 2^-21 of it, or half of f16's smallest step, 2^-25, which is 2^-34 of W at most.  2^(x - m) itself leaves f32 below
2^-126 where the scale is 2^100 at most: 2^-26, 2^-35 of W.  So a stored element of `most` misses 3 * 2^-35 most W for every
key, over the sum of the weights, whatever the other sequences' scales are.
"""
import numpy as np
import pytest

import test_gpu_long_context as base
from heliopause_amd import hip_kernels as H

pytestmark = pytest.mark.gpu

U = base.U
FULL = {"i8": 127.0, "e4m3": 448.0}


def attend(pool, q, scale, lists=None, stride=0):
    """The kernel's output, and what is exact of it: out, mass = sum p |v|, W / sum p, score sizes, keys."""
    t = base._torch()
    n, Hq, D = q.shape
    d_q = base.dev(q)
    got = t.full((n, Hq, D), 7.0, device="cuda")
    d_lists = None if lists is None else base.dev(np.asarray(lists, np.int32))
    H.block_attention_device(pool.cache(), pool.blocks(), Hq, d_q.data_ptr(), 0, got.data_ptr(), 0, scale=scale,
                             d_selected=base.ptr(d_lists), budget=0 if lists is None else len(lists[0]))
    base.sync()
    stored = [x.float().cpu().numpy().astype(np.float64) for x in (pool.keys, pool.values)]
    scales = [s.cpu().numpy().astype(np.float64) for s in pool.scales]
    out, mass, top, size, count = np.zeros(q.shape), np.zeros(q.shape), np.zeros((n, Hq)), np.zeros((n, Hq)), np.zeros((n, Hq))
    for s in range(n):
        for h in range(Hq):
            kvh = h // (Hq // pool.kv)
            if lists is None:
                at = np.arange(pool.lengths[s])
            else:
                at = np.concatenate([np.arange(b * pool.block, min((b + 1) * pool.block, pool.lengths[s])) for b in lists[s * pool.kv + kvh]])
            page, slot = pool.pages[s, at // pool.page], at % pool.page
            ks, vs = (x[page, kvh, slot // pool.block] for x in scales)
            k, v = stored[0][page, kvh, slot] * ks[:, None], stored[1][page, kvh, slot]
            x = k @ q[s, h].astype(np.float64) * scale
            p = np.exp(x - x.max())
            out[s, h], mass[s, h] = (p * vs) @ v / p.sum(), (p * vs) @ np.abs(v) / p.sum()
            top[s, h], count[s, h] = (p * vs).max() / p.sum(), len(at)
            size[s, h] = (np.abs(k) @ np.abs(q[s, h].astype(np.float64))).max() * scale
    return base.values(got), out, mass, top, size, count


def check(pool, got, out, mass, top, size, count, tied=False):
    """tied: keys of the same stored bits and scales have the same score to the bit, and the others have no weight."""
    d = 0.0 if tied else size * (2.0 ** -20 + (pool.D + 1) * U)
    weight = 2 * (d + 2.0 ** -20) + 2.0 ** -21 + 2 * (count + 64) * U + 4 * U
    absolute = 3 * 2.0 ** -35 * FULL[pool.type] * top * count
    bound = 1.01 * (mass * np.broadcast_to(weight, count.shape)[..., None] + absolute[..., None]) + 2.0 ** -149
    base.check(got, out, bound)


def value_scales(pool, s, exponents):
    for i, e in enumerate(exponents):
        page, b = pool.pages[s, i * pool.block // pool.page], i * pool.block % pool.page // pool.block
        pool.scales[1][int(page), :, b] = 2.0 ** e


@pytest.mark.parametrize("type", ["i8", "e4m3"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_each_sequence_by_its_own_scales(hip, type, D):
    """Tiny scales only beside a sequence of large ones: both to the same share of their own."""
    rng = np.random.default_rng(D)
    pool = base.Pool(rng, [64, 200, 64, 5], 2, D, 32, 16, type, spare=0)
    value_scales(pool, 0, [-100, -100, -99, -100])
    value_scales(pool, 1, [100, 99, 98, 100, 97, 100, 100, 99, 98, 99, 100, 100, 98])
    value_scales(pool, 2, [-60, -61, -62, -60])
    q = (rng.standard_normal((4, 4, D)) * 2).astype(np.float32)
    check(pool, *attend(pool, q, D ** -0.5))
    check(pool, *attend(pool, q, D ** -0.5, [[0, 2], [3, 1], [5, 12], [4, 0], [2, 0], [3, 3], [0, 0], [0, 0]]))


@pytest.mark.parametrize("type", ["i8", "e4m3"])
@pytest.mark.parametrize("apart,ahead", [(20, 10), (40, 30), (60, 70), (100, 40), (100, 120)])
def test_small_blocks_beside_large_ones(hip, type, apart, ahead):
    """Blocks whose scales are 2^apart below the others' and whose keys' scores are `ahead` (to base 2) above; the values of
    the large blocks are zeros in every other channel, which show the small ones alone."""
    t = base._torch()
    rng = np.random.default_rng(apart + ahead)
    D = 64
    pool = base.Pool(rng, [160], 1, D, 32, 16, type, spare=0)
    large = rng.permutation(10)[:5]
    value_scales(pool, 0, [apart if b in large else 0 for b in range(10)])
    pool.scales[0].fill_(1.0)
    # a score is 64 * 32 q scale for the small blocks' keys, and 0 for the large ones'
    keys, values = pool.keys.float(), pool.values.float()
    for b in range(10):
        rows = pool.pages[0, b // 2], 0, slice(b % 2 * 16, b % 2 * 16 + 16)
        keys[rows] = 0.0 if b in large else 32.0
        if b in large:
            values[rows + (slice(0, None, 2),)] = 0.0
    pool.keys.copy_(keys.to(pool.keys.dtype))
    pool.values.copy_(values.to(pool.values.dtype))
    t.cuda.synchronize()
    q = np.full((1, 2, D), ahead * np.log(2) / (64 * 32), np.float32)
    got, out, mass, top, size, count = attend(pool, q, 1.0)
    check(pool, got, out, mass, top, size, count)
    if ahead - apart > -22:  # (the bound tells the small blocks' share from nothing)
        assert (np.abs(out[..., ::2]) > 100 * 3 * 2.0 ** -35 * FULL[type] * (top * count)[..., None]).mean() > 0.9


def equal_scores(type, e, sign, D, n):
    """Scores of 2^e (to base 2) and up to 1.9 times that.  All keys of a head alike, so that all weigh the same whatever
    their blocks' value scales; in the last sequence every third block's keys score half as much, and take all or
    nothing."""
    rng = np.random.default_rng(e)
    lengths = [n, 33, n, n]
    pool = base.Pool(rng, lengths, 1, D, 32, 16, type, spare=0)
    pool.keys.fill_(64.0 if type == "e4m3" else 64)
    pool.scales[0].fill_(1.0)
    blocks = -(-n // 16)
    value_scales(pool, 0, rng.choice([20, -30, 5, 16, -14], blocks))
    value_scales(pool, 1, [-30, 20, -100])
    value_scales(pool, 2, rng.integers(-100, 101, blocks))
    value_scales(pool, 3, rng.integers(-100, 101, blocks))
    for b in range(0, blocks, 3):
        pool.scales[0][int(pool.pages[3, b // 2]), 0, b % 2] = 0.5
    q = (np.array([1.0, 1.25, 1.5, 1.9])[None, :, None] * np.full((4, 4, D), sign)).astype(np.float32)
    scale = 2.0 ** e * np.log(2) / (64 * D)
    check(pool, *attend(pool, q, scale), tied=True)
    some = sorted(rng.permutation(blocks)[:4])
    check(pool, *attend(pool, q, scale, [some, [2, 0, 1, 1], some, some]), tied=True)


@pytest.mark.parametrize("type", ["i8", "e4m3"])
@pytest.mark.parametrize("e", [10, 16, 20, 22])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("D,n", [(64, 100), (128, 5000), (256, 700)])
def test_equal_scores_whatever_the_value_scales(hip, type, e, sign, D, n):
    """The sum of the weights has its share of every key, those of blocks whose scale is 2^200 below another's too."""
    equal_scores(type, e, sign, D, n)


@pytest.mark.parametrize("type", ["i8", "e4m3"])
@pytest.mark.parametrize("e", [24, 25, 26, 27, 28, 29, 30, 31, 33, 60])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("D,n", [(64, 100), (128, 5000), (256, 700)])
def test_value_scales_under_large_scores(hip, type, e, sign, D, n):
    """Scores whose steps in f32 are 2 to 2^37, so that a scale's exponent is less than a step of them."""
    equal_scores(type, e, sign, D, n)

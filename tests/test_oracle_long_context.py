"""The plain forms of the operators of long contexts (oracle/long_context.py) against what follows from their definitions.
CPU only."""
import numpy as np
import pytest

from oracle import long_context as L
from oracle import serving as S


def test_pages_are_neither_lost_nor_dealt_twice():
    """A hundred random steps: every page is on the stack or named once; positions and slots agree with the table."""
    rng = np.random.default_rng(1)
    n, width, page, count = 9, 12, 16, 60
    pages, lengths = np.full((n, width), -1, np.int32), np.zeros(n, np.int64)
    free, free_count = rng.permutation(count).astype(np.int32), count
    for step in range(100):
        new = rng.integers(0, 40, n) * (rng.random(n) < 0.5)
        new = np.minimum(new, width * page - lengths)
        keep = np.where(rng.random(n) < 0.2, -1, 0)
        new = np.where(keep < 0, np.minimum(new, 20), new)
        got = L.plan(pages, lengths, new, keep, free, free_count, page, count, 500)
        pages, lengths, free, free_count = got["pages"], got["lengths"], got["free"], got["free_count"]
        named = pages[pages >= 0]
        assert sorted([*named, *free[:free_count]]) == list(range(count))
        for s in range(n):
            rows = np.flatnonzero(got["sequences"] == s)
            assert len(rows) == new[s] and list(got["positions"][rows]) == list(range(lengths[s] - new[s], lengths[s]))
            for t in rows:
                p = got["positions"][t]
                entry = pages[s, p // page]
                assert got["slots"][t] == (entry * page + p % page if entry >= 0 else -1)
        if got["missing"].any():  # the batch is cleared
            lengths[:] = 0
            got = L.plan(pages, lengths, np.zeros(n), np.full(n, -1), free, free_count, page, count, 0)
            pages, free, free_count = got["pages"], got["free"], got["free_count"]
            assert free_count == count and (pages == -1).all()


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
def test_scales_hold_their_blocks(kind):
    rng = np.random.default_rng(2)
    for most in [*np.exp(rng.uniform(-60, 60, 500)), 448.0, 448.0 * 2.0 ** -7, np.nextafter(448.0, 500), 127.0]:
        s = L.block_scale(kind, most)
        # (A * (1 / 127) * 127 is A but for the last bits)
        assert most <= L.MOST[kind] * s * (1 + 2.0 ** -50) and most > L.MOST[kind] * s * (0.5 if kind == "e4m3" else 0.999)
        assert L.grown_scale(kind, s, most * 0.99) == s
        g = L.grown_scale(kind, s, most * 1.2)
        assert g >= s and most * 1.2 <= L.MOST[kind] * g * (1 + 2.0 ** -50)
    assert L.block_scale(kind, 0.0) == 2.0 ** -100 and L.block_scale(kind, 1e38) == 2.0 ** 100


def test_outward():
    rng = np.random.default_rng(3)
    x = np.concatenate([rng.standard_normal(4000) * np.exp(rng.uniform(-80, 80, 4000)), [0.0, -0.0, 1.0, 1.00390625, 1e-45]]).astype(np.float32)
    lo, hi = L.outward(x, False), L.outward(x, True)
    assert (lo <= x).all() and (x <= hi).all() and (lo.view(np.uint32) & 0xffff == 0).all() and (hi.view(np.uint32) & 0xffff == 0).all()
    assert (hi - lo <= np.abs(x) * 2.0 ** -6.99 + 2.0 ** -133).all()
    assert L.outward(np.float32([np.nan, np.inf, -np.inf, 3.4e38]), True).tolist() == [L.BF16_MOST, L.BF16_MOST, -L.BF16_MOST, L.BF16_MOST]


def test_no_key_left_out_has_a_higher_bound():
    """A block's score is at least any of its keys' scores with any of the group's queries, and none that is left out is
    above one that is taken; with a budget for all, all are taken."""
    rng = np.random.default_rng(4)
    kv, D, page, block, n = 2, 16, 32, 16, 300
    count = -(-n // page)
    pages = rng.permutation(count).astype(np.int32)[None]
    keys = rng.standard_normal((count, kv, page, D)).astype(np.float32)
    q = rng.standard_normal((1, 4, D))
    got = L.bounds(keys, [n], pages, page, count, block, {(0, b) for b in range(-(-n // block))})
    bound = np.zeros((count, kv, page // block, 2, D))
    for (p, b), (lo, hi) in got.items():
        bound[p, :, b, 0], bound[p, :, b, 1] = lo, hi
    for budget in (1, 5, 19):
        rows = L.select(q, bound, [n], pages, page, count, block, budget, 0, 0)
        for h, taken in enumerate(rows):
            score = []
            for b in range(19):
                lo, hi = bound[pages[0, b // 2], h, b % 2]
                score.append(max(np.maximum(r * lo, r * hi).sum() for r in q[0, 2 * h:2 * h + 2]))
                end = min(n, b * block + block)
                k = keys[pages[0, b // 2], h, b * block % page:end - 1 - (end - 1) // page * page + 1]
                assert (k @ q[0, 2 * h:2 * h + 2].T).max() <= score[-1] + 1e-9
            assert len(taken) == min(budget, 19) and taken == sorted(taken)
            assert min(score[b] for b in taken) >= max([score[b] for b in range(19) if b not in taken], default=-np.inf)


def test_attention_over_all_blocks_is_the_paged_attention():
    rng = np.random.default_rng(5)
    pages = rng.permutation(12).astype(np.int32).reshape(2, 6)
    keys, values = rng.standard_normal((2, 12, 2, 16, 8))
    q = rng.standard_normal((2, 4, 8))
    want = S.paged_attention(q, keys, values, [90, 33], pages, 16, 12, 0, 0.3)
    lists = [list(range(6))] * 2 + [[0, 1, 2]] * 2
    for got in (L.block_attention(q, keys, values, [90, 33], pages, 16, 12, 0, 0.3),
                L.block_attention(q, keys, values, [90, 33], pages, 16, 12, 0, 0.3, lists, 16)):
        assert all(np.allclose(x, y, rtol=1e-12) for x, y in zip(got, want))

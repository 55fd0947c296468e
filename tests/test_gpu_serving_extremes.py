"""The operators over several sequences where their numbers are extreme: weights far below the largest, scores and scales
far from one, infinities among what counts; and the rules ahead of a sampler.

Bounds are those of test_gpu_serving.py's head, with what a case changes about them beside it.  Scores that the cases
below make are sums of one non-zero exact product, and far enough apart (or the same) that f32's rounding of them leaves
every weight 0 or 1 to below f32's step.
"""
import numpy as np
import pytest

import test_gpu_serving as base
from heliopause_amd import hip_kernels as H

pytestmark = pytest.mark.gpu

U, ELEM = base.U, base.ELEM
dev, dtype_of, half_step, sync, values = base.dev, base.dtype_of, base.half_step, base.sync, base.values


@pytest.fixture(scope="module")
def S(oracle):
    from oracle import serving

    return serving


def tensor(a, type):
    return base._torch().from_numpy(np.ascontiguousarray(a, dtype=np.float32)).cuda().to(dtype_of(type))


def packed(q, k, v, offsets, *, type, out=None, scale=1.0, window=0):
    """q, k, v device tensors [rows][heads][D]: the output as float64."""
    t = base._torch()
    out = out or type
    rows, heads, D = q.shape
    got = t.full((rows, heads, D), 7.0, dtype=dtype_of(out), device="cuda")
    off = dev(np.asarray(offsets, np.int32))
    sync()
    H.packed_attention_device(len(offsets) - 1, off.data_ptr(), rows, heads, k.shape[1], D, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                              ELEM[type], got.data_ptr(), ELEM[out], scale=scale, sliding_window=window)
    sync()
    return values(got)


def paged(pool, q, *, q_type="f32", out="f32", scale=1.0, window=0):
    t = base._torch()
    heads = q.shape[1]
    x = tensor(q, q_type)
    got = t.full(tuple(x.shape), 7.0, dtype=dtype_of(out), device="cuda")
    sync()
    H.paged_attention_device(pool.cache(), heads, x.data_ptr(), ELEM[q_type], got.data_ptr(), ELEM[out], scale=scale, sliding_window=window)
    sync()
    return values(got)


def place(pool, sequence, keys, vals):
    """Rows [position][kv head][D] of a sequence into its pages (as stored)."""
    t = base._torch()
    for rows, to in ((keys, pool.keys), (vals, pool.values)):
        x = t.from_numpy(np.ascontiguousarray(rows, dtype=np.float32)).cuda().to(to.dtype)
        for p in range(0, len(rows), pool.page):
            n = min(pool.page, len(rows) - p)
            to[int(pool.pages[sequence, p // pool.page]), :, :n] = x[p:p + n].transpose(0, 1)


# (D, heads, many rows) that take each form of the packed kernel: few blocks split their keys over two groups of waves,
# those of 2800 rows do not.
FORMS = [(64, 1, False), (64, 32, True), (128, 1, False), (128, 16, True), (256, 1, False), (256, 16, True)]


# ---- small weights -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("D,heads,many", FORMS)
@pytest.mark.parametrize("type", ["f16", "bf16"])
def test_packed_weights_far_below_the_largest(hip, S, type, D, heads, many):
    """A first key that outweighs each of the others by 2^22 to 2^28, and so many others that they count: their values
    are 1 and its value is 0, so the output is the share that they have.  An f16 weight is off by half a subnormal step
    at most, 2^-32 of the running maximum; the others' sum by n of those."""
    n = 6000
    rng = np.random.default_rng(D)
    k = np.zeros((n, 1, D))
    k[0, 0, 0], k[1:, 0, 1] = 16.0, rng.integers(-32, 33, n - 1) / 16.0
    q = np.zeros((n, heads, D))
    q[:, :, 0], q[:, :, 1] = 25.0 * np.log(2.0) / 16.0, np.log(2.0)
    v = np.ones((n, 1, D))
    v[0] = 0.0
    q, k, v = (tensor(x, type) for x in (q, k, v))
    got = packed(q, k, v, [0, n], type=type, out="f32")
    at = sorted({n - 1, n - 2, n // 2 + 7, 1000, 130, 33, 1, 0} | set(rng.integers(0, n, 6).tolist()))
    ref = S.packed_attention(values(q), values(k), values(v), [0, n], 0, 1.0, set(at))
    u = base._torch().finfo(dtype_of(type)).eps / 2
    for row in at:
        r, mass, size, keys = ref[row]
        weight = 2 * (size * D * U + 2.0 ** -20) + 2 * (keys + 64) * U
        bound = 1.01 * (mass * weight[:, None] + u * (mass + np.abs(r))) + half_step("f32", r) + (2.0 ** -32 * keys if type == "f16" else 0.0)
        base.check(got[row], r, bound)
    assert got[n - 1].min() > 2.0 ** -15  # (they do count)


# ---- large scores and scales ---------------------------------------------------------------------------------------------

def ranked(rng, n, ties):
    """n whole numbers 1 .. 200 (a key's score in steps), the largest so far twice here and there."""
    x = rng.integers(1, 200, n).astype(np.float64)
    for i in range(ties, n, ties):
        x[i] = x[:i].max()
    return x


def of_the_best(scores, rows):
    """Mean of the rows [key][D] whose score is the largest."""
    return rows[scores == scores.max()].mean(0)


@pytest.mark.parametrize("power", [20, 22, 23, 25, 26, 27, 28, 29, 32, 60, 110])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("type", ["f16", "bf16"])
def test_packed_large_scores(hip, type, sign, power):
    """Scores of about 2^power, above or below zero: the best key has the weight, or the best ones share it.  Off by the
    weights' rounding (none: 1) and that of sums and quotient, 2^-20 of the value."""
    rng = np.random.default_rng(power)
    for D, heads, many in FORMS:
        lengths = [1500, 1300] if many else [150, 70]
        n = sum(lengths)
        rank = np.concatenate([ranked(rng, m, 17) for m in lengths])
        k, q = np.zeros((n, 1, D)), np.zeros((n, heads, D))
        k[:, 0, 3] = rank if sign > 0 else 256 - rank
        q[:, :, 3] = sign
        v = rng.integers(-8, 9, (n, 1, D)).astype(np.float64)
        got = packed(*(tensor(x, type) for x in (q, k, v)), [0, lengths[0], n], type=type, out="f32", scale=2.0 ** (power - 8), window=90)
        for begin, rows in ((0, lengths[0]), (lengths[0], lengths[1])):
            for i in range(0, rows, 1 if n < 300 else 37):
                first = max(0, i - 89)
                ref = of_the_best(rank[begin + first:begin + i + 1], v[begin + first:begin + i + 1, 0])
                assert np.all(np.abs(got[begin + i] - ref) <= 2.0 ** -20 * 8), (D, i)


@pytest.mark.parametrize("power", [20, 22, 25, 26, 27, 28, 29, 32, 60, 110])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("type", ["f16", "bf16", "e4m3"])
def test_paged_large_scores(hip, type, sign, power):
    """The same over pages, whole and split over workgroups.  (e4m3 holds the whole numbers up to 16: ranks below that)"""
    rng = np.random.default_rng(power)
    for D in (64, 128, 256):
        lengths = [1, 33, 150, 3000]
        pool = base.Pool(rng, lengths, 1, D, 16, type, scales=(1.0, 1.0))
        ranks = []
        for s, n in enumerate(lengths):
            rank = ranked(rng, n, 17)
            rank = np.ceil(rank / 14.0) if type == "e4m3" else rank
            k, v = np.zeros((n, 1, D)), rng.integers(-8, 9, (n, 1, D)).astype(np.float64)
            k[:, 0, 3] = rank if sign > 0 else (16 if type == "e4m3" else 256) - rank
            place(pool, s, k, v)
            ranks.append((rank, v))
        q = np.zeros((len(lengths), 3, D))
        q[:, :, 3] = sign
        got = paged(pool, q, scale=2.0 ** (power - (4 if type == "e4m3" else 8)))
        for s, (rank, v) in enumerate(ranks):
            assert np.all(np.abs(got[s] - of_the_best(rank, v[:, 0])) <= 2.0 ** -20 * 8), (D, s)


@pytest.mark.parametrize("size,scale", [(2.0 ** 13, 2.0 ** 120), (1e20, 2.0 ** 90), (2.0 ** 127, 64.0), (2.0 ** 127, 2.0 ** 120), (2.0 ** 100, 2.0 ** 20)])
@pytest.mark.parametrize("type,q_type", [("f16", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("e4m3", "f32")])
def test_paged_large_queries_at_large_scales(hip, type, q_type, size, scale):
    """Keys of zeros score 0 whatever the query and the scale are, and share the weight; one key against the query's
    direction then has none, one along it all (where its score is within f32)."""
    rng = np.random.default_rng(1)
    for D in (64, 128, 256):
        lengths = [40, 300, 40, 1, 300]
        pool = base.Pool(rng, lengths, 1, D, 16, type, scales=(1.0, 1.0))
        q = np.full((len(lengths), 2, D), size)
        refs = []
        for s, n in enumerate(lengths):
            k, v = np.zeros((n, 1, D)), rng.integers(-8, 9, (n, 1, D)).astype(np.float64)
            refs.append(v[:, 0].mean(0))
            if s == 1:
                k[7, 0, 5] = -1.0
                refs[-1] = np.delete(v[:, 0], 7, 0).mean(0)
            if s == 4 and size * scale <= 2.0 ** 133:
                k[299, 0, 5] = 2.0 ** -6
                refs[-1] = v[299, 0]
            place(pool, s, k, v)
        got = paged(pool, q, q_type=q_type, scale=scale)
        # (weights 1 in two parts, exact; sums of up to 300 whole numbers exact; the quotient)
        assert np.all(np.abs(got - np.stack(refs)[:, None]) <= 2.0 ** -20 * 8), D


def test_paged_scores_of_ordinary_size_from_far_factors(hip, S):
    """bf16 keys of some 2^-125 under queries and a scale whose product is past f32's range."""
    rng = np.random.default_rng(2)
    lengths = [1, 40, 400]
    pool = base.Pool(rng, lengths, 2, 128, 16, "bf16")
    for s, n in enumerate(lengths):
        place(pool, s, rng.uniform(1, 4, (n, 2, 128)) * rng.choice([-1, 1], (n, 2, 128)) * 2.0 ** -126, rng.standard_normal((n, 2, 128)))
    q = np.zeros((3, 4, 128))
    q[:, :, [3, 40, 77]] = rng.uniform(1, 2, (3, 4, 3)) * rng.choice([-1, 1], (3, 4, 3)) * 2.0 ** 101
    got = paged(pool, q, scale=2.0 ** 30)
    ref, mass, size, count = S.paged_attention(values(tensor(q, "f32")), values(pool.keys), values(pool.values), pool.lengths,
                                               pool.pages, pool.page, pool.count, 0, 2.0 ** 30)
    base.check(got, ref, base.paged_bound("f32", "bf16", ref, mass, size, count, 128))


# ---- infinities that count ---------------------------------------------------------------------------------------------

@pytest.mark.parametrize("D,heads,many", FORMS)
@pytest.mark.parametrize("type", ["f16", "bf16"])
def test_packed_rows_whose_every_score_is_minus_infinity(hip, type, D, heads, many):
    """Row 0 and those behind it up to the first finite score: softmax of nothing but -inf is NaN, not a row without
    keys; later rows have the finite keys' values alone."""
    n = 2800 if many else 100
    k, q = np.zeros((n, 1, D)), np.ones((n, heads, D))
    k[:3, 0, 1], k[50, 0, 2] = -np.inf, -np.inf
    v = np.full((n, 1, D), 5.0)
    v[:3] = v[50] = 3.0
    got = packed(*(tensor(x, type) for x in (q, k, v)), [0, n], type=type, scale=0.125)
    assert np.isnan(got[:3]).all() and np.all(got[3:] == 5.0)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("type", ["f16", "bf16"])
@pytest.mark.parametrize("odd", [np.inf, -np.inf, np.nan])
def test_packed_value_whose_weight_is_nothing(hip, type, D, odd):
    """A value that is no number under a weight that rounds to 0: its column is no number for every row that sees it,
    wherever the tiles and blocks lie (the rows ahead of it in the batch move them), and stays for those that do not."""
    lead_of = {}
    for heads, lead in ((1, 0), (1, 1), (1, 40), (1, 77), (32 if D == 64 else 16, 2403), (32 if D == 64 else 16, 2500)):
        n = 300
        k, q = np.zeros((lead + n, 1, D)), np.zeros((lead + n, heads, D))
        k[lead, 0, 0], q[:, :, 0] = 30.0, 30.0     # the first key has the weight
        v = np.full((lead + n, 1, D), 2.0)
        v[lead + 100, 0, 6] = odd
        offsets = [0, n] if lead == 0 else [0, lead, lead + n]
        got = packed(*(tensor(x, type) for x in (q, k, v)), offsets, type=type)[lead:]
        assert np.all(got[:100] == 2.0) and np.all(np.delete(got, 6, 2) == 2.0)
        assert not np.isfinite(got[100:, :, 6]).any()
        lead_of[heads, lead] = got[:, 0, 6]
    first = lead_of[1, 0]
    assert all(np.array_equal(first, x, equal_nan=True) for x in lead_of.values())


@pytest.mark.parametrize("D", [64, 128, 256])
def test_paged_rows_whose_every_score_is_minus_infinity(hip, D):
    """f16 keys of -inf under queries of 1 + 2^-12, both of whose f16 parts are above zero: the scores are -inf.  Where
    all are, the row is NaN; where one is not, its value; where there is no key, zeros.  Rows that one workgroup has
    whole, and rows in many parts."""
    lengths = [1, 40, 200, 5000, 40, 200, 5000, 5000, 70, 0, 5000]
    pool = base.Pool(np.random.default_rng(4), lengths, 1, D, 16, "f16")
    one = {4: 39, 5: 3, 6: 4999, 7: 2500}  # sequence: its one finite key
    for s, n in enumerate(lengths):
        if not n:
            continue
        k, v = np.zeros((n, 1, D)), np.full((n, 1, D), 3.0)
        k[:, 0, 1] = -np.inf
        if s in one:
            k[one[s], 0, 1], v[one[s]] = 1.0, 5.0
        place(pool, s, k, v)
    pool.pages[8] = -1                      # no page at all
    pool.pages[10, :300] = -1               # only the last keys are there, all of them -inf
    pool.upload()
    got = paged(pool, np.full((len(lengths), 11, D), 1.0 + 2.0 ** -12))
    for s in range(len(lengths)):
        if s in (8, 9):
            assert np.all(got[s] == 0.0), s
        elif s in one:
            assert np.all(got[s] == 5.0), s
        else:
            assert np.isnan(got[s]).all(), s


def test_paged_value_whose_weight_is_nothing(hip):
    for type in ("f16", "bf16"):
        pool = base.Pool(np.random.default_rng(3), [300, 300], 1, 64, 16, type)
        for s in range(2):
            k, v = np.zeros((300, 1, 64)), np.full((300, 1, 64), 2.0)
            k[5, 0, 0] = 30.0
            v[100 + 150 * s, 0, 6] = np.inf
            place(pool, s, k, v)
        q = np.zeros((2, 3, 64))
        q[:, :, 0] = 30.0
        got = paged(pool, q)
        assert np.all(np.delete(got, 6, 2) == 2.0) and not np.isfinite(got[:, :, 6]).any()


# ---- the rules ahead of a sampler ------------------------------------------------------------------------------------------

def capped(oracle, x, cap):
    return np.array([oracle.softcap(float(v), cap) for v in np.asarray(x, np.float32).ravel()], np.float32).reshape(np.shape(x))


@pytest.mark.parametrize("rows,n", [(1, 5), (3, 2049), (2, 6000)])
@pytest.mark.parametrize("cap", [30.0, 0.7])
@pytest.mark.parametrize("in_place", [False, True])
def test_rules_cap_the_logits_first(hip, oracle, S, rows, n, cap, in_place):
    """To the bit: cap * tanh(logit / cap) as the top-k forms it, then the rules on that."""
    t = base._torch()
    rng = np.random.default_rng(n)
    logits = (rng.standard_normal((rows, n)) * 40).astype(np.float32)
    logits[0, :4] = np.inf, -np.inf, 0.0, np.nan
    history = rng.integers(0, n, (rows, 50)).astype(np.int32)
    told, r, f = np.full(rows, 50, np.int32), rng.uniform(0.8, 1.4, rows).astype(np.float32), rng.uniform(0, 1, rows).astype(np.float32)
    ids, bias, counts = rng.integers(0, n, (rows, 3)).astype(np.int32), rng.standard_normal((rows, 3)).astype(np.float32), np.full(rows, 3, np.int32)
    allowed = rng.integers(0, 2 ** 32, (rows, (n + 31) // 32), dtype=np.uint64).astype(np.uint32)
    x = dev(logits)
    out = x if in_place else t.zeros_like(x)
    d = [dev(a) for a in (history, told, r, f, ids, bias, counts, allowed.view(np.int32))]
    p = [a.data_ptr() for a in d]
    sync()
    H.logit_rules_device(rows, n, x.data_ptr(), out.data_ptr(), d_history=p[0], history_stride=50, d_history_lengths=p[1],
                         d_repetition=p[2], d_frequency=p[3], d_bias_ids=p[4], d_bias_values=p[5], d_bias_counts=p[6], bias_stride=3,
                         d_allowed=p[7], softcap=cap)
    sync()
    ref = S.logit_rules(capped(oracle, logits, cap), history, told, None, r, f, None, ids, bias, counts, allowed)
    got = out.cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    assert np.array_equal(got.view(np.uint32)[~np.isnan(ref)], ref.view(np.uint32)[~np.isnan(ref)])


def test_masked_tokens_have_no_weight_under_a_softcap(hip, oracle):
    """Rules with the cap, top-k without one, sampler: what the mask forbids is never a number again and is never
    sampled, and where nothing is masked the candidates are those of the top-k's own cap, to the bit."""
    t = base._torch()
    rng = np.random.default_rng(5)
    rows, n, k = 4, 5000, 40
    logits = (rng.standard_normal((rows, n)) * 20).astype(np.float32)
    allowed = np.full((rows, (n + 31) // 32), 0xFFFFFFFF, np.uint32)
    few = {1: [17], 2: [3, 4999], 3: list(range(100, 130))}  # row: the tokens that its mask leaves
    for row, tokens in few.items():
        allowed[row] = 0
        for i in tokens:
            allowed[row, i // 32] |= np.uint32(1 << (i % 32))
            logits[row, i] = -20.0 - i % 7
    x, m = dev(logits), dev(allowed.view(np.int32))
    ruled = t.zeros_like(x)
    ids, vals = (t.zeros((2, rows, k), dtype=d, device="cuda") for d in (t.int32, t.float32))
    state, tokens, kept = (t.zeros(c, dtype=t.int32, device="cuda") for c in (1, rows, rows))
    probs = t.full((rows, k), -1.0, dtype=t.float64, device="cuda")
    sync()
    H.logit_rules_device(rows, n, x.data_ptr(), ruled.data_ptr(), d_allowed=m.data_ptr(), softcap=30.0)
    L = H.lib()
    H.assertHipOk(L.hp_hip_topk_device(ruled.data_ptr(), rows, n, k, 0.0, ids[0].data_ptr(), vals[0].data_ptr(), None), "topk")
    H.assertHipOk(L.hp_hip_topk_device(x.data_ptr(), rows, n, k, 30.0, ids[1].data_ptr(), vals[1].data_ptr(), None), "topk")
    drawn = [set() for _ in range(rows)]
    for _ in range(200):
        H.sample_device(ids[0].data_ptr(), vals[0].data_ptr(), rows, k, k, {"doSample": True, "topK": k, "temperature": 1.5, "topP": 1.0},
                        state.data_ptr(), tokens.data_ptr(), probs.data_ptr(), kept.data_ptr(), 0)
        sync()
        for row, token in enumerate(tokens.tolist()):
            drawn[row].add(token)
    ids, vals, probs = ids.cpu().numpy(), vals.cpu().numpy(), probs.cpu().numpy()
    assert np.array_equal(ids[0, 0], ids[1, 0]) and np.array_equal(vals[0, 0].view(np.uint32), vals[1, 0].view(np.uint32))
    for row, left in few.items():
        there = np.isfinite(vals[0, row])
        assert sorted(ids[0, row][there]) == left and np.all(vals[0, row][~there] == -np.inf)
        assert np.array_equal(vals[0, row][there], np.sort(capped(oracle, logits[row, left], 30.0))[::-1])
        assert np.all(probs[row][~there] == 0.0) and abs(probs[row][there].sum() - 1.0) < 1e-12
        assert drawn[row] <= set(left)

"""The operators over several sequences against their 64-bit forms (oracle/serving.py).

Bounds.  A rounding is off by half a step, u = finfo(type).eps / 2 relative (and half of the smallest subnormal near
zero); U = 2^-24 is f32's.

* append: a row of D <= 256 elements: the sum of squares is a tree and a run of 8 f32 sums of f32 products (at most
  8 + 5 + 1 roundings on a term), halved by the root, then root, division and two products: below 12 U of a normed
  element.  A rotated one is two products with a rounded cosine or sine (2 U each) and a sum: x' is off by at most 12 U
  + 3 U of |x cos| + |y sin|, taken as 16 U (|x| + |y|).  E4M3 divides by its scale through a reciprocal, 2 U more.
  Then the output type's half step.
* paged attention: with A = sum p |v|: a score's terms are exact products of the key with the query's parts (which miss
  2^-21 of an element and 2^-28 of the row's largest) added in f32 over D elements: off by d = S (2^-20 + D U), S the
  largest sum |scale q k|; exp2 and its argument add 2^-20 to a weight.  Both sums have these weights: 2 (d + 2^-20).  A
  weight's two parts miss 2^-17 of it (bf16 pages) or 2^-21; n + 64 f32 sums add (n + 64) U A in the numerator and as
  much in the denominator.
* packed attention: the same with one part a weight: the numerator's and denominator's weights are the same rounded
  ones, so what a rounding moves is u |v - out| <= u (A + |out|); masked weights are exactly 0.  Scores are sums of
  exact products.
* logit rules: to the bit.
"""
import numpy as np
import pytest

from heliopause_amd import hip_kernels as H

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ELEM = {"f32": 0, "f16": 1, "bf16": 2, "e4m3": 3}


def _torch():
    import torch

    return torch


def dtype_of(name):
    t = _torch()
    return {"f32": t.float32, "f16": t.float16, "bf16": t.bfloat16, "e4m3": t.float8_e4m3fn}[name]


def half_step(name, ref):
    t = _torch()
    info = t.finfo(dtype_of(name))
    return np.maximum(np.abs(ref) * (info.eps / 2), info.tiny * info.eps / 2)


def dev(a):
    return _torch().from_numpy(np.ascontiguousarray(a)).cuda()


def values(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def sync():
    _torch().cuda.synchronize()


def check(got, ref, bound):
    got, ref, bound = np.broadcast_arrays(got, ref, bound)
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    wrong = ~(np.abs(got - ref) <= bound) & np.isfinite(ref)
    assert not wrong.any(), (np.argwhere(wrong)[:5], got[wrong][:5], ref[wrong][:5], bound[wrong][:5])
    inf = np.isinf(ref)
    assert np.array_equal(got[inf], ref[inf])


class Pool:
    """Pages [page][kv head][slot][D] of a type, filled with values or NaN, and a batch's tables."""

    def __init__(self, rng, lengths, kv, D, page, type, *, fill="values", spare=2, extra=1, joined=False, scales=(0.25, 0.5)):
        t = _torch()
        self.kv, self.D, self.page, self.type = kv, D, page, type
        need = [max(0, -(-n // page)) for n in lengths]
        self.width = max(1, max(need) + extra)
        self.count = sum(need) + spare
        order = rng.permutation(self.count)
        self.pages = np.full((len(lengths), self.width), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.pages[s, :n] = order[at:at + n]
            at += n
        self.scales = scales if type == "e4m3" else (1.0, 1.0)
        shape = (self.count, 2 if joined else 1, kv, page, D)

        def filled():
            x = rng.standard_normal(shape) * (40.0 if type == "e4m3" else 1.0)
            if fill == "nan":
                x[:] = np.nan
            return t.from_numpy(x.astype(np.float32)).cuda().to(dtype_of(type))

        if joined:  # keys and values of a page side by side
            both = filled()
            self.keys, self.values = both[:, 0], both[:, 1]
            self.both, self.stride = both, 2 * kv * page * D
        else:
            self.keys, self.values, self.stride = filled()[:, 0], filled()[:, 0], 0
        self.lengths = np.asarray(lengths, np.int32)
        self.upload()

    def upload(self):
        self.d_pages, self.d_lengths = dev(self.pages), dev(self.lengths)

    def cache(self):
        return H.paged_cache(self.keys.data_ptr(), self.values.data_ptr(), ELEM[self.type], page_count=self.count,
                             page_size=self.page, head_count_kv=self.kv, head_dim=self.D,
                             d_pages=self.d_pages.data_ptr(), d_lengths=self.d_lengths.data_ptr(),
                             sequence_count=len(self.lengths), pages_per_sequence=self.width,
                             key_scale=self.scales[0], value_scale=self.scales[1], page_stride=self.stride)


# ---- append -----------------------------------------------------------------------------------------------------------

def run_append(oracle_mod, seed, new, lengths, *, Hq=4, kv=2, D=64, page=16, type="f16", out="f16", norm=True, rope=None,
               factors=False, shared_v=False, no_q=False, strided=False, joined=False, packed=True, tail=2, kv_out=True,
               spoil=None, stream=0, base=10000.0):
    t = _torch()
    rng = np.random.default_rng(seed)
    rope = D if rope is None else rope
    offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.int32) if packed else None
    T = int(sum(new)) + tail if packed else len(lengths)
    pool = Pool(rng, [min(max(n, 0), 100000) for n in lengths], kv, D, page, type, joined=joined)
    pool.lengths = np.asarray(lengths, np.int32)
    if spoil:
        spoil(pool)
    pool.upload()
    before = values(pool.keys), values(pool.values)
    if strided:  # one projection's rows, with a gap behind
        rows = (rng.standard_normal((T, Hq + 2 * kv + 1, D)) * 2).astype(np.float32)
        d_rows = dev(rows)
        q, k, v = rows[:, :Hq], rows[:, Hq:Hq + kv], rows[:, Hq + kv:Hq + 2 * kv]
        ptr = [d_rows.data_ptr() + 4 * D * o for o in (0, Hq, Hq + kv)]
        strides = dict.fromkeys(("q_stride", "k_stride", "v_stride"), (Hq + 2 * kv + 1) * D)
    else:
        q, k, v = ((rng.standard_normal((T, n, D)) * 2).astype(np.float32) for n in (Hq, kv, kv))
        keep = [dev(x) for x in (q, k, v)]
        ptr, strides = [x.data_ptr() for x in keep], {}
    qn, kn = ((1 + 0.1 * rng.standard_normal(D)).astype(np.float32) for _ in range(2))
    f = np.exp(rng.uniform(0, 2, rope // 2)).astype(np.float32) if factors else None
    d_qn, d_kn, d_f = dev(qn), dev(kn), None if f is None else dev(f)
    outs = [t.full((T, n, D), 7.0, dtype=dtype_of(out), device="cuda") for n in (Hq, kv, kv)]
    d_off = None if offsets is None else dev(offsets)
    H.paged_append_device(pool.cache(), T, 0 if no_q else Hq, 0 if no_q else ptr[0], ptr[1], 0 if shared_v else ptr[2],
                          0 if no_q else outs[0].data_ptr(), ELEM[out], d_offsets=0 if d_off is None else d_off.data_ptr(),
                          d_q_norm=d_qn.data_ptr() if norm else 0, d_k_norm=d_kn.data_ptr() if norm else 0,
                          norm_values=norm, rope_dims=rope, rope_freq_base=base,
                          d_rope_freq_factors=0 if d_f is None else d_f.data_ptr(),
                          d_k_out=outs[1].data_ptr() if kv_out else 0, d_v_out=outs[2].data_ptr() if kv_out else 0,
                          stream=stream, **strides)
    sync()
    rows = oracle_mod.append(None if no_q else q, k, None if shared_v else v, pool.lengths, offsets, pool.pages, page,
                             pool.count, q_norm=qn if norm else None, k_norm=kn if norm else None, norm_values=norm,
                             rope_dims=rope, base=base, factors=f)

    def row_bound(x, rotated):
        b = np.abs(x)
        if rotated and rope:  # a rotation keeps the pair's length: |x| + |y| <= sqrt 2 of it
            h = rope // 2
            pair = np.sqrt(x[:, :h] ** 2 + x[:, h:rope] ** 2) * 1.4143
            b = np.concatenate([pair, pair, b[:, rope:]], 1)
        return 16 * U * b

    written = {}
    seen = set()
    for row, rq, rk, rv, page_id, slot in rows:
        seen.add(row)
        for o, ref, rot in ((outs[0], rq, True), (outs[1], rk, True), (outs[2], rv, False)):
            if ref is None or (o is not outs[0] and not kv_out):
                continue
            check(values(o[row]), ref, row_bound(ref, rot) * 1.01 + half_step(out, ref))
        if page_id >= 0:
            written[(page_id, slot)] = (rk, rv)
    for row in range(T):
        if row not in seen:  # left as it was
            assert all(bool((o[row] == 7.0).all()) for o in outs)
    now = values(pool.keys), values(pool.values)
    for which in range(2):
        expected, bound = before[which].copy(), np.zeros_like(before[which])
        for (p, slot), refs in written.items():
            ref = refs[which] / pool.scales[which]
            b = (row_bound(refs[which], which == 0) / pool.scales[which]) + 2 * U * np.abs(ref)
            if type == "e4m3":
                ref = np.clip(ref, -448, 448)
            expected[p, :, slot], bound[p, :, slot] = ref, b * 1.01 + half_step(type, ref)
        check(now[which], expected, bound)
    return written


@pytest.fixture(scope="module")
def S(oracle):
    from oracle import serving

    return serving


@pytest.mark.parametrize("D,Hq,kv", [(64, 4, 2), (128, 6, 1), (256, 8, 2), (128, 5, 5)])
@pytest.mark.parametrize("type,out", [("f16", "f16"), ("bf16", "f32"), ("e4m3", "bf16")])
def test_append_prompts(hip, S, D, Hq, kv, type, out):
    written = run_append(S, D + kv, [3, 0, 17, 1, 40], [3, 0, 37, 5000, 41], Hq=Hq, kv=kv, D=D, type=type, out=out)
    assert len(written) == 61


@pytest.mark.parametrize("D,rope,factors,norm", [(64, 0, False, True), (64, 8, True, False), (128, 24, False, True),
                                                 (128, 64, True, True), (256, 256, True, False), (256, 136, False, True)])
def test_append_rotations(hip, S, D, rope, factors, norm):
    run_append(S, rope, [9, 2], [1009, 123456], D=D, rope=rope, factors=factors, norm=norm, out="f32", page=64)


@pytest.mark.parametrize("kw", [{"shared_v": True}, {"no_q": True, "Hq": 4}, {"strided": True}, {"joined": True},
                                {"kv_out": False}, {"shared_v": True, "norm": False}, {"base": 1e6, "rope": 32}])
def test_append_forms(hip, S, kw):
    run_append(S, 5, [2, 7, 1], [2, 30, 70], type="bf16", out="bf16", **kw)


def test_append_one_token_each(hip, S):
    lengths = [1, 0, 17, 16, -4, 333, 48]
    written = run_append(S, 11, None, lengths, packed=False, D=256, Hq=8, kv=2, out="f32", kv_out=False)
    assert len(written) == 5


def test_append_many_tokens_and_sequences(hip, S):
    """A search over more than 64 sequences in two rounds, and empty ones among them."""
    rng = np.random.default_rng(3)
    new = rng.integers(0, 90, 150)
    new[10:20] = 0
    run_append(S, 12, list(new), list(new + rng.integers(0, 50, 150)), D=64, Hq=2, kv=1, rope=16, kv_out=False)


def test_append_absent_and_bad_pages(hip, S):
    """Entries that name no page drop the row, whatever they are; positions behind the table are left alone."""
    def spoil(pool):
        pool.pages[0, 0] = -1
        pool.pages[1, 0] = pool.count
        pool.pages[2, 1] = np.iinfo(np.int32).max
        pool.pages[3, 0] = np.iinfo(np.int32).min
        # its last three rows have no place; the three before them have one on the table's last entry, which names no page
        pool.lengths[4] = pool.width * pool.page + 3

    written = run_append(S, 13, [5, 20, 20, 3, 6], [5, 20, 20, 3, 6], spoil=spoil)
    assert len(written) == 4 + 16


@pytest.mark.parametrize("scale", [1.0, 0.01])
def test_append_e4m3_range(hip, scale):
    """Every 16-bit f16 value through an e4m3 cache: to nearest even, saturated, NaN kept; scale a power of two or not."""
    t = _torch()
    x = np.arange(65536, dtype=np.uint16).view(np.float16).astype(np.float32).reshape(-1, 1, 64)
    n = x.shape[0]
    keys, vals = (t.zeros((n // 16, 1, 16, 64), dtype=t.float8_e4m3fn, device="cuda") for _ in range(2))
    pages, lengths, offsets = dev(np.arange(n // 16, dtype=np.int32)), dev(np.array([n], np.int32)), dev(np.array([0, n], np.int32))
    c = H.paged_cache(keys.data_ptr(), vals.data_ptr(), 3, page_count=n // 16, page_size=16, head_count_kv=1, head_dim=64,
                      d_pages=pages.data_ptr(), d_lengths=lengths.data_ptr(), sequence_count=1, pages_per_sequence=n // 16,
                      key_scale=scale, value_scale=scale)
    d = dev(x)
    H.paged_append_device(c, n, 0, 0, d.data_ptr(), 0, 0, 0, d_offsets=offsets.data_ptr())
    sync()
    inv = (np.float32(1.0) / np.float32(scale)).astype(np.float32)
    with np.errstate(all="ignore"):
        s = np.clip((x * inv).astype(np.float32), np.float32(-448), np.float32(448))
    ref = t.from_numpy(s).to(t.float8_e4m3fn).float().numpy().reshape(-1)
    for pool in (keys, vals):
        got = pool.float().cpu().numpy().reshape(-1)
        assert np.array_equal(np.isnan(got), np.isnan(ref))
        assert np.array_equal(got[~np.isnan(ref)], ref[~np.isnan(ref)])


# ---- paged attention -----------------------------------------------------------------------------------------------------

def paged_bound(name, type, ref, mass, size, count, D):
    d = size * (2.0 ** -20 + D * U)
    weight = 2 * (d + 2.0 ** -20) + (2.0 ** -17 if type == "bf16" else 2.0 ** -21) + 2 * (count + 64) * U
    return 1.01 * mass * weight[..., None] + half_step(name, ref) + 1e-30


def run_paged(S, pool, Hq, q_type="f32", out="f32", window=0, scale=None, rng=None, q_times=2.0, strides=False, stream=0):
    t = _torch()
    n, D = len(pool.lengths), pool.D
    scale = D ** -0.5 if scale is None else scale
    gap = 2 if strides else 0
    full = t.from_numpy((rng.standard_normal((n, Hq + gap, D)) * q_times).astype(np.float32)).cuda().to(dtype_of(q_type))
    got = t.full((n, Hq + 2 * gap, D), 7.0, dtype=dtype_of(out), device="cuda")
    H.paged_attention_device(pool.cache(), Hq, full.data_ptr(), ELEM[q_type], got.data_ptr(), ELEM[out], scale=scale,
                             sliding_window=window, q_stride=(Hq + gap) * D if strides else 0,
                             output_stride=(Hq + 2 * gap) * D if strides else 0, stream=stream)
    sync()
    q = values(full[:, :Hq])
    ref, mass, size, count = S.paged_attention(q, values(pool.keys) * pool.scales[0], values(pool.values) * pool.scales[1],
                                               pool.lengths, pool.pages, pool.page, pool.count, window, scale)
    assert bool((got[:, Hq:] == 7.0).all())
    check(values(got[:, :Hq]), ref, paged_bound(out, pool.type, ref, mass, size, count, D))
    return got[:, :Hq]


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 127, 128, 129, 160, 161, 255, 257, 400, 3, 1000]


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("type,q_type,out", [("f16", "f32", "f32"), ("bf16", "f32", "f32"), ("e4m3", "f32", "f32"),
                                             ("bf16", "bf16", "bf16"), ("f16", "f16", "f16"), ("e4m3", "bf16", "f16"),
                                             ("bf16", "f16", "f32")])
def test_paged_types(hip, S, D, type, q_type, out):
    rng = np.random.default_rng(D)
    run_paged(S, Pool(rng, LENGTHS, 2, D, 16, type), 8, q_type, out, rng=rng)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("type,q_type", [("f16", "f32"), ("bf16", "f32"), ("bf16", "bf16"), ("e4m3", "f16")])
def test_paged_wide_tables(hip, S, D, type, q_type):
    """Tables with room for more than the caches hold: the loads go past them."""
    rng = np.random.default_rng(D)
    run_paged(S, Pool(rng, [1, 0, 129, 700, 64], 2, D, 16, type, extra=(33 << 20) // (2 * 2 * D * 5 * 16)), 8, q_type, rng=rng)


def test_paged_offsets_past_32_bits(hip, S):
    """Pages two gigabytes apart."""
    t = _torch()
    rng = np.random.default_rng(14)
    pool = Pool(rng, [40, 17], 1, 64, 16, "f16", spare=0, extra=0)
    stride = 1 << 30  # elements
    far = t.empty(pool.count * stride, dtype=t.float16, device="cuda")
    keys, values_ = far.view(pool.count, stride)[:, :1024], far.view(pool.count, stride)[:, 1 << 29:(1 << 29) + 1024]
    keys.copy_(pool.keys.reshape(pool.count, -1))
    values_.copy_(pool.values.reshape(pool.count, -1))
    pool.keys, pool.values, pool.stride = keys.view(pool.count, 1, 16, 64), values_.view(pool.count, 1, 16, 64), stride
    run_paged(S, pool, 2, rng=rng)
    # and a row appended there
    row = dev(np.ones((2, 1, 64), np.float32))
    H.paged_append_device(pool.cache(), 2, 0, 0, row.data_ptr(), 0, 0, 0)
    sync()
    for s, n in enumerate((40, 17)):
        assert bool((pool.keys[pool.pages[s, (n - 1) // 16], 0, (n - 1) % 16] == 1).all())
        assert bool((pool.values[pool.pages[s, (n - 1) // 16], 0, (n - 1) % 16] == 1).all())


@pytest.mark.parametrize("Hq,kv", [(1, 1), (2, 1), (3, 1), (7, 1), (8, 1), (9, 1), (16, 1), (21, 1), (5, 5), (14, 2), (40, 8)])
def test_paged_groups(hip, S, Hq, kv):
    rng = np.random.default_rng(Hq)
    run_paged(S, Pool(rng, [1, 130, 0, 700], kv, 64, 32, "f16"), Hq, rng=rng)


@pytest.mark.parametrize("window", [1, 5, 16, 17, 100, 128, 129, 1000, 2 ** 31 - 1])
@pytest.mark.parametrize("page", [16, 128])
def test_paged_windows(hip, S, window, page):
    """Windows that begin inside a tile and a page, with the pages before them given back and their slots NaN."""
    rng = np.random.default_rng(window)
    pool = Pool(rng, [1, 40, 129, 300, 777], 1, 128, page, "bf16")
    for s, n in enumerate(pool.lengths):
        pool.pages[s, :max(0, int(n) - window) // page] = -1
    pool.upload()
    run_paged(S, pool, 4, window=window, rng=rng)


@pytest.mark.parametrize("type", ["f16", "bf16", "e4m3"])
def test_paged_masked_places_hold_nan_and_inf(hip, S, type):
    """Slots behind the length, before the window, and all of page 0 (which absent pages read in its place)."""
    t = _torch()
    rng = np.random.default_rng(9)
    lengths = [1, 17, 130, 250, 64]
    pool = Pool(rng, lengths, 2, 64, 16, type, spare=3)
    free = next(p for p in range(pool.count) if p not in pool.pages)
    pool.pages[pool.pages == 0] = free  # page 0 is nobody's
    window, odd = 100, float("nan") if type == "e4m3" else float("inf")
    for p in (pool.keys, pool.values):
        p[0] = float("nan")
        for s, n in enumerate(lengths):
            for i in range(pool.width * 16):
                page = pool.pages[s, i // 16]
                if page >= 0 and (i >= n or i < n - window):
                    p[page, :, i % 16] = odd if i % 2 else float("nan")
    pool.pages[3, 10] = -1          # a hole in the middle
    pool.pages[2, 7] = pool.count   # and one past the pool
    pool.pages[4, :] = -7           # a sequence without a page
    pool.upload()
    got = run_paged(S, pool, 6, window=window, rng=rng)
    assert bool((got[4] == 0).all())


def test_paged_values_that_are_seen_propagate(hip):
    """An infinite value that counts is never a number again where it reaches (two parts of a weight times an infinity:
    that or a NaN), a NaN key makes its rows NaN; the other elements, heads and rows stay."""
    t = _torch()
    rng = np.random.default_rng(10)
    pool = Pool(rng, [200, 200], 2, 64, 16, "f16")
    pool.values[pool.pages[0, 3], 0, 5, 7] = float("inf")
    pool.keys[pool.pages[1, 2], 1, 1, 0] = float("nan")
    q = t.ones((2, 4, 64), device="cuda")
    out = t.zeros_like(q)
    H.paged_attention_device(pool.cache(), 4, q.data_ptr(), 0, out.data_ptr(), 0, scale=0.125)
    sync()
    o = out.cpu().numpy()
    assert not np.isfinite(o[0, :2, 7]).any() and np.isfinite(np.delete(o[0], 7, 1)).all() and np.isfinite(o[0, 2:]).all()
    assert np.isnan(o[1, 2:]).all() and np.isfinite(o[1, :2]).all()


@pytest.mark.parametrize("type", ["f16", "bf16", "e4m3"])
@pytest.mark.parametrize("times", [1e-30, 1e-4, 300.0, 1e20])
def test_paged_query_sizes(hip, S, type, times):
    """Queries far from 1, with the scale that brings the scores back (their parts must not leave the operand's range)."""
    rng = np.random.default_rng(4)
    run_paged(S, Pool(rng, [3, 200], 1, 64, 16, type), 3, rng=rng, q_times=times, scale=float(np.float32(0.125 / times)))


def test_paged_long_and_many(hip, S):
    """One context over every workgroup, among short ones; then more sequences than threads scan at once."""
    rng = np.random.default_rng(6)
    run_paged(S, Pool(rng, [70000, 1, 513], 1, 128, 64, "f16"), 2, rng=rng)
    run_paged(S, Pool(rng, list(rng.integers(0, 300, 600)), 1, 64, 16, "bf16"), 2, "bf16", "bf16", rng=rng)


def test_paged_strides_and_joined_pages(hip, S):
    rng = np.random.default_rng(7)
    run_paged(S, Pool(rng, [100, 33, 0], 2, 128, 32, "f16", joined=True), 4, "f16", "f32", rng=rng, strides=True)


def test_paged_lengths_past_the_table(hip, S):
    rng = np.random.default_rng(8)
    pool = Pool(rng, [64, 32], 1, 64, 16, "f16", extra=0)
    pool.lengths = np.array([2 ** 31 - 1, -(2 ** 31)], np.int32)
    pool.upload()
    run_paged(S, pool, 1, rng=rng)


def test_paged_agrees_with_the_ring(hip):
    """Next to the framework's ring attention on the same keys: page 4096 slots long, one sequence."""
    t = _torch()
    rng = np.random.default_rng(12)
    kc, vc = (t.from_numpy(rng.standard_normal((1, 2, 4096, 256)).astype(np.float16)).cuda() for _ in range(2))
    q = t.from_numpy(rng.standard_normal((8, 256)).astype(np.float16).astype(np.float32) * 0.25).cuda()
    position, lengths, pages = dev(np.array([2999], np.int32)), dev(np.array([3000], np.int32)), dev(np.zeros((1, 1), np.int32))
    ring, paged = t.zeros_like(q), t.zeros_like(q)
    H.gqa_attention_device(H.attention_config(8, 2, 4096), q.data_ptr(), kc.data_ptr(), vc.data_ptr(), position.data_ptr(), ring.data_ptr())
    c = H.paged_cache(kc.data_ptr(), vc.data_ptr(), 1, page_count=1, page_size=4096, head_count_kv=2, head_dim=256,
                      d_pages=pages.data_ptr(), d_lengths=lengths.data_ptr(), sequence_count=1, pages_per_sequence=1)
    H.paged_attention_device(c, 8, q.data_ptr(), 0, paged.data_ptr(), 0, scale=1.0)
    sync()
    a, b = values(ring), values(paged)
    # the ring rounds its output to f16 (2^-11) and sums in f32 in another order (scores to +-16: 16 * 300 U)
    assert np.max(np.abs(a - b)) <= np.max(np.abs(b)) * (2.0 ** -11 + 16 * 300 * U)


# ---- packed attention ------------------------------------------------------------------------------------------------------

def run_packed(S, lengths, Hq, kv, D, type="f16", out=None, window=0, scale=None, seed=0, tail=3, joined=False, lead=0,
               spoil=None, stream=0, sample=None):
    t = _torch()
    out = out or type
    rng = np.random.default_rng(seed)
    scale = D ** -0.5 if scale is None else scale
    offsets = (lead + np.concatenate([[0], np.cumsum(lengths)])).astype(np.int32)
    T = int(offsets[-1]) + tail
    rows = t.from_numpy((rng.standard_normal((T, Hq + 2 * kv, D)) * 1.5).astype(np.float32)).cuda().to(dtype_of(type))
    q, k, v = rows.split([Hq, kv, kv], 1)
    if not joined:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    if spoil:
        spoil(q, k, v)
    got = t.full((T, Hq, D), 7.0, dtype=dtype_of(out), device="cuda")
    d_off = dev(offsets)
    H.packed_attention_device(len(lengths), d_off.data_ptr(), T, Hq, kv, D, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                              ELEM[type], got.data_ptr(), ELEM[out], scale=scale, sliding_window=window,
                              q_stride=q.stride(0), k_stride=k.stride(0), v_stride=v.stride(0), stream=stream)
    sync()
    rows = None if sample is None else set(rng.choice(T, sample, replace=False)) | set(int(e) - 1 for e in offsets[1:])
    ref = S.packed_attention(values(q), values(k), values(v), offsets, window, scale, rows)
    o, seen = values(got), np.abs(values(v)[:offsets[-1]])
    largest = seen[np.isfinite(seen)].max(initial=0.0)
    u = _torch().finfo(dtype_of(type)).eps / 2
    for row in range(T):
        if row not in ref:
            if rows is None or not lead <= row < offsets[-1]:
                assert np.all(o[row] == 7.0), row
            continue
        r, mass, size, n = ref[row]
        with np.errstate(all="ignore"):
            d = size * D * U
            weight = 2 * (d + 2.0 ** -20) + 2 * (n + 64) * U
            bound = 1.01 * (mass * weight[:, None] + u * (mass + np.abs(r))) + half_step(out, r) + 1e-30
            if type == "f16":  # weights below 2^-14 have f16's subnormal step, 2^-25 at most, of a sum of at least one
                bound = bound + 2.0 ** -25 * n * largest
        check(o[row], r, np.where(np.isfinite(r), bound, 0.0))
    return got


PACKED = [1, 2, 31, 32, 33, 0, 63, 64, 65, 127, 128, 129, 200]


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("type", ["f16", "bf16"])
def test_packed_lengths(hip, S, D, type):
    run_packed(S, PACKED, 2, 1, D, type, seed=D)


@pytest.mark.parametrize("Hq,kv", [(1, 1), (3, 1), (8, 2), (5, 5), (14, 2), (16, 16)])
def test_packed_heads(hip, S, Hq, kv):
    run_packed(S, [70, 5], Hq, kv, 64, "bf16", out="f32", seed=Hq)


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 64, 65, 100, 128, 2 ** 31 - 1])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_packed_windows(hip, S, window, D):
    run_packed(S, [300, 7, 129], 1, 1, D, "f16", window=window, seed=window % 1000)


@pytest.mark.parametrize("Hq,kv,D,lengths", [(16, 8, 64, [2100, 300, 2000]), (16, 2, 128, [1000, 77, 600]), (10, 5, 256, [3500, 3000, 200])])
@pytest.mark.parametrize("window", [0, 333])
def test_packed_blocks_that_fill_the_card(hip, S, Hq, kv, D, lengths, window):
    """Batches large enough for whole blocks (the small ones above split their keys over two groups of waves)."""
    def spoil(q, k, v):
        v[lengths[0] - 3, 0, 5], v[lengths[0] - 2, 0, 6] = float("inf"), float("nan")

    run_packed(S, lengths, Hq, kv, D, "bf16", window=window, sample=60, spoil=spoil, seed=D)


def test_packed_forms(hip, S):
    run_packed(S, [140, 30], 4, 2, 128, "bf16", joined=True)
    run_packed(S, [33, 2], 4, 2, 128, "f16", out="f32", lead=5)  # rows ahead of the first sequence stay too
    run_packed(S, [0, 0, 0], 2, 1, 64)
    run_packed(S, [1], 2, 1, 64, tail=0)
    run_packed(S, [700], 2, 1, 128, "bf16", scale=1.0)            # scores to +-60: a few keys hold the weight


def test_packed_many_sequences(hip, S):
    rng = np.random.default_rng(1)
    lengths = list(rng.integers(0, 12, 300))
    lengths[100] = 150
    run_packed(S, lengths, 2, 2, 64, "bf16", seed=2)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("type", ["f16", "bf16"])
def test_packed_later_rows_do_not_reach_back(hip, S, type, D):
    """Infinities and NaNs in a sequence's later keys and values, behind it and before a window: rows that do not see
    them are as if they were not there; rows that do have what the formula gives."""
    def spoil(q, k, v):
        k[50, 0] = float("nan")       # every later row of the sequence is NaN
        v[100, 0, 3] = float("inf")   # column 3 from row 100 on
        v[101, 0, 4] = float("-inf")
        v[130, 0, 5] = float("nan")
        v[131, 0, 3] = float("-inf")  # inf - inf
        k[200:], v[200:] = float("nan"), float("nan")  # behind the last sequence

    def spoil_window(q, k, v):
        v[10, 0, 1], k[11, 0] = float("nan"), float("inf")

    run_packed(S, [60, 140], 2, 1, D, type, spoil=spoil)
    run_packed(S, [200], 2, 1, D, type, window=40, spoil=spoil_window)


def test_packed_strides_past_32_bits(hip, S):
    """Rows sixteen megabytes apart: the last ones lie past four gigabytes."""
    t = _torch()
    T, stride = 300, (1 << 23)
    far = t.empty(T * stride, dtype=t.float16, device="cuda").view(T, stride)
    near = t.randn(T, 3, 64, device="cuda").half()
    far[:, :192] = near.view(T, -1)
    offsets = dev(np.array([0, 300], np.int32))
    outs = [t.zeros(T, 1, 64, dtype=t.float16, device="cuda") for _ in range(2)]
    for x, o, step in ((far, outs[0], stride), (near, outs[1], 192)):
        p = x.data_ptr()
        H.packed_attention_device(1, offsets.data_ptr(), T, 1, 1, 64, p, p + 128, p + 256, 1, o.data_ptr(), 1, scale=0.125,
                                  q_stride=step, k_stride=step, v_stride=step)
    sync()
    assert t.equal(*outs) and bool(outs[0].any())


def test_packed_bad_offsets_stay_inside(hip):
    """Offsets that fall, or point outside the batch, name no row outside it (the result of their sequences is open)."""
    t = _torch()
    q = t.ones((70, 2, 64), dtype=t.float16, device="cuda")
    out = t.zeros_like(q)
    for bad in ([0, 1000, 2000], [-50, 20, 10], [60, 30, 70], [2 ** 31 - 1, 0, 5], [0, -5, -9]):
        d = dev(np.array(bad, np.int32))
        H.packed_attention_device(2, d.data_ptr(), 70, 2, 2, 64, q.data_ptr(), q.data_ptr(), q.data_ptr(), 1, out.data_ptr(), 1)
    sync()
    assert bool(((out == 0) | (out == 1)).all())


# ---- logit rules ---------------------------------------------------------------------------------------------------------

def run_rules(S, rows, n, *, history=0, biases=0, mask=None, stride=0, in_place=False, seed=0, prompts=True, params=True,
              edit=None, stream=0):
    t = _torch()
    rng = np.random.default_rng(seed)
    wide = stride or n
    logits = (rng.standard_normal((rows, wide)) * 4).astype(np.float32)
    arg, kw = {}, {}
    if history:
        arg["history"] = (n * rng.random((rows, history)) ** 3).astype(np.int32)
        arg["history"][rng.random((rows, history)) < 0.05] = -1
        arg["history"][:, -1] = n
        arg["lengths"] = rng.integers(0, history + 3, rows).astype(np.int32)
        arg["lengths"][0] = history
        if prompts:
            arg["prompts"] = rng.integers(-2, history + 2, rows).astype(np.int32)
        if params:
            arg["repetition"], arg["frequency"], arg["presence"] = (rng.uniform(a, b, rows).astype(np.float32) for a, b in ((0.7, 1.5), (-0.5, 0.7), (-1, 1)))
    if biases:
        arg["bias_ids"] = rng.integers(-2, n + 2, (rows, biases)).astype(np.int32)
        arg["bias_ids"][:, biases // 2] = arg["bias_ids"][:, 0]  # the same token twice: the last counts
        arg["bias_values"] = (rng.standard_normal((rows, biases)) * 3).astype(np.float32)
        arg["bias_counts"] = rng.integers(0, biases + 3, rows).astype(np.int32)
        arg["bias_counts"][0] = biases
    if mask is not None:
        arg["allowed"] = np.packbits(rng.random((rows, (n + 31) // 32 * 32)) < mask, axis=1, bitorder="little").view(np.uint32)
        arg["allowed"][-1] = 0  # a row without any
    if edit:
        edit(logits, arg)
    d = {k: dev(v.view(np.int32) if v.dtype == np.uint32 else v) for k, v in arg.items()}
    names = {"history": "d_history", "lengths": "d_history_lengths", "prompts": "d_prompt_lengths", "repetition": "d_repetition",
             "frequency": "d_frequency", "presence": "d_presence", "bias_ids": "d_bias_ids", "bias_values": "d_bias_values",
             "bias_counts": "d_bias_counts", "allowed": "d_allowed"}
    x = dev(logits)
    out = x if in_place else t.full((rows, wide), 7.0, device="cuda")
    H.logit_rules_device(rows, n, x.data_ptr(), out.data_ptr(), history_stride=history, bias_stride=biases,
                         logits_stride=stride, output_stride=stride, stream=stream,
                         **{names[k]: v.data_ptr() for k, v in d.items()})
    sync()
    got = out.cpu().numpy()
    ref = S.logit_rules(logits[:, :n], **arg)
    assert np.array_equal(got[:, :n].view(np.uint32)[~np.isnan(ref)], ref.view(np.uint32)[~np.isnan(ref)])
    assert np.isnan(got[:, :n][np.isnan(ref)]).all()
    assert np.array_equal(got[:, n:], logits[:, n:] if in_place else np.full((rows, wide - n), 7.0, np.float32))


@pytest.mark.parametrize("n", [1, 3, 4, 31, 33, 255, 1023, 1024, 1025, 4097, 32000, 50257])
def test_rules_widths(hip, S, n):
    run_rules(S, 3, n, history=40, biases=5, mask=0.5, seed=n)


@pytest.mark.parametrize("rows,n", [(1, 262144), (20, 100003), (300, 20011), (70, 65536)])
def test_rules_slices(hip, S, rows, n):
    """Many slices, at row widths that start rows anywhere."""
    run_rules(S, rows, n, history=100, biases=7, mask=0.9, seed=rows)


@pytest.mark.parametrize("kw", [{}, {"history": 1}, {"history": 300, "prompts": False}, {"history": 50, "params": False},
                                {"biases": 1}, {"biases": 70}, {"mask": 0.0}, {"mask": 1.0}, {"history": 9, "mask": 0.3},
                                {"stride": 1311}, {"stride": 1312, "in_place": True, "history": 20, "biases": 3},
                                {"in_place": True, "mask": 0.5, "history": 5000}])
def test_rules_alone_and_together(hip, S, kw):
    run_rules(S, 4, 1303, **kw)


def test_rules_rows_past_32_bits(hip):
    t = _torch()
    stride, n = 1 << 30, 5000
    x = t.empty(3 * stride, device="cuda").view(3, stride)
    x[:, :n] = 2.0
    history, one = dev(np.array([[7], [8], [9]], np.int32)), dev(np.ones(3, np.int32))
    r = dev(np.full(3, 4.0, np.float32))
    H.logit_rules_device(3, n, x.data_ptr(), x.data_ptr(), d_history=history.data_ptr(), history_stride=1,
                         d_history_lengths=one.data_ptr(), d_repetition=r.data_ptr(), logits_stride=stride, output_stride=stride)
    sync()
    ref = t.full((3, n), 2.0, device="cuda")
    ref[[0, 1, 2], [7, 8, 9]] = 0.5
    assert t.equal(x[:, :n], ref)


def test_rules_odd_values(hip, S):
    """NaN, infinities and zeros in the logits, a token that fills the history, parameters that change nothing."""
    def edit(logits, arg):
        logits[0, :8] = [np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-40, 3e38, -3e38]
        arg["history"][0, :8] = range(8)
        arg["history"][1] = 5
        arg["repetition"][2], arg["frequency"][2], arg["presence"][2] = 1.0, 0.0, 0.0

    run_rules(S, 3, 500, history=3000, mask=0.7, edit=edit)


@pytest.mark.parametrize("scale", [2.0 ** 120, 2.0 ** -149])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_largest_and_smallest_scales(hip, S, D, scale):
    """Queries of zeros: every key weighs the same at the largest scale; at the smallest they do whatever the query."""
    rng = np.random.default_rng(7)
    times = 0.0 if scale > 1 else 1.0
    for type, scales in (("f16", (1.0, 1.0)), ("e4m3", (2.0 ** -20, 0.5))):
        run_paged(S, Pool(rng, [1, 40, 0, 333], 2, D, 16, type, scales=scales), 4, rng=rng, q_times=times, window=100,
                  scale=scale)

    def zeros(q, k, v):
        q *= times
    run_packed(S, [1, 100, 65], 2, 1, D, "bf16", scale=scale, spoil=zeros, seed=D, window=40)


@pytest.mark.parametrize("Hq,kv,D", [(4, 1, 64), (12, 1, 128), (8, 2, 256), (6, 1, 64), (2, 2, 256)])
@pytest.mark.parametrize("out", ["f32", "f16"])
def test_packed_heads_that_share_a_workgroup(hip, S, Hq, kv, D, out):
    """Four, two and one heads a workgroup over its whole range of rows, in batches that fill the card (one walk over
    the keys) and in small ones (two), with rows that end inside a block and a window that begins inside a tile."""
    heads = -(-1400 // (Hq * 25)) * Hq  # blocks of 128 rows over 3200 rows past every limit of the split
    run_packed(S, [1, 31, 32, 33, 2000, 0, 97, 1006], heads, heads // Hq * kv, D, "f16", out, window=75, seed=Hq, sample=60)
    run_packed(S, [1, 31, 32, 33, 97], Hq, kv, D, "f16", out, window=40, seed=Hq, joined=True)

"""The operators of long contexts against their plain forms (oracle/long_context.py).

Bounds.  U = 2^-24 is f32's half step.  Page plans, key bounds and selections are equal.

* append: rows are off as the paged append's are, below 16 U of a normed and rotated pair, with the angle's share: a turn
  reduced to f32 is 2^-25 off at most, 2 pi 2^-25 < 4 U of a pair, sine and cosine 2 U each as there: 20 U.  A scale is the
  largest element's product with 1 / 127: its error and two U (i8), or the same power of two.  A stored element is the rounding
  of x (1 / scale): half a step, with the row's error and 2 U.  What a block held moves to f32(stored f32(old / new)), to
  the bit.
* attention: as the paged attention's (tests/test_gpu_serving.py), with U for the product with the key scale and 2 U for
  that of a weight with its scale's part.  A weight's last part is a multiple of f16's smallest step: it misses 2^-25 of
  2^10 times the largest weight with its scale, 2^-35 of that for every key and stored element (pages of f16 and of 8
  bits; bf16 has f32's range).  A key of weight 2^-36 whose value stands alone among zeros counts as 0.
"""
import numpy as np
import pytest

from heliopause_amd import hip_kernels as H

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ELEM = {"f32": 0, "f16": 1, "bf16": 2, "e4m3": 3, "i8": 4}
MOST = {"i8": 127.0, "e4m3": 448.0}


def _torch():
    import torch

    return torch


def dtype_of(name):
    t = _torch()
    return {"f32": t.float32, "f16": t.float16, "bf16": t.bfloat16, "e4m3": t.float8_e4m3fn, "i8": t.int8}[name]


def half_step(name, ref):
    info = _torch().finfo(dtype_of(name))
    return np.maximum(np.abs(ref) * (info.eps / 2), info.tiny * info.eps / 2)


def dev(a):
    return _torch().from_numpy(np.ascontiguousarray(a)).cuda()


def values(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def ptr(t):
    return 0 if t is None else t.data_ptr()


def sync():
    _torch().cuda.synchronize()


def check(got, ref, bound):
    got, ref, bound = np.broadcast_arrays(got, ref, bound)
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    wrong = ~(np.abs(got - ref) <= bound) & np.isfinite(ref)
    assert not wrong.any(), (np.argwhere(wrong)[:5], got[wrong][:5], ref[wrong][:5], bound[wrong][:5])
    inf = np.isinf(ref)
    assert np.array_equal(got[inf], ref[inf])


@pytest.fixture(scope="module")
def L(oracle):
    from oracle import long_context

    return long_context


class Pool:
    """Pages of a type, their blocks' scales and bounds, and a batch's tables.  Slots and blocks that no sequence has
    filled hold what must not count: NaN where the type has one, and NaN scales."""

    def __init__(self, rng, lengths, kv, D, page, block, type, *, scaled=None, extra=1, spare=2, joined=False, spread=0.3):
        t = _torch()
        self.kv, self.D, self.page, self.block, self.type, self.per = kv, D, page, block, type, page // block
        self.lengths = np.asarray(lengths, np.int32)
        need = [max(0, -(-n // page)) for n in lengths]
        self.width = max(1, max(need) + extra)
        self.count = sum(need) + spare
        order = rng.permutation(self.count)
        self.pages = np.full((len(lengths), self.width), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            self.pages[s, :n] = order[at:at + n]
            at += n
        self.scaled = (type in MOST) if scaled is None else scaled
        shape = (2, self.count, kv, page, D)
        x = rng.standard_normal(shape).astype(np.float32)
        live = np.zeros((self.count, page), bool)
        for s, n in enumerate(lengths):
            for p in range(max(0, n)):
                live[self.pages[s, p // page], p % page] = True
        self.live = live
        x = np.clip(np.rint(x * 40), -127, 127) if type == "i8" else np.clip(x * 120, -448, 448) if type == "e4m3" else x
        if type != "i8":
            x[:, ~live[:, None, :, None].repeat(kv, 1).repeat(D, 3)] = np.nan
        both = t.from_numpy(x).cuda().to(dtype_of(type))
        if joined:  # keys and values of a page side by side
            both = both.transpose(0, 1).contiguous()
            self.keys, self.values, self.stride = both[:, 0], both[:, 1], 2 * kv * page * D
        else:
            self.keys, self.values, self.stride = both[0], both[1], 0
        self.both = both
        scales = np.exp(spread * rng.standard_normal((2, self.count, kv, self.per))).astype(np.float32) / MOST.get(type, 1) * 3
        scales[:, ~live.reshape(self.count, self.per, block).any(2)[:, None].repeat(kv, 1)] = np.nan
        self.scales = [dev(s) if self.scaled else None for s in scales]
        self.bounds = t.full((self.count, kv, self.per, 2, D), float("nan"), dtype=t.bfloat16, device="cuda")
        self.whole = (0.25, 0.5) if type == "e4m3" and not self.scaled else (1.0, 1.0)
        self.upload()

    def upload(self):
        self.d_pages, self.d_lengths = dev(self.pages), dev(self.lengths)

    def cache(self):
        return H.paged_cache(self.keys.data_ptr(), self.values.data_ptr(), ELEM[self.type], page_count=self.count,
                             page_size=self.page, head_count_kv=self.kv, head_dim=self.D, d_pages=self.d_pages.data_ptr(),
                             d_lengths=self.d_lengths.data_ptr(), sequence_count=len(self.lengths),
                             pages_per_sequence=self.width, key_scale=self.whole[0], value_scale=self.whole[1],
                             page_stride=self.stride)

    def blocks(self):
        return H.cache_blocks(self.block, d_key_scales=ptr(self.scales[0]), d_value_scales=ptr(self.scales[1]),
                              d_key_bounds=self.bounds.data_ptr())

    def real(self, which):
        """What the keys (0) or values (1) stand for, f32 products."""
        x = (self.keys, self.values)[which].float().cpu().numpy()
        if self.scaled:
            return x * self.scales[which].cpu().numpy().repeat(self.block, 2)[..., None]
        return x * np.float32(self.whole[which])


# ---- page plans -----------------------------------------------------------------------------------------------------------

def run_plan(L, pages, lengths, new, keep, free, free_count, page_size, page_count, rows, *, in_place=False, stream=0, maps=True,
             sums=True):
    t = _torch()
    want = L.plan(pages, lengths, new, keep, free, free_count, page_size, page_count, rows)
    i32 = lambda a: None if a is None else dev(np.asarray(a, np.int32))  # noqa: E731
    d_pages, d_lengths, d_new, d_keep, d_free, d_count = (i32(a) for a in (pages, lengths, new, keep, free, [free_count]))
    S, W = pages.shape
    out = d_lengths if in_place else t.full((S,), -7, dtype=t.int32, device="cuda")
    offsets, missing = (t.full((n,), -7, dtype=t.int32, device="cuda") for n in (S + 1, S))
    seq, pos = (t.full((rows + 1,), -7, dtype=t.int32, device="cuda") for _ in range(2))
    slots = t.full((rows + 1,), -7, dtype=t.int64, device="cuda")
    H.page_plan_device(S, W, page_size, page_count, ptr(d_pages), ptr(d_lengths), ptr(out), ptr(d_free), ptr(d_count),
                       d_new_tokens=ptr(d_new), d_keep_from=ptr(d_keep), d_offsets=ptr(offsets) if sums else 0,
                       d_missing=ptr(missing) if sums else 0, token_count=rows, d_sequences=ptr(seq) if maps else 0,
                       d_positions=ptr(pos) if maps else 0, d_slots=ptr(slots), stream=stream)
    sync()
    assert np.array_equal(d_pages.cpu().numpy(), want["pages"])
    assert np.array_equal(out.cpu().numpy(), want["lengths"])
    assert int(d_count) == want["free_count"]
    assert np.array_equal(d_free.cpu().numpy(), want["free"])
    if sums:
        assert np.array_equal(offsets.cpu().numpy(), want["offsets"])
        assert np.array_equal(missing.cpu().numpy(), want["missing"])
    for got, name in ((seq, "sequences"), (pos, "positions"), (slots, "slots")) if maps else ((slots, "slots"),):
        assert np.array_equal(got[:rows].cpu().numpy(), want[name]), name
        assert int(got[rows]) == -7
    return want


def table(rng, lengths, page_size, width, spare):
    need = [min(width, max(0, -(-int(n) // page_size))) for n in lengths]
    count = sum(need) + spare
    order = rng.permutation(count).astype(np.int32)
    pages = np.full((len(lengths), width), -1, np.int32)
    at = 0
    for s, n in enumerate(need):
        pages[s, :n] = order[at:at + n]
        at += n
    free = np.full(count, -1, np.int32)
    free[:spare] = order[at:]
    return pages, free, count


@pytest.mark.parametrize("page_size", [16, 64, 4096])
@pytest.mark.parametrize("spare", [0, 3, 200])
@pytest.mark.parametrize("decode", [False, True])
def test_plans(hip, L, page_size, spare, decode):
    rng = np.random.default_rng(page_size + spare)
    lengths = [0, 1, page_size - 1, page_size, page_size + 1, 5 * page_size, 3 * page_size + 7, -4, 2 * page_size, 0]
    new = None if decode else [3, 0, 1, 2 * page_size, page_size, 0, 70 * page_size, 5, -2, 1]
    keep = [0, 0, 0, -1, page_size, 3 * page_size + 1, 10 ** 9, 0, -5, -1]
    pages, free, count = table(rng, lengths, page_size, 80, spare)
    rows = len(lengths) if decode else sum(max(0, n) for n in new) + 5
    for k in (None, keep):
        run_plan(L, pages, lengths, new, k, free, spare, page_size, count, rows)
    run_plan(L, pages, lengths, new, keep, free, spare, page_size, count, rows, in_place=True, maps=False, sums=False)
    run_plan(L, pages, lengths, new, keep, free, spare, page_size, count, rows // 2)


@pytest.mark.parametrize("S", [1, 63, 65, 1025, 3000])
def test_plans_of_many_sequences(hip, L, S):
    rng = np.random.default_rng(S)
    lengths = rng.integers(0, 200, S)
    pages, free, count = table(rng, lengths, 16, 20, 5 * S)
    new = rng.integers(0, 60, S) * (rng.random(S) < 0.7)
    keep = np.where(rng.random(S) < 0.3, -1, rng.integers(0, 150, S))
    run_plan(L, pages, lengths, new, keep, free, 5 * S, 16, count, int(new.sum()) + 3)
    run_plan(L, pages, lengths, None, keep, free, S // 2, 16, count, S)


@pytest.mark.parametrize("S,rows", [(40, 9000), (700, 20000), (5000, 30000)])
@pytest.mark.parametrize("back", [False, True])
def test_large_plans(hip, L, S, rows, back):
    """More rows than one workgroup takes, long rows of the table, sequences without new tokens, with gaps in their tables,
    and with all their pages there; few free pages in the end."""
    rng = np.random.default_rng(S)
    lengths = rng.integers(0, 3000, S)
    pages, free, count = table(rng, lengths, 16, 260, rows // 16)
    weight = rng.random(S) * (rng.random(S) < 0.6)
    new = rng.multinomial(rows, weight / weight.sum())
    keep = np.where(rng.random(S) < 0.3, -1, rng.integers(0, 2000, S)) if back else None
    first = run_plan(L, pages, lengths, new, keep, free, rows // 16, 16, count, rows + 100)
    again = first["pages"].copy()
    again[rng.random(again.shape) < 0.02] = -1  # some gaps
    run_plan(L, again, lengths, new, keep, first["free"], int(first["free_count"]), 16, count, rows + 100)


def test_plans_with_bad_entries(hip, L):
    """Entries and free pages that name no page, gaps, tokens past the table's end, a stack that overflows or has a bad
    count; nothing outside the arrays is touched."""
    rng = np.random.default_rng(5)
    lengths = [40, 100, 16, 1000, 2 ** 31 - 5]
    pages, free, count = table(rng, [40, 100, 16, 96, 0], 16, 6, 4)
    pages[0, 1], pages[1, 3], pages[2, 0], pages[3, 5] = count, -5, 2 ** 31 - 1, -2 ** 31
    free[1] = count + 3
    run_plan(L, pages, lengths, [30, 20, 64, 9, 3], None, free, 4, 16, count, 140)
    run_plan(L, pages, lengths, [30, 20, 64, 9, 0], [-1, 32, -1, 64, 0], free, 4, 16, count, 140)
    run_plan(L, pages, [40, 100, 16, 96, 0], [30, 20, 64, 9, 0], [-1, -1, -1, -1, -1], free, 10 ** 6, 16, count, 140)
    run_plan(L, pages, [40, 100, 16, 96, 0], [30, 20, 64, 9, 0], None, free, -3, 16, count, 140)


def test_a_plan_taken_again(hip, L):
    """A step that lacked pages, again with the lengths as they were and more pages free: what was dealt stays."""
    rng = np.random.default_rng(6)
    pages, free, count = table(rng, [20, 5], 16, 12, 3)
    free = np.concatenate([free, np.full(20, -1, np.int32)])
    count += 20
    first = run_plan(L, pages, [20, 5], [100, 60], None, free, 3, 16, count, 160)
    assert first["missing"].sum() == 7
    more = first["free"].copy()
    more[:12] = np.arange(count - 12, count)
    again = run_plan(L, first["pages"], [20, 5], [100, 60], None, more, 12, 16, count, 160)
    assert again["missing"].sum() == 0 and again["free_count"] == 5
    assert (again["slots"] >= 0).sum() == 160


# ---- append ---------------------------------------------------------------------------------------------------------------

def run_append(L, seed, new, lengths, *, Hq=4, kv=2, D=64, page=32, block=16, type="i8", out="f16", norm=True, rope=None,
               factors=False, shared_v=False, no_q=False, strided=False, joined=False, packed=True, tail=2, kv_out=True,
               spoil=None, times=2.0, stream=0, inputs=None):
    from oracle import serving as S

    t = _torch()
    rng = np.random.default_rng(seed)
    rope = D if rope is None else rope
    offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.int32) if packed else None
    T = int(sum(new)) + tail if packed else len(lengths)
    pool = Pool(rng, [min(max(n, 0), 100000) for n in lengths], kv, D, page, block, type, joined=joined)
    if type == "e4m3":
        pool.scales = [t.exp2(t.ceil(t.log2(s))) for s in pool.scales]
    pool.lengths = np.asarray(lengths, np.int32)
    if spoil:
        spoil(pool)
    pool.upload()
    before = [values(x) for x in (pool.keys, pool.values)]
    old = [s.cpu().numpy().copy() for s in pool.scales]
    if inputs is not None:
        q, k, v = inputs
    else:
        q, k, v = ((rng.standard_normal((T, n, D)) * times).astype(np.float32) for n in (Hq, kv, kv))
    if strided:  # one projection's rows, with a gap behind
        rows = np.concatenate([q, k, v, np.zeros((T, 1, D), np.float32)], 1)
        keep = dev(rows)
        at = [keep.data_ptr() + 4 * D * o for o in (0, Hq, Hq + kv)]
        strides = dict.fromkeys(("q_stride", "k_stride", "v_stride"), (Hq + 2 * kv + 1) * D)
    else:
        keep = [dev(x) for x in (q, k, v)]
        at, strides = [x.data_ptr() for x in keep], {}
    qn, kn = ((1 + 0.1 * rng.standard_normal(D)).astype(np.float32) for _ in range(2))
    f = np.exp(rng.uniform(0, 2, rope // 2)).astype(np.float32) if factors else None
    d_qn, d_kn, d_f, d_off = dev(qn), dev(kn), None if f is None else dev(f), None if offsets is None else dev(offsets)
    outs = [t.full((T, n, D), 7.0, dtype=dtype_of(out), device="cuda") for n in (Hq, kv, kv)]
    H.block_append_device(pool.cache(), pool.blocks(), T, 0 if no_q else Hq, 0 if no_q else at[0], at[1], 0 if shared_v else at[2],
                          0 if no_q else ptr(outs[0]), ELEM[out], d_offsets=ptr(d_off), d_q_norm=ptr(d_qn) if norm else 0,
                          d_k_norm=ptr(d_kn) if norm else 0, norm_values=norm, rope_dims=rope, d_rope_freq_factors=ptr(d_f),
                          d_k_out=ptr(outs[1]) if kv_out else 0, d_v_out=ptr(outs[2]) if kv_out else 0, stream=stream, **strides)
    sync()
    rows = S.append(None if no_q else q, k, None if shared_v else v, pool.lengths, offsets, pool.pages, page, pool.count,
                    q_norm=qn if norm else None, k_norm=kn if norm else None, norm_values=norm, rope_dims=rope, factors=f)

    def row_bound(x, rotated):
        b = np.abs(x)
        if rotated and rope:
            h = rope // 2
            pair = np.sqrt(x[:, :h] ** 2 + x[:, h:rope] ** 2) * 1.4143
            b = np.concatenate([pair, pair, b[:, rope:]], 1)
        return 20.2 * U * b

    placed, seen = {}, set()
    for row, rq, rk, rv, page_id, slot in rows:
        seen.add(row)
        for o, ref, rot in ((outs[0], rq, True), (outs[1], rk, True), (outs[2], rv, False)):
            if ref is None or (o is not outs[0] and not kv_out):
                continue
            check(values(o[row]), ref, row_bound(ref, rot) + half_step(out, ref))
        if page_id >= 0:
            placed.setdefault((page_id, slot // block), {})[slot] = (rk, rv)
    for row in range(T):
        if row not in seen:  # left as it was
            assert all(bool((o[row] == 7.0).all()) for o in outs)
    for which, bits in ((0, pool.keys), (1, pool.values)):
        now, scales = values(bits), pool.scales[which].cpu().numpy()
        expected, bound, same = before[which].copy(), np.zeros_like(now), old[which].copy()
        for (p, b), slots in placed.items():
            first = min(slots)
            for h in range(kv):
                ref = {i: r[which][h] for i, r in slots.items()}
                off = {i: row_bound(r[which], which == 0)[h] for i, r in slots.items()}
                most, slack = max(np.abs(r).max() for r in ref.values()), max(o.max() for o in off.values())
                fresh = first % block == 0
                had = float(old[which][p, h, b])
                wants = [L.block_scale(type, m) if fresh else L.grown_scale(type, had, m) for m in (most - slack, most + slack)]
                s = float(scales[p, h, b])
                if wants[0] == wants[1]:
                    assert s == wants[0] if wants[0] == had else abs(s - wants[0]) <= 2.02 * (U * s)
                else:
                    assert wants[0] * (1 - 2.02 * U) <= s <= wants[1] * (1 + 2.02 * U), (s, wants, had)
                same[p, h, b] = s
                if s != had and not fresh:  # what was there moved
                    ratio = np.float32(had) / np.float32(s)
                    held = before[which][p, h, b * block:first].astype(np.float32) * ratio
                    expected[p, h, b * block:first] = np.rint(held) if type == "i8" else values(t.from_numpy(held).to(dtype_of(type)))
                for i, r in ref.items():
                    x = np.clip(r / s, -MOST[type], MOST[type])
                    expected[p, h, i] = x
                    step = 0.5 if type == "i8" else half_step(type, x)
                    bound[p, h, i] = step * 1.0001 + off[i] / s + 3 * U * np.abs(x)
        check(now, expected, bound)
        assert np.array_equal(same, scales, equal_nan=True)
    return placed


@pytest.mark.parametrize("D,Hq,kv", [(64, 4, 2), (128, 6, 1), (256, 8, 2), (128, 5, 5)])
@pytest.mark.parametrize("type,out,block", [("i8", "f16", 16), ("i8", "f32", 32), ("e4m3", "bf16", 16), ("e4m3", "f32", 32)])
def test_append_prompts(hip, L, D, Hq, kv, type, out, block):
    placed = run_append(L, D + kv, [3, 0, 17, 1, 40], [3, 0, 37, 5000, 41], Hq=Hq, kv=kv, D=D, type=type, out=out, block=block)
    assert sum(len(s) for s in placed.values()) == 61


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("type", ["i8", "e4m3"])
def test_append_block_sizes(hip, L, D, block, type):
    """Every number of passes over a block's rows; blocks whole, begun and ended within."""
    run_append(L, D + block, [300, 5, 129], [300, 200, 150], D=D, block=block, page=128, type=type, Hq=2, kv=1, kv_out=False)


@pytest.mark.parametrize("D,rope,factors,norm", [(64, 0, False, True), (64, 8, True, False), (128, 24, False, True),
                                                 (128, 64, True, True), (256, 256, True, False), (256, 136, False, True)])
@pytest.mark.parametrize("packed", [True, False])
def test_append_rotations(hip, L, D, rope, factors, norm, packed):
    new = [9, 2] if packed else None
    run_append(L, rope, new, [1009, 23456], D=D, rope=rope, factors=factors, norm=norm, out="f32", packed=packed, page=64)


@pytest.mark.parametrize("kw", [{"shared_v": True}, {"no_q": True}, {"strided": True}, {"joined": True}, {"kv_out": False},
                                {"shared_v": True, "norm": False}, {"times": 40.0, "norm": False}, {"times": 1e-3, "norm": False}])
@pytest.mark.parametrize("type", ["i8", "e4m3"])
def test_append_forms(hip, L, kw, type):
    run_append(L, 5, [2, 7, 1], [2, 30, 70], type=type, out="bf16", **kw)


@pytest.mark.parametrize("D,Hq,kv", [(64, 14, 2), (128, 16, 1), (256, 8, 2)])
@pytest.mark.parametrize("type", ["i8", "e4m3"])
def test_append_one_token_each(hip, L, D, Hq, kv, type):
    lengths = [1, 0, 17, 16, -4, 333, 48]
    placed = run_append(L, 11, None, lengths, packed=False, D=D, Hq=Hq, kv=kv, type=type, out="f32", kv_out=False)
    assert len(placed) == 5


def test_append_many_sequences(hip, L):
    rng = np.random.default_rng(3)
    new = rng.integers(0, 90, 150)
    new[10:20] = 0
    run_append(L, 12, list(new), list(new + rng.integers(0, 50, 150)), D=64, Hq=2, kv=1, rope=16, kv_out=False)


def test_append_absent_and_bad_pages(hip, L):
    def spoil(pool):
        pool.pages[0, 0] = -1
        pool.pages[1, 0] = pool.count
        pool.pages[2, 1] = np.iinfo(np.int32).max
        pool.pages[3, 0] = np.iinfo(np.int32).min
        pool.lengths[4] = pool.width * pool.page + 3

    placed = run_append(L, 13, [5, 40, 40, 3, 6], [5, 40, 40, 3, 6], spoil=spoil)
    assert sum(len(s) for s in placed.values()) == 8 + 32


@pytest.mark.parametrize("type", ["i8", "e4m3"])
def test_a_block_token_by_token(hip, L, type):
    """Elements that grow from token to token: a scale grows time and again, and what the block holds stays within its
    steps.  With half a step of the scale at each growth, i8's at least 1.25 times the one before: 2.5 steps in all, and
    half of one of its own; e4m3's powers of two keep a value's relative half step, and a subnormal's half step (2^-10)
    of each scale, half the next one's."""
    t = _torch()
    rng = np.random.default_rng(1)
    D, block = 64, 64
    x = (rng.standard_normal((block, 1, D)) * 1.07 ** np.arange(block)[:, None, None]).astype(np.float32)
    keys, vals = (t.zeros((1, 1, block, D), dtype=dtype_of(type), device="cuda") for _ in range(2))
    scales = [t.full((1, 1, 1), float("nan"), device="cuda") for _ in range(2)]
    pages, d, grown = dev(np.zeros((1, 1), np.int32)), dev(x), 0
    for i in range(block):
        length = dev(np.array([i + 1], np.int32))
        c = H.paged_cache(ptr(keys), ptr(vals), ELEM[type], page_count=1, page_size=block, head_count_kv=1, head_dim=D,
                          d_pages=ptr(pages), d_lengths=ptr(length), sequence_count=1, pages_per_sequence=1)
        b = H.cache_blocks(block, d_key_scales=ptr(scales[0]), d_value_scales=ptr(scales[1]))
        was = float(scales[0])
        H.block_append_device(c, b, 1, 0, 0, d[i].data_ptr(), 0, 0, 0)
        sync()
        now = float(scales[0])
        grown += i > 0 and now != was
        assert not now < was
        s = np.float64(now)
        got, ref = values(keys)[0, 0, :i + 1] * s, x[:i + 1, 0].astype(np.float64)
        bound = 3.001 * s if type == "i8" else np.abs(ref) * 2.0 ** -4 * 1.001 + s * 2.0 ** -9
        assert (np.abs(got - ref) <= bound).all()
    assert grown >= 5 and t.equal(keys.view(t.uint8), vals.view(t.uint8))


@pytest.mark.parametrize("type", ["i8", "e4m3"])
def test_append_extremes(hip, L, type):
    """Zeros, numbers below and above the scales' range, infinities and NaN, block by block."""
    t = _torch()
    D, block = 64, 16
    x = np.random.default_rng(2).standard_normal((7 * block, 1, D)).astype(np.float32)
    x[:16] = 0.0
    x[16:32] *= 1e-38
    x[32:48] *= 1e37
    x[50, 0, 3], x[70, 0, 5], x[90, 0, 60] = np.inf, -np.inf, np.nan
    keys, vals = (t.zeros((7, 1, block, D), dtype=dtype_of(type), device="cuda") for _ in range(2))
    scales = [t.full((7, 1, 1), 5.0, device="cuda") for _ in range(2)]
    pages, d = dev(np.arange(7, dtype=np.int32)[None]), dev(x)
    b = H.cache_blocks(block, d_key_scales=ptr(scales[0]), d_value_scales=ptr(scales[1]))

    def append(rows, first, length):
        n, off = dev(np.array([length], np.int32)), dev(np.array([0, rows], np.int32))
        c = H.paged_cache(ptr(keys), ptr(vals), ELEM[type], page_count=7, page_size=block, head_count_kv=1, head_dim=D,
                          d_pages=ptr(pages), d_lengths=ptr(n), sequence_count=1, pages_per_sequence=7)
        H.block_append_device(c, b, rows, 0, 0, d[first].data_ptr(), 0, 0, 0, d_offsets=ptr(off))
        sync()
        return scales[0].cpu().numpy().reshape(-1), values(keys)

    s, k = append(112, 0, 112)
    assert s[0] == 2.0 ** -100 and not k[0].any()
    assert s[1] == 2.0 ** -100 and not k[1].any()
    assert s[2] == 2.0 ** 100 and np.array_equal(np.abs(k[2][0, :, :4]), np.full((16, 4), MOST[type]))
    assert np.isnan(s[3:6]).all() and np.isfinite(s[6])
    # a poisoned block stays so until it begins anew (its first position is among the rows)
    s, _ = append(2, 96, 84)
    assert np.isnan(s[5])
    s, _ = append(2, 96, 66)
    assert np.isfinite(s[4]) and np.isnan(s[5])
    s, _ = append(2, 96, 82)
    assert np.isfinite(s[5])
    s, _ = append(16, 96, 64)
    assert np.isfinite(s[3])


# ---- bounds and selection ---------------------------------------------------------------------------------------------------

def run_bounds(L, pool, new=None, tail=3):
    lengths, packed = pool.lengths, new is not None
    before = values(pool.bounds)
    offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.int32) if packed else None
    d_off = dev(offsets) if packed else None
    H.block_bounds_device(pool.cache(), pool.blocks(), int(offsets[-1]) + tail if packed else len(lengths), d_offsets=ptr(d_off))
    sync()
    touched = set()
    for s, n in enumerate(lengths):
        for p in range(max(0, n - (new[s] if packed else 1)), n):
            if p < pool.width * pool.page:
                touched.add((s, p // pool.block))
    with np.errstate(all="ignore"):
        want = L.bounds(pool.real(0), lengths, pool.pages, pool.page, pool.count, pool.block, touched)
    expected = before.copy()
    for (page, b), (lo, hi) in want.items():
        expected[page, :, b, 0], expected[page, :, b, 1] = lo, hi
    assert np.array_equal(values(pool.bounds), expected, equal_nan=True)
    return len(want)


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 127, 128, 129, 160, 161, 255, 257, 400, 3, 1000]


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("type,scaled", [("f16", False), ("bf16", False), ("e4m3", False), ("e4m3", True), ("i8", True)])
@pytest.mark.parametrize("page,block", [(16, 16), (128, 16), (64, 64), (128, 128)])
def test_bounds(hip, L, D, type, scaled, page, block):
    rng = np.random.default_rng(D)
    pool = Pool(rng, LENGTHS, 2, D, page, block, type, scaled=scaled, joined=page == 64)
    run_bounds(L, pool)
    assert run_bounds(L, pool, [min(n, 1 + 7 * i) for i, n in enumerate(LENGTHS)]) >= 19  # (sequences with new tokens)


@pytest.mark.parametrize("type", ["f16", "bf16", "e4m3"])
def test_bounds_of_odd_keys(hip, L, type):
    """Infinities, NaN, zeros of both signs, subnormals, and f16 values between two of bf16."""
    t = _torch()
    pool = Pool(np.random.default_rng(4), [64, 40], 1, 64, 32, 16, type, scaled=False)
    k = pool.keys
    page = pool.pages
    k[page[0, 0], 0, 3, 5] = float("nan")
    if type != "e4m3":
        k[page[0, 0], 0, 17, 6], k[page[0, 1], 0, 2, 7], k[page[0, 1], 0, 3, 7] = float("inf"), float("-inf"), float("nan")
        k[page[1, 0], 0, :16, 8] = 2.0 ** -24
        k[page[1, 0], 0, :16, 9] = -1.0 - 2.0 ** -10
    k[page[0, 1], 0, 16:, 1] = 0.0
    k[page[0, 1], 0, 20, 1] = -0.0
    run_bounds(L, pool, [64, 40])
    assert t.isfinite(pool.bounds[page[0, :2].tolist()]).all()


def test_bounds_of_poisoned_and_absent_blocks(hip, L):
    pool = Pool(np.random.default_rng(6), [64, 50, 70], 2, 64, 32, 16, "i8")
    pool.scales[0][pool.pages[0, 1], 1, 0] = float("nan")
    pool.pages[1, 0], pool.pages[2, 2] = -1, pool.count
    pool.lengths[0] = pool.width * pool.page + 9
    pool.upload()
    H.block_bounds_device(pool.cache(), pool.blocks(), 300, d_offsets=ptr(dev(np.array([0, 120, 170, 240], np.int32))))
    sync()
    b = values(pool.bounds)
    assert (np.abs(b[pool.pages[0, 1], 1, 0]) > 3e38).all() and (np.abs(b[pool.pages[0, 1], 0, 0]) < 100).all()
    named = {int(p) for p in (pool.pages[0, 0], pool.pages[0, 1], pool.pages[1, 1], pool.pages[2, 0], pool.pages[2, 1])}
    assert all(np.isnan(b[p]).all() for p in range(pool.count) if p not in named)


def run_select(L, pool, Hq, budget, first, last, rng=None, q_type="f32", q=None, gap=0, counts=True, stream=0):
    t = _torch()
    n, D = len(pool.lengths), pool.D
    if q is None:
        q = t.from_numpy((rng.standard_normal((n, Hq + gap, D)) * 2).astype(np.float32)).cuda().to(dtype_of(q_type))
    selected = t.full((n * pool.kv + 1, budget), -7, dtype=t.int32, device="cuda")
    d_counts = t.full((n * pool.kv + 1,), -7, dtype=t.int32, device="cuda")
    H.block_select_device(pool.cache(), pool.blocks(), Hq, ptr(q), ELEM[q_type], budget, ptr(selected), ptr(d_counts) if counts else 0,
                          first_blocks=first, last_blocks=last, q_stride=(Hq + gap) * D if gap else 0, stream=stream)
    sync()
    want = L.select(values(q[:, :Hq]), pool.bounds.float().cpu().numpy(), pool.lengths, pool.pages, pool.page, pool.count,
                    pool.block, budget, first, last)
    got = selected.cpu().numpy()
    for row, blocks in enumerate(want):
        assert list(got[row]) == blocks + [-1] * (budget - len(blocks)), (row, got[row], blocks)
    assert (got[-1] == -7).all()
    assert list(d_counts.cpu().numpy()) == [len(b) for b in want] + [-7] if counts else bool((d_counts == -7).all())
    return selected, d_counts, want


def bounded(pool, rng, spread=1.0):
    """Bounds of every block, as random keys have them."""
    t = _torch()
    x = rng.standard_normal((pool.count, pool.kv, pool.per, 2, pool.D)) * spread
    x.sort(axis=3)
    pool.bounds = t.from_numpy(x.astype(np.float32)).cuda().to(t.bfloat16)
    return pool


@pytest.mark.parametrize("D,Hq,kv", [(64, 14, 2), (128, 4, 1), (128, 10, 5), (256, 8, 2), (256, 3, 3), (64, 16, 1)])
@pytest.mark.parametrize("q_type", ["f32", "f16", "bf16"])
def test_select(hip, L, D, Hq, kv, q_type):
    rng = np.random.default_rng(D + Hq)
    pool = bounded(Pool(rng, [0, 1, 500, 2000, 16, 17, 3000, -3], kv, D, 32, 16, "i8"), rng)
    for budget, first, last in ((1, 0, 0), (1, 1, 0), (7, 1, 2), (40, 0, 1), (500, 3, 3)):
        run_select(L, pool, Hq, budget, first, last, rng, q_type)
    run_select(L, pool, Hq, 9, 1, 1, rng, q_type, gap=2, counts=False)


@pytest.mark.parametrize("blocks", [1, 63, 64, 65, 1000, 1024, 1025, 5000])
def test_select_from_many(hip, L, blocks):
    rng = np.random.default_rng(blocks)
    pool = bounded(Pool(rng, [16 * blocks - 3], 1, 64, 64, 16, "i8"), rng)
    for budget in (1, 2, 64, 1023, 1024):
        run_select(L, pool, 2, max(budget, 2), 1, 1, rng)


@pytest.mark.parametrize("blocks", [300, 3000, 20000])
@pytest.mark.parametrize("alike", ["all", "few", "nearly"])
def test_select_where_many_are_alike(hip, L, blocks, alike):
    """Blocks of equal bounds, of a few kinds, and of bounds of which one element differs by the last bit of bf16 under a
    query element of 2^-20: all within what single precision can tell apart."""
    t = _torch()
    rng = np.random.default_rng(blocks)
    pool = bounded(Pool(rng, [16 * blocks], 1, 64, 128, 16, "i8", extra=0), rng)
    b = pool.bounds.float().cpu().numpy()
    flat = np.empty((blocks, 2, 64), np.float32)
    kinds = rng.integers(0, {"all": 1, "few": 5, "nearly": 1}[alike], blocks)
    flat[:] = b[pool.pages[0, 0], 0, :1]
    flat[:, :, 5] += kinds[:, None] * np.float32(0.5)
    if alike == "nearly":
        flat[:, :, 9] = (1 + rng.integers(0, 100, blocks)[:, None] * 2.0 ** -7).astype(np.float32)
    for i in range(blocks):
        b[pool.pages[0, i // 8], 0, i % 8] = flat[i]
    pool.bounds = t.from_numpy(b).cuda().to(t.bfloat16)
    q = rng.standard_normal((1, 2, 64)).astype(np.float32)
    q[:, :, 9] = 2.0 ** -20
    for budget in (1, 70, 299):
        run_select(L, pool, 2, budget, 0, 1, q=dev(q))


@pytest.mark.parametrize("times", [2.0 ** 100, 2.0 ** -120, 3e38, 1e-45])
def test_select_of_large_and_small_numbers(hip, L, times):
    """Scores past f32's range and below its normal numbers."""
    rng = np.random.default_rng(3)
    pool = bounded(Pool(rng, [3000, 40], 2, 128, 64, 32, "i8"), rng)
    big = bounded(Pool(rng, [3000, 40], 2, 128, 64, 32, "i8"), rng, spread=1e36)
    q = (np.clip(rng.standard_normal((2, 6, 128)), -1, 1) * times).astype(np.float32)
    for p in (pool, big):
        run_select(L, p, 6, 20, 1, 1, q=dev(q))


def test_select_ties_and_odd_scores(hip, L):
    """Equal scores go to the first blocks; zeros of both signs are equal; scores that differ in their last bits only;
    infinite and NaN queries; the largest bounds."""
    t = _torch()
    rng = np.random.default_rng(9)
    pool = bounded(Pool(rng, [900, 900, 900, 900], 1, 64, 64, 16, "i8", extra=0), rng)
    q = rng.standard_normal((4, 2, 64)).astype(np.float32)
    b = values(pool.bounds).astype(np.float32)
    p = pool.pages
    b[p[0]] = b[p[0, 0], :, :1]  # every block alike
    b[p[1]] = 0.0
    b[p[1]][:, :, ::2] = -0.0
    q[1, :, ::2] *= -1
    q[2, 0, 3], q[2, 1, 9], q[2, 1, 10] = np.inf, -np.inf, np.nan
    b[p[2, 3], 0, 1] = [[-3e38] * 64, [3e38] * 64]
    b[p[3]] = 1.0  # two elements tell the blocks apart, by 2^-30 of the score
    q[3] = 1.0
    q[3, :, 0] = 2.0 ** -24
    for i in range(14):
        b[p[3, i], 0, :, :, 0] = (1 + (i * 5) % 14 * np.arange(1, 5)[:, None]).astype(np.float32)
    pool.bounds = t.from_numpy(b).cuda().to(t.bfloat16)
    for budget in (1, 5, 30):
        run_select(L, pool, 2, budget, 0, 0, q=dev(q))


def test_select_absent_pages(hip, L):
    rng = np.random.default_rng(10)
    pool = bounded(Pool(rng, [700, 300, 64], 2, 64, 32, 16, "i8"), rng)
    pool.pages[0, :12], pool.pages[0, 21], pool.pages[1, 4], pool.pages[2, :2] = -1, pool.count, 2 ** 31 - 1, -9
    pool.lengths[1] = pool.width * pool.page + 77
    pool.upload()
    for budget in (2, 9, 60):
        run_select(L, pool, 4, budget, 1, 1, rng)


# ---- attention ----------------------------------------------------------------------------------------------------------------

def attention_bound(pool, name, ref, mass, size, count):
    d = size * (2.0 ** -20 + (pool.D + 1) * U)
    weight = 2 * (d + 2.0 ** -20) + (2.0 ** -17 if pool.type == "bf16" else 2.0 ** -21) + 2 * (count + 64) * U + 4 * U
    bound = 1.01 * mass * weight[..., None] + half_step(name, ref) + 1e-30
    if pool.type != "bf16":
        most = MOST[pool.type] * float(np.nanmax(pool.scales[1].cpu().numpy())) if pool.scaled else np.nanmax(np.abs(pool.real(1)))
        bound = bound + 1.01 * (count * 2.0 ** -35 * most)[..., None]
    return bound


def run_attention(L, pool, Hq, q_type="f32", out="f32", window=0, scale=None, rng=None, q_times=2.0, strides=False, lists=None,
                  counts=None, budget=0, stream=0, q=None, bound=None):
    """lists: [S * kv][budget] with what counts decided by `counts` (None: all)."""
    t = _torch()
    n, D = len(pool.lengths), pool.D
    scale = D ** -0.5 if scale is None else scale
    gap = 2 if strides else 0
    full = q if q is not None else t.from_numpy((rng.standard_normal((n, Hq + gap, D)) * q_times).astype(np.float32)).cuda().to(dtype_of(q_type))
    got = t.full((n, Hq + 2 * gap, D), 7.0, dtype=dtype_of(out), device="cuda")
    d_lists = None if lists is None else dev(np.asarray(lists, np.int32))
    d_counts = None if counts is None else dev(np.asarray(counts, np.int32))
    H.block_attention_device(pool.cache(), pool.blocks(), Hq, ptr(full), ELEM[q_type], ptr(got), ELEM[out], scale=scale,
                             sliding_window=window, d_selected=ptr(d_lists), d_counts=ptr(d_counts), budget=budget,
                             q_stride=(Hq + gap) * D if strides else 0, output_stride=(Hq + 2 * gap) * D if strides else 0, stream=stream)
    sync()
    chosen = None
    if lists is not None:
        chosen = [row[:max(0, min(budget, c))] for row, c in zip(np.asarray(lists), [budget] * len(lists) if counts is None else counts)]
    ref, mass, size, count = L.block_attention(values(full[:, :Hq]), pool.real(0).astype(np.float64), pool.real(1).astype(np.float64),
                                               pool.lengths, pool.pages, pool.page, pool.count, window, scale, chosen, pool.block)
    assert bool((got[:, Hq:] == 7.0).all())
    check(values(got[:, :Hq]), ref, attention_bound(pool, out, ref, mass, size, count) if bound is None else bound(ref, mass))
    return got[:, :Hq], ref


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("type", ["i8", "e4m3"])
@pytest.mark.parametrize("q_type,out", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("page,block", [(16, 16), (64, 32), (128, 128)])
def test_scaled_attention(hip, L, D, type, q_type, out, page, block):
    rng = np.random.default_rng(D)
    run_attention(L, Pool(rng, LENGTHS, 2, D, page, block, type, spread=1.0), 8, q_type, out, rng=rng)


@pytest.mark.parametrize("Hq,kv,D", [(1, 1, 64), (7, 1, 128), (9, 1, 64), (16, 1, 256), (24, 2, 128), (10, 5, 64)])
@pytest.mark.parametrize("type", ["i8", "e4m3"])
def test_scaled_attention_heads(hip, L, Hq, kv, D, type):
    rng = np.random.default_rng(Hq)
    run_attention(L, Pool(rng, [1, 130, 0, 513], kv, D, 32, 16, type), Hq, rng=rng, strides=True)


@pytest.mark.parametrize("window", [1, 15, 16, 17, 100, 5000])
@pytest.mark.parametrize("type", ["i8", "e4m3"])
def test_scaled_attention_windows(hip, L, window, type):
    rng = np.random.default_rng(window)
    pool = Pool(rng, LENGTHS, 2, 128, 32, 32, type)
    for s, n in enumerate(LENGTHS):  # pages that the window has passed are given back
        pool.pages[s, :max(0, n - window) // pool.page] = -1
    pool.upload()
    run_attention(L, pool, 4, window=window, rng=rng)


@pytest.mark.parametrize("type", ["i8", "e4m3"])
def test_scaled_attention_wide_tables_and_joined_pages(hip, L, type):
    rng = np.random.default_rng(3)
    run_attention(L, Pool(rng, [1, 0, 129, 700, 64], 2, 64, 16, 16, type, extra=(33 << 20) // (2 * 64 * 2 * 5 * 16)), 8, rng=rng)
    run_attention(L, Pool(rng, [1, 0, 129, 700, 64], 2, 64, 64, 16, type, joined=True), 8, rng=rng)


@pytest.mark.parametrize("type", ["i8", "e4m3"])
def test_scales_far_apart(hip, L, type):
    """Blocks of values 2^100 apart, the small ones under the heavy keys: the weights of each block count with its own
    scale, whatever the others' are.  One sequence has tiny scales only."""
    t = _torch()
    rng = np.random.default_rng(8)
    pool = Pool(rng, [64, 64, 64, 200], 1, 64, 16, 16, type, spare=0)
    e = np.array([[0, -60, 60, -100], [-100, -100, -100, -100], [100, 99, 98, 100], [0, 0, 0, 0]])
    for s in range(3):
        for i in range(4):
            pool.scales[1][pool.pages[s, i]] = 2.0 ** e[s, i]
    run = lambda: run_attention(L, pool, 4, rng=rng, bound=lambda ref, mass: mass * 2.0 ** -12 + 2.0 ** -96)  # noqa: E731
    run()
    # a scale of 0 is nothing but zeros
    pool.scales[1][pool.pages[0, 2]] = 0.0
    run()
    # keys' scales as far apart: scores of nearly 0 beside others
    pool.scales[0][pool.pages[2, 1]] = 2.0 ** -100
    run()
    assert t.isfinite(pool.scales[1]).all()


def test_a_poisoned_block_shows(hip, L):
    """A NaN scale of a block reaches the heads that attend to it, and no other sequence or KV head."""
    t = _torch()
    rng = np.random.default_rng(12)
    for which in (0, 1):
        pool = Pool(rng, [100, 100, 100], 2, 64, 32, 16, "i8")
        pool.scales[which][pool.pages[1, 1], 0, 1] = float("nan")
        q = dev(rng.standard_normal((3, 4, 64)).astype(np.float32))
        got = t.zeros((3, 4, 64), device="cuda")
        H.block_attention_device(pool.cache(), pool.blocks(), 4, ptr(q), 0, ptr(got), 0)
        sync()
        bad = t.isnan(got).all(-1)
        assert bad.tolist() == [[False] * 4, [True, True, False, False], [False] * 4]
        assert t.isfinite(got[~bad]).all()
        # outside a window, behind the end and on absent pages it does not
        pool.lengths[1] = 48
        pool.upload()
        H.block_attention_device(pool.cache(), pool.blocks(), 4, ptr(q), 0, ptr(got), 0)
        pool.lengths[1] = 100
        pool.upload()
        again = t.zeros((3, 4, 64), device="cuda")
        H.block_attention_device(pool.cache(), pool.blocks(), 4, ptr(q), 0, ptr(again), 0, sliding_window=36)
        pool.pages[1, 1] = -1
        pool.upload()
        third = t.zeros((3, 4, 64), device="cuda")
        H.block_attention_device(pool.cache(), pool.blocks(), 4, ptr(q), 0, ptr(third), 0)
        sync()
        assert all(t.isfinite(x).all() for x in (got, again, third))


def test_scaled_attention_offsets_past_32_bits(hip, L):
    t = _torch()
    rng = np.random.default_rng(14)
    pool = Pool(rng, [40, 17], 1, 64, 32, 16, "i8", spare=0, extra=0)
    stride = (1 << 31) + 4096
    far = t.zeros(pool.count * stride, dtype=t.int8, device="cuda")
    keys, vals = (far.view(pool.count, stride)[:, o:o + 2048] for o in (0, 1 << 30))
    keys.copy_(pool.keys.reshape(pool.count, -1))
    vals.copy_(pool.values.reshape(pool.count, -1))
    pool.keys, pool.values, pool.stride = keys.view(pool.count, 1, 32, 64), vals.view(pool.count, 1, 32, 64), stride
    run_attention(L, pool, 2, rng=rng)
    run_bounds(L, pool)
    run_attention(L, pool, 2, rng=rng, lists=[[0, 2], [0, 1]], budget=2)
    row = dev(np.full((2, 1, 64), 0.25, np.float32))
    was = [x.clone() for x in (pool.keys, pool.values)]
    H.block_append_device(pool.cache(), pool.blocks(), 2, 0, 0, ptr(row), 0, 0, 0)
    sync()
    for now, old, scales in zip((pool.keys, pool.values), was, pool.scales):
        for s, n in enumerate(pool.lengths):
            page, slot = int(pool.pages[s, (n - 1) // 32]), (n - 1) % 32
            scale = float(scales[page, 0, slot // 16])
            assert (np.abs(values(now[page, 0, slot]) * scale - 0.25) <= 0.5001 * scale).all()
            old[page, 0, slot] = now[page, 0, slot]
            if slot % 16 == 0:
                continue
        assert t.equal(now, old)


SELECTED = [("f16", False, "f32"), ("f16", False, "f16"), ("bf16", False, "f32"), ("bf16", False, "bf16"), ("e4m3", False, "f32"),
            ("e4m3", True, "bf16"), ("i8", True, "f32")]


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("type,scaled,q_type", SELECTED)
@pytest.mark.parametrize("page,block", [(16, 16), (128, 32), (64, 64)])
def test_selected_attention(hip, L, D, type, scaled, q_type, page, block):
    """Lists of every length, with entries that name no block, blocks behind the end and on absent pages; what they leave
    out holds NaN where the type has one."""
    rng = np.random.default_rng(D + block)
    pool = Pool(rng, LENGTHS, 2, D, page, block, type, scaled=scaled)
    budget = 11
    lists = np.full((len(LENGTHS) * 2, budget), -1, np.int32)
    counts = np.zeros(len(LENGTHS) * 2, np.int32)
    for row in range(len(lists)):
        n = -(-LENGTHS[row // 2] // block)
        some = sorted(rng.permutation(n)[:rng.integers(0, budget + 1)]) if n else []
        lists[row, :len(some)], counts[row] = some, len(some)
    lists[30, 3], lists[31, 0], lists[32, 5], lists[33, 1] = -1, 10 ** 6, 2 ** 31 - 1, -2 ** 31
    pool.pages[17, 1] = -1
    pool.pages[19, 0] = pool.count
    pool.upload()
    run_attention(L, pool, 8, q_type, rng=rng, lists=lists, counts=counts, budget=budget)
    counts[5], counts[6], counts[34], counts[36] = -3, 0, 500, 2 ** 31 - 1
    run_attention(L, pool, 8, q_type, rng=rng, lists=lists, counts=counts, budget=budget)
    run_attention(L, pool, 8, q_type, rng=rng, lists=lists, budget=budget, strides=True)


@pytest.mark.parametrize("type,scaled", [("bf16", False), ("i8", True)])
def test_selected_attention_of_many_rows(hip, L, type, scaled):
    """More (sequence, KV head) rows than lanes, groups of more than eight heads, long lists."""
    rng = np.random.default_rng(2)
    lengths = list(rng.integers(1, 300, 50)) + [4000]
    pool = Pool(rng, lengths, 3, 64, 16, 16, type, scaled=scaled)
    lists = np.full((len(lengths) * 3, 250), -1, np.int32)
    for row in range(len(lists)):
        n = -(-lengths[row // 3] // 16)
        lists[row, :n] = rng.permutation(n)
    counts = [min(250, -(-lengths[r // 3] // 16)) for r in range(len(lists))]
    run_attention(L, pool, 27, rng=rng, lists=lists, counts=counts, budget=250)


def test_a_block_named_twice_counts_twice(hip, L):
    rng = np.random.default_rng(2)
    pool = Pool(rng, [100], 1, 64, 32, 16, "i8")
    run_attention(L, pool, 2, rng=rng, lists=[[1, 4, 4, 6]], budget=4)


def test_masks_that_leave_nothing(hip, L):
    t = _torch()
    rng = np.random.default_rng(2)
    for type in ("i8", "bf16"):
        pool = Pool(rng, [0, 50, -2, 60], 1, 64, 16, 16, type)
        pool.pages[1, :] = -1
        pool.upload()
        lists = [[-1, -1], [0, 1], [0, 3], [70, -1]]
        got, _ = run_attention(L, pool, 2, rng=rng, lists=lists, budget=2)
        assert not got.any()
        if type == "i8":
            got, _ = run_attention(L, pool, 2, rng=rng)
            assert not got[:3].any() and bool(t.isfinite(got).all()) and got[3].any()


def test_odd_queries(hip, L):
    """Large and tiny queries and scales; a NaN or infinite query shows in its own head."""
    t = _torch()
    rng = np.random.default_rng(20)
    pool = Pool(rng, [100, 33], 1, 64, 16, 16, "i8")
    for times, scale in ((2.0 ** 90, 2.0 ** -95), (2.0 ** -90, 2.0 ** 88), (2.0 ** 60, 2.0 ** -60)):
        run_attention(L, pool, 2, rng=rng, q_times=times, scale=scale)
    q = rng.standard_normal((2, 2, 64)).astype(np.float32)
    q[0, 1, 7], q[1, 0, 3] = np.nan, np.inf
    got = t.zeros((2, 2, 64), device="cuda")
    d = dev(q)
    H.block_attention_device(pool.cache(), pool.blocks(), 2, ptr(d), 0, ptr(got), 0)
    sync()
    assert t.isnan(got).all(-1).tolist() == [[False, True], [True, False]]

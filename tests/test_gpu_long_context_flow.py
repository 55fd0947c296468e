"""The operators of long contexts in use: requests come, go on and end, their pages dealt on the device, their tokens into
pages of 8 bits, their attention over the blocks that the bounds select; captured and replayed with the lengths that the
plan itself moves on; on several streams."""
import numpy as np
import pytest

from heliopause_amd import hip_kernels as H

pytestmark = pytest.mark.gpu

HQ, KV, D, PAGE, BLOCK, WIDTH, POOL, BUDGET = 6, 2, 64, 32, 16, 10, 48, 5
SCALE = D ** -0.5


def _torch():
    import torch

    return torch


def dev(a):
    return _torch().from_numpy(np.ascontiguousarray(a)).cuda()


class Service:
    """The device state of a batch of `n` sequences, and a step of it."""

    def __init__(self, n, type, seed, pool=POOL):
        t = _torch()
        self.n, self.type, self.pool = n, type, pool
        z = lambda *s, dtype=t.int32: t.zeros(s, dtype=dtype, device="cuda")  # noqa: E731
        e = {"i8": t.int8, "e4m3": t.float8_e4m3fn, "f16": t.float16}[type]
        self.id = {"i8": H.HP_ELEM_I8, "e4m3": H.HP_ELEM_E4M3, "f16": H.HP_ELEM_F16}[type]
        self.keys, self.values = (z(pool, KV, PAGE, D, dtype=e) for _ in range(2))
        if type != "i8":
            self.keys.fill_(float("nan"))
            self.values.fill_(float("nan"))
        self.scales = [z(pool, KV, PAGE // BLOCK, dtype=t.float32).fill_(float("nan")) for _ in range(2)] if type != "f16" else [None] * 2
        self.bounds = z(pool, KV, PAGE // BLOCK, 2, D, dtype=t.bfloat16).fill_(float("nan"))
        self.pages, self.lengths = z(n, WIDTH).fill_(-1), z(n)
        self.free = dev(np.random.default_rng(seed).permutation(pool).astype(np.int32))
        self.free_count, self.missing = z(1).fill_(pool), z(n)
        self.keep = z(n)
        self.selected, self.counts = z(n, KV, BUDGET), z(n, KV)
        self.out, self.whole = z(n, HQ, D, dtype=t.float32), z(n, HQ, D, dtype=t.float32)
        self.q_in, self.k_in, self.v_in = (z(n, h, D, dtype=t.float32) for h in (HQ, KV, KV))
        self.q16 = z(n, HQ, D, dtype=t.float16)
        p = lambda x: 0 if x is None else x.data_ptr()  # noqa: E731
        self.p = p
        self.cache = H.paged_cache(p(self.keys), p(self.values), self.id, page_count=pool, page_size=PAGE, head_count_kv=KV,
                                   head_dim=D, d_pages=p(self.pages), d_lengths=p(self.lengths), sequence_count=n,
                                   pages_per_sequence=WIDTH)
        self.blocks = H.cache_blocks(BLOCK, d_key_scales=p(self.scales[0]), d_value_scales=p(self.scales[1]),
                                     d_key_bounds=p(self.bounds))

    def _append(self, rows, q, k, v, q_out, stream, **kw):
        if self.type == "f16":
            H.paged_append_device(self.cache, rows, HQ, self.p(q), self.p(k), self.p(v), self.p(q_out), H.HP_ELEM_F16, rope_dims=D,
                                  norm_values=True, stream=stream, **kw)
        else:
            H.block_append_device(self.cache, self.blocks, rows, HQ, self.p(q), self.p(k), self.p(v), self.p(q_out), H.HP_ELEM_F16,
                                  rope_dims=D, norm_values=True, stream=stream, **kw)

    def prompts(self, new, keep, rng, stream=0):
        """Requests' new tokens, packed; the caller's rows of queries, keys and values."""
        t = _torch()
        rows = int(sum(new)) + 2
        q, k, v = (dev(rng.standard_normal((rows, h, D)).astype(np.float32)) for h in (HQ, KV, KV))
        q_out = t.zeros((rows, HQ, D), dtype=t.float16, device="cuda")
        d_new, d_keep = dev(np.asarray(new, np.int32)), dev(np.asarray(keep, np.int32))
        offsets, slots = t.zeros(self.n + 1, dtype=t.int32, device="cuda"), t.zeros(rows, dtype=t.int64, device="cuda")
        t.cuda.synchronize()
        H.page_plan_device(self.n, WIDTH, PAGE, self.pool, self.p(self.pages), self.p(self.lengths), self.p(self.lengths),
                           self.p(self.free), self.p(self.free_count), d_new_tokens=self.p(d_new), d_keep_from=self.p(d_keep),
                           d_offsets=self.p(offsets), d_missing=self.p(self.missing), token_count=rows, d_slots=self.p(slots), stream=stream)
        self._append(rows, q, k, v, q_out, stream, d_offsets=self.p(offsets))
        H.block_bounds_device(self.cache, self.blocks, rows, d_offsets=self.p(offsets), stream=stream)
        t.cuda.synchronize()
        return offsets, slots

    def feed(self, rng):
        for x in (self.q_in, self.k_in, self.v_in):
            x.copy_(dev(rng.standard_normal(tuple(x.shape)).astype(np.float32)))

    def step(self, stream=0):
        """One token of every sequence that has some; nothing here depends on a length."""
        H.page_plan_device(self.n, WIDTH, PAGE, self.pool, self.p(self.pages), self.p(self.lengths), self.p(self.lengths),
                           self.p(self.free), self.p(self.free_count), d_keep_from=self.p(self.keep), d_missing=self.p(self.missing),
                           stream=stream)
        self._append(self.n, self.q_in, self.k_in, self.v_in, self.q16, stream)
        H.block_bounds_device(self.cache, self.blocks, self.n, stream=stream)
        H.block_select_device(self.cache, self.blocks, HQ, self.p(self.q16), H.HP_ELEM_F16, BUDGET, self.p(self.selected),
                              self.p(self.counts), first_blocks=1, last_blocks=1, stream=stream)
        H.block_attention_device(self.cache, self.blocks, HQ, self.p(self.q16), H.HP_ELEM_F16, self.p(self.out), H.HP_ELEM_F32,
                                 scale=SCALE, d_selected=self.p(self.selected), d_counts=self.p(self.counts), budget=BUDGET, stream=stream)
        if self.type == "f16":
            H.paged_attention_device(self.cache, HQ, self.p(self.q16), H.HP_ELEM_F16, self.p(self.whole), H.HP_ELEM_F32, scale=SCALE, stream=stream)
        else:
            H.block_attention_device(self.cache, self.blocks, HQ, self.p(self.q16), H.HP_ELEM_F16, self.p(self.whole), H.HP_ELEM_F32,
                                     scale=SCALE, stream=stream)

    def state(self):
        got = [x.cpu() for x in (self.pages, self.lengths, self.free, self.free_count, self.missing, self.selected, self.counts, self.out, self.whole)]
        return got + [x.view(_torch().uint8).cpu() for x in (self.keys, self.values, self.bounds)] + [s.cpu() for s in self.scales if s is not None]

    def real(self, which):
        x = (self.keys, self.values)[which].float().cpu().numpy().astype(np.float64)
        s = self.scales[which]
        return x if s is None else x * s.cpu().numpy().astype(np.float64).repeat(BLOCK, 2)[..., None]


def same(a, b):
    t = _torch()
    return all(t.equal(x, y) or (x.is_floating_point() and t.equal(t.isnan(x), t.isnan(y)) and t.equal(x.nan_to_num(), y.nan_to_num()))
               for x, y in zip(a, b))


def check_attention(s, oracle):
    """Both attentions against the 64-bit form over what the pages hold."""
    from oracle import long_context as L

    q = s.q16.float().cpu().numpy().astype(np.float64)
    keys, values = s.real(0), s.real(1)
    lengths, pages = s.lengths.cpu().numpy(), s.pages.cpu().numpy()
    lists = s.selected.cpu().numpy().reshape(s.n * KV, BUDGET)
    bounds = s.bounds.float().cpu().numpy()
    want = L.select(q, bounds, lengths, pages, PAGE, s.pool, BLOCK, BUDGET, 1, 1)
    assert [[b for b in row if b >= 0] for row in lists.tolist()] == want
    for out, chosen in ((s.out, want), (s.whole, None)):
        ref, mass, size, count = L.block_attention(q, keys, values, lengths, pages, PAGE, s.pool, 0, SCALE, chosen, BLOCK)
        # (the bound of the attention's own tests: scores 2^-20 off, weights 2^-21, n + 64 sums of f32)
        bound = mass * (2 * size * (2.0 ** -20 + 66 * 2.0 ** -24) + 2.0 ** -18 + 2 * (count + 64) * 2.0 ** -24)[..., None] * 1.01
        got = out.cpu().numpy()
        assert np.isfinite(got).all()
        assert (np.abs(got - ref) <= bound + count[..., None] * 2.0 ** -26 + 1e-30).all()


@pytest.mark.parametrize("type", ["i8", "e4m3", "f16"])
def test_requests_come_go_on_and_end(hip, oracle, type):
    t = _torch()
    rng = np.random.default_rng(5)
    s = Service(4, type, 1)
    s.prompts([70, 3, 0, 150], [0, 0, 0, 0], rng)
    assert s.lengths.tolist() == [70, 3, 0, 150] and int(s.free_count) == POOL - 3 - 1 - 5
    for _ in range(35):
        s.feed(rng)
        t.cuda.synchronize()
        s.step()
        t.cuda.synchronize()
    assert s.lengths.tolist() == [105, 38, 0, 185] and int(s.free_count) == POOL - 4 - 2 - 6
    check_attention(s, oracle)
    assert not s.out[2].any() and not s.whole[2].any()
    # sequence 0 has its next turn, 1 and 3 end, new requests take 1 and 2
    offsets, slots = s.prompts([40, 64, 33, 0], [0, -1, 0, -1], rng)
    assert s.lengths.tolist() == [145, 64, 33, 0] and offsets.tolist() == [0, 40, 104, 137, 137]
    assert int(s.free_count) == POOL - 5 - 2 - 2 and (slots[:137] >= 0).all() and (slots[137:] == -1).all()
    named = s.pages[s.pages >= 0]
    assert len(named) == len(named.unique()) and not np.intersect1d(named.cpu(), s.free[:int(s.free_count)].cpu()).size
    for _ in range(3):
        s.feed(rng)
        t.cuda.synchronize()
        s.step()
        t.cuda.synchronize()
        check_attention(s, oracle)
    # a window gives the first pages of sequence 0 back
    s.keep.copy_(dev(np.array([70, 0, 0, 0], np.int32)))
    s.feed(rng)
    t.cuda.synchronize()
    s.step()
    t.cuda.synchronize()
    assert s.pages[0, :2].tolist() == [-1, -1] and int(s.free_count) == POOL - 3 - 3 - 2
    check_attention(s, oracle)


@pytest.mark.parametrize("type", ["i8", "e4m3", "f16"])
def test_captured_steps_move_on_by_themselves(hip, type):
    """A captured step replayed over page and block borders, with other work between the replays, leaves what eager steps
    leave, to the bit, every time."""
    t = _torch()
    a, b = Service(5, type, 2), Service(5, type, 2)
    for s in (a, b):
        s.prompts([30, 95, 0, 1, 64], [0] * 5, np.random.default_rng(7))
    stream = t.cuda.Stream()
    feed = np.random.default_rng(8)
    a.feed(np.random.default_rng(9))
    b.feed(np.random.default_rng(9))
    t.cuda.synchronize()
    with t.cuda.stream(stream):
        a.step(stream.cuda_stream)  # sizes the stream's scratch
    b.step()
    t.cuda.synchronize()
    g = t.cuda.CUDAGraph()
    with t.cuda.graph(g, stream=stream):
        a.step(stream.cuda_stream)
    for i in range(40):
        for s in (a, b):
            s.feed(np.random.default_rng(100 + i))
        t.cuda.synchronize()
        g.replay()
        t.cuda.synchronize()
        b.step()
        t.cuda.synchronize()
        junk = t.randn(1 << 20, device="cuda").sum()  # (the program's own work in between)
        del junk
        if i % 8 == 0 or i == 39:
            assert same(a.state(), b.state()), i
    assert a.lengths.tolist() == [71, 136, 0, 42, 105]
    del feed


def test_steps_on_two_streams_at_once(hip):
    """Batches on streams of their own, queued without a wait between them, leave what each leaves alone."""
    t = _torch()
    streams = [t.cuda.Stream() for _ in range(2)]
    both = [Service(7, "i8", 3), Service(7, "f16", 4)]
    alone = [Service(7, "i8", 3), Service(7, "f16", 4)]
    for s in both + alone:
        s.prompts([40, 7, 0, 90, 128, 1, 33], [0] * 7, np.random.default_rng(1))
        s.feed(np.random.default_rng(2))
    t.cuda.synchronize()
    for _ in range(20):
        for s, stream in zip(both, streams):
            s.step(stream.cuda_stream)
    t.cuda.synchronize()
    for s in alone:
        for _ in range(20):
            s.step()
        t.cuda.synchronize()
    for x, y in zip(both, alone):
        assert same(x.state(), y.state())


def test_too_few_pages(hip, oracle):
    """A prompt that finds too few pages: its rows there are dropped, its places left out of the attention, and nothing else
    is touched; when pages come free the same prompt is taken again."""
    t = _torch()
    s = Service(2, "i8", 5, pool=4)
    s.prompts([40, 100], [0, 0], np.random.default_rng(1))
    assert s.missing.tolist() == [0, 2] and int(s.free_count) == 0
    s.feed(np.random.default_rng(2))
    t.cuda.synchronize()
    s.step()
    t.cuda.synchronize()
    check_attention(s, oracle)
    s.lengths.copy_(dev(np.array([41, 0], np.int32)))  # the second request steps back; the first ends
    s.prompts([0, 100], [-1, 0], np.random.default_rng(1))
    assert s.missing.tolist() == [0, 0] and int(s.free_count) == 0 and s.lengths.tolist() == [0, 100]
    s.step()
    t.cuda.synchronize()
    check_attention(s, oracle)


def test_scratch_is_sized_before_a_capture(hip):
    t = _torch()
    s = Service(3, "i8", 6)
    s.prompts([40, 7, 3], [0] * 3, np.random.default_rng(1))
    stream = t.cuda.Stream()
    g = t.cuda.CUDAGraph()
    with t.cuda.stream(stream):
        with pytest.raises(RuntimeError, match="scratch must be sized"):
            g.capture_begin()
            try:
                s.step(stream.cuda_stream)
            finally:
                g.capture_end()

"""The operators over several sequences in use: prompts and next tokens of a batch through projections, cache,
attention, head, rules, top-k and sampler; captured and replayed; on two streams."""
import numpy as np
import pytest

from heliopause_amd import hip_kernels as H
from heliopause_amd import synthetic as S

pytestmark = pytest.mark.gpu

HQ, KV, D, HIDDEN, VOCAB, PAGE, WIDTH = 4, 2, 64, 512, 1000, 16, 12
POOL = 40


def dev(a):
    import torch

    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


class Model:
    """One attention block's projections and a head, on random blocks."""

    def __init__(self):
        self.h = {}
        for name, t, rows, k in (("q", "Q4_K", HQ * D, HIDDEN), ("k", "Q4_K", KV * D, HIDDEN), ("v", "Q6_K", KV * D, HIDDEN),
                                 ("o", "Q4_K", HIDDEN, HQ * D), ("head", "Q6_K", VOCAB, HIDDEN)):
            self.h[name] = H.createHipQuantizedWeightHandle(t, S.weight_blocks(t, S.derive(7, name), rows, k), k, rows)

    def release(self):
        for h in self.h.values():
            H.releaseHipQuantizedWeightHandle(h)


class Batch:
    """Buffers of a batch of `n` sequences with up to `rows` new tokens."""

    def __init__(self, n, rows):
        import torch

        z = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device="cuda")  # noqa: E731
        self.n, self.rows = n, rows
        self.hidden, self.q, self.k, self.v = z(rows, HIDDEN), z(rows, HQ, D), z(rows, KV, D), z(rows, KV, D)
        self.q16, self.k16, self.v16 = (z(rows, h, D, dtype=torch.float16) for h in (HQ, KV, KV))
        self.attn, self.o = z(rows, HQ, D), z(rows, HIDDEN)
        self.logits, self.ruled = z(rows, VOCAB), z(rows, VOCAB)
        self.ids, self.vals = z(rows, 8, dtype=torch.int32), z(rows, 8)
        self.rng, self.tokens, self.kept = z(1, dtype=torch.int32), z(rows, dtype=torch.int32), z(rows, dtype=torch.int32)
        self.probs = z(rows, 8, dtype=torch.float64)
        self.history, self.told = z(rows, 32, dtype=torch.int32), z(rows, dtype=torch.int32)
        self.repetition, self.frequency = z(rows), z(rows)
        self.repetition.fill_(1.3)
        self.frequency.fill_(0.25)
        self.allowed = z(rows, (VOCAB + 31) // 32, dtype=torch.int32)
        self.allowed.fill_(-1)
        self.pages, self.lengths, self.offsets = z(n, WIDTH, dtype=torch.int32), z(n, dtype=torch.int32), z(n + 1, dtype=torch.int32)


def pools():
    import torch

    return [torch.full((POOL, KV, PAGE, D), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2)]


def step(m, b, kv, stream, prompts):
    """One pass of the batch, every launch on `stream`."""
    rows = b.rows
    H.matmul_multi_device([m.h[n].handle for n in "qkv"], b.hidden.data_ptr(), HIDDEN, rows,
                          [b.q.data_ptr(), b.k.data_ptr(), b.v.data_ptr()], [rows * HQ * D, rows * KV * D, rows * KV * D], stream)
    c = H.paged_cache(kv[0].data_ptr(), kv[1].data_ptr(), H.HP_ELEM_F16, page_count=POOL, page_size=PAGE, head_count_kv=KV,
                      head_dim=D, d_pages=b.pages.data_ptr(), d_lengths=b.lengths.data_ptr(), sequence_count=b.n,
                      pages_per_sequence=WIDTH)
    H.paged_append_device(c, rows, HQ, b.q.data_ptr(), b.k.data_ptr(), b.v.data_ptr(), b.q16.data_ptr(), H.HP_ELEM_F16,
                          d_offsets=b.offsets.data_ptr() if prompts else 0, norm_values=True, rope_dims=D,
                          d_k_out=b.k16.data_ptr(), d_v_out=b.v16.data_ptr(), stream=stream)
    if prompts:
        H.packed_attention_device(b.n, b.offsets.data_ptr(), rows, HQ, KV, D, b.q16.data_ptr(), b.k16.data_ptr(), b.v16.data_ptr(),
                                  H.HP_ELEM_F16, b.attn.data_ptr(), H.HP_ELEM_F32, scale=2.0 ** -9, stream=stream)
    else:
        H.paged_attention_device(c, HQ, b.q16.data_ptr(), H.HP_ELEM_F16, b.attn.data_ptr(), H.HP_ELEM_F32, scale=2.0 ** -9, stream=stream)
    H.matmul_multi_device([m.h["o"].handle], b.attn.data_ptr(), HQ * D, rows, [b.o.data_ptr()], [rows * HIDDEN], stream)
    H.matmul_multi_device([m.h["head"].handle], b.o.data_ptr(), HIDDEN, rows, [b.logits.data_ptr()], [rows * VOCAB], stream)
    H.logit_rules_device(rows, VOCAB, b.logits.data_ptr(), b.ruled.data_ptr(), d_history=b.history.data_ptr(), history_stride=32,
                         d_history_lengths=b.told.data_ptr(), d_repetition=b.repetition.data_ptr(),
                         d_frequency=b.frequency.data_ptr(), d_allowed=b.allowed.data_ptr(), stream=stream)
    H.assertHipOk(H.lib().hp_hip_topk_device(b.ruled.data_ptr(), rows, VOCAB, 8, 0.0, b.ids.data_ptr(), b.vals.data_ptr(), stream or None), "topk")
    H.sample_device(b.ids.data_ptr(), b.vals.data_ptr(), rows, 8, 8, {"doSample": False, "topK": 1, "temperature": 1.0, "topP": 1.0},
                    b.rng.data_ptr(), b.tokens.data_ptr(), b.probs.data_ptr(), b.kept.data_ptr(), stream)


def outputs(b):
    return [t.cpu().numpy().copy() for t in (b.q16, b.attn, b.logits, b.ruled, b.ids, b.tokens)]


def table_of(rng, n):
    """Nine pages for each of n sequences."""
    pages = rng.permutation(POOL)[:n * 9].reshape(n, 9).astype(np.int32)
    return dev(np.pad(pages, ((0, 0), (0, WIDTH - 9)), constant_values=-1))


def fill(b, rng):
    b.hidden.copy_(dev(rng.standard_normal((b.rows, HIDDEN)).astype(np.float32)))
    b.history.copy_(dev(rng.integers(0, VOCAB, (b.rows, 32)).astype(np.int32)))
    b.told.copy_(dev(rng.integers(0, 33, b.rows).astype(np.int32)))
    b.allowed.copy_(dev(rng.integers(-2 ** 31, 2 ** 31, tuple(b.allowed.shape)).astype(np.int32)))


@pytest.fixture(scope="module")
def model(hip):
    m = Model()
    yield m
    m.release()


def test_prompts_then_tokens(hip, model):
    """Prompts of 40, 0 and 21 tokens and then one token each: the last token's attention over the pages is the packed
    attention's last row of the prompt with that token behind it, and the token sampled greedily is the best that the
    rules leave."""
    import torch

    from oracle import serving as O

    rng = np.random.default_rng(1)
    lens = [40, 0, 21]
    prompt, kv = Batch(3, 61 + 2), pools()
    table = np.full((3, WIDTH), -1, np.int32)
    free = list(rng.permutation(POOL))
    for s, n in enumerate(lens):
        for i in range((n + 1 + PAGE - 1) // PAGE):
            table[s, i] = free.pop()
    fill(prompt, rng)
    prompt.pages.copy_(dev(table))
    prompt.lengths.copy_(dev(np.array(lens, np.int32)))
    prompt.offsets.copy_(dev(np.array([0, 40, 40, 61], np.int32)))
    step(model, prompt, kv, 0, True)
    nxt = Batch(3, 3)
    fill(nxt, rng)
    nxt.pages.copy_(dev(table))
    nxt.lengths.copy_(dev(np.array([n + 1 for n in lens], np.int32)))
    torch.cuda.synchronize()
    step(model, nxt, kv, 0, False)
    # the prompts with their next tokens behind them, packed
    whole = Batch(3, 64)
    order = [*range(40), None, None, *range(40, 61), None]
    hidden, at = prompt.hidden.cpu().numpy(), 0
    rows = []
    for o in order:
        rows.append(hidden[o] if o is not None else nxt.hidden[at].cpu().numpy())
        at += o is None
    whole.hidden.copy_(dev(np.stack(rows)))
    whole.allowed.fill_(-1)
    other = pools()
    wide = np.full((3, WIDTH), -1, np.int32)
    wide[0, :3], wide[1, :1], wide[2, :2] = [0, 1, 2], [3], [4, 5]
    whole.pages.copy_(dev(wide))
    whole.lengths.copy_(nxt.lengths)
    whole.offsets.copy_(dev(np.array([0, 41, 42, 64], np.int32)))
    torch.cuda.synchronize()
    step(model, whole, other, 0, True)
    torch.cuda.synchronize()
    # (64 columns and 3 columns run different projection kernels, 1e-4 apart, which moves a 16-bit rounding of q, k and v
    # by a step of 2^-11 of the value; scores here stay below 2, so weights move by 2^-9 and outputs by that of the
    # largest value, with a step of the values' own)
    last = [40, 41, 63]
    got, ref = nxt.attn.cpu().numpy(), whole.attn.cpu().numpy()[last]
    assert np.isfinite(got).all()
    assert np.max(np.abs(got - ref)) <= 2.0 ** -8 * np.max(np.abs(whole.v16.float().cpu().numpy()))
    for b in (prompt, nxt):
        logits = b.logits.cpu().numpy()
        ruled = O.logit_rules(logits, b.history.cpu().numpy(), b.told.cpu().numpy(), None, b.repetition.cpu().numpy(),
                              b.frequency.cpu().numpy(), None, allowed=b.allowed.cpu().numpy().view(np.uint32))
        assert np.array_equal(b.ruled.cpu().numpy().view(np.uint32), ruled.view(np.uint32))
        assert np.array_equal(b.tokens.cpu().numpy(), ruled.argmax(1))


def test_captured_step_replays(hip, model):
    """Two captured steps (prompts, next tokens) on one stream share its scratch; each replay, with other inputs, lengths
    and pages and eager work in between, is what an eager call gives."""
    import torch

    stream = torch.cuda.Stream()
    rng = np.random.default_rng(2)
    batches = [Batch(3, 30), Batch(4, 4)]
    kv, graphs = pools(), []

    def fresh(b, prompts, r):
        fill(b, rng)
        b.pages.copy_(table_of(rng, b.n))
        if prompts:
            cut = np.sort(rng.integers(0, 31, 2))
            off = np.array([0, *cut, 28 + r % 3], np.int32)
            off[1:3] = np.minimum(off[1:3], off[3])
            b.offsets.copy_(dev(off))
            b.lengths.copy_(dev(np.diff(off).astype(np.int32)))
        else:
            b.lengths.copy_(dev(rng.integers(0, 9 * PAGE + 1, b.n).astype(np.int32)))
        for p in kv:
            p.copy_(torch.from_numpy(rng.standard_normal(tuple(p.shape)).astype(np.float16)))
        for t in (b.q16, b.k16, b.v16, b.attn):
            t.zero_()
        torch.cuda.synchronize()

    for b, prompts in zip(batches, (True, False)):
        fresh(b, prompts, 0)
        with torch.cuda.stream(stream):
            step(model, b, kv, stream.cuda_stream, prompts)  # sizes the stream's scratch
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            step(model, b, kv, stream.cuda_stream, prompts)
        graphs.append(g)
    for r in range(4):
        for b, prompts, g in zip(batches, (True, False), graphs):
            fresh(b, prompts, r)
            before = [p.clone() for p in kv]
            g.replay()
            torch.cuda.synchronize()
            got, got_kv = outputs(b), [p.clone() for p in kv]
            for p, q in zip(kv, before):
                p.copy_(q)
            for t in (b.q16, b.k16, b.v16, b.attn, b.logits, b.ruled):
                t.zero_()
            torch.cuda.synchronize()
            step(model, b, kv, 0, prompts)
            torch.cuda.synchronize()
            for x, y in zip(got, outputs(b)):
                assert np.array_equal(x, y, equal_nan=x.dtype.kind == "f"), (r, prompts)
            assert all(torch.equal(x, y) for x, y in zip(got_kv, kv))


def test_capture_needs_a_sized_stream(hip):
    """The attention's scratch is not allocated under capture: the call is refused, and the capture goes on."""
    import torch

    stream = torch.cuda.Stream()
    b, kv = Batch(2, 2), pools()
    b.lengths.fill_(20)
    c = H.paged_cache(kv[0].data_ptr(), kv[1].data_ptr(), H.HP_ELEM_F16, page_count=POOL, page_size=PAGE, head_count_kv=KV,
                      head_dim=D, d_pages=b.pages.data_ptr(), d_lengths=b.lengths.data_ptr(), sequence_count=2, pages_per_sequence=WIDTH)
    p = H.HipPagedAttention(b.q.data_ptr(), b.attn.data_ptr(), 0, 0, HQ, 0, 0, 0, 1.0, 0)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        assert H.lib().hp_hip_paged_attention_device(c, p, stream.cuda_stream) == H.HP_ERR_ARG
        assert "before graph capture" in H.last_error()
        H.logit_rules_device(2, VOCAB, b.logits.data_ptr(), b.ruled.data_ptr(), stream=stream.cuda_stream)
    b.logits.fill_(3.0)
    g.replay()
    torch.cuda.synchronize()
    assert bool((b.ruled == 3.0).all())


def test_two_streams(hip, model):
    """Steps of two batches queued on two streams at once are those of one after the other."""
    import torch

    rng = np.random.default_rng(3)
    streams, work = [torch.cuda.Stream() for _ in range(2)], []
    for n in (3, 4):
        b, kv = Batch(n, n), pools()
        fill(b, rng)
        b.pages.copy_(table_of(rng, n))
        b.lengths.copy_(dev(rng.integers(1, 9 * PAGE + 1, n).astype(np.int32)))
        for p in kv:
            p.copy_(torch.from_numpy(rng.standard_normal(tuple(p.shape)).astype(np.float16)))
        torch.cuda.synchronize()
        step(model, b, kv, 0, False)
        torch.cuda.synchronize()
        work.append((b, kv, outputs(b)))
    for _ in range(20):
        for (b, kv, _), s in zip(work, streams):
            step(model, b, kv, s.cuda_stream, False)
    torch.cuda.synchronize()
    for b, _, ref in work:
        for x, y in zip(outputs(b), ref):
            assert np.array_equal(x, y)


def test_calls_are_counted_and_profiled(hip):
    b = Batch(2, 2)
    before = H.hipResidentWeightStats()["kernelLaunches"]
    H.profile(True)
    H.logit_rules_device(2, VOCAB, b.logits.data_ptr(), b.ruled.data_ptr())
    ms, n = H.profile_read(H.HP_KERNEL_SAMPLE)
    H.profile(False)
    assert n == 1 and ms > 0 and H.hipResidentWeightStats()["kernelLaunches"] == before + 1


def test_empty_batches_do_nothing(hip):
    import torch

    b, kv = Batch(2, 2), pools()
    out = torch.full((2, HQ, D), 7.0, device="cuda")
    c = H.paged_cache(kv[0].data_ptr(), kv[1].data_ptr(), H.HP_ELEM_F16, page_count=POOL, page_size=PAGE, head_count_kv=KV,
                      head_dim=D, d_pages=b.pages.data_ptr(), d_lengths=b.lengths.data_ptr(), sequence_count=0, pages_per_sequence=WIDTH)
    H.paged_append_device(c, 0, HQ, b.q.data_ptr(), b.k.data_ptr(), b.v.data_ptr(), out.data_ptr(), 0)
    H.paged_attention_device(c, HQ, b.q.data_ptr(), 0, out.data_ptr(), 0)
    H.packed_attention_device(0, b.offsets.data_ptr(), 2, HQ, KV, D, b.q16.data_ptr(), b.k16.data_ptr(), b.v16.data_ptr(), 1, out.data_ptr(), 0)
    H.packed_attention_device(2, b.offsets.data_ptr(), 0, HQ, KV, D, b.q16.data_ptr(), b.k16.data_ptr(), b.v16.data_ptr(), 1, out.data_ptr(), 0)
    H.logit_rules_device(0, VOCAB, b.logits.data_ptr(), out.data_ptr())
    torch.cuda.synchronize()
    assert bool((out == 7.0).all())

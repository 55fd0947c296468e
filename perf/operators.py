"""What a program that serves several conversations at once has this framework do between the projections, as timed
cases.  Kinds of work:

* ``append``: a batch's new queries, keys and values from the projections: head norms, position rotation, and the
  keys and values into the sequences' pages (one new token a sequence, or whole prompts packed end to end);
* ``decode``: attention of one new token of every sequence over its pages;
* ``prompt``: causal attention over whole prompts packed end to end;
* ``logits``: repetition, frequency and presence penalties, biases and the grammar's mask on the head's logits.

Sizes are those of the model that the benchmark and the tests use (8 query heads over 2 KV heads of 256, vocabulary
262144, contexts of 4096) and generic ones (heads of 64 and 128, longer contexts, batches).  The lengths of a case's
sequences are its own (``ragged``), the values are the seed's.
"""
import math

import numpy as np
import torch

own = False  # True: the framework's kernels; False: the plain forms

EPSILON = 1e-6
FREQ_BASE = 10000.0
ELEM = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}
TYPE_ID = {"f32": 0, "f16": 1, "bf16": 2, "e4m3": 3}  # HP_ELEM_* of include/hp_hip.h
KEY_SCALE, VALUE_SCALE = 0.03125, 0.015625  # of an e4m3 cache: stored = value / scale
E4M3_MOST = 448.0
PAD_ROWS = 3  # rows behind the last sequence of a packed batch, which stay as they were

APPEND = {"heads": 8, "kv_heads": 2, "head_dim": 256, "rope_dims": 256, "factors": False, "norm": True, "page": 16,
          "cache": "f16", "out": "f16", "sequences": 1, "tokens": 0, "context": 4096, "ragged": 1}
DECODE = {"heads": 8, "kv_heads": 2, "head_dim": 256, "page": 16, "cache": "f16", "q": "f32", "sequences": 1,
          "context": 4096, "window": 0, "scale": 0.0625, "ragged": 1}
PROMPT = {"heads": 8, "kv_heads": 2, "head_dim": 256, "type": "f16", "sequences": 1, "tokens": 77, "window": 0,
          "scale": 0.0625, "joined": False, "ragged": 1}
LOGITS = {"rows": 1, "vocab": 262144, "history": 2048, "biases": 16, "mask": True, "ragged": 1}


def listed():
    """Smallest to largest per kind."""
    return [
        # one conversation's next token in the benchmark's model: latency alone
        dict(APPEND, name="append-one", kind="append"),
        # a batch's next tokens, partial rotation with frequency factors, an fp8 cache
        dict(APPEND, name="append-batch", kind="append", heads=32, kv_heads=8, head_dim=128, rope_dims=64,
             factors=True, page=64, cache="e4m3", out="bf16", sequences=201, context=9000),
        # prompts arriving together, their keys and values also handed to the prompt attention
        dict(APPEND, name="append-prompts", kind="append", heads=32, kv_heads=8, head_dim=128, rope_dims=128,
             norm=False, page=32, cache="bf16", out="bf16", sequences=11, tokens=16000, context=4096),
        # one conversation of the benchmark's model, f32 activations as its projections give them
        dict(DECODE, name="decode-one", kind="decode"),
        # a serving batch of ragged contexts, 16-bit activations
        dict(DECODE, name="decode-batch", kind="decode", heads=32, kv_heads=8, head_dim=128, page=64, cache="bf16",
             q="bf16", sequences=48, context=8192, scale=0.125),
        # two very long contexts: few rows, a long axis
        dict(DECODE, name="decode-long", kind="decode", heads=16, kv_heads=4, head_dim=128, page=128, cache="f16",
             q="f32", sequences=2, context=131072, scale=0.125),
        # a large batch on an fp8 cache whose layers slide a window (the pages before it are given back)
        dict(DECODE, name="decode-window", kind="decode", page=32, cache="e4m3", q="f32", sequences=130, context=4096,
             window=1024),
        # a question of a few words
        dict(PROMPT, name="prompt-short", kind="prompt"),
        # ragged prompts of a serving batch, Q/K/V as one projection leaves them
        dict(PROMPT, name="prompt-ragged", kind="prompt", heads=32, kv_heads=8, head_dim=128, type="bf16",
             sequences=15, tokens=12345, scale=0.125, joined=True),
        # a long document
        dict(PROMPT, name="prompt-long", kind="prompt", heads=16, kv_heads=4, head_dim=128, type="bf16", sequences=1,
             tokens=16384, scale=0.125),
        # one conversation's logits under a grammar
        dict(LOGITS, name="logits-one", kind="logits"),
        # a serving batch's logits, an odd vocabulary, long histories
        dict(LOGITS, name="logits-batch", kind="logits", rows=128, vocab=151669, history=6000, biases=300),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "decode", "prompt", "logits"])
    heads, kv_heads, dim = rng.choice([(8, 2, 256), (32, 8, 128), (16, 4, 128), (16, 16, 64), (14, 2, 64), (5, 5, 128),
                                       (16, 1, 128), (4, 1, 256), (40, 8, 128), (10, 5, 256)])
    model = {"heads": heads, "kv_heads": kv_heads, "head_dim": dim}
    ragged = rng.randrange(1, 1 << 20)
    page = rng.choice([16, 32, 64, 128])
    cache = rng.choice(["f16", "bf16", "e4m3"])
    if kind == "append":
        rope = rng.choice([0, dim // 4, dim // 2, dim, dim])
        prompts = rng.random() < 0.5
        tokens = _log(rng, 30, 9000) if prompts else 0
        return dict(APPEND, kind=kind, **model, rope_dims=rope, factors=rope > 0 and rng.random() < 0.5,
                    norm=rng.random() < 0.5, page=page, cache=cache, out=rng.choice(["f32", "f16", "bf16"]),
                    sequences=rng.randrange(1, 17) if prompts else _log(rng, 1, 300), tokens=tokens,
                    context=_log(rng, 40, 9000), ragged=ragged)
    if kind == "decode":
        context = _log(rng, 16, 100000)
        most = max(1, min(300, int(3.0e8 / (context * kv_heads * dim))))
        window = _log(rng, 8, context) if rng.random() < 0.3 else 0
        return dict(DECODE, kind=kind, **model, page=page, cache=cache, q=rng.choice(["f32", "f16", "bf16"]),
                    sequences=_log(rng, 1, most), context=context, window=window, scale=dim ** -0.5, ragged=ragged)
    if kind == "prompt":
        tokens = _log(rng, 20, 12000)
        return dict(PROMPT, kind=kind, **model, type=rng.choice(["f16", "bf16"]),
                    sequences=rng.randrange(max(1, tokens * tokens * heads // (1 << 31)), 24), tokens=tokens,
                    window=_log(rng, 8, tokens) if rng.random() < 0.25 else 0, scale=dim ** -0.5,
                    joined=rng.random() < 0.5, ragged=ragged)
    vocab = rng.choice([262144, 32000, 128256, 50257, 100003, 151669])
    return dict(LOGITS, kind=kind, rows=_log(rng, 1, 70), vocab=vocab, history=_log(rng, 1, 8000),
                biases=rng.choice([0, 1, 30, 300]), mask=rng.random() < 0.6, ragged=ragged)


# ---- lengths ------------------------------------------------------------------------------------------------------
def _shares(case):
    """How the prompts of a packed batch share its tokens: lengths within a factor of about seven of one another, one
    of them empty where there are many."""
    n, total = case["sequences"], case["tokens"]
    r = np.random.RandomState(case["ragged"])
    weight = r.uniform(0.25, 1.75, n)
    if n > 6:
        weight[n // 2] = 0.0
    cut = np.floor(np.cumsum(weight) / weight.sum() * total + 0.5).astype(np.int64)
    cut[-1] = total
    return np.diff(np.concatenate([[0], cut]))


def _contexts(case):
    """Tokens that each sequence has in its pages, the new one among them: from one to the longest; in a batch the
    last rows are padding (length 0)."""
    n = case["sequences"]
    r = np.random.RandomState(case["ragged"])
    length = np.maximum(1, np.floor(np.exp(r.uniform(math.log(max(1.0, case["context"] / 8)), math.log(case["context"] + 0.5), n)))).astype(np.int64)
    length[0] = case["context"]
    if n > 4:
        length[1], length[-1] = 1, 0
    return length


def _append_lengths(case):
    """(new tokens, tokens in the pages afterwards) of each sequence."""
    if not case["tokens"]:
        length = _contexts(case)
        return np.minimum(length, 1), length
    new = _shares(case)
    r = np.random.RandomState(case["ragged"] + 1)
    past = np.where(r.uniform(size=len(new)) < 0.5, 0, r.randint(0, case["context"], len(new)))  # half go on from a turn before
    return new, new + past


# ---- inputs -------------------------------------------------------------------------------------------------------
class _State:
    pass


def _generator(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + case["ragged"])
    return g


def _normal(g, shape, dtype=torch.float32, times=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * times).to(dtype)


def _ints(values):
    return torch.from_numpy(np.asarray(values, np.int32)).cuda()


def _pages(s, case, length, g):
    """A pool of pages a little larger than the sequences need, dealt out in no order; the table's entries past a
    sequence's last page, and the pages that a sliding window has passed, name no page (-1)."""
    page = case["page"]
    need = -(-length // page)
    width = max(1, int(need.max())) + 1
    pool = int(need.sum()) + 3
    order = torch.randperm(pool, generator=g, device="cuda").cpu().numpy()
    table = np.full((len(length), width), -1, np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += int(n)
        if case.get("window"):
            table[i, :max(0, int(length[i]) - case["window"]) // page] = -1
    s.table, s.lengths, s.pool = _ints(table), _ints(length), pool


def _cache(g, s, case, times):
    shape = (s.pool, case["kv_heads"], case["page"], case["head_dim"])
    if case["cache"] == "e4m3":
        return (torch.randn(shape, generator=g, device="cuda") * times).clamp(-E4M3_MOST, E4M3_MOST).to(ELEM["e4m3"])
    return _normal(g, shape, ELEM[case["cache"]])


def prepare(case, seed):
    s, g = _State(), _generator(case, seed)
    s.case = case
    {"append": _prepare_append, "decode": _prepare_decode, "prompt": _prepare_prompt, "logits": _prepare_logits}[case["kind"]](s, case, g)
    torch.cuda.current_stream().synchronize()
    return s


def _prepare_append(s, case, g):
    heads, kv, dim = case["heads"], case["kv_heads"], case["head_dim"]
    new, length = _append_lengths(case)
    _pages(s, case, length, g)
    s.packed = case["tokens"] > 0
    s.rows = case["tokens"] + PAD_ROWS if s.packed else case["sequences"]
    s.offsets = _ints(np.concatenate([[0], np.cumsum(new)])) if s.packed else None
    s.q, s.k, s.v = (_normal(g, (s.rows, n, dim), times=2.0) for n in (heads, kv, kv))
    s.q_norm, s.k_norm = ((1.0 + 0.1 * _normal(g, (dim,)) for _ in range(2)) if case["norm"] else (None, None))
    s.factors = torch.exp(torch.rand(case["rope_dims"] // 2, generator=g, device="cuda") * 2.0) if case["factors"] else None
    s.keys, s.values = _cache(g, s, case, 30.0), _cache(g, s, case, 60.0)
    out = ELEM[case["out"]]
    s.q_out = torch.zeros((s.rows, heads, dim), dtype=out, device="cuda")
    s.k_out, s.v_out = ((torch.zeros((s.rows, kv, dim), dtype=out, device="cuda") for _ in range(2)) if s.packed else (None, None))


def _prepare_decode(s, case, g):
    _pages(s, case, _contexts(case), g)
    s.q = _normal(g, (case["sequences"], case["heads"], case["head_dim"]), ELEM[case["q"]], 2.0)
    s.keys, s.values = _cache(g, s, case, 1.0 / KEY_SCALE), _cache(g, s, case, 1.0 / VALUE_SCALE)
    s.out = torch.zeros_like(s.q)


def _prepare_prompt(s, case, g):
    heads, kv, dim, dtype = case["heads"], case["kv_heads"], case["head_dim"], ELEM[case["type"]]
    rows = case["tokens"] + PAD_ROWS
    s.offsets = _ints(np.concatenate([[0], np.cumsum(_shares(case))]))
    if case["joined"]:  # one projection's rows: queries, keys, values side by side
        s.q, s.k, s.v = _normal(g, (rows, heads + 2 * kv, dim), dtype, 1.5).split([heads, kv, kv], dim=1)
    else:
        s.q, s.k, s.v = (_normal(g, (rows, n, dim), dtype, 1.5) for n in (heads, kv, kv))
    s.longest = int(_shares(case).max())
    s.out = torch.zeros((rows, heads, dim), dtype=dtype, device="cuda")


def _prepare_logits(s, case, g):
    rows, n = case["rows"], case["vocab"]
    r = np.random.RandomState(case["ragged"])
    s.logits = _normal(g, (rows, n), times=4.0)
    seen = np.minimum(case["history"], np.floor(np.exp(r.uniform(0, math.log(case["history"] + 1.0), rows)))).astype(np.int64)
    seen[0] = case["history"]
    if rows > 2:
        seen[1] = 0
    s.seen, s.prompt = _ints(seen), _ints(seen // 3)
    # a text's tokens: a few come often, most once
    u = torch.rand((rows, case["history"]), generator=g, device="cuda")
    s.history = (n * u ** 4).to(torch.int32).clamp_(0, n - 1)
    s.repetition = 1.0 + 0.3 * torch.rand(rows, generator=g, device="cuda")
    s.frequency = 0.5 * torch.rand(rows, generator=g, device="cuda")
    s.presence = 0.5 * torch.rand(rows, generator=g, device="cuda")
    s.bias_ids = s.bias_values = s.bias_counts = None
    if case["biases"]:
        s.bias_ids = (n * torch.rand((rows, case["biases"]), generator=g, device="cuda", dtype=torch.float64)).to(torch.int32)
        s.bias_values = _normal(g, (rows, case["biases"]), times=3.0)
        s.bias_counts = _ints(r.randint(0, case["biases"] + 1, rows))
    s.allowed = None
    if case["mask"]:  # a grammar leaves few tokens in most states and nearly all in others; one row here is left none
        share = torch.from_numpy(np.where(r.uniform(size=rows) < 0.5, 1e-3, 0.97)).cuda()
        bits = torch.rand((rows, (n + 31) // 32, 32), generator=g, device="cuda") < share[:, None, None]
        if rows > 3:
            bits[2] = False
        s.allowed = (bits.to(torch.int64) << torch.arange(32, device="cuda")).sum(-1).to(torch.int32)
    s.out = torch.zeros_like(s.logits)


# ---- the framework's calls ------------------------------------------------------------------------------------------
_stream = None


def _the_stream():
    """The stream that a pass is queued on: the current one, so that what comes before and after it in the program keeps
    its order.  Torch's default stream has no handle that the framework's calls take (0 is the framework's own), so a
    program on that one moves to a stream of its own, behind what it has queued."""
    global _stream
    current = torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())  # (current_stream() takes 3 us of a call of 7)
    if current == 0:
        if _stream is None:
            _stream = torch.cuda.Stream()
        _stream.wait_stream(torch.cuda.current_stream())
        torch.cuda.set_stream(_stream)
        current = _stream.cuda_stream
    return current


def _p(t):
    return 0 if t is None else t.data_ptr()


def _paged_cache(H, s, case):
    c = H.paged_cache(_p(s.keys), _p(s.values), TYPE_ID[case["cache"]], page_count=s.pool, page_size=case["page"],
                      head_count_kv=case["kv_heads"], head_dim=case["head_dim"], d_pages=_p(s.table),
                      d_lengths=_p(s.lengths), sequence_count=case["sequences"], pages_per_sequence=s.table.shape[1])
    if case["cache"] == "e4m3":
        c.key_scale, c.value_scale = KEY_SCALE, VALUE_SCALE
    return c


def _own(s, case):
    from heliopause_amd import hip_kernels as H

    q = _the_stream()
    if case["kind"] == "append":
        H.paged_append_device(_paged_cache(H, s, case), s.rows, case["heads"], _p(s.q), _p(s.k), _p(s.v), _p(s.q_out),
                              TYPE_ID[case["out"]], d_offsets=_p(s.offsets), d_q_norm=_p(s.q_norm),
                              d_k_norm=_p(s.k_norm), norm_values=case["norm"], epsilon=EPSILON,
                              rope_dims=case["rope_dims"], rope_freq_base=FREQ_BASE, d_rope_freq_factors=_p(s.factors),
                              d_k_out=_p(s.k_out), d_v_out=_p(s.v_out), stream=q)
        return _append_outputs(s)
    if case["kind"] == "decode":
        H.paged_attention_device(_paged_cache(H, s, case), case["heads"], _p(s.q), TYPE_ID[case["q"]], _p(s.out),
                                 TYPE_ID[case["q"]], scale=case["scale"], sliding_window=case["window"], stream=q)
        return s.out
    if case["kind"] == "prompt":
        t = TYPE_ID[case["type"]]
        H.packed_attention_device(case["sequences"], _p(s.offsets), s.q.shape[0], case["heads"], case["kv_heads"],
                                  case["head_dim"], _p(s.q), _p(s.k), _p(s.v), t, _p(s.out), t, scale=case["scale"],
                                  sliding_window=case["window"], q_stride=s.q.stride(0), k_stride=s.k.stride(0),
                                  v_stride=s.v.stride(0), stream=q)
        return s.out
    H.logit_rules_device(case["rows"], case["vocab"], _p(s.logits), _p(s.out), d_history=_p(s.history),
                         history_stride=case["history"], d_history_lengths=_p(s.seen), d_prompt_lengths=_p(s.prompt),
                         d_repetition=_p(s.repetition), d_frequency=_p(s.frequency), d_presence=_p(s.presence),
                         d_bias_ids=_p(s.bias_ids), d_bias_values=_p(s.bias_values), d_bias_counts=_p(s.bias_counts),
                         bias_stride=case["biases"], d_allowed=_p(s.allowed),
                         allowed_stride=0 if s.allowed is None else s.allowed.shape[1], stream=q)
    return s.out


# ---- the plain forms ------------------------------------------------------------------------------------------------
def _append_outputs(s):
    return {name: t for name, t in (("q", s.q_out), ("k", s.k_out), ("v", s.v_out), ("keys", s.keys), ("values", s.values)) if t is not None}


def _rms(x, weight):
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPSILON)
    return y if weight is None else y * weight


def _rotate(x, cos, sin, dims):
    """Pairs (u, u + dims / 2) of each head by the token's angles; the rest as it is."""
    half = dims // 2
    a, b = x[..., :half], x[..., half:dims]
    return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., dims:]], -1)


def _stored(x, case, scale):
    if case["cache"] == "e4m3":
        return (x / scale).clamp(-E4M3_MOST, E4M3_MOST).to(ELEM["e4m3"])
    return x.to(ELEM[case["cache"]])


def _plain_append(s, case):
    row = torch.arange(s.rows, device="cuda")
    if s.packed:
        seq = torch.searchsorted(s.offsets[1:].contiguous(), row, right=True)
        live = seq < case["sequences"]
        seq = seq.clamp(max=case["sequences"] - 1)
        position = s.lengths[seq] - s.offsets[seq + 1] + row
    else:
        seq, position = row, s.lengths - 1
        live = position >= 0
    row, seq, position = row[live], seq[live], position[live].long()
    q, k, v = s.q[row], s.k[row], s.v[row]
    if case["norm"]:
        q, k, v = _rms(q, s.q_norm), _rms(k, s.k_norm), _rms(v, None)
    if case["rope_dims"]:
        half = case["rope_dims"] // 2
        frequency = FREQ_BASE ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
        if s.factors is not None:
            frequency = frequency / s.factors.double()
        angle = position.double()[:, None, None] * frequency
        cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
        q, k = _rotate(q, cos, sin, case["rope_dims"]), _rotate(k, cos, sin, case["rope_dims"])
    page = s.table[seq, position // case["page"]].long()
    slot = position % case["page"]
    for pool, x, scale in ((s.keys, k, KEY_SCALE), (s.values, v, VALUE_SCALE)):
        bits = torch.uint8 if case["cache"] == "e4m3" else torch.int16
        pool.view(bits)[page, :, slot] = _stored(x, case, scale).view(bits)
    s.q_out[row] = q.to(s.q_out.dtype)
    if s.packed:
        s.k_out[row] = k.to(s.k_out.dtype)
        s.v_out[row] = v.to(s.v_out.dtype)
    return _append_outputs(s)


def _softmax(scores, mask):
    """Over the last axis, 0 where the mask is false; a row without any is all 0."""
    scores = scores.masked_fill_(~mask, -math.inf)
    most = scores.amax(-1, keepdim=True)
    p = scores.sub_(torch.where(most == -math.inf, torch.zeros_like(most), most)).exp_()
    total = p.sum(-1, keepdim=True)
    return p.div_(torch.where(total == 0, torch.ones_like(total), total))


def _gathered(pool, s, case, scale):
    """The sequences' rows of a pool in order, [sequence][kv head][position][dim], in 32 bits."""
    pages = s.table.clamp(min=0).long()
    bits = torch.uint8 if case["cache"] == "e4m3" else torch.int16
    x = pool.view(bits)[pages].view(pool.dtype).float()  # [sequence][page][head][slot][dim]
    if case["cache"] == "e4m3":
        x = x * scale
    return x.permute(0, 2, 1, 3, 4).reshape(case["sequences"], case["kv_heads"], -1, case["head_dim"])


def _plain_decode(s, case):
    n, kv, dim = case["sequences"], case["kv_heads"], case["head_dim"]
    k, v = _gathered(s.keys, s, case, KEY_SCALE), _gathered(s.values, s, case, VALUE_SCALE)
    q = s.q.float().reshape(n, kv, case["heads"] // kv, dim)
    scores = torch.matmul(q, k.transpose(-1, -2)) * case["scale"]
    at = torch.arange(k.shape[2], device="cuda")
    seen = at < s.lengths[:, None]
    if case["window"]:
        seen &= at >= s.lengths[:, None] - case["window"]
    out = torch.matmul(_softmax(scores, seen[:, None, None]), v)
    return out.reshape(n, case["heads"], dim).to(s.out.dtype)


def _plain_prompt(s, case):
    heads, kv, dim, longest = case["heads"], case["kv_heads"], case["head_dim"], s.longest
    at = torch.arange(longest, device="cuda")
    length = (s.offsets[1:] - s.offsets[:-1])[:, None]
    there = at < length
    row = (s.offsets[:-1, None] + at).clamp(max=case["tokens"] - 1).long()
    q = s.q[row].float().reshape(-1, longest, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(-1, kv, heads // kv * longest, dim)
    k, v = (t[row].float().permute(0, 2, 1, 3).contiguous() for t in (s.k, s.v))
    scores = torch.matmul(q, k.transpose(-1, -2)).mul_(case["scale"])
    seen = (at <= at[:, None]) & there[:, None, :]
    if case["window"]:
        seen &= at > at[:, None] - case["window"]
    p = _softmax(scores.view(-1, kv, heads // kv, longest, longest), seen[:, None, None])
    out = torch.matmul(p.view(-1, kv, heads // kv * longest, longest), v)
    out = out.view(-1, kv, heads // kv, longest, dim).permute(0, 3, 1, 2, 4).reshape(-1, longest, heads, dim)
    s.out[row[there]] = out[there].to(s.out.dtype)
    return s.out


def _counts(ids, valid, n):
    """How often each of the n tokens is among the valid ids of its row."""
    count = torch.zeros((ids.shape[0], n), device="cuda")
    return count.scatter_add_(1, ids.clamp(0, n - 1).long(), valid.float())


def _plain_logits(s, case):
    n = case["vocab"]
    at = torch.arange(case["history"], device="cuda")
    told = at < s.seen[:, None]
    seen = _counts(s.history, told, n) > 0
    count = _counts(s.history, told & (at >= s.prompt[:, None]), n)
    x = s.logits
    r = s.repetition[:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - s.frequency[:, None] * count
    x = x - torch.where(count > 0, s.presence[:, None], torch.zeros_like(x[:, :1]))
    if s.bias_ids is not None:  # the last entry of a token counts
        at = torch.arange(case["biases"], device="cuda")
        which = torch.zeros((case["rows"], n), dtype=torch.int64, device="cuda")
        which.scatter_reduce_(1, s.bias_ids.long(), torch.where(at < s.bias_counts[:, None], at + 1, torch.zeros_like(at)), "amax")
        bias = torch.cat([torch.zeros_like(s.bias_values[:, :1]), s.bias_values], 1).gather(1, which)
        x = torch.where(which > 0, x + bias, x)
    if s.allowed is not None:
        at = torch.arange(n, device="cuda")
        x = x.masked_fill((s.allowed[:, at // 32] >> (at % 32).to(torch.int32)) & 1 == 0, -math.inf)
    return x


def run(s):
    case = s.case
    if own:
        return _own(s, case)
    return {"append": _plain_append, "decode": _plain_decode, "prompt": _plain_prompt, "logits": _plain_logits}[case["kind"]](s, case)


# ---- the definition in 64 bits --------------------------------------------------------------------------------------
def _wide(t):
    return None if t is None else t.detach().double()


def _exact_attention(q, k, v, first, last, scale):
    """Row i of q ([rows][heads][dim], with k and v [keys][kv heads][dim]) over its keys first[i] .. last[i]."""
    out = torch.zeros_like(q)
    group = q.shape[1] // k.shape[1]
    at = torch.arange(k.shape[0], device=q.device)
    masked = (at < first[:, None]) | (at > last[:, None])
    for h in range(q.shape[1]):
        e = q[:, h] @ k[:, h // group].T * scale
        e[masked] = -math.inf
        e = torch.exp(e - e.max(1, keepdim=True).values.clamp(min=-1e300))
        out[:, h] = e @ v[:, h // group] / e.sum(1, keepdim=True).clamp(min=1e-300)
    return out


def _exact_row(x, weight, position, case, factors):
    """One tensor's rows [token][head][dim]: norm (weight: a vector, True for none, None for no norm), rotation (position
    None: none)."""
    if weight is not None:
        x = x / torch.sqrt(torch.sum(x ** 2, -1, keepdim=True) / x.shape[-1] + EPSILON)
        if weight is not True:
            x = x * weight
    dims = case["rope_dims"]
    if position is not None and dims:
        x = x.clone()
        for u in range(dims // 2):
            turn = position * math.pow(FREQ_BASE, -2.0 * u / dims)
            if factors is not None:
                turn = turn / factors[u]
            z = torch.complex(x[..., u], x[..., u + dims // 2]) * torch.polar(torch.ones_like(turn), turn)[:, None]
            x[..., u], x[..., u + dims // 2] = z.real, z.imag
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        new, length = _append_lengths(case)
        rows, seqs, positions = [], [], []
        for i, (n, total) in enumerate(zip(new, length)):
            start = int(new[:i].sum()) if s.packed else i
            rows += range(start, start + int(n))
            seqs += [i] * int(n)
            positions += range(int(total - n), int(total))
        rows, position = torch.tensor(rows, device="cuda"), torch.tensor(positions, device="cuda", dtype=torch.float64)
        norm = case["norm"]
        q = _exact_row(_wide(s.q)[rows], _wide(s.q_norm) if norm else None, position, case, _wide(s.factors))
        k = _exact_row(_wide(s.k)[rows], _wide(s.k_norm) if norm else None, position, case, _wide(s.factors))
        v = _exact_row(_wide(s.v)[rows], True if norm else None, None, case, None)
        table = s.table.cpu().numpy()
        where = torch.tensor([int(table[i, p // case["page"]]) for i, p in zip(seqs, positions)], device="cuda")
        slot = torch.tensor([p % case["page"] for p in positions], device="cuda")
        got = {}
        for name, x, buffer in (("q", q, s.q_out), ("k", k, s.k_out), ("v", v, s.v_out)):
            if buffer is not None:
                got[name] = _wide(buffer)
                got[name][rows] = x
        for name, x, pool, scale in (("keys", k, s.keys, KEY_SCALE), ("values", v, s.values, VALUE_SCALE)):
            got[name] = pool.double()
            got[name][where, :, slot] = (x / scale).clamp(-E4M3_MOST, E4M3_MOST) if case["cache"] == "e4m3" else x
        return got
    if case["kind"] == "decode":
        out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
        length, table = s.lengths.tolist(), s.table.long()
        for i, n in enumerate(length):
            if not n:
                continue
            start = max(0, n - case["window"]) if case["window"] else 0
            at = torch.arange(start, n, device="cuda")
            page, slot = table[i, at // case["page"]], at % case["page"]
            k, v = (p.view(torch.uint8 if p.dtype == ELEM["e4m3"] else torch.int16)[page, :, slot].view(p.dtype).double() for p in (s.keys, s.values))
            if case["cache"] == "e4m3":
                k, v = k * KEY_SCALE, v * VALUE_SCALE
            last = torch.full((1,), len(at), device="cuda")
            out[i:i + 1] = _exact_attention(_wide(s.q[i:i + 1]), k, v, torch.zeros_like(last), last, case["scale"])
        return out
    if case["kind"] == "prompt":
        out = _wide(s.out)
        cut = s.offsets.tolist()
        for a, b in zip(cut, cut[1:]):
            if a == b:
                continue
            last = torch.arange(b - a, device="cuda")
            first = last - case["window"] + 1 if case["window"] else torch.zeros_like(last)
            out[a:b] = _exact_attention(*(_wide(t[a:b]) for t in (s.q, s.k, s.v)), first, last, case["scale"])
        return out
    out = _wide(s.logits)
    n = case["vocab"]
    for i in range(case["rows"]):
        told = s.history[i, :int(s.seen[i])].long()
        row, r = out[i], float(s.repetition[i])
        seen = torch.unique(told)
        row[seen] = torch.where(row[seen] > 0, row[seen] / r, row[seen] * r)
        count = torch.bincount(told[int(s.prompt[i]):], minlength=n).double()
        row -= float(s.frequency[i]) * count + float(s.presence[i]) * (count > 0)
        if s.bias_ids is not None:
            c = int(s.bias_counts[i])
            last = dict(zip(s.bias_ids[i, :c].tolist(), s.bias_values[i, :c].double().tolist()))
            if last:
                row[torch.tensor(list(last), device="cuda")] += torch.tensor(list(last.values()), dtype=torch.float64, device="cuda")
        if s.allowed is not None:
            words = s.allowed[i].cpu().numpy().view(np.uint8)
            row[torch.from_numpy(np.unpackbits(words, bitorder="little")[:n] == 0).cuda()] = -math.inf
    return out


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "logits":
        rows, n = case["rows"], case["vocab"]
        r = 8.0 * n + (n / 8.0 if case["mask"] else 0.0) + 2.0 * case["history"] + 4.0 * case["biases"]
        return {"bytes": rows * r, "flops": 4.0 * rows * n}
    heads, kv, dim = case["heads"], case["kv_heads"], case["head_dim"]
    if kind == "append":
        new = int(_append_lengths(case)[0].sum())
        out = BYTES[case["out"]] * (heads + (2 * kv if case["tokens"] else 0)) + 2 * BYTES[case["cache"]] * kv
        return {"bytes": new * dim * (4.0 * (heads + 2 * kv) + out), "flops": new * dim * (heads + 2 * kv) * 8.0}
    if kind == "decode":
        length = _contexts(case)
        keys = float((np.minimum(length, case["window"]) if case["window"] else length).sum())
        return {"bytes": 2.0 * keys * kv * dim * BYTES[case["cache"]] + 2.0 * case["sequences"] * heads * dim * BYTES[case["q"]],
                "flops": 4.0 * keys * heads * dim}
    length = _shares(case).astype(np.float64)
    w = np.minimum(length, case["window"]) if case["window"] else length
    pairs = float((w * (w + 1) / 2 + (length - w) * w).sum())
    return {"bytes": case["tokens"] * dim * 2.0 * (2 * heads + 2 * kv), "flops": 4.0 * pairs * heads * dim}

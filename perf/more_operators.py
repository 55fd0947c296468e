"""What a program that serves long conversations from 8-bit pages, or attends to a part of them only, has this framework do
around the paged cache, as timed cases.  Kinds of work:

* ``plan``: the step's page tables, lengths, row offsets and slot maps from the requests' lengths, on the device: pages
  that are no longer needed go back, new ones are dealt;
* ``append``: a batch's new queries, keys and values from the projections into pages of 8 bits with a scale for each block
  of positions and KV head (one new token a sequence, or prompts packed end to end);
* ``decode``: attention of one new token of every sequence over such pages;
* ``bounds``: the least and largest key elements of the blocks that new tokens lie in;
* ``sparse``: a token's attention over the blocks that these bounds select for its queries: the new token's block
  refreshed, the selection, the attention.

Sizes are those of the model that the benchmark and the tests use (8 query heads over 2 KV heads of 256, contexts of 4096)
and generic ones (heads of 64 and 128, longer contexts, batches).  The lengths of a case's sequences are its own
(``ragged``), the values are the seed's.
"""
import math

import numpy as np
import torch

own = False  # True: the framework's kernels; False: the plain forms

EPSILON = 1e-6
FREQ_BASE = 10000.0
ELEM = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "i8": torch.int8}
BYTES = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1, "i8": 1}
TYPE_ID = {"f32": 0, "f16": 1, "bf16": 2, "e4m3": 3, "i8": 4}  # HP_ELEM_* of include/hp_hip.h
MOST = {"e4m3": 448.0, "i8": 127.0}  # the largest stored value
SCALE_LOW, SCALE_HIGH = 2.0 ** -100, 2.0 ** 100
GROWTH = 1.25  # least growth of an i8 block's scale
BF16_MOST = float(torch.finfo(torch.bfloat16).max)
PAD_ROWS = 3  # rows behind the last sequence of a packed batch

PLAN = {"page": 64, "sequences": 201, "tokens": 0, "context": 9000, "window": 0, "short": 0, "ragged": 1}
APPEND = {"heads": 8, "kv_heads": 2, "head_dim": 256, "rope_dims": 256, "factors": False, "norm": True, "page": 16,
          "block": 16, "cache": "e4m3", "out": "f16", "sequences": 1, "tokens": 0, "context": 4096, "ragged": 1}
DECODE = {"heads": 8, "kv_heads": 2, "head_dim": 256, "page": 16, "block": 16, "cache": "i8", "q": "f32", "sequences": 1,
          "context": 4096, "window": 0, "scale": 0.0625, "ragged": 1}
BOUNDS = {"kv_heads": 2, "head_dim": 256, "page": 64, "block": 64, "cache": "f16", "sequences": 1, "tokens": 0,
          "context": 4096, "ragged": 1}
SPARSE = {"heads": 8, "kv_heads": 2, "head_dim": 256, "page": 64, "block": 64, "cache": "f16", "q": "f32",
          "sequences": 1, "tokens": 0, "context": 32768, "budget": 32, "first": 1, "last": 2, "scale": 0.0625, "ragged": 1}


def listed():
    """Smallest to largest per kind."""
    return [
        # the next tokens of a serving batch whose layers slide a window: the pages before it go back
        dict(PLAN, name="plan-step", kind="plan", window=4096),
        # an offline batch: new requests in the place of finished ones, next turns of others
        dict(PLAN, name="plan-prompts", kind="plan", page=16, sequences=256, tokens=700001, context=4000),
        # one conversation's next token in the benchmark's model: latency alone
        dict(APPEND, name="append-one", kind="append"),
        # a batch's next tokens, from projections that leave them normed and rotated, into i8 blocks of 64
        dict(APPEND, name="append-batch", kind="append", heads=32, kv_heads=8, head_dim=128, rope_dims=0, norm=False,
             page=64, block=64, cache="i8", out="bf16", sequences=201, context=9000),
        # prompts arriving together, their keys and values also handed to the prompt attention
        dict(APPEND, name="append-prompts", kind="append", heads=32, kv_heads=8, head_dim=128, rope_dims=128, page=32,
             block=32, out="bf16", sequences=11, tokens=16000, context=4096),
        # one conversation of the benchmark's model, f32 activations as its projections give them
        dict(DECODE, name="decode-one", kind="decode"),
        # a serving batch of ragged contexts, 16-bit activations
        dict(DECODE, name="decode-batch", kind="decode", heads=32, kv_heads=8, head_dim=128, page=64, block=64, q="bf16",
             sequences=48, context=8192, scale=0.125),
        # the prompts of a batch, behind their append
        dict(BOUNDS, name="bounds-prompts", kind="bounds", kv_heads=8, head_dim=128, cache="bf16", sequences=11,
             tokens=16000),
        # a long document in the benchmark's model, fp8 pages with scales
        dict(BOUNDS, name="bounds-long", kind="bounds", page=128, block=32, cache="e4m3", tokens=100000, context=200),
        # one conversation of the benchmark's model, an eighth of its context
        dict(SPARSE, name="sparse-one", kind="sparse", budget=64),
        # a serving batch of ragged long contexts, 64 blocks of each
        dict(SPARSE, name="sparse-batch", kind="sparse", heads=32, kv_heads=8, head_dim=128, cache="bf16", q="bf16",
             sequences=24, budget=64, scale=0.125),
        # two very long contexts in i8 pages, small blocks
        dict(SPARSE, name="sparse-long", kind="sparse", heads=16, kv_heads=4, head_dim=128, page=128, block=32,
             cache="i8", sequences=2, context=262144, budget=256, scale=0.125),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "append", "decode", "bounds", "sparse"])
    heads, kv_heads, dim = rng.choice([(8, 2, 256), (32, 8, 128), (16, 4, 128), (16, 16, 64), (14, 2, 64), (5, 5, 128),
                                       (16, 1, 128), (4, 1, 256), (40, 8, 128), (10, 5, 256)])
    model = {"heads": heads, "kv_heads": kv_heads, "head_dim": dim}
    ragged = rng.randrange(1, 1 << 20)
    page = rng.choice([16, 32, 64, 128])
    block = rng.choice([b for b in (16, 32, 64, 128) if b <= page])
    if kind == "plan":
        tokens = _log(rng, 50, 500000) if rng.random() < 0.6 else 0
        return dict(PLAN, kind=kind, page=page, sequences=_log(rng, 1, 400), tokens=tokens, context=_log(rng, 40, 20000),
                    window=_log(rng, 16, 5000) if not tokens and rng.random() < 0.5 else 0,
                    short=_log(rng, 1, 40) if rng.random() < 0.3 else 0, ragged=ragged)
    if kind == "append":
        cache = rng.choice(["i8", "e4m3", "e4m3"])
        # (an i8 element next to a border is another whole number after the last bit of a norm or a rotation: i8 rows
        # come normed and rotated here)
        rope = 0 if cache == "i8" else rng.choice([0, dim // 4, dim // 2, dim, dim])
        prompts = rng.random() < 0.5
        tokens = _log(rng, 30, 9000) if prompts else 0
        return dict(APPEND, kind=kind, **model, rope_dims=rope, factors=rope > 0 and rng.random() < 0.5,
                    norm=cache != "i8" and rng.random() < 0.5, page=page, block=block, cache=cache,
                    out=rng.choice(["f32", "f16", "bf16"]),
                    sequences=rng.randrange(1, 17) if prompts else _log(rng, 1, 300), tokens=tokens,
                    context=_log(rng, 40, 9000), ragged=ragged)
    if kind == "decode":
        context = _log(rng, 16, 100000)
        most = max(1, min(300, int(3.0e8 / (context * kv_heads * dim))))
        window = _log(rng, 8, context) if rng.random() < 0.3 else 0
        return dict(DECODE, kind=kind, **model, page=page, block=block, cache=rng.choice(["i8", "e4m3"]),
                    q=rng.choice(["f32", "f16", "bf16"]), sequences=_log(rng, 1, most), context=context, window=window,
                    scale=dim ** -0.5, ragged=ragged)
    if kind == "bounds":
        prompts = rng.random() < 0.6
        return dict(BOUNDS, kind=kind, kv_heads=kv_heads, head_dim=dim, page=page, block=block,
                    cache=rng.choice(["f16", "bf16", "i8", "e4m3"]),
                    sequences=rng.randrange(1, 17) if prompts else _log(rng, 1, 300),
                    tokens=_log(rng, 30, 30000) if prompts else 0, context=_log(rng, 40, 9000), ragged=ragged)
    context = _log(rng, 100, 150000)
    most = max(1, min(100, int(2.0e8 / (context * kv_heads * dim))))
    return dict(SPARSE, kind=kind, **model, page=page, block=block, cache=rng.choice(["f16", "bf16", "i8", "e4m3"]),
                q=rng.choice(["f32", "f16", "bf16"]), sequences=_log(rng, 1, most), context=context,
                budget=_log(rng, 4, max(4, min(512, 8192 // block))), first=rng.randrange(0, 3), last=rng.randrange(0, 3),
                scale=dim ** -0.5, ragged=ragged)


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
    """Tokens of each sequence: from one to the longest; in a batch the last rows are padding (length 0)."""
    n = case["sequences"]
    r = np.random.RandomState(case["ragged"])
    length = np.maximum(1, np.floor(np.exp(r.uniform(math.log(max(1.0, case["context"] / 8)), math.log(case["context"] + 0.5), n)))).astype(np.int64)
    length[0] = case["context"]
    if n > 4:
        length[1], length[-1] = 1, 0
    return length


def _new_lengths(case):
    """(new tokens, tokens in the pages with them) of each sequence."""
    if not case["tokens"]:
        length = _contexts(case)
        return np.minimum(length, 1), length
    new = _shares(case)
    r = np.random.RandomState(case["ragged"] + 1)
    past = np.where(r.uniform(size=len(new)) < 0.5, 0, r.randint(0, case["context"], len(new)))  # half go on from a turn before
    return new, new + past


def _plan_lengths(case):
    """(tokens before the step, new ones, first position that stays: -1 where the sequence is over)."""
    if not case["tokens"]:
        length = _contexts(case)
        keep = np.maximum(0, length + 1 - case["window"]) if case["window"] else np.zeros_like(length)
        return length, np.minimum(length, 1), keep
    new = _shares(case)
    r = np.random.RandomState(case["ragged"] + 1)
    length = r.randint(0, case["context"], len(new))
    return length, new, np.where(r.uniform(size=len(new)) < 0.6, -1, 0)


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


def _scaled(case):
    return case["cache"] in MOST


def _scales(g, s, case, size):
    """Of each block and KV head, so that the block's values are some `size` and differ from block to block."""
    shape = (s.pool, case["kv_heads"], case["page"] // case["block"])
    return torch.exp(0.3 * torch.randn(shape, generator=g, device="cuda")) * (size * 3.0 / MOST[case["cache"]])


def _pool(g, s, case, channels=None):
    """One pool of pages: values of about 1 (stored ones of 8 bits fill their range), some elements larger than others
    where `channels` says so, as keys have them."""
    shape = (s.pool, case["kv_heads"], case["page"], case["head_dim"])
    x = torch.randn(shape, generator=g, device="cuda")
    if channels is not None:
        x.mul_(channels)
    if case["cache"] == "i8":
        return x.mul_(40.0).round_().clamp_(-127, 127).to(torch.int8)
    if case["cache"] == "e4m3":
        return x.mul_(150.0).clamp_(-448.0, 448.0).to(ELEM["e4m3"])
    return x.to(ELEM[case["cache"]])


def _caches(g, s, case):
    channels = 0.5 + 1.5 * torch.rand(case["head_dim"], generator=g, device="cuda") ** 4
    s.keys, s.values = _pool(g, s, case, channels), _pool(g, s, case)
    s.key_scales = s.value_scales = None
    if _scaled(case):
        s.key_scales, s.value_scales = _scales(g, s, case, 1.0), _scales(g, s, case, 1.0)


def prepare(case, seed):
    s, g = _State(), _generator(case, seed)
    s.case = case
    {"plan": _prepare_plan, "append": _prepare_append, "decode": _prepare_decode, "bounds": _prepare_bounds,
     "sparse": _prepare_sparse}[case["kind"]](s, case, g)
    torch.cuda.current_stream().synchronize()
    return s


def _prepare_plan(s, case, g):
    page, n = case["page"], case["sequences"]
    length, new, keep = _plan_lengths(case)
    after = np.where(keep < 0, 0, length) + new
    s.width = max(1, int(-(-np.maximum(length, after).max() // page))) + 1
    held = -(-length // page)
    s.pool = int(held.sum() + (-(-after // page)).sum()) + 5
    order = torch.randperm(s.pool, generator=g, device="cuda").cpu().numpy().astype(np.int32)
    table = np.full((n, s.width), -1, np.int32)
    at = 0
    for i, m in enumerate(held):
        table[i, :m] = order[at:at + m]
        at += int(m)
        if case["window"]:  # given back in the steps before, but for the last two
            gone = max(0, int(keep[i]) // page - 2)
            table[i, :gone] = -1
    free = np.setdiff1d(order, table)
    free = free[np.argsort(np.argsort(order)[free])] if len(free) else free
    if case["short"]:  # fewer free pages than the step wants
        free = free[:case["short"]]
    stack = np.full(s.pool, -1, np.int32)
    stack[:len(free)] = free
    s.table, s.free, s.free_count = _ints(table), _ints(stack), _ints([len(free)])
    s.lengths, s.keep = _ints(length), _ints(keep) if case["window"] or case["tokens"] else None
    s.new = _ints(new) if case["tokens"] else None
    s.rows = case["tokens"] + PAD_ROWS if case["tokens"] else n
    s.after, s.missing, s.offsets = _ints(length), _ints(np.zeros(n)), _ints(np.zeros(n + 1))
    s.sequences, s.positions = _ints(np.zeros(s.rows)), _ints(np.zeros(s.rows))
    s.slots = torch.zeros(s.rows, dtype=torch.int64, device="cuda")


def _prepare_append(s, case, g):
    heads, kv, dim = case["heads"], case["kv_heads"], case["head_dim"]
    new, length = _new_lengths(case)
    _pages(s, case, length, g)
    s.packed = case["tokens"] > 0
    s.rows = case["tokens"] + PAD_ROWS if s.packed else case["sequences"]
    s.offsets = _ints(np.concatenate([[0], np.cumsum(new)])) if s.packed else None
    s.q, s.k, s.v = (_normal(g, (s.rows, n, dim), times=2.0) for n in (heads, kv, kv))
    s.q_norm, s.k_norm = ((1.0 + 0.1 * _normal(g, (dim,)) for _ in range(2)) if case["norm"] else (None, None))
    s.factors = torch.exp(torch.rand(case["rope_dims"] // 2, generator=g, device="cuda") * 2.0) if case["factors"] else None
    _caches(g, s, case)
    if case["cache"] == "e4m3":  # as earlier appends leave them: powers of two
        s.key_scales, s.value_scales = (torch.exp2(torch.ceil(torch.log2(x))) for x in (s.key_scales, s.value_scales))
    out = ELEM[case["out"]]
    s.q_out = torch.zeros((s.rows, heads, dim), dtype=out, device="cuda")
    s.k_out, s.v_out = ((torch.zeros((s.rows, kv, dim), dtype=out, device="cuda") for _ in range(2)) if s.packed else (None, None))


def _prepare_decode(s, case, g):
    _pages(s, case, _contexts(case), g)
    s.q = _normal(g, (case["sequences"], case["heads"], case["head_dim"]), ELEM[case["q"]], 2.0)
    _caches(g, s, case)
    s.out = torch.zeros_like(s.q)


def _prepare_bounds(s, case, g):
    new, length = _new_lengths(case)
    _pages(s, case, length, g)
    _caches(g, s, case)
    s.packed = case["tokens"] > 0
    s.rows = case["tokens"] + PAD_ROWS if s.packed else case["sequences"]
    s.offsets = _ints(np.concatenate([[0], np.cumsum(new)])) if s.packed else None
    s.bounds = _normal(g, (s.pool, case["kv_heads"], case["page"] // case["block"], 2, case["head_dim"]), torch.bfloat16)


def _prepare_sparse(s, case, g):
    kv, dim, page, block = case["kv_heads"], case["head_dim"], case["page"], case["block"]
    _pages(s, case, _contexts(case), g)
    s.packed, s.rows, s.offsets = False, case["sequences"], None
    s.q = _normal(g, (case["sequences"], case["heads"], dim), ELEM[case["q"]], 2.0)
    _caches(g, s, case)
    s.bounds = torch.empty((s.pool, kv, page // block, 2, dim), dtype=torch.bfloat16, device="cuda")
    step = max(1, (1 << 28) // (kv * page * dim))
    for at in range(0, s.pool, step):  # as the steps before left them
        x = _real(s.keys[at:at + step], None if s.key_scales is None else s.key_scales[at:at + step], case)
        x = x.reshape(-1, kv, page // block, block, dim)
        s.bounds[at:at + step] = torch.stack([_outward(x.amin(3), False), _outward(x.amax(3), True)], 3)
    s.selected = torch.zeros((case["sequences"], kv, case["budget"]), dtype=torch.int32, device="cuda")
    s.counts = torch.zeros((case["sequences"], kv), dtype=torch.int32, device="cuda")
    s.out = torch.zeros_like(s.q)


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


def _views(H, s, case):
    """The descriptions of the cache and of what is kept of its blocks, which a program makes once for its buffers."""
    if not hasattr(s, "views"):
        c = H.paged_cache(_p(s.keys), _p(s.values), TYPE_ID[case["cache"]], page_count=s.pool, page_size=case["page"],
                          head_count_kv=case["kv_heads"], head_dim=case["head_dim"], d_pages=_p(s.table),
                          d_lengths=_p(s.lengths), sequence_count=case["sequences"], pages_per_sequence=s.table.shape[1])
        s.views = c, H.cache_blocks(case["block"], d_key_scales=_p(s.key_scales), d_value_scales=_p(s.value_scales),
                                    d_key_bounds=_p(getattr(s, "bounds", None)))
    return s.views


def _own(s, case):
    from heliopause_amd import hip_kernels as H

    q = _the_stream()
    if case["kind"] == "plan":
        H.page_plan_device(case["sequences"], s.width, case["page"], s.pool, _p(s.table), _p(s.lengths), _p(s.after),
                           _p(s.free), _p(s.free_count), d_new_tokens=_p(s.new), d_keep_from=_p(s.keep),
                           d_offsets=_p(s.offsets), d_missing=_p(s.missing), token_count=s.rows,
                           d_sequences=_p(s.sequences), d_positions=_p(s.positions), d_slots=_p(s.slots), stream=q)
        return _plan_outputs(s)
    cache, blocks = _views(H, s, case)
    if case["kind"] == "append":
        H.block_append_device(cache, blocks, s.rows, case["heads"], _p(s.q), _p(s.k), _p(s.v), _p(s.q_out),
                              TYPE_ID[case["out"]], d_offsets=_p(s.offsets), d_q_norm=_p(s.q_norm),
                              d_k_norm=_p(s.k_norm), norm_values=case["norm"], epsilon=EPSILON,
                              rope_dims=case["rope_dims"], rope_freq_base=FREQ_BASE, d_rope_freq_factors=_p(s.factors),
                              d_k_out=_p(s.k_out), d_v_out=_p(s.v_out), stream=q)
        return _append_outputs(s)
    if case["kind"] == "decode":
        H.block_attention_device(cache, blocks, case["heads"], _p(s.q), TYPE_ID[case["q"]], _p(s.out),
                                 TYPE_ID[case["q"]], scale=case["scale"], sliding_window=case["window"], stream=q)
        return s.out
    H.block_bounds_device(cache, blocks, s.rows, d_offsets=_p(s.offsets), stream=q)
    if case["kind"] == "bounds":
        return s.bounds
    H.block_select_device(cache, blocks, case["heads"], _p(s.q), TYPE_ID[case["q"]], case["budget"], _p(s.selected),
                          _p(s.counts), first_blocks=case["first"], last_blocks=case["last"], stream=q)
    H.block_attention_device(cache, blocks, case["heads"], _p(s.q), TYPE_ID[case["q"]], _p(s.out), TYPE_ID[case["q"]],
                             scale=case["scale"], d_selected=_p(s.selected), d_counts=_p(s.counts),
                             budget=case["budget"], stream=q)
    return _sparse_outputs(s)


# ---- the plain forms ------------------------------------------------------------------------------------------------
def _plan_outputs(s):
    return {"table": s.table, "lengths": s.after, "free": s.free, "free_count": s.free_count, "missing": s.missing,
            "offsets": s.offsets, "sequences": s.sequences, "positions": s.positions, "slots": s.slots}


def _plain_plan(s, case):
    page, n, width = case["page"], case["sequences"], s.width
    table, length = s.table.long(), s.lengths.long().clamp(min=0)
    at = torch.arange(width, device="cuda")
    named = (table >= 0) & (table < s.pool)
    count = s.free_count.long().clamp(0, s.pool)
    # back: in order of sequence and position, on top of the free pages
    if s.keep is not None:
        keep = s.keep.long()[:, None]
        back = (keep < 0) | ((at + 1) * page <= keep)
        length = torch.where(keep[:, 0] < 0, torch.zeros_like(length), length)
        to = count + torch.cumsum((back & named).view(-1), 0) - 1
        to = torch.where((back & named).view(-1) & (to < s.pool), to, s.pool)
        stack = torch.cat([s.free, s.free[:1]]).long().scatter_(0, to, table.view(-1))[:s.pool]
        count = (count + (back & named).sum()).clamp(max=s.pool)
        table = torch.where(back, torch.full_like(table, -1), table)
        named &= ~back
    else:
        stack = s.free.long()
    new = (length > 0).long() if s.new is None else s.new.long().clamp(min=0)
    after = length + new
    # dealt: the new positions' pages that have no name yet, from the top of the stack
    want = (at >= ((length + page - 1) // page)[:, None]) & (at < ((after + page - 1) // page)[:, None]) & ~named
    rank = torch.cumsum(want.view(-1), 0).view(n, width) - 1
    dealt = stack[(count - 1 - rank).clamp(0, s.pool - 1)]
    dealt = torch.where((rank < count) & (dealt >= 0) & (dealt < s.pool), dealt, torch.full_like(dealt, -1))
    table = torch.where(want, dealt, table)
    s.missing.copy_((want & (dealt < 0)).sum(1))
    s.free_count.copy_(count - torch.minimum(count, want.sum()))
    s.free.copy_(stack)
    s.table.copy_(table)
    s.after.copy_(after)
    s.offsets.copy_(torch.cat([torch.zeros_like(new[:1]), torch.cumsum(new, 0)]))
    # each row's place
    row = torch.arange(s.rows, device="cuda")
    if s.new is None:
        seq, position, there = row, after - 1, new > 0
    else:
        offsets = s.offsets.long()
        seq = torch.searchsorted(offsets[1:].contiguous(), row, right=True)
        there = seq < n
        seq = seq.clamp(max=n - 1)
        position = length[seq] + row - offsets[seq]
    entry = table[seq, (position // page).clamp(0, width - 1)]
    none = torch.full_like(row, -1)
    slot = torch.where((position // page < width) & (entry >= 0) & (entry < s.pool), entry * page + position % page, none)
    s.sequences.copy_(torch.where(there, seq, none))
    s.positions.copy_(torch.where(there, position, none))
    s.slots.copy_(torch.where(there, slot, none))
    return _plan_outputs(s)


def _append_outputs(s):
    return {name: t for name, t in (("q", s.q_out), ("k", s.k_out), ("v", s.v_out), ("keys", s.keys), ("values", s.values),
                                    ("key_scales", s.key_scales), ("value_scales", s.value_scales)) if t is not None}


def _rms(x, weight):
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPSILON)
    return y if weight is None else y * weight


def _rotate(x, cos, sin, dims):
    """Pairs (u, u + dims / 2) of each head by the token's angles; the rest as it is."""
    half = dims // 2
    a, b = x[..., :half], x[..., half:dims]
    return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., dims:]], -1)


def _rows(s, case):
    """(row, sequence, position) of the new tokens that belong to a sequence."""
    row = torch.arange(s.rows, device="cuda")
    if s.packed:
        seq = torch.searchsorted(s.offsets[1:].contiguous(), row, right=True)
        live = seq < case["sequences"]
        seq = seq.clamp(max=case["sequences"] - 1)
        position = s.lengths[seq] - s.offsets[seq + 1] + row
    else:
        seq, position = row, s.lengths - 1
        live = position >= 0
    return row[live], seq[live], position[live].long()


def _block_scale(most, case):
    """The scale of a block whose largest element is `most`."""
    if case["cache"] == "i8":
        scale = most / MOST["i8"]
    else:  # the least power of two under which 448 reaches it: 448 = 0.875 * 2^9
        m, e = torch.frexp(most)
        scale = torch.ldexp(torch.ones_like(most), torch.where(m <= 0.875, e - 9, e - 8)) * (m > 0)
    return scale.clamp(SCALE_LOW, SCALE_HIGH)


def _stored(x, case):
    most = MOST[case["cache"]]
    x = x.round() if case["cache"] == "i8" else x
    return x.clamp(-most, most).to(ELEM[case["cache"]])


def _store_blocks(x, page, slot, pool, scales, case):
    """Rows x [token][kv head][dim] into their pages, with the scales of the blocks they lie in."""
    kv, block, per = case["kv_heads"], case["block"], case["page"] // case["block"]
    where = page * per + slot // block
    touched, which = torch.unique(where, return_inverse=True)
    at_page, at_block = touched // per, touched % per
    most = torch.zeros((len(touched), kv), device="cuda").scatter_reduce_(
        0, which[:, None].expand(-1, kv), x.abs().amax(-1), "amax")
    begin = torch.full((len(touched),), block, device="cuda").scatter_reduce_(0, which, slot % block, "amin")
    old = scales[at_page, :, at_block]
    fresh = _block_scale(most, case)
    grown = torch.maximum(fresh, old * GROWTH).clamp(SCALE_LOW, SCALE_HIGH) if case["cache"] == "i8" else fresh
    first = (begin == 0)[:, None]
    grows = ~first & (most > old * MOST[case["cache"]])
    scale = torch.where(first, fresh, torch.where(grows, grown, old))
    # what the blocks hold already moves to the new scale
    bits = pool.view(torch.uint8)
    slots = at_block[:, None] * block + torch.arange(block, device="cuda")
    held = bits[at_page[:, None], :, slots].view(pool.dtype)  # [block][slot][kv head][dim]
    moved = _stored(held.float() * (old / scale)[:, None, :, None], case)
    moves = grows[:, None, :] & (torch.arange(block, device="cuda") < begin[:, None])[:, :, None]
    bits[at_page[:, None], :, slots] = torch.where(moves[..., None], moved.view(torch.uint8), held.view(torch.uint8))
    scales[at_page, :, at_block] = scale
    bits[page, :, slot] = _stored(x * (1.0 / scale)[which][:, :, None], case).view(torch.uint8)


def _plain_append(s, case):
    row, seq, position = _rows(s, case)
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
    page, slot = s.table[seq, position // case["page"]].long(), position % case["page"]
    _store_blocks(k, page, slot, s.keys, s.key_scales, case)
    _store_blocks(v, page, slot, s.values, s.value_scales, case)
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


def _real(pool, scales, case):
    """What a pool's pages stand for, in 32 bits."""
    x = pool.float()
    if scales is not None:
        x = x * scales.repeat_interleave(case["block"], 2)[..., None]
    return x


def _bits(pool):
    return pool.view(torch.uint8 if pool.element_size() == 1 else torch.int16)


def _gathered(pool, scales, s, case):
    """The sequences' rows of a pool in order, [sequence][kv head][position][dim], in 32 bits."""
    n, kv, width, dim = case["sequences"], case["kv_heads"], s.table.shape[1], case["head_dim"]
    pages = s.table.clamp(min=0).long().view(-1)
    x = _real(_bits(pool)[pages].view(pool.dtype), None if scales is None else scales[pages], case)
    return x.view(n, width, kv, case["page"], dim).permute(0, 2, 1, 3, 4).reshape(n, kv, -1, dim)


def _plain_decode(s, case):
    n, kv, dim = case["sequences"], case["kv_heads"], case["head_dim"]
    k, v = _gathered(s.keys, s.key_scales, s, case), _gathered(s.values, s.value_scales, s, case)
    q = s.q.float().reshape(n, kv, case["heads"] // kv, dim)
    scores = torch.matmul(q, k.transpose(-1, -2)) * case["scale"]
    at = torch.arange(k.shape[2], device="cuda")
    seen = at < s.lengths[:, None]
    if case["window"]:
        seen &= at >= s.lengths[:, None] - case["window"]
    out = torch.matmul(_softmax(scores, seen[:, None, None]), v)
    return out.reshape(n, case["heads"], dim).to(s.out.dtype)


def _outward(x, up):
    """x in bf16, the nearest value that is not below (up) or not above it."""
    x = x.clamp(-BF16_MOST, BF16_MOST)
    y = x.to(torch.bfloat16)
    bits, value = y.view(torch.int16), y.float()
    away = ~torch.signbit(value) if up else torch.signbit(value)  # a larger magnitude is further out
    moved = torch.where(away, bits + 1, bits - 1).to(torch.int16)
    return torch.where(value < x if up else value > x, moved, bits).view(torch.bfloat16)


def _plain_bounds(s, case):
    block, page, dim = case["block"], case["page"], case["head_dim"]
    _, seq, position = _rows(s, case)
    key = torch.unique(seq * (s.table.shape[1] * page // block) + position // block)
    seq, b = key // (s.table.shape[1] * page // block), key % (s.table.shape[1] * page // block)
    first = b * block
    at_page, at_block = s.table[seq, first // page].long(), first % page // block
    slots = first[:, None] % page + torch.arange(block, device="cuda")
    x = _bits(s.keys)[at_page[:, None], :, slots].view(s.keys.dtype).float()  # [block][slot][kv head][dim]
    if s.key_scales is not None:
        x = x * s.key_scales[at_page, :, at_block][:, None, :, None]
    live = (first[:, None] + torch.arange(block, device="cuda") < s.lengths[seq][:, None])[:, :, None, None]
    least = _outward(torch.where(live, x, math.inf).amin(1), False)
    most = _outward(torch.where(live, x, -math.inf).amax(1), True)
    s.bounds[at_page, :, at_block] = torch.stack([least, most], 2)
    return s.bounds


def _sparse_outputs(s):
    return {"out": s.out, "selected": s.selected, "counts": s.counts, "bounds": s.bounds}


def _select(s, case):
    n, kv, dim, block, page, budget = (case[x] for x in ("sequences", "kv_heads", "head_dim", "block", "page", "budget"))
    per = page // block
    total = s.table.shape[1] * per
    b = torch.arange(total, device="cuda")
    entry = s.table[:, b // per].long()
    live = (b * block < s.lengths[:, None]) & (entry >= 0) & (entry < s.pool)
    bound = s.bounds[entry.clamp(min=0), :, (b % per)[None]].double()  # [sequence][block][kv head][2][dim]
    q = s.q.double().view(n, kv, case["heads"] // kv, dim)
    least, most = bound[:, :, :, 0].permute(0, 2, 3, 1).contiguous(), bound[:, :, :, 1].permute(0, 2, 3, 1).contiguous()
    score = (torch.matmul(q.clamp(min=0), most) + torch.matmul(q.clamp(max=0), least)).amax(2)  # [sequence][kv head][block]
    blocks = (s.lengths.long() + block - 1) // block
    always = (b < case["first"]) | (b >= blocks[:, None] - case["last"])
    score = torch.where(always[:, None], math.inf, score)
    score = torch.where(live[:, None], score, -math.inf)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices
    count = live.sum(1).clamp(max=budget)[:, None].expand(n, kv)
    order = torch.nn.functional.pad(order, (0, max(0, budget - total)))[..., :budget]
    order = torch.where(torch.arange(budget, device="cuda") < count[..., None], order, total).sort(-1).values
    s.selected.copy_(torch.where(order < total, order, -1))
    s.counts.copy_(count)


def _taken(pool, scales, page, slot, case):
    """Rows [sequence][kv head][position][dim] of a pool, in 32 bits."""
    h = torch.arange(case["kv_heads"], device="cuda")[None, :, None]
    x = _bits(pool)[page, h, slot].view(pool.dtype).float()
    return x if scales is None else x * scales[page, h, slot // case["block"]][..., None]


def _plain_sparse(s, case):
    n, kv, dim, block = case["sequences"], case["kv_heads"], case["head_dim"], case["block"]
    _plain_bounds(s, case)
    _select(s, case)
    at = (s.selected.long()[..., None] * block + torch.arange(block, device="cuda")).view(n, kv, -1)
    seen = (at >= 0) & (at < s.lengths[:, None, None])
    at = at.clamp(min=0)
    page = torch.gather(s.table.long()[:, None].expand(n, kv, -1), 2, at // case["page"]).clamp(min=0)
    k = _taken(s.keys, s.key_scales, page, at % case["page"], case)
    v = _taken(s.values, s.value_scales, page, at % case["page"], case)
    q = s.q.float().reshape(n, kv, case["heads"] // kv, dim)
    scores = torch.matmul(q, k.transpose(-1, -2)) * case["scale"]
    out = torch.matmul(_softmax(scores, seen[:, :, None]), v)
    s.out.copy_(out.reshape(n, case["heads"], dim))
    return _sparse_outputs(s)


def run(s):
    case = s.case
    if own:
        return _own(s, case)
    return {"plan": _plain_plan, "append": _plain_append, "decode": _plain_decode, "bounds": _plain_bounds,
            "sparse": _plain_sparse}[case["kind"]](s, case)


# ---- the definition in 64 bits --------------------------------------------------------------------------------------
def _wide(t):
    return None if t is None else t.detach().double()


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


def _exact_append(s, case):
    new, length = _new_lengths(case)
    page, block, kind = case["page"], case["block"], case["cache"]
    rows, position = [], []
    for i, (n, total) in enumerate(zip(new, length)):
        start = int(new[:i].sum()) if s.packed else i
        rows += range(start, start + int(n))
        position += range(int(total - n), int(total))
    rows, position = torch.tensor(rows, device="cuda"), torch.tensor(position, device="cuda", dtype=torch.float64)
    norm, factors = case["norm"], _wide(s.factors)
    q = _exact_row(_wide(s.q)[rows], _wide(s.q_norm) if norm else None, position, case, factors)
    k = _exact_row(_wide(s.k)[rows], _wide(s.k_norm) if norm else None, position, case, factors)
    v = _exact_row(_wide(s.v)[rows], True if norm else None, None, case, None)
    got = {}
    for name, x, buffer in (("q", q, s.q_out), ("k", k, s.k_out), ("v", v, s.v_out)):
        if buffer is not None:
            got[name] = _wide(buffer)
            got[name][rows] = x
    table = s.table.cpu().numpy()
    for name, x, pool, scales in (("keys", k, s.keys, s.key_scales), ("values", v, s.values, s.value_scales)):
        codes, scale = pool.double(), scales.double()
        at = 0
        for i, (n, total) in enumerate(zip(new, length)):
            p = int(total - n)
            while p < total:
                end = min(int(total), p - p % block + block)
                y = x[at:at + end - p]
                where, b, slot = int(table[i, p // page]), p % page // block, p % page
                most = y.abs().amax((0, 2))
                if kind == "i8":
                    wanted = most / 127.0
                else:
                    wanted = torch.exp2(torch.ceil(torch.log2(most / 448.0)))
                if p % block:
                    old = scale[where, :, b].clone()
                    grown = torch.maximum(wanted, 1.25 * old) if kind == "i8" else wanted
                    wanted = torch.where(most > old * MOST[kind], grown, old)
                    codes[where, :, slot - p % block:slot] *= (old / wanted)[:, None, None]
                scale[where, :, b] = wanted
                codes[where, :, slot:slot + end - p] = (y / wanted[:, None]).transpose(0, 1)
                at, p = at + end - p, end
        got[name] = None if kind == "i8" else codes  # (i8's are whole numbers, next to borders either)
        got[name[:-1] + "_scales"] = scale
    return got


def _exact_keys(pool, scales, page, slot, head, case):
    x = _bits(pool)[page, head, slot].view(pool.dtype).double()
    return x if scales is None else x * scales[page, head, slot // case["block"]].double()[:, None]


def _exact_head(q, s, case, i, h, at):
    """Queries [group][dim] of KV head h of sequence i over the positions `at`."""
    page, slot = s.table[i].long()[at // case["page"]], at % case["page"]
    k = _exact_keys(s.keys, s.key_scales, page, slot, h, case)
    v = _exact_keys(s.values, s.value_scales, page, slot, h, case)
    e = q @ k.T * case["scale"]
    p = torch.exp(e - e.max(1, keepdim=True).values)
    return p @ v / p.sum(1, keepdim=True)


def _exact_bounds(s, case):
    """The bounds themselves, which bf16 rounds outward."""
    new, length = _new_lengths(case)
    page, block = case["page"], case["block"]
    got = s.bounds.double()
    for i, (n, total) in enumerate(zip(new, length)):
        for b in range(int(total - n) // block, -(-int(total) // block) if n else 0):
            at = torch.arange(b * block, min(int(total), b * block + block), device="cuda")
            where = int(s.table[i, b * block // page])
            x = _bits(s.keys)[where, :, at % page].view(s.keys.dtype).double()
            if s.key_scales is not None:
                x = x * s.key_scales[where, :, b * block % page // block].double()[:, None, None]
            got[where, :, b * block % page // block, 0] = x.min(1).values
            got[where, :, b * block % page // block, 1] = x.max(1).values
    return got


def _exact_selected(q, s, case, i, h):
    """The blocks of sequence i that the queries [group][dim] of KV head h take, from bounds that are up to date."""
    block, per, length = case["block"], case["page"] // case["block"], int(s.lengths[i])
    n = -(-length // block)
    b = torch.arange(n, device="cuda")
    bound = s.bounds[s.table[i].long()[b // per], h, b % per].double()
    middle, radius = (bound[:, 1] + bound[:, 0]) / 2, (bound[:, 1] - bound[:, 0]) / 2
    score = (middle @ q.T + radius @ q.abs().T).max(1).values
    score[(b < case["first"]) | (b >= n - case["last"])] = math.inf
    best = sorted(range(n), key=lambda x, v=score.tolist(): (-v[x], x))[:case["budget"]]
    return sorted(best)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "plan":
        return None  # whole numbers
    if kind == "append":
        return _exact_append(s, case)
    if kind == "bounds":
        return _exact_bounds(s, case)
    n, kv, group = case["sequences"], case["kv_heads"], case["heads"] // case["kv_heads"]
    if kind == "sparse":
        bounds = _exact_bounds(s, case)
        _plain_bounds(s, case)
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    for i, length in enumerate(s.lengths.tolist()):
        for h in range(kv if length else 0):
            q = s.q[i, h * group:(h + 1) * group].double()
            if kind == "sparse":
                b = torch.tensor(_exact_selected(q, s, case, i, h), device="cuda")
                at = (b[:, None] * case["block"] + torch.arange(case["block"], device="cuda")).view(-1)
                at = at[at < length]
            else:
                at = torch.arange(max(0, length - case["window"]) if case["window"] else 0, length, device="cuda")
            out[i, h * group:(h + 1) * group] = _exact_head(q, s, case, i, h, at)
    if kind == "sparse":
        return {"out": out, "selected": None, "counts": None, "bounds": bounds}
    return out


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def work(case):
    kind, page = case["kind"], case["page"]
    if kind == "plan":
        length, new, keep = _plan_lengths(case)
        after = np.where(keep < 0, 0, length) + new
        back = np.where(keep < 0, -(-length // page), keep // page if case["window"] else 0)
        entries = float(back.sum() + (-(-after // page) - np.where(keep < 0, 0, length) // page).sum())
        rows = case["tokens"] or case["sequences"]
        return {"bytes": 16.0 * rows + 8.0 * entries + 24.0 * case["sequences"], "flops": 8.0 * rows}
    kv, dim, block, e = case["kv_heads"], case["head_dim"], case["block"], BYTES[case["cache"]]
    if kind == "append":
        heads = case["heads"]
        new, length = _new_lengths(case)
        blocks = float(sum((n > 0) * (-(-n // block)) for n in new))
        new = int(new.sum())
        out = BYTES[case["out"]] * (heads + (2 * kv if case["tokens"] else 0)) + 2 * kv
        return {"bytes": new * dim * (4.0 * (heads + 2 * kv) + out) + 8.0 * kv * blocks,
                "flops": new * dim * (heads + 2 * kv) * 8.0}
    if kind == "bounds":
        new, length = _new_lengths(case)
        begin, blocks = (length - new) // block, -(-length // block)  # of the blocks that have new tokens
        keys = float(np.where(new > 0, length - begin * block, 0).sum())
        count = float(np.where(new > 0, blocks - begin, 0).sum())
        return {"bytes": kv * dim * (keys * e + 4.0 * count), "flops": 2.0 * keys * kv * dim}
    heads, length = case["heads"], _contexts(case)
    per_key = 2.0 * kv * dim * e + (8.0 * kv / block if _scaled(case) else 0.0)
    rows = 2.0 * case["sequences"] * heads * dim * BYTES[case["q"]]
    if kind == "decode":
        keys = float((np.minimum(length, case["window"]) if case["window"] else length).sum())
        return {"bytes": keys * per_key + rows, "flops": 4.0 * keys * heads * dim}
    blocks = -(-length // block)
    last = float((length - np.maximum(0, blocks - 1) * block).sum())  # keys of the block that is refreshed
    keys = float(np.minimum(length, case["budget"] * block).sum())
    return {"bytes": keys * per_key + rows + kv * dim * (4.0 * float(blocks.sum()) + e * last),
            "flops": 4.0 * keys * heads * dim + 4.0 * float(blocks.sum()) * heads * dim}

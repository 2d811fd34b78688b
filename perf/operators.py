"""The serving operators around the paged Q8 cache, as measurable cases.

Four operators of a server that answers many conversations at once:

* ``packed``: the prompts of several sequences, of different lengths and after
  different amounts of earlier context, appended to the cache and attended to
  causally in one call (tq_hip_prefill_packed_async);
* ``weights``: the decode step of a batch that also adds every cached token's
  attention weight to a running total (tq_hip_decode_step_weights_async);
* ``evict``: those totals choose which tokens a cache of bounded size keeps
  (tq_hip_kv_evict_async);
* ``logits``: penalties for repeated tokens, biases and a grammar's mask on the
  logits, and the token that is best after them (tq_hip_logits_process).

The head shapes are the benchmark's: 8 query / 2 kv heads of 64 (the small
parity shape), 32 / 8 of 128 (the 8B class) and 64 / 8 of 128 (the 70B class);
draw() adds one head per group and groups of three.

What is quantized (queries, keys and values as block_q8: 32 codes and a scale)
is defined by its fp32 arithmetic, bit for bit, so codes are compared as whole
bytes; everything after the codes is real arithmetic.
"""
import ctypes as C
import math
import random

import numpy as np
import torch

own = False

QK = 32
PAGE = 16
THETA = 500000.0
VOCAB = 128256
SHAPES = {"small": (8, 2, 64), "8b": (32, 8, 128), "70b": (64, 8, 128), "single": (16, 16, 128), "triple": (24, 8, 64)}
SPARE = 5     # rows of the output behind the last packed sequence


# ---- the cases -------------------------------------------------------------

def listed():
    return [
        # three short messages at once on the smallest shape: latency
        {"name": "packed-small", "op": "packed", "shape": "small", "n": 3, "low": 1, "high": 33, "context": 0},
        # new conversations that arrived together
        {"name": "packed-8b-prompts", "op": "packed", "shape": "8b", "n": 16, "low": 64, "high": 2048, "context": 0},
        # the next turns of running conversations
        {"name": "packed-8b-turns", "op": "packed", "shape": "8b", "n": 24, "low": 8, "high": 512, "context": 4000},
        # a few long documents on the large shape
        {"name": "packed-70b-documents", "op": "packed", "shape": "70b", "n": 4, "low": 1024, "high": 4096,
         "context": 0},
        # one short conversation's step: latency
        {"name": "weights-small", "op": "weights", "shape": "small", "n": 1, "low": 256, "high": 256},
        # a serving batch of very different lengths
        {"name": "weights-8b-batch64", "op": "weights", "shape": "8b", "n": 64, "low": 512, "high": 8192},
        # long contexts on the large shape
        {"name": "weights-70b-16k", "op": "weights", "shape": "70b", "n": 16, "low": 16384, "high": 16384},
        # a full cache of a running batch gives up one token for each new one
        {"name": "evict-8b-one", "op": "evict", "shape": "8b", "n": 32, "low": 2049, "high": 2049, "keep": 2048,
         "sinks": 4, "recent": 256},
        # a batch of long prompts is cut down to the budget
        {"name": "evict-8b-half", "op": "evict", "shape": "8b", "n": 64, "low": 2500, "high": 4096, "keep": 2048,
         "sinks": 4, "recent": 256},
        # one long document on the large shape, cut to a quarter
        {"name": "evict-70b-32k", "op": "evict", "shape": "70b", "n": 1, "low": 32768, "high": 32768, "keep": 8192,
         "sinks": 4, "recent": 1024},
        # one conversation's next token
        {"name": "logits-one", "op": "logits", "rows": 1, "vocab": VOCAB, "pad": 0, "history": 600, "bias": 8,
         "grammar": False},
        # a serving batch under grammars
        {"name": "logits-batch64", "op": "logits", "rows": 64, "vocab": VOCAB, "pad": 0, "history": 4096, "bias": 32,
         "grammar": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["packed", "weights", "evict", "logits"])
    if op == "logits":
        return {"op": op, "rows": _log_int(rng, 1, 64), "vocab": _log_int(rng, 1000, VOCAB), "pad": rng.choice([0, 0, 1, 64]),
                "history": _log_int(rng, 1, 4096), "bias": rng.choice([0, rng.randint(1, 64)]),
                "grammar": rng.random() < 0.5}
    shape = rng.choice(["small", "8b", "8b", "70b", "single", "triple"])
    nq, nkv, hd = SHAPES[shape]
    if op == "packed":
        n, context = _log_int(rng, 1, 32), rng.choice([0, _log_int(rng, 1, 4000)])
        high = _log_int(rng, 2, 2048)
        # at most the largest listed case's padded scores
        high = min(high, int(math.sqrt(4 * 64 * 4096 * 4096 / (2 * n * nq))))
        if context:
            context = min(context, max(1, 4 * 64 * 4096 * 4096 // (2 * n * nq * high)))
        return {"op": op, "shape": shape, "n": n, "low": rng.randint(0, high), "high": high, "context": context}
    n = _log_int(rng, 1, 64)
    high = _log_int(rng, 64, min(16384, 262144 * 8 // (n * nkv)))
    low = high if rng.random() < 0.4 else rng.randint(max(1, high // 16), high)
    case = {"op": op, "shape": shape, "n": n, "low": low, "high": high}
    if op == "evict":
        keep = rng.randint(max(1, high // 8), high)
        recent = rng.randint(0, keep // 2)
        case.update(keep=keep, recent=recent, sinks=rng.randint(0, min(8, keep - recent)))
    return case


def _lengths(case):
    """The sequences' lengths: the case's own, for every seed."""
    if case["low"] == case["high"]:
        return [case["high"]] * case["n"]
    r = random.Random(case["n"] * 1000003 + case["low"] * 101 + case["high"])
    return [case["high"]] + [r.randint(case["low"], case["high"]) for _ in range(case["n"] - 1)]


def _contexts(case):
    """Tokens that each packed sequence already has."""
    r = random.Random(case["n"] * 7919 + case["context"])
    return [r.randint(0, case["context"]) for _ in range(case["n"])]


def work(case):
    if case["op"] == "logits":
        cells = case["rows"] * case["vocab"]
        n = cells * 8 + case["rows"] * (4 * case["history"] + 8 * case["bias"] + 4)
        return {"bytes": n + (cells // 8 if case["grammar"] else 0), "flops": 0}
    nq, nkv, hd = SHAPES[case["shape"]]
    row = 2 * nkv * (hd // QK) * 36          # a token's keys and values in the cache
    lens = _lengths(case)
    if case["op"] == "packed":
        rows, before = sum(lens), _contexts(case)
        pairs = sum(n * b + n * (n + 1) // 2 for n, b in zip(lens, before))
        read = sum(b * row for n, b in zip(lens, before) if n)
        return {"bytes": read + rows * (row + 4 * (2 * nq * hd + 2 * nkv * hd + hd)), "flops": 4 * nq * hd * pairs}
    if case["op"] == "weights":
        n = case["n"]
        return {"bytes": sum(lens) * (row + 8 * nkv) + n * (row + 4 * (2 * nq * hd + 2 * nkv * hd + hd)),
                "flops": 4 * nq * hd * sum(lens)}
    # totals and positions are read, those that are kept written; the tokens kept from behind the budget move:
    # the window's, and their share of the others where totals do not go by position
    moved = 0.0
    keep, sinks, recent = case["keep"], case["sinks"], case["recent"]
    for n in lens:
        if n > keep:
            last = min(recent, n - keep)
            free = n - sinks - recent
            moved += last + (n - keep - last) * (keep - sinks - recent) / free
    kept = sum(min(n, keep) for n in lens)
    return {"bytes": nkv * 8 * (sum(lens) + kept) + 2 * row * moved, "flops": 0}


# ---- inputs ----------------------------------------------------------------

def _generator(seed, part):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 64 + part) & 0x7FFFFFFFFFFF)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _int32(values):
    return torch.as_tensor(np.asarray(values, np.int32)).cuda()


def _rope(pos, hd):
    """cos and sin rows of the given positions: angles in 64 bits."""
    i = torch.arange(hd // 2, device="cuda", dtype=torch.float64)
    angle = torch.as_tensor(np.asarray(pos, np.float64)).cuda()[:, None] * THETA ** (-2.0 * i / hd)
    return angle.cos().float().contiguous(), angle.sin().float().contiguous()


def _pool(seed, shape, pages):
    """A cache's pages [pages][kv head][K|V][16 tokens][block][36 bytes]: quantized normal rows, keys with channels of
    different sizes."""
    _, nkv, hd = SHAPES[shape]
    g = _generator(seed, 1)
    size = torch.ones(2, 1, hd // QK, QK, device="cuda")
    size[0] = (0.4 * _randn(g, 1, hd // QK, QK)).exp()
    pool = torch.empty(pages, nkv, 2, PAGE, hd // QK, 36, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // (nkv * 2 * PAGE * hd))
    for p in range(0, pages, step):
        x = _randn(g, min(step, pages - p), nkv, 2, PAGE, hd // QK, QK) * size
        d = x.abs().amax(-1, keepdim=True) / 127
        pool[p:p + step, ..., 4:] = (x / d).round().to(torch.int8).view(torch.uint8)
        pool[p:p + step, ..., :4] = d.view(torch.uint8)
    return pool


def _tables(seed, capacity):
    """Page lists of sequences that hold `capacity` tokens, on scattered pages."""
    need = [max(1, -(-c // PAGE)) for c in capacity]
    ids = np.random.RandomState(seed & 0x7FFFFFFF).permutation(sum(need)).astype(np.int32)
    at = np.concatenate([[0], np.cumsum(need)])
    return [ids[a:b] for a, b in zip(at[:-1], at[1:])]


def _table(pages):
    """The lists as one tensor, short ones filled up with page 0."""
    t = np.zeros((len(pages), max(len(p) for p in pages)), np.int64)
    for i, p in enumerate(pages):
        t[i, :len(p)] = p
    return torch.from_numpy(t).cuda()


_stream = None


def _user_stream():
    """The one stream that this program works on."""
    global _stream
    if _stream is None:
        _stream = torch.cuda.Stream()
    return _stream.cuda_stream


class _Memory:
    """Device memory of the framework's, seen by torch."""

    def __init__(self, base, nbytes, keep):
        self.keep = keep
        self.__cuda_array_interface__ = {"shape": (nbytes,), "typestr": "|u1", "data": (base, False), "version": 2}


def _handle(s, pages):
    """The framework's cache with the same contents, and its pool in place of the plain one."""
    from tailorquantkernel_amd import native
    native.init(0)
    nq, nkv, hd = s["heads"]
    kv = native.PagedKV(nq, nkv, hd, s["pool"].shape[0], len(pages), max(len(p) for p in pages))
    for i, p in enumerate(pages):
        kv.set_pages(i, p)
    base, nbytes, _ = kv.pool()
    pool = torch.as_tensor(_Memory(base, nbytes, kv), device="cuda").view(s["pool"].shape)
    pool.copy_(s["pool"])
    s.update(native=native, lib=native.load(), kv=kv, pool=pool, stream=_user_stream())


def _workspace(nbytes):
    return torch.empty(max(16, nbytes), dtype=torch.uint8, device="cuda")


def _prepare_packed(s, case, seed):
    nq, nkv, hd = s["heads"]
    lens, before = _lengths(case), _contexts(case)
    rows, g = sum(lens), _generator(seed, 2)
    pages = _tables(seed, [n + b for n, b in zip(lens, before)])
    s["pool"] = _pool(seed, case["shape"], sum(len(p) for p in pages))
    s["q"], s["k"], s["v"] = (_randn(g, rows, h * hd) for h in (nq, nkv, nkv))
    at = [b + i for n, b in zip(lens, before) for i in range(n)]
    s["cos"], s["sin"] = _rope(at, hd)
    s["out"] = torch.full((rows + SPARE, nq * hd), 0.5, device="cuda")
    s["table"] = _table(pages)
    s["seq"] = torch.as_tensor([i for i, n in enumerate(lens) for _ in range(n)], dtype=torch.int64).cuda()
    s["at"] = torch.as_tensor(at, dtype=torch.int64).cuda()
    s["before"] = torch.as_tensor(before).cuda()
    s["longest"] = max(lens)
    s["pos0"], s["start"] = np.asarray(before, np.int32), np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
    if own:
        _handle(s, pages)
        s["ws"] = _workspace(s["lib"].tq_hip_prefill_packed_ws_bytes(s["kv"].h, case["n"], s["pos0"].ctypes.data,
                                                                     s["start"].ctypes.data))


def _prepare_weights(s, case, seed):
    nq, nkv, hd = s["heads"]
    lens, n, g = _lengths(case), case["n"], _generator(seed, 2)
    pages = _tables(seed, lens)
    s["pool"] = _pool(seed, case["shape"], sum(len(p) for p in pages))
    s["q"], s["k"], s["v"] = (_randn(g, n, h * hd) for h in (nq, nkv, nkv))
    s["cos"], s["sin"] = _rope([m - 1 for m in lens], hd)
    s["out"] = torch.zeros(n, nq * hd, device="cuda")
    s["pos"], s["max_pos"] = _int32([m - 1 for m in lens]), max(lens) - 1
    s["stride"] = max(lens) + 3
    # totals of earlier steps: a few tokens hold most of the weight
    s["total"] = (1.5 * _randn(g, n, nkv, s["stride"])).exp() * 0.05
    s["where"] = torch.arange(s["stride"], dtype=torch.int32, device="cuda").repeat(n, nkv, 1)
    s["table"] = _table(pages)
    if own:
        _handle(s, pages)
        s["ws"] = _workspace(s["lib"].tq_hip_decode_step_weights_ws_bytes(s["kv"].h, n, s["max_pos"]))


def _prepare_evict(s, case, seed):
    _, nkv, hd = s["heads"]
    lens, n, g = _lengths(case), case["n"], _generator(seed, 2)
    pages = _tables(seed, lens)
    s["pool"] = _pool(seed, case["shape"], sum(len(p) for p in pages))
    s["len"], s["max_len"], s["stride"] = _int32(lens), max(lens), max(lens)
    s["next"] = _int32([m + 100 for m in lens])     # a hundred tokens were evicted earlier
    s["total"] = (1.5 * _randn(g, n, nkv, s["stride"])).exp() * 0.05
    where = torch.arange(s["stride"], dtype=torch.int32, device="cuda")
    s["where"] = torch.where(where < 50, where, where + 100).repeat(n, nkv, 1)
    s["total_kept"], s["where_kept"] = torch.zeros_like(s["total"]), torch.zeros_like(s["where"])
    s["rules"] = (case["keep"], case["sinks"], case["recent"])
    s["table"] = _table(pages)
    if own:
        _handle(s, pages)
        s["ws"] = _workspace(s["lib"].tq_hip_kv_evict_ws_bytes(s["kv"].h, n, s["max_len"], case["keep"]))


def _prepare_logits(s, case, seed):
    rows, vocab, g = case["rows"], case["vocab"], _generator(seed, 2)
    stride, width = vocab + case["pad"], case["history"]
    s["vocab"] = vocab
    s["logits"] = 3 * _randn(g, rows, stride)
    s["out"], s["token"] = torch.zeros(rows, stride, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda")
    # frequent tokens come again: ids by a power law, each row its own
    u = torch.rand(rows, width, generator=g, device="cuda")
    s["history"] = ((u ** 3 * vocab).long() * 7919 % vocab).int()
    ends = torch.rand(rows, 2, generator=g, device="cuda")
    s["length"] = (width * (0.5 + 0.5 * ends[:, 0])).ceil().int()
    s["length"][0] = width
    s["prompt"] = (s["length"] * ends[:, 1]).int()
    s["repetition"] = 1 + 0.3 * torch.rand(rows, generator=g, device="cuda")
    s["presence"] = 0.5 * torch.rand(rows, generator=g, device="cuda")
    s["frequency"] = 0.2 * torch.rand(rows, generator=g, device="cuda")
    s["bias"] = s["mask"] = None
    if case["bias"]:
        ids = torch.randint(0, vocab, (rows, case["bias"]), generator=g, device="cuda", dtype=torch.int32)
        ids[:, -1] = ids[:, 0]       # the last entry of an id counts
        s["bias"] = (ids, 4 * _randn(g, rows, case["bias"]),
                     torch.full((rows,), case["bias"], dtype=torch.int32, device="cuda"))
    if case["grammar"]:
        # a grammar's states: anything, most words, a handful of symbols
        share = torch.tensor([1.0, 0.6, 0.0005], device="cuda")[torch.randint(0, 3, (rows,), generator=g, device="cuda")]
        words = -(-vocab // 32)
        bits = torch.rand(rows, words, 32, generator=g, device="cuda") < share[:, None, None]
        value = (bits.long() << torch.arange(32, device="cuda")).sum(-1)
        s["mask"] = torch.where(value >= 2 ** 31, value - 2 ** 32, value).int()
    if own:
        from tailorquantkernel_amd import native
        native.init(0)
        s.update(native=native, lib=native.load(), stream=_user_stream())
        s["ws"] = _workspace(s["lib"].tq_hip_logits_ws_bytes(rows, vocab))


def prepare(case, seed):
    s = {"op": case["op"], "heads": SHAPES[case["shape"]] if "shape" in case else None}
    {"packed": _prepare_packed, "weights": _prepare_weights, "evict": _prepare_evict,
     "logits": _prepare_logits}[case["op"]](s, case, seed)
    torch.cuda.synchronize()
    return s


# ---- the plain forms -------------------------------------------------------

def _rotate(x, cos, sin):
    """RoPE of rows x [rows][heads][hd], halves paired."""
    a, b = x.chunk(2, -1)
    c, s = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * s, a * s + b * c], -1)


def _quantize(x):
    """Scales and codes (as floats) of the 32-value blocks of x [..., hd]."""
    x = x.unflatten(-1, (-1, QK))
    # divided by a tensor: torch multiplies by the reciprocal of a number, which rounds otherwise
    d = x.abs().amax(-1, keepdim=True) / torch.full((), 127.0, device="cuda")
    inverse = torch.where(d != 0, 1 / d, torch.zeros_like(d))
    return d, (x * inverse).round()


def _append(pool, pages, slots, k, v):
    """Rows k and v [rows][kv heads][hd] into the given pages and slots."""
    for_cache = [torch.cat([d.view(torch.uint8), q.to(torch.int8).view(torch.uint8)], -1)
                 for d, q in (_quantize(k), _quantize(v))]
    pool[pages, :, 0, slots], pool[pages, :, 1, slots] = for_cache


def _gather(pool, table):
    """Keys and values [2][n][kv heads][tokens][hd] of the pages of each sequence."""
    got = pool[table]
    x = got[..., 4:].contiguous().view(torch.int8).float() * got[..., :4].contiguous().view(torch.float32)
    n, pages, nkv, _, _, nb, _ = x.shape
    return x.permute(3, 0, 2, 1, 4, 5, 6).reshape(2, n, nkv, pages * PAGE, nb * QK)


def _values_of_codes(x):
    d, codes = _quantize(x)
    return (d * codes).flatten(-2)


def _softmax(scores):
    """exp(scores) over its sum along the last axis, in place; every row has a score that is not masked."""
    scores -= scores.amax(-1, keepdim=True)
    scores.exp_()
    scores /= scores.sum(-1, keepdim=True)
    return scores


def _plain_packed(s):
    nq, nkv, hd = s["heads"]
    group, n = nq // nkv, s["table"].shape[0]
    rows = s["q"].shape[0]
    k = _rotate(s["k"].view(rows, nkv, hd), s["cos"], s["sin"])
    _append(s["pool"], s["table"][s["seq"], s["at"] // PAGE], s["at"] % PAGE, k, s["v"].view(rows, nkv, hd))
    keys, values = _gather(s["pool"], s["table"])
    q = _values_of_codes(_rotate(s["q"].view(rows, nq, hd), s["cos"], s["sin"]))
    index = s["at"] - s["before"][s["seq"]]
    padded = torch.zeros(n, s["longest"], nq, hd, device="cuda")
    padded[s["seq"], index] = q
    padded = padded.view(n, s["longest"], nkv, group, hd).permute(0, 2, 3, 1, 4).reshape(n, nkv, -1, hd)
    scores = (padded @ keys.transpose(-1, -2)).view(n, nkv, group, s["longest"], -1)
    scores *= hd ** -0.5
    token = torch.arange(scores.shape[-1], device="cuda")
    last = s["before"][:, None] + torch.arange(s["longest"], device="cuda")
    scores.masked_fill_((token > last[..., None])[:, None, None], -math.inf)
    out = _softmax(scores).view(n, nkv, -1, scores.shape[-1]) @ values
    out = out.view(n, nkv, group, s["longest"], hd).permute(0, 3, 1, 2, 4)
    s["out"][:rows] = out[s["seq"], index].reshape(rows, nq * hd)
    return {"out": s["out"], "cache": s["pool"]}


def _plain_weights(s):
    nq, nkv, hd = s["heads"]
    group, n = nq // nkv, s["table"].shape[0]
    pos = s["pos"].long()
    k = _rotate(s["k"].view(n, nkv, hd), s["cos"], s["sin"])
    _append(s["pool"], s["table"].gather(1, pos[:, None] // PAGE)[:, 0], pos % PAGE, k, s["v"].view(n, nkv, hd))
    keys, values = _gather(s["pool"], s["table"])
    q = _values_of_codes(_rotate(s["q"].view(n, nq, hd), s["cos"], s["sin"])).view(n, nkv, group, hd)
    scores = q @ keys.transpose(-1, -2)
    scores *= hd ** -0.5
    token = torch.arange(scores.shape[-1], device="cuda")
    scores.masked_fill_((token > pos[:, None])[:, None, None], -math.inf)
    p = _softmax(scores)
    s["out"].copy_((p @ values).view(n, nq * hd))
    added = p.sum(2)[..., :s["stride"]]
    total, where = s["total"][..., :added.shape[-1]], s["where"][..., :added.shape[-1]]
    token, new = token[:added.shape[-1]], pos[:, None, None]
    total.copy_(torch.where(token < new, total + added, torch.where(token == new, added, total)))
    where.copy_(torch.where(token == new, token.int(), where))
    return {"out": s["out"], "total": s["total"], "where": s["where"], "cache": s["pool"]}


def _plain_evict(s):
    keep, sinks, recent = s["rules"]
    n, nkv, width = s["total"].shape
    token = torch.arange(width, device="cuda")
    real = token < s["len"][:, None, None]
    safe = (s["where"] < sinks) | (s["where"] >= (s["next"] - recent)[:, None, None])
    key = torch.where(safe, torch.full_like(s["total"], math.inf), s["total"])
    # real tokens first, the largest totals first, ties by slot
    order = torch.where(real, key, torch.full_like(key, -math.inf)).sort(dim=-1, descending=True, stable=True).indices
    chosen = torch.zeros_like(key, dtype=torch.bool).scatter_(-1, order[..., :keep], True) & real
    inside = token < keep
    hole, mover = real & inside & ~chosen, chosen & ~inside
    # the i-th hole takes the i-th token from behind the budget
    i, h, to = hole.nonzero(as_tuple=True)
    source = mover.nonzero(as_tuple=True)[2]
    for_kept = [(s["total_kept"], s["total"]), (s["where_kept"], s["where"])]
    kept = chosen & inside
    moved = [torch.where(kept, old, new) for new, old in for_kept]
    for_moved = [x[i, h, source] for _, x in for_kept]
    moved[0][i, h, to], moved[1][i, h, to] = for_moved
    s["total_kept"].copy_(moved[0])
    s["where_kept"].copy_(moved[1])
    rows = s["pool"][s["table"][i, source // PAGE], h, :, source % PAGE]
    s["pool"][s["table"][i, to // PAGE], h, :, to % PAGE] = rows
    return {"total": s["total_kept"], "where": s["where_kept"], "cache": s["pool"]}


def _plain_logits(s):
    vocab = s["vocab"]
    x = s["logits"][:, :vocab]
    ids = s["history"].long()
    place = torch.arange(ids.shape[1], device="cuda")
    there = place < s["length"][:, None]
    count = torch.zeros(x.shape, dtype=torch.int32, device="cuda")
    seen = count.scatter_add(1, ids, there.int()) > 0
    count = count.scatter_add(1, ids, (there & (place >= s["prompt"][:, None])).int())
    by = s["repetition"][:, None]
    y = torch.where(seen, torch.where(x > 0, x / by, x * by), x)
    y = y - s["frequency"][:, None] * count
    y = y - torch.where(count > 0, s["presence"][:, None], torch.zeros_like(y))
    if s["bias"] is not None:
        ids, value, length = s["bias"]
        place = torch.arange(ids.shape[1], device="cuda")
        place = torch.where(place < length[:, None], place, torch.full_like(place, -1)).expand(ids.shape)
        last = torch.full(x.shape, -1, device="cuda").scatter_reduce(1, ids.long(), place, "amax")
        y = torch.where(last >= 0, y + value.gather(1, last.clamp(min=0)), y)
    if s["mask"] is not None:
        bit = torch.arange(32, device="cuda", dtype=torch.int32)
        allowed = ((s["mask"][..., None] >> bit) & 1).flatten(1)[:, :vocab] != 0
        y = torch.where(allowed, y, torch.full_like(y, -math.inf))
    s["out"][:, :vocab] = y
    best = y.amax(-1, keepdim=True)
    token = torch.arange(vocab, device="cuda")
    first = torch.where(y == best, token, torch.full_like(token, vocab)).amin(-1)
    s["token"].copy_(torch.where(best[:, 0] > -math.inf, first, torch.full_like(first, -1)))
    return {"out": s["out"], "token": s["token"]}


# ---- a pass ----------------------------------------------------------------

def _run_own(s):
    lib, st = s["lib"], s["stream"]
    ws, ws_bytes = s["ws"].data_ptr(), s["ws"].numel()
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    if s["op"] == "logits":
        bias = s["bias"] or (None, None, None)
        rules = s["native"].LogitsRules(
            ptr(s["history"]), s["history"].shape[1], ptr(s["length"]), ptr(s["prompt"]), ptr(s["repetition"]),
            ptr(s["presence"]), ptr(s["frequency"]), ptr(bias[0]), ptr(bias[1]),
            bias[0].shape[1] if s["bias"] else 0, ptr(bias[2]), ptr(s["mask"]),
            s["mask"].shape[1] if s["mask"] is not None else 0)
        rc = lib.tq_hip_logits_process(ptr(s["logits"]), s["logits"].shape[1], s["logits"].shape[0], s["vocab"],
                                       C.byref(rules), ptr(s["out"]), s["out"].shape[1], ptr(s["token"]), ws, ws_bytes,
                                       st)
        s["native"].check(rc, "tq_hip_logits_process")
        return {"out": s["out"], "token": s["token"]}
    kv = s["kv"].h
    if s["op"] == "packed":
        rc = lib.tq_hip_prefill_packed_async(kv, len(s["pos0"]), None, s["pos0"].ctypes.data, s["start"].ctypes.data,
                                             ptr(s["q"]), ptr(s["k"]), ptr(s["v"]), ptr(s["cos"]), ptr(s["sin"]),
                                             ptr(s["out"]), ws, ws_bytes, st)
        s["native"].check(rc, "tq_hip_prefill_packed_async")
        return {"out": s["out"], "cache": s["pool"]}
    n = s["total"].shape[0]
    if s["op"] == "weights":
        rc = lib.tq_hip_decode_step_weights_async(kv, n, None, ptr(s["pos"]), s["max_pos"], ptr(s["q"]), ptr(s["k"]),
                                                  ptr(s["v"]), ptr(s["cos"]), ptr(s["sin"]), ptr(s["out"]), None,
                                                  ptr(s["total"]), ptr(s["where"]), s["stride"], ws, ws_bytes, st)
        s["native"].check(rc, "tq_hip_decode_step_weights_async")
        return {"out": s["out"], "total": s["total"], "where": s["where"], "cache": s["pool"]}
    rc = lib.tq_hip_kv_evict_async(kv, n, None, ptr(s["len"]), s["max_len"], ptr(s["next"]), *s["rules"],
                                   ptr(s["total"]), ptr(s["where"]), ptr(s["total_kept"]), ptr(s["where_kept"]),
                                   s["stride"], ws, ws_bytes, st)
    s["native"].check(rc, "tq_hip_kv_evict_async")
    return {"total": s["total_kept"], "where": s["where_kept"], "cache": s["pool"]}


def run(state):
    if own:
        return _run_own(state)
    return {"packed": _plain_packed, "weights": _plain_weights, "evict": _plain_evict,
            "logits": _plain_logits}[state["op"]](state)


# ---- from the definitions, in 64 bits ---------------------------------------

def _exact_rows(x, heads, cos, sin):
    """Rows rotated where cos is given; the rotation's products and sums are fp32's by definition."""
    x = x.double().reshape(x.shape[0], heads, -1)
    if cos is None:
        return x
    half = x.shape[-1] // 2
    c, s = cos.double()[:, None], sin.double()[:, None]
    f = lambda t: t.float().double()  # noqa: E731
    low, high = x[..., :half], x[..., half:]
    return torch.cat((f(f(low * c) - f(high * s)), f(f(low * s) + f(high * c))), dim=2)


def _exact_codes(x):
    """What the block_q8 of rows x stand for: scale and inverse are fp32's by definition, codes to the nearest, ties to even."""
    blocks = x.reshape(*x.shape[:-1], -1, QK)
    scale = (blocks.abs().max(dim=-1, keepdim=True).values / 127.0).float()
    inverse = torch.where(scale > 0, (1.0 / scale.double()).float(), scale)
    codes = torch.round((blocks * inverse.double()).float())
    return (scale.double() * codes.double()).reshape(x.shape)


def _exact_cached(pool, pages, count):
    """Keys and values [kv heads][count][hd] that a sequence's pages hold."""
    raw = pool[torch.as_tensor(np.asarray(pages, np.int64)).cuda()]
    scale = raw[..., 0:4].contiguous().view(torch.float32).double()
    x = raw[..., 4:36].contiguous().view(torch.int8).double() * scale
    x = x.flatten(-2)                                   # [pages][kv heads][2][16][hd]
    k, v = (x[:, :, w].transpose(0, 1).flatten(1, 2)[:, :count] for w in (0, 1))
    return k, v


def _exact_attention(case, s, q, k, v, pos):
    """Rows q [m][heads][hd] at positions pos on keys k and values v [kv heads][tokens][hd]: outputs and weights."""
    nq, nkv, hd = s["heads"]
    out = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    weights = []
    token = torch.arange(k.shape[1], device="cuda")
    hidden = token[None, :] > pos[:, None]
    for h in range(nq):
        scores = (q[:, h] @ k[h // (nq // nkv)].t().contiguous()) / math.sqrt(hd)
        scores = scores.masked_fill(hidden, -math.inf)
        w = torch.exp(scores - scores.max(dim=1, keepdim=True).values)
        w = w / w.sum(dim=1, keepdim=True)
        out[:, h] = w @ v[h // (nq // nkv)]
        if case["op"] == "weights":
            weights.append(w[0])
    return out, weights


def _exact_sequences(case, seed):
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    nq, nkv, hd = s["heads"]
    lens, packed = _lengths(case), case["op"] == "packed"
    before = _contexts(case) if packed else [m - 1 for m in lens]
    pages = _tables(seed, [n + b for n, b in zip(lens, before)] if packed else lens)
    out = s["out"].double()
    total = None if packed else s["total"].double()
    at = 0
    for i, (m, b) in enumerate(zip(lens, before)):
        m = m if packed else 1
        if m == 0:
            continue
        rows = slice(at, at + m)
        at += m
        cos, sin = s["cos"][rows], s["sin"][rows]
        k, v = _exact_cached(s["pool"], pages[i], b)
        k = torch.cat((k, _exact_codes(_exact_rows(s["k"][rows], nkv, cos, sin)).transpose(0, 1)), dim=1)
        v = torch.cat((v, _exact_codes(_exact_rows(s["v"][rows], nkv, None, None)).transpose(0, 1)), dim=1)
        q = _exact_codes(_exact_rows(s["q"][rows], nq, cos, sin))
        o, w = _exact_attention(case, s, q, k, v, torch.arange(b, b + m, device="cuda"))
        out[rows] = o.reshape(m, nq * hd)
        if not packed:
            for h in range(nkv):
                mine = sum(w[h * (nq // nkv):(h + 1) * (nq // nkv)])
                total[i, h, :b] += mine[:b]
                total[i, h, b] = mine[b]
    return {"out": out, "cache": None} if packed else {"out": out, "total": total, "where": None, "cache": None}


def _exact_evict(case, seed):
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    total, where = s["total"].double().cpu().numpy(), s["where"].cpu().numpy()
    kept = np.zeros_like(total)
    for i, m in enumerate(_lengths(case)):
        upto = int(s["next"][i])
        for h in range(total.shape[1]):
            t, p = total[i, h, :m].copy(), where[i, h, :m]
            t[(p < case["sinks"]) | (p >= upto - case["recent"])] = np.inf
            best = np.sort(np.lexsort((np.arange(m), -t))[:case["keep"]])
            inside, behind = best[best < case["keep"]], best[best >= case["keep"]]
            holes = np.setdiff1d(np.arange(min(m, case["keep"])), inside)
            kept[i, h, inside], kept[i, h, holes] = total[i, h, inside], total[i, h, behind]
    return {"total": torch.from_numpy(kept), "where": None, "cache": None}


def _exact_logits(case, seed):
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    vocab = case["vocab"]
    out = np.zeros(s["out"].shape)
    a = {k: v.cpu().numpy() for k, v in s.items() if isinstance(v, torch.Tensor)}
    for r in range(case["rows"]):
        x = a["logits"][r, :vocab].astype(np.float64)
        text = a["history"][r, :a["length"][r]]
        seen = np.unique(text)
        by = float(a["repetition"][r])
        x[seen] = np.where(x[seen] > 0, x[seen] / by, x[seen] * by)
        said, times = np.unique(text[a["prompt"][r]:], return_counts=True)
        x[said] -= float(a["frequency"][r]) * times + float(a["presence"][r])
        if s["bias"] is not None:
            ids, value = s["bias"][0][r].tolist(), s["bias"][1][r].tolist()
            for t, b in dict(zip(ids, value)).items():
                x[t] += b
        if s["mask"] is not None:
            allowed = np.unpackbits(a["mask"][r].view(np.uint8), bitorder="little")[:vocab]
            x[allowed == 0] = -np.inf
        out[r, :vocab] = x
    return {"out": torch.from_numpy(out), "token": None}


def exact(case, seed):
    if case["op"] == "logits":
        return _exact_logits(case, seed)
    if case["op"] == "evict":
        return _exact_evict(case, seed)
    return _exact_sequences(case, seed)

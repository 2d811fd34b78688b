"""Operators for long contexts around the paged Q8 cache, as measurable cases.

* ``angles``: cos and sin rows of any positions, with the scalings that carry a
  model past the length it was trained on (tq_hip_rope_rows);
* ``rope``: the query and key heads of a fused projection, normalized and
  rotated in one pass, either pair layout, whole heads or a part of them
  (tq_hip_norm_rope);
* ``shared``: the decode step of a batch whose sequences begin with the same
  pages, a system prompt or a document, read once for all of a group
  (tq_hip_decode_step_shared_async);
* ``bounds``: the largest and smallest key of each block of cached tokens,
  channel by channel (tq_hip_kv_bounds_async);
* ``select``: the blocks whose keys can score highest with a query
  (tq_hip_kv_select_async);
* ``blocks``: the decode step over the selected blocks alone, which also keeps
  the bounds of the block that takes the new token
  (tq_hip_decode_step_blocks_async).

The head shapes are the benchmark's: 8 query / 2 kv heads of 64 (the small
parity shape), 32 / 8 of 128 (the 8B class) and 64 / 8 of 128 (the 70B class);
draw() adds one head per group and groups of three.

What is quantized (queries, keys and values as block_q8: 32 codes and a scale)
and the rounding of the bounds (bf16, outward) are defined bit for bit; a
block's score is real arithmetic in 64 bits.
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
EPS = 1e-6
SHAPES = {"small": (8, 2, 64), "8b": (32, 8, 128), "70b": (64, 8, 128), "single": (16, 16, 128), "triple": (24, 8, 64)}
SCALINGS = ("plain", "linear", "ntk", "bands", "yarn")
TRAINED, FACTOR = 8192, 8.0         # positions a model was trained on, and how far it is carried past them
BANDS, RAMP = (1.0, 4.0), (1.0, 32.0)   # turns over TRAINED: below the first scaled, above the second not


# ---- the cases -------------------------------------------------------------

def listed():
    return [
        # one decode step's rows of a serving batch, for all layers: latency
        {"name": "angles-step64", "op": "angles", "n": 64, "rot": 128, "scaling": "bands", "far": 65536},
        # the positions of many packed prompts
        {"name": "angles-prompts", "op": "angles", "n": 32768, "rot": 128, "scaling": "yarn", "far": 65536},
        # a serving batch's step between the projection and the cache: latency
        {"name": "rope-step64", "op": "rope", "shape": "8b", "n": 64, "rot": 128, "layout": "half", "norm": True,
         "scaling": "bands", "far": 65536},
        # long prompts on the large shape, pairs side by side, half of the head
        {"name": "rope-prompts", "op": "rope", "shape": "70b", "n": 4096, "rot": 64, "layout": "interleaved",
         "norm": True, "scaling": "yarn", "far": 65536},
        # a batch of conversations under one system prompt
        {"name": "shared-8b-system", "op": "shared", "shape": "8b", "n": 64, "groups": 1, "lone": 0, "prefix": 4096,
         "low": 16, "high": 512},
        # questions about a few long documents on the large shape
        {"name": "shared-70b-documents", "op": "shared", "shape": "70b", "n": 48, "groups": 3, "lone": 0,
         "prefix": 16384, "low": 32, "high": 1024},
        # the next turns of running conversations
        {"name": "bounds-8b-turns", "op": "bounds", "shape": "8b", "n": 24, "low": 8, "high": 512, "context": 4000,
         "block": 16},
        # long documents just cached
        {"name": "bounds-70b-32k", "op": "bounds", "shape": "70b", "n": 8, "low": 32768, "high": 32768, "context": 0,
         "block": 64},
        # one long conversation: latency
        {"name": "select-8b-one", "op": "select", "shape": "8b", "n": 1, "low": 16384, "high": 16384, "block": 16,
         "keep": 128, "sinks": 1, "recent": 8},
        # a batch of long contexts on the large shape
        {"name": "select-70b-32k", "op": "select", "shape": "70b", "n": 16, "low": 32768, "high": 32768, "block": 64,
         "keep": 64, "sinks": 1, "recent": 4},
        # one long conversation, an eighth of it attended to: latency
        {"name": "blocks-8b-one", "op": "blocks", "shape": "8b", "n": 1, "low": 16384, "high": 16384, "block": 16,
         "keep": 128},
        # a batch of long contexts on the large shape
        {"name": "blocks-70b-32k", "op": "blocks", "shape": "70b", "n": 16, "low": 30000, "high": 32768, "block": 64,
         "keep": 64},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["angles", "rope", "shared", "bounds", "select", "blocks"])
    if op == "angles":
        return {"op": op, "n": _log_int(rng, 1, 32768), "rot": 2 * rng.randint(1, 64), "scaling": rng.choice(SCALINGS),
                "far": _log_int(rng, 100, 1000000)}
    shape = rng.choice(["small", "8b", "8b", "70b", "single", "triple"])
    nq, nkv, hd = SHAPES[shape]
    if op == "rope":
        return {"op": op, "shape": shape, "n": _log_int(rng, 1, min(16384, 4096 * 72 * 128 // ((nq + nkv) * hd))),
                "rot": rng.choice([hd, hd // 2, 2 * rng.randint(1, hd // 2)]),
                "layout": rng.choice(["half", "interleaved"]), "norm": rng.random() < 0.6,
                "scaling": rng.choice(SCALINGS), "far": _log_int(rng, 100, 1000000)}
    if op == "shared":
        n = _log_int(rng, 2, 64)
        groups = rng.randint(1, max(1, min(4, n // 2)))
        lone = rng.choice([0, 0, rng.randint(0, min(4, n - groups))])
        high = _log_int(rng, 1, 1024)
        return {"op": op, "shape": shape, "n": n, "groups": groups, "lone": lone,
                "prefix": PAGE * _log_int(rng, 1, 16384 // PAGE), "low": rng.randint(1, high), "high": high}
    if op == "bounds":
        n = _log_int(rng, 1, 64)
        high = _log_int(rng, 1, min(32768, 8 * 32768 * 8 // (n * nkv)))
        return {"op": op, "shape": shape, "n": n, "low": rng.randint(1, high), "high": high,
                "context": rng.choice([0, _log_int(rng, 1, 4000)]), "block": rng.choice([16, 32, 48, 64, 128])}
    n, block = _log_int(rng, 1, 32), rng.choice([16, 32, 48, 64, 128])
    most = min(32768, 16 * 32768 * 8 // (n * nkv))
    budget = max(4, 16 * 4096 * 8 // (n * nkv * block))
    # a selection is made among blocks enough
    high = _log_int(rng, 32 * block if op == "select" else 64, most)
    low = high if rng.random() < 0.4 else rng.randint(max(1, high // 16), high)
    blocks = -(-high // block)
    case = {"op": op, "shape": shape, "n": n, "low": low, "high": high, "block": block}
    if op == "blocks":
        return {**case, "keep": _log_int(rng, 1, min(512, blocks, budget))}
    keep = _log_int(rng, 4, min(512, blocks // 2))
    return {**case, "keep": keep, "sinks": rng.randint(0, 2), "recent": rng.randint(1, max(1, keep // 2 - 2))}


def _lengths(case):
    """The sequences' lengths (of shared, behind the prefix; of bounds, the new tokens): the case's own, for every seed."""
    if case["low"] == case["high"]:
        return [case["high"]] * case["n"]
    r = random.Random(case["n"] * 1000003 + case["low"] * 101 + case["high"])
    return [case["high"]] + [r.randint(case["low"], case["high"]) for _ in range(case["n"] - 1)]


def _contexts(case):
    """Tokens whose blocks have bounds already."""
    r = random.Random(case["n"] * 7919 + case["context"])
    return [r.randint(0, case["context"]) for _ in range(case["n"])]


def _groups(case):
    """First queries of the groups (and the end of the last), and the groups' common tokens."""
    r = random.Random(case["n"] * 31 + case["groups"] * 7 + case["prefix"])
    n, m = case["n"] - case["lone"], case["groups"]
    cuts = sorted(r.sample(range(1, n), m - 1)) if m > 1 else []
    prefix = [case["prefix"]] + [PAGE * r.randint(1, case["prefix"] // PAGE) for _ in range(m - 1)]
    return [0] + cuts + [n], prefix


def _own_prefix(case):
    """Common tokens in front of each query's own."""
    start, prefix = _groups(case)
    at = [0] * case["n"]
    for a, b, p in zip(start[:-1], start[1:], prefix):
        at[a:b] = [p] * (b - a)
    return at


def _row(case):
    """Bytes of a token's keys and values in the cache."""
    _, nkv, hd = SHAPES[case["shape"]]
    return 2 * nkv * (hd // QK) * 36


def work(case):
    n = case["n"]
    if case["op"] == "angles":
        return {"bytes": n * (4 + 4 * case["rot"]), "flops": 0}
    nq, nkv, hd = SHAPES[case["shape"]]
    if case["op"] == "rope":
        return {"bytes": n * (4 + 8 * (nq + nkv) * hd), "flops": 0}
    lens, row, step = _lengths(case), _row(case), 4 * (2 * nq * hd + 2 * nkv * hd + hd)
    if case["op"] == "shared":
        prefix = _own_prefix(case)
        return {"bytes": (sum(_groups(case)[1]) + sum(lens)) * row + n * (row + step),
                "flops": 4 * nq * hd * (sum(lens) + sum(prefix))}
    block = case["block"]
    if case["op"] == "bounds":
        first = [c // block for c in _contexts(case)]
        whole = [c + m for c, m in zip(_contexts(case), lens)]
        return {"bytes": sum((m - f * block) * row // 2 + (-(-m // block) - f) * nkv * hd * 4
                             for m, f in zip(whole, first)), "flops": 0}
    if case["op"] == "select":
        return {"bytes": sum(-(-m // block) for m in lens) * nkv * hd * 4 + n * (4 * nq * hd + 4 * nkv * case["keep"]),
                "flops": 0}
    seen = sum(min(m, (case["keep"] - 1) * block + (m - 1) % block + 1) for m in lens)
    return {"bytes": seen * row + n * (row + step + 4 * nkv * case["keep"]), "flops": 4 * nq * hd * seen}


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


def _shared_tables(case, seed):
    """Page lists of a shared case: the group's pages, then the sequence's own."""
    start, prefix = _groups(case)
    lens = _lengths(case)
    parts = _tables(seed, prefix + lens)
    lists = list(parts[len(prefix):])
    for g, (a, b) in enumerate(zip(start[:-1], start[1:])):
        for i in range(a, b):
            lists[i] = np.concatenate([parts[g], lists[i]])
    return lists, sum(len(p) for p in parts)


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


def _library(s):
    from tailorquantkernel_amd import native
    native.init(0)
    s.update(native=native, lib=native.load(), stream=_user_stream())


def _handle(s, pages):
    """The framework's cache with the same contents, and its pool in place of the plain one."""
    _library(s)
    nq, nkv, hd = s["heads"]
    kv = s["native"].PagedKV(nq, nkv, hd, s["pool"].shape[0], len(pages), max(len(p) for p in pages))
    for i, p in enumerate(pages):
        kv.set_pages(i, p)
    base, nbytes, _ = kv.pool()
    pool = torch.as_tensor(_Memory(base, nbytes, kv), device="cuda").view(s["pool"].shape)
    pool.copy_(s["pool"])
    s.update(kv=kv, pool=pool)


def _workspace(nbytes):
    return torch.empty(max(16, nbytes), dtype=torch.uint8, device="cuda")


def _scaling(case):
    """(scaling, factor, trained length, low, high) of a case's positions."""
    low, high = {"bands": BANDS, "yarn": RAMP}.get(case["scaling"], (0.0, 0.0))
    return case["scaling"], FACTOR, TRAINED, low, high


def _rope_struct(s, case):
    n, (scaling, factor, trained, low, high) = s["native"], _scaling(case)
    kind = dict(zip(SCALINGS, (n.ROPE_PLAIN, n.ROPE_LINEAR, n.ROPE_NTK, n.ROPE_BANDS, n.ROPE_YARN)))[scaling]
    layout = n.ROPE_INTERLEAVED if case.get("layout") == "interleaved" else n.ROPE_HALF
    return n.Rope(case["rot"], layout, kind, trained, THETA, factor, low, high, 0.0)


def _prepare_angles(s, case, seed):
    g, n, half = _generator(seed, 2), case["n"], case["rot"] // 2
    s["pos"] = torch.randint(0, case["far"], (n,), generator=g, device="cuda", dtype=torch.int32)
    s["cos"], s["sin"] = torch.zeros(n, half, device="cuda"), torch.zeros(n, half, device="cuda")
    if own:
        _library(s)
        s["rope"] = _rope_struct(s, case)


def _prepare_rope(s, case, seed):
    nq, nkv, hd = s["heads"]
    g, n = _generator(seed, 2), case["n"]
    s["pos"] = torch.randint(0, case["far"], (n,), generator=g, device="cuda", dtype=torch.int32)
    # rows of a fused projection: q, k and v one behind the other
    s["rows"] = 2 * _randn(g, n, (nq + 2 * nkv) * hd)
    s["q_norm"] = s["k_norm"] = None
    if case["norm"]:
        s["q_norm"], s["k_norm"] = 1 + 0.2 * _randn(g, hd), 1 + 0.2 * _randn(g, hd)
    s["q_out"], s["k_out"] = torch.zeros(n, nq * hd, device="cuda"), torch.zeros(n, nkv * hd, device="cuda")
    if own:
        _library(s)
        s["rope"] = _rope_struct(s, case)


def _prepare_step(s, case, seed, last):
    """A step's q, k, v, cos, sin and output rows; last: the new tokens' positions."""
    nq, nkv, hd = s["heads"]
    n, g = case["n"], _generator(seed, 2)
    s["q"], s["k"], s["v"] = (_randn(g, n, h * hd) for h in (nq, nkv, nkv))
    s["cos"], s["sin"] = _rope(last, hd)
    s["out"] = torch.zeros(n, nq * hd, device="cuda")
    s["pos"], s["max_pos"] = _int32(last), max(last)


def _prepare_shared(s, case, seed):
    pages, total = _shared_tables(case, seed)
    s["pool"] = _pool(seed, case["shape"], total)
    before = _own_prefix(case)
    _prepare_step(s, case, seed, [p + m - 1 for p, m in zip(before, _lengths(case))])
    start, prefix = _groups(case)
    s["groups"] = (len(prefix), np.asarray(start, np.int32), np.asarray(prefix, np.int32))
    # for the plain form: each lone query is a group without common tokens
    counts = [b - a for a, b in zip(start[:-1], start[1:])] + [1] * case["lone"]
    heads = start[:-1] + list(range(start[-1], case["n"]))
    s["before"] = torch.as_tensor(before).cuda()
    s["group"] = torch.as_tensor([g for g, c in enumerate(counts) for _ in range(c)]).cuda()
    s["member"] = torch.as_tensor([j for c in counts for j in range(c)]).cuda()
    s["most"] = max(counts)
    common = -(-case["prefix"] // PAGE)
    s["prefix_table"] = _table([pages[i][:common] for i in heads])
    s["group_prefix"] = torch.as_tensor([before[i] for i in heads]).cuda()
    s["own_table"] = _table([p[b // PAGE:] for p, b in zip(pages, before)])
    if own:
        _handle(s, pages)
        m, start, prefix = s["groups"]
        s["ws"] = _workspace(s["lib"].tq_hip_decode_step_shared_ws_bytes(s["kv"].h, case["n"], s["max_pos"], m,
                                                                         start.ctypes.data, prefix.ctypes.data))


def _prepare_bounds(s, case, seed):
    _, nkv, hd = s["heads"]
    before, n = _contexts(case), case["n"]
    lens = [b + m for b, m in zip(before, _lengths(case))]
    pages = _tables(seed, lens)
    s["pool"] = _pool(seed, case["shape"], sum(len(p) for p in pages))
    s["table"], s["block"] = _table(pages), case["block"]
    s["from"], s["len"], s["max_len"] = _int32(before), _int32(lens), max(lens)
    s["stride"] = -(-max(lens) // case["block"]) + 1
    s["bounds"] = torch.full((n, nkv, s["stride"], 2, hd), 0.5, dtype=torch.bfloat16, device="cuda")
    if own:
        _handle(s, pages)


def _prepare_select(s, case, seed):
    nq, nkv, hd = s["heads"]
    lens, n, g = _lengths(case), case["n"], _generator(seed, 2)
    s["block"], s["rules"] = case["block"], (case["keep"], case["sinks"], case["recent"])
    last = [m - 1 for m in lens]
    s["q"] = _randn(g, n, nq * hd)
    s["cos"], s["sin"] = _rope(last, hd)
    s["pos"], s["max_pos"] = _int32(last), max(last)
    s["stride"] = max(last) // case["block"] + 1
    # a block's keys lie around its own centre, as a passage of text is about something
    size = (0.4 * _randn(g, nkv, 1, hd)).exp()
    centre, half = 0.5 * _randn(g, n, nkv, s["stride"], hd), 1.5 + 0.3 * _randn(g, n, nkv, s["stride"], hd)
    s["bounds"] = torch.stack([centre + half.abs(), centre - half.abs()], 3).mul_(size[..., None, :]).bfloat16()
    del centre, half
    s["list"] = torch.zeros(n, nkv, case["keep"], dtype=torch.int32, device="cuda")
    if own:
        _library(s)
        s["kv"] = s["native"].PagedKV(nq, nkv, hd, 1, n, -(-max(lens) // PAGE))
        s["ws"] = _workspace(s["lib"].tq_hip_kv_select_ws_bytes(s["kv"].h, n, s["max_pos"], case["block"], case["keep"]))


def _prepare_blocks(s, case, seed):
    _, nkv, hd = s["heads"]
    lens, n, block, keep = _lengths(case), case["n"], case["block"], case["keep"]
    pages = _tables(seed, lens)
    s["pool"] = _pool(seed, case["shape"], sum(len(p) for p in pages))
    _prepare_step(s, case, seed, [m - 1 for m in lens])
    # as a selection leaves them: the last block, and others in order
    g = _generator(seed, 3)
    count = ((s["pos"] // block) + 1).long()
    rank = torch.rand(n, nkv, int(count.max()), generator=g, device="cuda")
    at = torch.arange(rank.shape[-1], device="cuda")
    rank = torch.where(at == (count - 1)[:, None, None], torch.full_like(rank, 2.0), rank)
    rank = torch.where(at < count[:, None, None], rank, torch.full_like(rank, -1.0))
    chosen = rank.topk(min(keep, rank.shape[-1]), dim=-1)
    ids = torch.where(chosen.values >= 0, chosen.indices, torch.full_like(chosen.indices, 1 << 30)).sort(-1).values
    s["list"] = torch.full((n, nkv, keep), -1, dtype=torch.int32, device="cuda")
    s["list"][..., :ids.shape[-1]] = torch.where(ids < 1 << 30, ids, torch.full_like(ids, -1)).int()
    s["block"], s["keep"], s["table"] = block, keep, _table(pages)
    s["stride"] = s["max_pos"] // block + 2
    centre, half = _randn(g, n, nkv, s["stride"], hd), _randn(g, n, nkv, s["stride"], hd).abs()
    s["bounds"] = torch.stack([centre + half, centre - half], 3).bfloat16()
    if own:
        _handle(s, pages)
        s["ws"] = _workspace(s["lib"].tq_hip_decode_step_blocks_ws_bytes(s["kv"].h, n, s["max_pos"], block, keep))


def prepare(case, seed):
    s = {"op": case["op"], "heads": SHAPES[case["shape"]] if "shape" in case else None, "case": dict(case)}
    {"angles": _prepare_angles, "rope": _prepare_rope, "shared": _prepare_shared, "bounds": _prepare_bounds,
     "select": _prepare_select, "blocks": _prepare_blocks}[case["op"]](s, case, seed)
    torch.cuda.synchronize()
    return s


# ---- the plain forms -------------------------------------------------------

def _plain_rows(case, pos):
    """cos and sin [rows][rot / 2] of positions: angles in 64 bits, rounded once."""
    scaling, factor, trained, low, high = _scaling(case)
    rot = case["rot"]
    i = torch.arange(rot // 2, device="cuda", dtype=torch.float64)
    theta = THETA * factor ** (rot / (rot - 2)) if scaling == "ntk" and rot > 2 else THETA
    f = theta ** (-2 * i / rot)
    magnitude = 1.0
    if scaling == "linear":
        f = f / factor
    if scaling == "bands":
        turns = trained * f / (2 * math.pi)
        share = ((turns - low) / (high - low)).clamp(0, 1)
        f = f * share + f / factor * (1 - share)
    if scaling == "yarn":
        first, last = (rot * math.log(trained / (2 * math.pi * b)) / (2 * math.log(theta)) for b in (high, low))
        first, last = max(math.floor(first), 0), min(math.ceil(last), rot - 1)
        ramp = ((i - first) / max(last - first, 0.001)).clamp(0, 1)
        f = f * (1 - ramp) + f / factor * ramp
        magnitude = 0.1 * math.log(factor) + 1
    angle = pos.double()[:, None] * f
    return (angle.cos() * magnitude).float(), (angle.sin() * magnitude).float()


def _plain_angles(s):
    cos, sin = _plain_rows(s["case"], s["pos"])
    s["cos"].copy_(cos)
    s["sin"].copy_(sin)
    return {"cos": s["cos"], "sin": s["sin"]}


def _plain_turned(x, weight, cos, sin, rot, layout):
    """Heads x [rows][heads][hd], normalized where there are weights, their first rot values turned."""
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
    c, s = cos[:, None], sin[:, None]
    turned, rest = x[..., :rot], x[..., rot:]
    if layout == "half":
        a, b = turned.chunk(2, -1)
        return torch.cat([a * c - b * s, a * s + b * c, rest], -1)
    a, b = turned[..., 0::2], turned[..., 1::2]
    return torch.cat([torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2), rest], -1)


def _plain_rope(s):
    nq, nkv, hd = s["heads"]
    case, n = s["case"], s["rows"].shape[0]
    cos, sin = _plain_rows(case, s["pos"])
    q, k = s["rows"][:, :nq * hd].view(n, nq, hd), s["rows"][:, nq * hd:(nq + nkv) * hd].view(n, nkv, hd)
    s["q_out"].copy_(_plain_turned(q, s["q_norm"], cos, sin, case["rot"], case["layout"]).flatten(1))
    s["k_out"].copy_(_plain_turned(k, s["k_norm"], cos, sin, case["rot"], case["layout"]).flatten(1))
    return {"q": s["q_out"], "k": s["k_out"]}


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


def _values(rows):
    """What block_q8 rows [..., nb, 36] stand for: [..., hd]."""
    x = rows[..., 4:].contiguous().view(torch.int8).float() * rows[..., :4].contiguous().view(torch.float32)
    return x.flatten(-2)


def _gather(pool, table):
    """Keys and values [2][n][kv heads][tokens][hd] of the pages of each row of the table."""
    x = _values(pool[table])
    n, pages, nkv, _, _, hd = x.shape
    return x.permute(3, 0, 2, 1, 4, 5).reshape(2, n, nkv, pages * PAGE, hd)


def _values_of_codes(x):
    d, codes = _quantize(x)
    return (d * codes).flatten(-2)


def _softmax(scores):
    """exp(scores) over its sum along the last axis, in place; every row has a score that is not masked."""
    scores -= scores.amax(-1, keepdim=True)
    scores.exp_()
    scores /= scores.sum(-1, keepdim=True)
    return scores


def _step_rows(s):
    """A step's keys [n][nkv][hd], after RoPE, and queries [n][nkv][group][hd], as their codes stand for."""
    nq, nkv, hd = s["heads"]
    n = s["q"].shape[0]
    k = _rotate(s["k"].view(n, nkv, hd), s["cos"], s["sin"])
    q = _values_of_codes(_rotate(s["q"].view(n, nq, hd), s["cos"], s["sin"])).view(n, nkv, nq // nkv, hd)
    return k, s["v"].view(n, nkv, hd), q


def _plain_shared(s):
    nq, nkv, hd = s["heads"]
    n, group = s["q"].shape[0], nq // nkv
    pos, before = s["pos"].long(), s["before"]
    k, v, q = _step_rows(s)
    mine = pos - before
    _append(s["pool"], s["own_table"].gather(1, mine[:, None] // PAGE)[:, 0], mine % PAGE, k, v)
    keys, values = _gather(s["pool"], s["own_table"])
    own_scores = q @ keys.transpose(-1, -2) * hd ** -0.5
    token = torch.arange(keys.shape[2], device="cuda")
    own_scores.masked_fill_((token > mine[:, None])[:, None, None], -math.inf)
    # the common tokens, for all members of a group at once
    first_keys, first_values = _gather(s["pool"], s["prefix_table"])
    m, tokens = first_keys.shape[0], first_keys.shape[2]
    padded = torch.zeros(m, s["most"], nkv, group, hd, device="cuda")
    padded[s["group"], s["member"]] = q
    padded = padded.permute(0, 2, 1, 3, 4).reshape(m, nkv, -1, hd)
    scores = (padded @ first_keys.transpose(-1, -2)).view(m, nkv, s["most"], group, tokens)
    scores = scores.permute(0, 2, 1, 3, 4)[s["group"], s["member"]] * hd ** -0.5
    token = torch.arange(tokens, device="cuda")
    scores.masked_fill_((token >= before[:, None])[:, None, None], -math.inf)
    p = _softmax(torch.cat([scores, own_scores], -1))
    out = p[..., tokens:] @ values
    padded = torch.zeros(m, s["most"], nkv, group, tokens, device="cuda")
    padded[s["group"], s["member"]] = p[..., :tokens]
    padded = padded.permute(0, 2, 1, 3, 4).reshape(m, nkv, -1, tokens)
    first = (padded @ first_values).view(m, nkv, s["most"], group, hd).permute(0, 2, 1, 3, 4)
    s["out"].copy_((out + first[s["group"], s["member"]]).reshape(n, nq * hd))
    return {"out": s["out"], "cache": s["pool"]}


def _outward(high, low):
    """fp32 values in bf16, those of `high` rounded up and those of `low` down: [2 in front of the last axis]."""
    x = torch.stack([high, low], -2)
    bits = x.view(torch.int32)
    up = torch.tensor([[True], [False]], device="cuda")
    away = ((bits & 0xFFFF) != 0) & (up == (x > 0))
    return ((bits >> 16) + away.int()).to(torch.int16).view(torch.bfloat16)


def _plain_bounds(s):
    block, stride = s["block"], s["stride"]
    keys = _values(s["pool"][:, :, 0][s["table"]])           # [n][pages][kv head][16][hd]
    n, pages, nkv, _, hd = keys.shape
    keys = keys.permute(0, 2, 1, 3, 4).reshape(n, nkv, pages * PAGE, hd)[:, :, :s["max_len"]]
    there = torch.arange(keys.shape[2], device="cuda") < s["len"][:, None]
    there = there[:, None, :, None]
    blocks = -(-keys.shape[2] // block)
    room = (0, 0, 0, blocks * block - keys.shape[2])
    most = torch.nn.functional.pad(keys.masked_fill(~there, -math.inf), room, value=-math.inf)
    most = most.view(n, nkv, blocks, block, hd).amax(3)
    least = torch.nn.functional.pad(keys.masked_fill(~there, math.inf), room, value=math.inf)
    least = least.view(n, nkv, blocks, block, hd).amin(3)
    at = torch.arange(blocks, device="cuda")
    new = (at >= (s["from"] // block)[:, None]) & (at * block < s["len"][:, None])
    into = s["bounds"][:, :, :blocks]
    into.copy_(torch.where(new[:, None, :, None, None], _outward(most, least), into))
    return {"bounds": s["bounds"]}


def _plain_select(s):
    nq, nkv, hd = s["heads"]
    keep, sinks, recent = s["rules"]
    n = s["q"].shape[0]
    q = _rotate(s["q"].view(n, nq, hd), s["cos"], s["sin"]).view(n, nkv, nq // nkv, hd).double()
    by = torch.stack([q.clamp(min=0).sum(2), q.clamp(max=0).sum(2)], 2).flatten(2)     # [n][nkv][2 hd]
    score = (s["bounds"].flatten(3).double() @ by[..., None])[..., 0]
    at = torch.arange(score.shape[-1], device="cuda")
    count = (s["pos"] // s["block"] + 1)[:, None, None]
    safe = (at < sinks) | (at >= count - recent)
    score = torch.where(safe, torch.full_like(score, math.inf), score)
    score = torch.where(at < count, score, torch.full_like(score, -math.inf))
    order = score.sort(dim=-1, descending=True, stable=True).indices[..., :keep]
    none = score.shape[-1]
    order = torch.where(order < count, order, torch.full_like(order, none)).sort(-1).values
    s["list"][..., :order.shape[-1]] = torch.where(order < none, order, torch.full_like(order, -1)).int()
    s["list"][..., order.shape[-1]:] = -1
    return {"list": s["list"]}


def _plain_blocks(s):
    nq, nkv, hd = s["heads"]
    n, block = s["q"].shape[0], s["block"]
    pos = s["pos"].long()
    k, v, q = _step_rows(s)
    _append(s["pool"], s["table"].gather(1, pos[:, None] // PAGE)[:, 0], pos % PAGE, k, v)
    # the listed blocks' tokens of each kv head; entries of -1 and tokens past the new one are masked
    ids = s["list"].long()
    token = (ids[..., None] * block + torch.arange(block, device="cuda")).flatten(2)
    seen = (ids >= 0).repeat_interleave(block, -1) & (token <= pos[:, None, None])
    token = torch.where(seen, token, torch.zeros_like(token))
    pages = s["table"].gather(1, (token // PAGE).flatten(1)).view(token.shape)
    head = torch.arange(nkv, device="cuda")[:, None]
    rows = _values(s["pool"][pages, head, :, token % PAGE])        # [n][nkv][tokens][2][hd]
    scores = q @ rows[..., 0, :].transpose(-1, -2) * hd ** -0.5
    scores.masked_fill_(~seen[:, :, None], -math.inf)
    s["out"].copy_((_softmax(scores) @ rows[..., 1, :]).reshape(n, nq * hd))
    # the new key into its block's bounds, which begin with the block's first token
    d, codes = _quantize(k)
    key = (d * codes).flatten(-2)
    i, at = torch.arange(n, device="cuda"), pos // block
    was, new = s["bounds"][i, :, at], _outward(key, key)             # [n][nkv][2][hd]
    first = (pos % block == 0)[:, None, None]
    both = torch.stack([torch.where(first, new[..., 0, :], torch.maximum(was[..., 0, :], new[..., 0, :])),
                        torch.where(first, new[..., 1, :], torch.minimum(was[..., 1, :], new[..., 1, :]))], 2)
    s["bounds"][i, :, at] = both
    return {"out": s["out"], "cache": s["pool"], "bounds": s["bounds"]}


# ---- a pass ----------------------------------------------------------------

def _run_own(s):
    lib, st, op, check = s["lib"], s["stream"], s["op"], s["native"].check
    ptr = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    if op == "angles":
        check(lib.tq_hip_rope_rows(C.byref(s["rope"]), s["pos"].shape[0], ptr(s["pos"]), ptr(s["cos"]), ptr(s["sin"]),
                                   st), "tq_hip_rope_rows")
        return {"cos": s["cos"], "sin": s["sin"]}
    nq, nkv, hd = s["heads"]
    if op == "rope":
        rows, heads = s["rows"], s["native"].Heads
        q = heads(ptr(rows), nq, rows.shape[1], ptr(s["q_norm"]), ptr(s["q_out"]), nq * hd)
        k = heads(ptr(rows) + 4 * nq * hd, nkv, rows.shape[1], ptr(s["k_norm"]), ptr(s["k_out"]), nkv * hd)
        check(lib.tq_hip_norm_rope(C.byref(s["rope"]), hd, rows.shape[0], ptr(s["pos"]), C.byref(q), C.byref(k), EPS,
                                   st), "tq_hip_norm_rope")
        return {"q": s["q_out"], "k": s["k_out"]}
    kv = s["kv"].h
    if op == "bounds":
        check(lib.tq_hip_kv_bounds_async(kv, s["len"].shape[0], None, ptr(s["from"]), ptr(s["len"]), s["max_len"],
                                         s["block"], ptr(s["bounds"]), s["stride"], st), "tq_hip_kv_bounds_async")
        return {"bounds": s["bounds"]}
    n, ws, ws_bytes = s["q"].shape[0], s["ws"].data_ptr(), s["ws"].numel()
    if op == "select":
        check(lib.tq_hip_kv_select_async(kv, n, None, ptr(s["pos"]), s["max_pos"], s["block"], *s["rules"], ptr(s["q"]),
                                         ptr(s["cos"]), ptr(s["sin"]), ptr(s["bounds"]), s["stride"], ptr(s["list"]),
                                         ws, ws_bytes, st), "tq_hip_kv_select_async")
        return {"list": s["list"]}
    step = (ptr(s["q"]), ptr(s["k"]), ptr(s["v"]), ptr(s["cos"]), ptr(s["sin"]), ptr(s["out"]))
    if op == "shared":
        m, start, prefix = s["groups"]
        check(lib.tq_hip_decode_step_shared_async(kv, n, None, ptr(s["pos"]), s["max_pos"], m, start.ctypes.data,
                                                  prefix.ctypes.data, *step, ws, ws_bytes, st),
              "tq_hip_decode_step_shared_async")
        return {"out": s["out"], "cache": s["pool"]}
    check(lib.tq_hip_decode_step_blocks_async(kv, n, None, ptr(s["pos"]), s["max_pos"], s["block"], s["keep"],
                                              ptr(s["list"]), *step, ptr(s["bounds"]), s["stride"], ws, ws_bytes, st),
          "tq_hip_decode_step_blocks_async")
    return {"out": s["out"], "cache": s["pool"], "bounds": s["bounds"]}


def run(state):
    if own:
        return _run_own(state)
    return {"angles": _plain_angles, "rope": _plain_rope, "shared": _plain_shared, "bounds": _plain_bounds,
            "select": _plain_select, "blocks": _plain_blocks}[state["op"]](state)


# ---- from the definitions, in 64 bits ---------------------------------------

def _exact_frequencies(case):
    """Radians per position of each pair, and what cos and sin are multiplied by."""
    rot, s = case["rot"], FACTOR
    base, magnitude, out = THETA, 1.0, []
    if case["scaling"] == "ntk" and rot > 2:
        base = THETA * s ** (rot / (rot - 2.0))
    if case["scaling"] == "yarn":
        magnitude = 1.0 + 0.1 * math.log(s)
        edge = lambda turns: rot * math.log(TRAINED / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))  # noqa: E731
        lo, hi = max(0, math.floor(edge(RAMP[1]))), min(rot - 1, math.ceil(edge(RAMP[0])))
    for i in range(rot // 2):
        w = math.exp(-2.0 * i / rot * math.log(base))
        if case["scaling"] == "linear":
            w /= s
        elif case["scaling"] == "bands":
            t = TRAINED / (2.0 * math.pi / w)
            if t < BANDS[0]:
                w /= s
            elif t <= BANDS[1]:
                x = (t - BANDS[0]) / (BANDS[1] - BANDS[0])
                w = (1.0 - x) * w / s + x * w
        elif case["scaling"] == "yarn":
            x = min(1.0, max(0.0, (i - lo) / max(0.001, hi - lo)))
            w = x * (w / s) + (1.0 - x) * w
        out.append(w)
    return np.asarray(out), magnitude


def _exact_angles(case, s):
    w, magnitude = _exact_frequencies(case)
    angle = s["pos"].cpu().numpy().astype(np.float64)[:, None] * w[None, :]
    return magnitude * np.cos(angle), magnitude * np.sin(angle)


def _exact_rope(case, s):
    nq, nkv, hd = s["heads"]
    cos, sin = (torch.from_numpy(x).cuda()[:, None, :] for x in _exact_angles(case, s))
    rows, rot, n = s["rows"].double(), case["rot"], case["n"]
    got = []
    for at, heads, weight in ((0, nq, s["q_norm"]), (nq * hd, nkv, s["k_norm"])):
        x = rows[:, at:at + heads * hd].reshape(n, heads, hd).clone()
        if weight is not None:
            x = x / torch.sqrt(EPS + (x * x).sum(2, keepdim=True) / hd) * weight.double()
        pairs = torch.arange(rot // 2, device="cuda")
        lower, upper = (pairs, pairs + rot // 2) if case["layout"] == "half" else (2 * pairs, 2 * pairs + 1)
        a, b = x[..., lower], x[..., upper]
        x[..., lower], x[..., upper] = a * cos - b * sin, b * cos + a * sin
        got.append(x.reshape(n, heads * hd))
    return {"q": got[0], "k": got[1]}


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


def _exact_steps(case, s, seed):
    """Outputs of a step, one sequence after the other, over all its tokens or those of the listed blocks; the new keys."""
    nq, nkv, hd = s["heads"]
    pages = _shared_tables(case, seed)[0] if case["op"] == "shared" else _tables(seed, _lengths(case))
    out, new_keys = torch.empty(case["n"], nq, hd, dtype=torch.float64, device="cuda"), []
    for i in range(case["n"]):
        row, pos = slice(i, i + 1), int(s["pos"][i])
        cos, sin = s["cos"][row], s["sin"][row]
        k, v = _exact_cached(s["pool"], pages[i], pos)
        new = _exact_codes(_exact_rows(s["k"][row], nkv, cos, sin)).transpose(0, 1)
        new_keys.append(new[:, 0])
        k = torch.cat((k, new), dim=1)
        v = torch.cat((v, _exact_codes(_exact_rows(s["v"][row], nkv, None, None)).transpose(0, 1)), dim=1)
        q = _exact_codes(_exact_rows(s["q"][row], nq, cos, sin))[0]
        for h in range(nkv):
            mine = q[h * (nq // nkv):(h + 1) * (nq // nkv)]
            kh, vh = k[h], v[h]
            if case["op"] == "blocks":
                blocks = [b for b in s["list"][i, h].tolist() if b >= 0]
                at = [t for b in blocks for t in range(b * case["block"], min(pos + 1, (b + 1) * case["block"]))]
                at = torch.as_tensor(at, device="cuda")
                kh, vh = kh[at], vh[at]
            w = (mine @ kh.t().contiguous()) / math.sqrt(hd)
            w = torch.exp(w - w.max(dim=1, keepdim=True).values)
            out[i, h * (nq // nkv):(h + 1) * (nq // nkv)] = (w / w.sum(dim=1, keepdim=True)) @ vh
    return out.reshape(case["n"], nq * hd), new_keys


def _exact_bounds(case, s, seed):
    out, block = s["bounds"].double(), case["block"]
    before = _contexts(case)
    lens = [b + m for b, m in zip(before, _lengths(case))]
    for i, pages in enumerate(_tables(seed, lens)):
        k, _ = _exact_cached(s["pool"], pages, lens[i])
        for b in range(before[i] // block, -(-lens[i] // block)):
            keys = k[:, b * block:(b + 1) * block]
            out[i, :, b, 0], out[i, :, b, 1] = keys.max(dim=1).values, keys.min(dim=1).values
    return {"bounds": out}


def exact(case, seed):
    global own
    if case["op"] == "select":
        return None     # whole numbers: the plain form, in 64 bits, has them
    was, own = own, False
    s = prepare(case, seed)
    own = was
    if case["op"] == "angles":
        cos, sin = _exact_angles(case, s)
        return {"cos": torch.from_numpy(cos), "sin": torch.from_numpy(sin)}
    if case["op"] == "rope":
        return _exact_rope(case, s)
    if case["op"] == "bounds":
        return _exact_bounds(case, s, seed)
    out, keys = _exact_steps(case, s, seed)
    if case["op"] == "shared":
        return {"out": out, "cache": None}
    bounds = s["bounds"].double()
    for i, key in enumerate(keys):
        pos = int(s["pos"][i])
        at, first = pos // case["block"], pos % case["block"] == 0
        was = bounds[i, :, at].clone()
        bounds[i, :, at, 0] = key if first else torch.maximum(was[:, 0], key)
        bounds[i, :, at, 1] = key if first else torch.minimum(was[:, 1], key)
    return {"out": out, "cache": None, "bounds": bounds}

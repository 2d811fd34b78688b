"""Bounds of blocks of cached keys, the choice of blocks by them, and the decode
step over the chosen ones, against their definitions in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

from tests.hip_graphs import Graphs
from tests.serving import PAGE, QK, Cache, attention, quantized, rope_rows, rotated

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nat():
    from tailorquantkernel_amd import native
    native.init(0)
    return native


# ---- bounds ------------------------------------------------------------------

def outward(x, up):
    """fp32 values as bf16 bits, rounded up or down."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    away = ((u & 0xFFFF) != 0) & ((x > 0) if up else (x < 0))
    return ((u >> 16) + away).astype(np.uint16)


def value(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


def bounds_of(rows):
    """Keys' blocks rows [tokens][nkv][nb]: bounds [nkv][2][hd] as bf16 bits."""
    with np.errstate(invalid="ignore", over="ignore"):
        keys = (rows["q"].astype(np.float32) * rows["d"][..., None].astype(np.float32)).reshape(*rows.shape[:2], -1)
    nan = np.isnan(keys)
    most = np.where(nan, -np.inf, keys).astype(np.float32).max(0, initial=-np.inf)
    least = np.where(nan, np.inf, keys).astype(np.float32).min(0, initial=np.inf)
    return np.stack([outward(most, True), outward(least, False)], 1)


def expected_bounds(cache, was, block, seqs, start, lens, max_len):
    want = was.copy()
    for s, a, m in zip(seqs, start, lens):
        m = min(m, max_len)
        for b in range(max(a, 0) // block, -(-m // block)) if max(a, 0) < m else ():
            rows = cache.rows(s, min(m, (b + 1) * block))[b * block:, :, 0]
            want[s, :, b] = bounds_of(rows)
    return want


class Bounds:
    def __init__(self, cache, block, stride, seed=0):
        self.c, self.block, self.stride = cache, block, stride
        shape = (len(cache.pages), cache.nkv, stride, 2, cache.hd)
        self.host = np.random.default_rng(seed).integers(0, 0x7F00, shape).astype(np.uint16)   # finite numbers
        self.dev = cache.up(self.host)

    def make(self, lens, start=None, seqs=None, max_len=None, stream=None):
        c = self.c
        self.max_len = max_len or max(max(lens), 1)
        self.hold = [None if a is None else c.up(np.asarray(a, np.int32)) for a in (seqs, start, lens)]
        p = [None if b is None else b.ptr for b in self.hold]
        c.nat.check(c.lib.tq_hip_kv_bounds_async(c.kv.h, len(lens), p[0], p[1], p[2], self.max_len, self.block,
                                                 self.dev.ptr, self.stride, stream), "bounds")
        c.sync()
        return self.dev.download(self.host.shape, np.uint16)


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("block", [16, 48, 128, 1024])
def test_bounds(nat, oracle, hd, block):
    lens = [1, 15, 16, 17, 0, 300, 1500]
    c = Cache(nat, oracle, hd + block, 4, 2, hd, lens)
    b = Bounds(c, block, -(-1500 // block) + 2)
    want = expected_bounds(c, b.host, block, range(7), [0] * 7, lens, 1500)
    assert np.array_equal(b.make(lens), want)


@pytest.mark.parametrize("block", [16, 64])
def test_bounds_of_new_tokens(nat, oracle, block):
    """Only the blocks that hold new tokens are made again, from all their tokens."""
    lens, start = [200, 64, 65, 500, 33], [199, 64, 64, 130, -5]
    c = Cache(nat, oracle, block, 8, 2, 64, lens)
    b = Bounds(c, block, 40)
    want = expected_bounds(c, b.host, block, range(5), start, lens, 500)
    assert np.array_equal(b.make(lens, start), want)


def test_bounds_of_named_sequences_up_to_a_length(nat, oracle):
    lens = [100, 200, 300]
    c = Cache(nat, oracle, 1, 4, 4, 128, lens)
    b = Bounds(c, 32, 10)
    want = expected_bounds(c, b.host, 32, [2, 0], [0, 0], [300, 100], 150)
    assert np.array_equal(b.make([300, 100, 50, 60], seqs=[2, 0, 3, -1], max_len=150), want)


def test_bounds_of_many_sequences(nat, oracle):
    """More blocks than waves of a launch, and fewer."""
    lens = [int(x) for x in np.random.default_rng(9).integers(1, 200, 40)]
    c = Cache(nat, oracle, 4, 8, 8, 64, lens)
    b = Bounds(c, 16, 13)
    assert np.array_equal(b.make(lens), expected_bounds(c, b.host, 16, range(40), [0] * 40, lens, max(lens)))
    c = Cache(nat, oracle, 4, 1, 1, 32, [9000])
    b = Bounds(c, 16, 563)
    assert np.array_equal(b.make([9000]), expected_bounds(c, b.host, 16, [0], [0], [9000], 9000))


def test_bounds_of_keys_that_are_no_numbers(nat, oracle):
    c = Cache(nat, oracle, 2, 2, 2, 64, [64])
    k = c.pool[c.pages[0]]
    k["d"][0, :, 0, 3, 0], k["d"][1, :, 0, 5, 1], k["d"][2, :, 0, 7, 0] = np.nan, np.inf, -1.5
    k["d"][3, :, 0, :, 0] = np.nan                 # a block without a number in the first 32 channels
    k["d"][3, :, 0, 2, 1] = 3e38                   # code * scale overflows
    c.pool[c.pages[0]] = k
    c.upload()
    b = Bounds(c, 16, 4)
    got = b.make([64])
    assert np.array_equal(got, expected_bounds(c, b.host, 16, [0], [0], [64], 64))
    assert (value(got[0, :, 3, 0, :32]) == -np.inf).all() and (value(got[0, :, 3, 1, :32]) == np.inf).all()


def test_bounds_hold_every_key(nat, oracle):
    c = Cache(nat, oracle, 3, 2, 1, 128, [256])
    got = Bounds(c, 64, 4).make([256])
    from tests.serving import values
    keys = values(c.rows(0, 256)[:, :, 0]).reshape(4, 64, 1, 128)
    assert (value(got[0, 0, :, 0]) >= keys.max(1)[:, 0]).all() and (value(got[0, 0, :, 1]) <= keys.min(1)[:, 0]).all()


# ---- selection -----------------------------------------------------------------

def chosen(bounds, q, count, keep, sinks, recent, hd, group):
    """A kv head's list: bounds [blocks][2][hd] as bits, q [group][hd] after RoPE."""
    if count <= keep:
        return list(range(count)) + [-1] * (keep - count)
    m, q = value(bounds).astype(np.float64), q.astype(np.float64)
    up, down = np.where(q <= 0, 0.0, q).sum(0), np.where(q >= 0, 0.0, q).sum(0)
    with np.errstate(invalid="ignore"):
        s = m[:count, 0] @ up + m[:count, 1] @ down
    s = np.where(np.isnan(s), -np.inf, s)
    at = np.arange(count)
    free = at[(at >= sinks) & (at < count - recent)]
    best = free[np.lexsort((free, -s[free]))][:keep - sinks - recent]
    return sorted([*range(sinks), *best.tolist(), *range(count - recent, count)])


class Select:
    """Queries at pos over random bounds; a cache of one page (no key is read)."""

    def __init__(self, nat, oracle, seed, nq, nkv, hd, pos, block, keep, sinks=1, recent=1, seqs=None, rope=True,
                 max_seqs=None, max_pos=None):
        self.nat, self.lib, r = nat, nat.load(), np.random.default_rng(seed)
        self.nq, self.nkv, self.hd, self.n = nq, nkv, hd, len(pos)
        self.pos, self.seqs, self.rules = list(pos), seqs, (block, keep, sinks, recent)
        self.max_pos = max(max(pos), 0) if max_pos is None else max_pos
        self.stride = self.max_pos // block + 3
        seqs_n = max_seqs or self.n
        self.kv = nat.PagedKV(nq, nkv, hd, 1, seqs_n, self.max_pos // PAGE + 1)
        centre = r.standard_normal((seqs_n, nkv, self.stride, hd), dtype=np.float32)
        half = np.abs(r.standard_normal(centre.shape, dtype=np.float32))
        self.bounds = np.stack([outward(centre + half, True), outward(centre - half, False)], 3)
        self.q = r.standard_normal((self.n, nq, hd), dtype=np.float32)
        self.cos, self.sin = rope_rows(oracle, hd, [max(p, 0) for p in pos]) if rope else (None, None)
        self.turned = rotated(oracle, self.q, self.cos, self.sin)

    def upload(self):
        up = self.nat.DeviceBuffer.from_numpy
        self.dev = {k: None if a is None else up(np.ascontiguousarray(a)) for k, a in (
            ("seq", None if self.seqs is None else np.asarray(self.seqs, np.int32)), ("pos", np.asarray(self.pos, np.int32)),
            ("q", self.q), ("cos", self.cos), ("sin", self.sin), ("bounds", self.bounds),
            ("list", np.full((self.n, self.nkv, self.rules[1]), -7, np.int32)))}
        self.ws_bytes = self.lib.tq_hip_kv_select_ws_bytes(self.kv.h, self.n, self.max_pos, *self.rules[:2])
        assert self.ws_bytes > 0
        self.ws = up(np.full(self.ws_bytes, 0xFF, np.uint8))

    def launch(self, stream=None):
        p = {k: None if b is None else b.ptr for k, b in self.dev.items()}
        self.nat.check(self.lib.tq_hip_kv_select_async(
            self.kv.h, self.n, p["seq"], p["pos"], self.max_pos, *self.rules, p["q"], p["cos"], p["sin"], p["bounds"],
            self.stride, p["list"], self.ws.ptr, self.ws_bytes, stream), "select")

    def run(self):
        self.upload()
        self.launch()
        return self.result()

    def result(self):
        self.nat.check(self.lib.tq_hip_device_synchronize(), "sync")
        return self.dev["list"].download((self.n, self.nkv, self.rules[1]), np.int32)

    def expected(self):
        block, keep, sinks, recent = self.rules
        g = self.nq // self.nkv
        out = np.full((self.n, self.nkv, keep), -1, np.int32)
        for i, p in enumerate(self.pos):
            s = i if self.seqs is None else self.seqs[i]
            if p < 0 or not 0 <= s < self.bounds.shape[0]:
                continue
            for h in range(self.nkv):
                out[i, h] = chosen(self.bounds[s, h], self.turned[i, h * g:(h + 1) * g], p // block + 1, keep, sinks,
                                   recent, self.hd, g)
        return out


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("group", [1, 3, 4, 8])
def test_select_shapes(nat, oracle, hd, group):
    s = Select(nat, oracle, hd + group, 2 * group, 2, hd, [0, 15, 16, 300, 1023, 2500, 5000], 16, 20, 2, 3)
    assert np.array_equal(s.run(), s.expected())


@pytest.mark.parametrize("keep,sinks,recent", [(1, 0, 1), (2, 1, 1), (7, 0, 1), (64, 1, 4), (100, 50, 50), (312, 0, 1),
                                               (313, 2, 2), (600, 5, 9)])
def test_select_rules(nat, oracle, keep, sinks, recent):
    s = Select(nat, oracle, keep, 8, 2, 64, [5000, 4999, 40, 31], 16, keep, sinks, recent, rope=False)
    assert np.array_equal(s.run(), s.expected())


@pytest.mark.parametrize("blocks", [2, 63, 64, 65, 1023, 1024, 1025, 4095, 4096, 4097, 6000, 40000])
@pytest.mark.parametrize("keep", [1, 33, 500])
def test_select_lengths(nat, oracle, blocks, keep):
    """Either side of the length where scores get a launch of their own."""
    s = Select(nat, oracle, blocks, 2, 1, 32, [16 * blocks - 1, 16 * blocks - 16], 16, keep, 0, 1)
    assert np.array_equal(s.run(), s.expected())


@pytest.mark.parametrize("blocks", [511, 512, 513, 1030, 4096, 4097])
@pytest.mark.parametrize("hd", [32, 128])
def test_select_for_a_batch(nat, oracle, blocks, hd):
    """Heads enough that scores get no launch of their own, up to the length where they do."""
    pos = [16 * blocks - 1, *(int(p) for p in np.random.default_rng(blocks).integers(0, 16 * blocks, 15))]
    s = Select(nat, oracle, blocks, 8, 8, hd, pos, 16, 70, 2, 3, rope=False)
    assert np.array_equal(s.run(), s.expected())


def test_select_among_equals(nat, oracle):
    """Equal scores go to the lower block, also where many share the edge and where all do."""
    s = Select(nat, oracle, 1, 4, 2, 64, [6400, 6400, 6400, 6400], 16, 40, 1, 2, rope=False)
    s.bounds[1] = s.bounds[1, :, :1]                      # all alike
    s.bounds[2, :, 100:300] = s.bounds[2, :, 7:8]         # many alike
    s.bounds[3, :, 0:402:2] = s.bounds[3, :, 1:403:2]     # pairs
    got, want = s.run(), s.expected()
    assert np.array_equal(got, want)
    assert np.array_equal(got[1, 0, :38], np.arange(38))


def test_select_near_equals(nat, oracle):
    """Scores that differ in the last bit of a bound rank as they are: 2^-8 of one channel beside 64 sums."""
    s = Select(nat, oracle, 2, 1, 1, 64, [16 * 800 - 1], 16, 30, 0, 1, rope=False)
    s.q = s.turned = np.abs(s.q) + 0.5
    s.bounds[0, 0] = s.bounds[0, 0, 0]
    order = np.random.default_rng(3).permutation(790)
    s.bounds[0, 0, order, 0, 0] = 0x4000 + np.arange(790)     # one more each
    got = s.run()
    assert np.array_equal(got, s.expected())
    assert set(got[0, 0, :29]) == set(order[-29:])


def test_select_infinite_and_nan(nat, oracle):
    s = Select(nat, oracle, 4, 2, 2, 64, [16 * 50 - 1, 16 * 50 - 1, 16 * 50 - 1], 16, 10, 1, 1, rope=False)
    s.bounds[0, :, 7, 0], s.bounds[0, :, 9, 0], s.bounds[0, :, 11, 1] = 0x7FC0, 0x7F80, 0xFF80     # NaN, inf, -inf
    s.bounds[1, :, :, 0] = 0x7FC0                         # nothing but NaN: the lowest blocks
    s.q[2, 0, 3] = s.turned[2, 0, 3] = np.nan
    got = s.run()
    assert np.array_equal(got, s.expected())
    assert np.array_equal(got[1, 0], [*range(9), 49]) and np.array_equal(got[2, 0], [*range(9), 49])


def test_select_idle_and_unknown(nat, oracle):
    s = Select(nat, oracle, 5, 4, 2, 64, [1000, -1, 500, 600, 1000], 32, 6, 1, 1, seqs=[2, 0, 3, -1, 1], max_seqs=3)
    got = s.run()
    assert np.array_equal(got, s.expected()) and (got[[1, 2, 3]] == -1).all()


def test_select_captured(nat, oracle):
    g = Graphs()
    for blocks in (300, 5000):
        s = Select(nat, oracle, blocks, 4, 2, 32, [16 * blocks - 1] * 3, 16, 24)
        s.upload()
        graph = g.capture(s.launch)
        r = np.random.default_rng(1)
        for _ in range(3):
            s.pos = [int(p) for p in r.integers(0, 16 * blocks, 3)]
            s.q = s.turned = r.standard_normal(s.q.shape, dtype=np.float32)
            s.cos = np.ones_like(s.cos)
            s.sin = np.zeros_like(s.sin)
            for k, a in (("pos", np.asarray(s.pos, np.int32)), ("q", s.q), ("cos", s.cos), ("sin", s.sin)):
                s.dev[k].upload(a)
            g.replay(graph)
            assert np.array_equal(s.result(), s.expected())


# ---- the step ------------------------------------------------------------------

class Step:
    """Query i appends to sequence seqs[i] at pos[i] and attends to its listed blocks."""

    def __init__(self, cache, pos, block, keep, seqs=None, rope=True, max_pos=None, bounds=True):
        c, r = cache, cache.r
        self.c, self.pos, self.seqs, self.block, self.keep = c, list(pos), seqs, block, keep
        n = self.n = len(self.pos)
        self.max_pos = max(max(self.pos), 0) if max_pos is None else max_pos
        self.q = r.standard_normal((n, c.nq, c.hd), dtype=np.float32)
        self.k = r.standard_normal((n, c.nkv, c.hd), dtype=np.float32)
        self.v = r.standard_normal((n, c.nkv, c.hd), dtype=np.float32)
        self.cos, self.sin = rope_rows(c.oracle, c.hd, [max(p, 0) for p in pos]) if rope else (None, None)
        self.list = np.full((n, c.nkv, keep), -1, np.int32)
        for i, p in enumerate(self.pos):
            if p < 0:
                continue
            for h in range(c.nkv):
                last = p // block
                ids = np.sort(r.permutation(last)[:keep - 1])
                self.list[i, h, :len(ids) + 1] = [*ids, last]
        self.bounds = Bounds(c, block, self.max_pos // block + 2) if bounds else None
        self.dev = {k: None if a is None else c.up(a) for k, a in (
            ("q", self.q), ("k", self.k), ("v", self.v), ("cos", self.cos), ("sin", self.sin),
            ("pos", np.asarray(self.pos, np.int32)), ("seq", None if seqs is None else np.asarray(seqs, np.int32)),
            ("list", self.list), ("out", np.full((n, c.nq, c.hd), 3.0, np.float32)))}
        self.ws_bytes = c.lib.tq_hip_decode_step_blocks_ws_bytes(c.kv.h, n, self.max_pos, block, keep)
        assert self.ws_bytes > 0
        self.ws = c.up(np.full(self.ws_bytes, 0xFF, np.uint8))

    def launch(self, stream=None):
        p = {k: None if b is None else b.ptr for k, b in self.dev.items()}
        b = self.bounds
        self.c.nat.check(self.c.lib.tq_hip_decode_step_blocks_async(
            self.c.kv.h, self.n, p["seq"], p["pos"], self.max_pos, self.block, self.keep, p["list"], p["q"], p["k"],
            p["v"], p["cos"], p["sin"], p["out"], b.dev.ptr if b else None, b.stride if b else 0, self.ws.ptr,
            self.ws_bytes, stream), "step")

    def run(self):
        self.launch()
        return self.results()

    def results(self):
        self.c.sync()
        return self.dev["out"].download(self.q.shape, np.float32)

    def check(self, out):
        """Against the definition.  The output's bound is attention()'s with `term` for the roundings behind a tile's
        products (three bf16 parts keep 2^-25 of a term): the waves' and the splits' weights, each an exp2, a product, a
        sum of at most 64 and a division, 2^-24 each, 80 in all at most."""
        c = self.c
        kq = quantized(c.oracle, rotated(c.oracle, self.k, self.cos, self.sin))
        vq, qq = quantized(c.oracle, self.v), quantized(c.oracle, rotated(c.oracle, self.q, self.cos, self.sin))
        for i, p in enumerate(self.pos):
            s = i if self.seqs is None else self.seqs[i]
            if p < 0:
                assert (out[i] == 3.0).all()
                continue
            c.put(s, [p], np.stack([kq[i], vq[i]], 1)[None])
            every = c.rows(s, p + 1)
            ids = self.list[i, :, :min(self.keep, p // self.block + 1)]
            at = [np.concatenate([np.arange(b * self.block, min(p + 1, (b + 1) * self.block)) for b in row]) for row in ids]
            rows = np.stack([every[t, h] for h, t in enumerate(at)], 1)
            ref, bound, _, _ = attention(c, qq[i:i + 1], rows, [len(rows) - 1], term=80 * 2.0 ** -24)
            assert (np.abs(out[i] - ref[0]) <= bound[0]).all(), f"query {i}"
            if self.bounds:
                b, new = p // self.block, bounds_of(kq[i][None])
                if p % self.block:
                    was = self.bounds.host[s, :, b]
                    new = np.stack([outward(np.maximum(value(was[:, 0]), value(new[:, 0])), True),
                                    outward(np.minimum(value(was[:, 1]), value(new[:, 1])), False)], 1)
                self.bounds.host[s, :, b] = new
        if self.bounds:
            assert np.array_equal(self.bounds.dev.download(self.bounds.host.shape, np.uint16), self.bounds.host)
        assert c.download().tobytes() == c.pool.tobytes(), "cache"


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 6, 7, 8])
def test_step_shapes(nat, oracle, hd, group):
    lens = [1, 31, 0, 33, 300, 700]
    st = Step(Cache(nat, oracle, hd + group, 2 * group, 2, hd, lens, room=1), lens, 16, 9)
    st.check(st.run())


@pytest.mark.parametrize("length", [0, 15, 16, 47, 48, 255, 256, 257, 1500, 5000])
@pytest.mark.parametrize("block,keep", [(16, 1), (16, 64), (48, 5), (64, 16), (128, 3), (1024, 4)])
def test_step_of_one_sequence(nat, oracle, length, block, keep):
    """One split and several; the new token first, in the middle and last of its block."""
    st = Step(Cache(nat, oracle, length + block, 8, 2, 64, [length], room=1), [length], block, keep)
    st.check(st.run())


def test_step_over_a_long_list(nat, oracle):
    """More tokens than one work-group stages the pages of."""
    st = Step(Cache(nat, oracle, 1, 2, 1, 32, [40000], room=1), [40000], 64, 600)
    st.check(st.run())


def test_step_of_a_batch(nat, oracle):
    """Past the number of queries that are ranked by length, and one split each."""
    lens = [int(x) for x in np.random.default_rng(3).integers(0, 200, 140)]
    st = Step(Cache(nat, oracle, 2, 4, 2, 64, lens, room=1), lens, 16, 4)
    st.check(st.run())
    lens = lens[:60]
    st = Step(Cache(nat, oracle, 2, 8, 8, 32, lens, room=1), lens, 32, 3)
    st.check(st.run())


def test_step_options(nat, oracle):
    c = Cache(nat, oracle, 3, 8, 2, 64, [500, 600, 700], room=1)
    st = Step(c, [700, -1, 500], 32, 6, seqs=[2, 1, 0], rope=False, max_pos=900)
    st.check(st.run())
    st = Step(c, [499, 600], 32, 6, seqs=[0, 1], bounds=False)
    st.check(st.run())


def test_step_over_all_blocks_is_the_plain_step(nat, oracle):
    lens = [100, 37, 260]
    c = Cache(nat, oracle, 4, 8, 2, 128, lens, room=1)
    st = Step(c, lens, 16, 17)
    assert (st.list[2, 0] == np.arange(17)).all()
    out = st.run()
    st.check(out)
    plain = c.up(np.zeros(st.q.shape, np.float32))
    p = {k: b.ptr for k, b in st.dev.items() if b}
    nat.check(c.lib.tq_hip_decode_step_async(c.kv.h, 3, None, p["pos"], st.max_pos, p["q"], p["k"], p["v"], p["cos"],
                                             p["sin"], plain.ptr, None), "plain")
    c.sync()
    # (the plain step splits its weights in two bf16 parts, 2^-17 of the values)
    assert np.abs(plain.download(st.q.shape, np.float32) - out).max() < 2.0 ** -16 * np.abs(st.v).max() * 4


def test_step_captured_and_two_at_once(nat, oracle):
    g, other = Graphs(), Graphs()
    lens = [300, 301]
    a = Step(Cache(nat, oracle, 5, 8, 2, 64, lens, room=8), lens, 16, 8)
    b = Step(Cache(nat, oracle, 6, 8, 2, 64, [2000], room=8), [2000], 16, 100)
    ga, gb = g.capture(a.launch), other.capture(b.launch)
    for turn in range(3):
        g.hip.launch_graph(ga, g.stream)
        other.hip.launch_graph(gb, other.stream)
        g.sync()
        for st in (a, b):
            st.check(st.results())
        if turn < 2:
            for st in (a, b):
                st.pos = [p + 1 for p in st.pos]
                st.cos, st.sin = rope_rows(oracle, 64, st.pos)
                last = np.asarray([p // 16 for p in st.pos])
                for i in range(st.n):
                    st.list[i, :, -1] = last[i]
                for k, x in (("pos", np.asarray(st.pos, np.int32)), ("list", st.list), ("cos", st.cos), ("sin", st.sin)):
                    st.dev[k].upload(x)
                # the captured grid goes by max_pos: these stay below its last split
                assert max(st.pos) // 16 == st.max_pos // 16


# ---- together ------------------------------------------------------------------

def test_a_long_conversation(nat, oracle):
    """Prompts are cached, their bounds made; then steps that choose their blocks and attend to them.  The bounds that the
    steps keep are those of all tokens at once, and each list is the definition's."""
    lens, block, keep = [700, 90, 1], 16, 8
    c = Cache(nat, oracle, 7, 8, 2, 64, lens, room=40)
    most = max(lens) + 40
    bounds = Bounds(c, block, most // block + 2)
    bounds.make(lens)
    pos = list(lens)
    for _ in range(20):
        st = Step(c, pos, block, keep, max_pos=most, bounds=False)
        st.bounds = bounds
        bounds.host = bounds.dev.download(bounds.host.shape, np.uint16)
        sel = Select(nat, oracle, 0, 8, 2, 64, pos, block, keep, 1, 2, max_pos=most)
        sel.q, sel.cos, sel.sin, sel.bounds, sel.stride = st.q, st.cos, st.sin, bounds.host, bounds.stride
        sel.turned = rotated(oracle, st.q, st.cos, st.sin)
        st.list = sel.run()
        assert np.array_equal(st.list, sel.expected())
        st.dev["list"].upload(st.list)
        st.check(st.run())
        pos = [p + 1 for p in pos]
    kept = bounds.dev.download(bounds.host.shape, np.uint16)
    assert np.array_equal(bounds.make(pos), kept)


@pytest.mark.parametrize("sign", [1, -1])
def test_select_among_the_largest_scores(nat, oracle, sign):
    """Infinite scores beside finite ones of either sign and of very different sizes: the bins' range ends near 2^64."""
    s = Select(nat, oracle, 7, 1, 1, 64, [16 * 600 - 1], 16, 40, 0, 1, rope=False)
    r = np.random.default_rng(8)
    s.q = s.turned = np.abs(s.q) + 0.5
    size = (sign * np.exp2(r.integers(-120, 120, s.stride))).astype(np.float32)
    s.bounds[0, 0] = outward(size, True)[:, None, None]
    s.bounds[0, 0, r.permutation(590)[:9], 0] = 0x7F80
    assert np.array_equal(s.run(), s.expected())

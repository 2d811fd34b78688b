"""tq_hip_prefill_packed_async on the GPU: prompts of several sequences in one
call, against the definition in 64 bits (bounds derived at
tests.serving.attention) and, for the cache, byte for byte.

The dense kernel keeps each product of a weight and a value to 2^-20: two fp16
parts of each (2^-22), the product of the two lower ones left out (2^-22), V's
own rounding (2^-24); and a weight's parts end at 2^-24 of 2^11 times itself in
units of the largest V scale so far, a value at 127 of them, so that each key
adds up to 2^-28 of that scale.
"""
from __future__ import annotations

import numpy as np
import pytest

from tests.hip_graphs import Graphs
from tests.serving import Cache, attention, quantized, rope_rows, rotated

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nat():
    from tailorquantkernel_amd import native
    native.init(0)
    return native


class Packed:
    """Rows of several sequences: lens[i] new tokens of sequence seqs[i] after before[i] cached ones."""

    def __init__(self, nat, oracle, seed, nq, nkv, hd, lens, before, seqs=None, first=0, spare=2, rope=True, skew=0,
                 change=None):
        order = list(range(len(lens))) if seqs is None else seqs
        held, room = [0] * (max(order) + 1), [0] * (max(order) + 1)
        for s, n, b in zip(order, lens, before):
            held[s], room[s] = b, n
        self.c = c = Cache(nat, oracle, seed, nq, nkv, hd, held, room=max(room))
        r, self.lens, self.before, self.seqs, self.first = c.r, lens, before, seqs, first
        self.rows = sum(lens)
        self.start = (first + np.concatenate([[0], np.cumsum(lens)])).astype(np.int32)
        self.pos0 = np.asarray(before, np.int32)
        total = first + self.rows + spare
        make = lambda h: r.standard_normal((total, h, hd), dtype=np.float32)  # noqa: E731
        self.q, self.k, self.v = make(nq), make(nkv), make(nkv)
        self.cos = self.sin = None
        if rope:
            at = [0] * first + [b + j for n, b in zip(lens, before) for j in range(n)] + [0] * spare
            self.cos, self.sin = rope_rows(oracle, hd, at)
        if change:
            change(self)
        self.skew = skew
        up = lambda a: None if a is None else c.up(np.concatenate([np.zeros(skew, np.float32), a.reshape(-1)]))  # noqa: E731
        self.dev = {"q": up(self.q), "k": up(self.k), "v": up(self.v), "cos": up(self.cos), "sin": up(self.sin),
                    "out": up(np.full(self.q.shape, 9.0, np.float32))}
        self.seq_array = None if seqs is None else np.asarray(seqs, np.int32)
        self.ws_bytes = c.lib.tq_hip_prefill_packed_ws_bytes(c.kv.h, len(lens), self.pos0.ctypes.data,
                                                             self.start.ctypes.data)
        assert self.ws_bytes > 0
        self.ws = c.up(np.full(self.ws_bytes, 0xFF, np.uint8))

    def launch(self, stream=None):
        p = lambda k: self.dev[k].ptr + 4 * self.skew if self.dev[k] is not None else None  # noqa: E731
        return self.c.lib.tq_hip_prefill_packed_async(
            self.c.kv.h, len(self.lens), None if self.seq_array is None else self.seq_array.ctypes.data,
            self.pos0.ctypes.data, self.start.ctypes.data, p("q"), p("k"), p("v"), p("cos"), p("sin"), p("out"),
            self.ws.ptr, self.ws_bytes, stream)

    def results(self):
        self.c.sync()
        flat = self.dev["out"].download((self.skew + self.q.size,), np.float32)
        return flat[self.skew:].reshape(self.q.shape)

    def run(self):
        self.c.nat.check(self.launch(), "packed")
        return self.results()

    def check(self, out, dense=True, finite=True):
        c = self.c
        kq = quantized(c.oracle, rotated(c.oracle, self.k, self.cos, self.sin))
        vq = quantized(c.oracle, self.v)
        qq = quantized(c.oracle, rotated(c.oracle, self.q, self.cos, self.sin))
        written = np.zeros(out.shape[0], bool)
        for i, (n, b) in enumerate(zip(self.lens, self.before)):
            if n == 0:
                continue
            s = i if self.seqs is None else self.seqs[i]
            at = slice(self.start[i], self.start[i + 1])
            written[at] = True
            c.put(s, range(b, b + n), np.stack([kq[at], vq[at]], 2))
            rows = c.rows(s, b + n)
            if not finite:
                continue
            ref, bound, _, _ = attention(c, qq[at], rows, range(b, b + n), 2.0 ** -20 if dense else 2.0 ** -17)
            if dense:
                top = np.abs(rows[:, :, 1]["d"]).max((0, 2)).astype(np.float64)          # of each kv head
                bound += (b + n) * 2.0 ** -28 * np.repeat(top, c.nq // c.nkv)[None, :, None]
            err = np.abs(out[at] - ref)
            far = np.argwhere(~(err <= bound))
            assert len(far) == 0, (f"sequence {i} ({n} after {b}): {len(far)} values, up to {(err / bound).max():.3g} of "
                                   f"the bound; first at (row, head, column) {far[:4].tolist()}")
        assert (out[~written] == 9.0).all(), "rows of no sequence were written"
        assert c.download().tobytes() == c.pool.tobytes(), "cache"


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 6, 7, 8])
def test_dense_shapes(nat, oracle, hd, group):
    p = Packed(nat, oracle, hd * group, 2 * group, 2, hd, [1, 0, 5, 31, 33, 130, 257], [0, 7, 100, 16, 0, 33, 3])
    p.check(p.run())


@pytest.mark.parametrize("hd,nq,nkv", [(32, 8, 2), (256, 4, 2)])
def test_row_form_shapes(nat, oracle, hd, nq, nkv):
    """Head dims that the dense kernel does not have."""
    p = Packed(nat, oracle, hd, nq, nkv, hd, [1, 0, 40, 33], [0, 7, 300, 16])
    p.check(p.run(), dense=False)


@pytest.mark.parametrize("lens,before", [
    ([1], [0]), ([1], [1]), ([2], [31]), ([32], [0]), ([31], [1]), ([33], [31]), ([16], [16]), ([700], [0]),
    ([100], [3000]),                     # blocks cut into runs
    ([1, 1, 1], [2000, 15, 16]),         # single tokens
    ([600, 20, 5], [10, 900, 1500]),
    ([0, 0, 3], [5, 0, 0])])
def test_lengths(nat, oracle, lens, before):
    p = Packed(nat, oracle, sum(lens), 8, 2, 64, lens, before)
    p.check(p.run())


def test_one_kv_head_many_blocks(nat, oracle):
    p = Packed(nat, oracle, 1, 8, 1, 128, [900, 500], [0, 20])
    p.check(p.run())


def test_more_sequences_than_one_table(nat, oracle):
    r = np.random.default_rng(2)
    lens, before = r.integers(0, 40, 150).tolist(), r.integers(0, 90, 150).tolist()
    p = Packed(nat, oracle, 2, 4, 2, 64, lens, before)
    p.check(p.run())


def test_order_offset_and_spare_rows(nat, oracle):
    """Sequences in any order, rows before the first and behind the last that belong to none."""
    p = Packed(nat, oracle, 3, 8, 2, 64, [20, 50, 9], [30, 0, 64], seqs=[4, 0, 2], first=7, spare=11)
    p.check(p.run())


def test_without_rope(nat, oracle):
    p = Packed(nat, oracle, 4, 8, 2, 128, [70, 20], [0, 40], rope=False)
    p.check(p.run())


@pytest.mark.parametrize("skew", [1, 2])
def test_unaligned_rows(nat, oracle, skew):
    """Arrays off a 16-byte boundary attend row by row."""
    p = Packed(nat, oracle, 5, 8, 2, 64, [40, 20], [0, 40], skew=skew)
    p.check(p.run(), dense=False)


def test_row_form_in_groups(nat, oracle):
    """More rows than one decode launch of the row form takes."""
    p = Packed(nat, oracle, 6, 2, 1, 32, [2100, 30], [0, 5])
    p.check(p.run(), dense=False)


def test_values_of_many_sizes(nat, oracle):
    """V rows from 2^-12 to 2^12 in one sequence, and sequences a million times apart."""
    def change(p):
        p.v *= np.exp2(p.c.r.integers(-12, 13, p.v.shape[0]))[:, None, None].astype(np.float32)
        p.v[p.start[1]:p.start[2]] *= np.float32(1e-15)
        p.v[p.start[2]:] *= np.float32(1e15)
    p = Packed(nat, oracle, 7, 8, 2, 128, [150, 90, 60], [0, 0, 0], change=change)
    p.check(p.run())


@pytest.mark.parametrize("scale", [2.0 ** -100, 2.0 ** 120])
@pytest.mark.parametrize("nq,nkv,hd,lens,before", [
    (8, 2, 128, [700, 130], [0, 40]), (8, 2, 64, [100], [3000]), (2, 1, 64, [40, 500], [6000, 0])])
def test_values_near_the_ends_of_the_type(nat, oracle, nq, nkv, hd, lens, before, scale):
    """Sums of shifted weights times such values leave fp32's range, their means do not."""
    def change(p):
        p.v *= np.float32(scale)
        p.c.pool["d"][:, :, 1] *= np.float32(scale)
        p.c.upload()
    p = Packed(nat, oracle, 24, nq, nkv, hd, lens, before, change=change)
    p.check(p.run())


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 3e38])
def test_what_the_causal_mask_hides(nat, oracle, bad):
    """A later token's K and V change no earlier row, whatever they are."""
    args = (nat, oracle, 8, 8, 2, 64, [120, 40], [10, 0])
    clean = Packed(*args)
    want = clean.run()
    clean.check(want)

    def spoil(p):
        p.k[77, 0], p.v[77, 0], p.v[77, 1, :5], p.k[150, 1, 3], p.v[150] = bad, bad, bad, bad, bad
    p = Packed(*args, change=spoil)
    got = p.run()
    # rows before, to twice the bound of the clean ones (the tile's units may differ)
    seen = np.zeros(got.shape[0], bool)
    seen[77:120] = seen[150:160] = True
    limit = 2 * 2.0 ** -18 * np.abs(want).max()
    assert np.isfinite(got[~seen]).all()
    assert (np.abs(got - want)[~seen] <= limit).all()


def test_peaked_rows(nat, oracle):
    """One key that takes nearly everything, early and late in the row."""
    def change(p):
        p.k[40] = 8 * p.q[300, 0]
        p.k[290] = 8 * p.q[310, 3]
    p = Packed(nat, oracle, 9, 4, 1, 128, [320], [0], rope=False, change=change)
    p.check(p.run())


def test_agrees_with_single_calls(nat, oracle):
    """The cache bytes of one tq_hip_prefill_async per sequence, its outputs within both bounds."""
    args = (nat, oracle, 10, 8, 2, 128, [100, 64, 333], [0, 50, 20])
    a, b = Packed(*args), Packed(*args)
    out = a.run()
    size = 4 * a.c.hd
    for i, n in enumerate(b.lens):
        at = int(b.start[i])
        ptr = lambda k, heads, b=b, at=at: b.dev[k].ptr + at * heads * size  # noqa: E731
        nat.check(b.c.lib.tq_hip_prefill_async(b.c.kv.h, i, b.before[i], n, ptr("q", 8), ptr("k", 2), ptr("v", 2),
                                               b.dev["cos"].ptr + at * size // 2, b.dev["sin"].ptr + at * size // 2,
                                               ptr("out", 8), None), "prefill")
        b.c.sync()
    assert a.c.download().tobytes() == b.c.download().tobytes()
    a.check(out)
    b.check(b.results(), dense=False)


def test_captured_and_replayed(nat, oracle):
    p = Packed(nat, oracle, 11, 8, 2, 64, [100, 1, 60], [400, 30, 0])
    gr = Graphs()
    g = gr.capture(lambda s: nat.check(p.launch(s), "captured"))
    # the host arrays are read during the call only
    p.pos0[:], p.start[:] = 0, 0
    for seed in range(3):
        r = np.random.default_rng(seed)
        for k in "qkv":
            a = getattr(p, k)
            a[:] = r.standard_normal(a.shape, dtype=np.float32)
            p.dev[k].upload(a)
        p.dev["out"].upload(np.full(p.q.shape, 9.0, np.float32))
        gr.replay(g)
        p.start = np.concatenate([[0], np.cumsum(p.lens)]).astype(np.int32)
        p.check(p.results())


@pytest.mark.parametrize("before,dense", [(65500, True), (65520, False)])
def test_the_longest_sequences(nat, oracle, before, dense):
    """Up to 65,536 tokens take the dense kernel, one more the row form."""
    p = Packed(nat, oracle, 14, 2, 1, 64, [36, 20], [before, 3])
    p.check(p.run(), dense=dense)


@pytest.mark.parametrize("nq,nkv,hd", [(8, 2, 64), (16, 8, 128), (5, 1, 64)])
def test_prompts_and_single_tokens(nat, oracle, nq, nkv, hd):
    """Both forms in one call: long prompts, short turns and single tokens, in any order, other rows untouched."""
    r = np.random.default_rng(nq)
    lens = [1] * 30 + [150, 2, 300, 0, 7, 90]
    before = [int(x) for x in r.integers(0, 1500, 30)] + [10, 700, 0, 5, 1200, 33]
    mix = r.permutation(len(lens))
    lens, before = [lens[i] for i in mix], [before[i] for i in mix]
    seqs = [int(x) for x in r.permutation(len(lens))]
    p = Packed(nat, oracle, 16, nq, nkv, hd, lens, before, seqs=seqs, first=3, spare=4)
    p.check(p.run())


def test_prompts_and_single_tokens_captured(nat, oracle):
    lens, before = [1] * 40 + [200], [1200] * 40 + [0]
    p = Packed(nat, oracle, 17, 8, 4, 128, lens, before)
    gr = Graphs()
    g = gr.capture(lambda s: nat.check(p.launch(s), "captured"))
    for seed in range(3):
        r = np.random.default_rng(seed)
        for k in "qkv":
            a = getattr(p, k)
            a[:] = r.standard_normal(a.shape, dtype=np.float32)
            p.dev[k].upload(a)
        gr.replay(g)
        p.check(p.results())


@pytest.mark.parametrize("bad", [np.nan, np.inf, 3e38])
def test_what_the_causal_mask_hides_row_by_row(nat, oracle, bad):
    """A later token of a short turn changes no earlier row of it."""
    args = (nat, oracle, 18, 8, 2, 64, [6, 3], [900, 700])
    clean = Packed(*args)
    want = clean.run()
    clean.check(want)

    def spoil(p):
        p.k[4, 0], p.v[4, 0], p.v[4, 1, :5], p.k[8, 1, 3], p.v[8] = bad, bad, bad, bad, bad
    p = Packed(*args, change=spoil)
    got = p.run()
    p.check(got, finite=False)
    for at in (slice(0, 4), slice(6, 8)):
        assert got[at].tobytes() == want[at].tobytes()


# (form, new tokens, cached ones) of a few sequences, all in that form
FORMS = [("dense", [120, 40], [70, 0]), ("dense", [90], [3000]), ("rows", [6, 3], [900, 700])]


@pytest.mark.parametrize("form,lens,before", FORMS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_value_blocks_that_are_no_numbers(nat, oracle, form, lens, before, hd, bad):
    """One block of a key's values: only its own columns, in the rows that see the key, are no numbers."""
    def change(p):
        c, t = p.c, before[0] - 40
        c.pool[c.pages[0][t // 16], 0, 1, t % 16]["d"][-1] = bad       # an old key
        c.upload()
        p.v[2, 1, 5] = np.inf                                            # a new one, its first block
    p = Packed(nat, oracle, 25, 8, 2, hd, lens, before, change=change)
    got = p.run()
    p.check(got, finite=False)
    c = p.c
    qq = quantized(c.oracle, rotated(c.oracle, p.q, p.cos, p.sin))
    for i, (n, b) in enumerate(zip(lens, before)):
        rows, at = c.rows(i, b + n), slice(p.start[i], p.start[i + 1])
        odd = ~np.isfinite(rows[:, :, 1]["d"])                           # [key][kv head][block]
        assert odd.sum() == (2 if i == 0 else 0)
        rows["d"][:, :, 1][odd] = 0.0
        ref, bound, _, _ = attention(c, qq[at], rows, range(b, b + n), 2.0 ** -20 if form == "dense" else 2.0 ** -17)
        if form == "dense":
            top = rows[:, :, 1]["d"].max((0, 2)).astype(np.float64)
            bound += (b + n) * 2.0 ** -28 * np.repeat(top, 4)[None, :, None]
        seen = np.arange(b + n)[None, :] <= np.arange(b, b + n)[:, None]
        hit = np.einsum("rt,thb->rhb", seen.astype(int), odd.astype(int)) > 0
        hit = np.repeat(np.repeat(hit, 4, 1), 32, 2)                     # [row][head][column]
        assert hit.any() == (i == 0)
        assert not np.isfinite(got[at][hit]).any()
        assert (np.abs(got[at] - ref)[~hit] <= bound[~hit]).all()


class Shifted:
    """A device array one float off the boundary it would have."""

    def __init__(self, c, a):
        self.buf = c.up(np.concatenate([np.zeros(1, np.float32), a]))
        self.ptr = self.buf.ptr + 4

    def download(self, shape, dtype):
        return self.buf.download((shape[0] + 1,), dtype)[1:]


@pytest.mark.parametrize("shifted", [["out"], ["q"], ["k", "v"], ["cos", "sin"], ["q", "k", "v", "cos", "sin"]])
def test_some_arrays_off_the_boundary(nat, oracle, shifted):
    p = Packed(nat, oracle, 26, 8, 2, 64, [40, 20, 1], [0, 40, 900])
    for k in shifted:
        a = np.full(p.q.shape, 9.0, np.float32) if k == "out" else getattr(p, k)
        p.dev[k] = Shifted(p.c, a.reshape(-1))
    p.check(p.run(), dense=False)


@pytest.mark.parametrize("place", ["first", "last"])
def test_a_long_sequence_and_its_neighbours(nat, oracle, place):
    """One past the dense kernel's length goes row by row, the others as without it: bit for bit."""
    lens, before = [300, 150, 40], [0, 20, 5]
    others = slice(0, 3)
    if place == "last":
        lens, before = lens + [2], before + [65600]
    else:
        lens, before, others = [2] + lens, [65600] + before, slice(1, 4)
    p = Packed(nat, oracle, 27, 2, 1, 64, lens, before)
    out = p.run()
    p.check(out)
    seq = np.arange(4, dtype=np.int32)[others].copy()
    pos0, start = p.pos0[others].copy(), p.start[others.start:others.stop + 1].copy()
    nbytes = p.c.lib.tq_hip_prefill_packed_ws_bytes(p.c.kv.h, 3, pos0.ctypes.data, start.ctypes.data)
    p.dev["out"].upload(np.full(p.q.shape, 9.0, np.float32))
    ws = p.c.up(np.full(nbytes, 0xFF, np.uint8))
    nat.check(p.c.lib.tq_hip_prefill_packed_async(
        p.c.kv.h, 3, seq.ctypes.data, pos0.ctypes.data, start.ctypes.data, *(p.dev[k].ptr for k in (
            "q", "k", "v", "cos", "sin", "out")), ws.ptr, nbytes, None), "packed")
    alone = p.results()
    at = slice(int(start[0]), int(start[-1]))
    assert np.array_equal(alone[at].view(np.uint32), out[at].view(np.uint32))


@pytest.mark.parametrize("rope", [True, False])
@pytest.mark.parametrize("skew", [0, 1])
def test_row_form_order_offset_and_spare_rows(nat, oracle, rope, skew):
    """Short turns only: sequences in any order, rows that belong to none, with and without RoPE."""
    p = Packed(nat, oracle, 28, 6, 2, 64, [2, 0, 5, 1], [900, 3, 1300, 700], seqs=[5, 1, 0, 3], first=9, spare=6, rope=rope,
               skew=skew)
    p.check(p.run(), dense=False)


@pytest.mark.parametrize("nq,nkv,hd", [(3, 1, 128), (5, 1, 64), (12, 2, 128), (7, 1, 128)])
def test_cut_blocks_of_odd_groups(nat, oracle, nq, nkv, hd):
    """Runs of blocks that do not fill their rows, with values 2^40 apart from one stretch of keys to the next."""
    def change(p):
        rows = np.arange(4200) // 500 % 2
        for t in range(4200):
            if rows[t]:
                p.c.pool["d"][p.c.pages[0][t // 16], :, 1, t % 16] *= np.float32(2.0 ** -40)
        p.c.upload()
    p = Packed(nat, oracle, 29, nq, nkv, hd, [70, 40], [4200, 0], change=change)
    p.check(p.run())


def test_a_long_prompt_in_groups_beside_others(nat, oracle):
    """More rows than one decode launch takes, of a sequence past the dense kernel's length, between dense ones: the
    bits of a call of that sequence alone (the others' blocks may be cut another way: right in both)."""
    lens, before = [90, 2100, 50], [0, 64000, 7]
    p = Packed(nat, oracle, 30, 2, 1, 64, lens, before)
    out = p.run()
    p.check(out, finite=False)
    blank = np.full(p.q.shape, 9.0, np.float32)
    ptrs = [p.dev[k].ptr for k in ("q", "k", "v", "cos", "sin", "out")]
    got = np.zeros_like(out)
    for i in range(3):
        seq, pos0, start = np.asarray([i], np.int32), p.pos0[i:i + 1].copy(), p.start[i:i + 2].copy()
        nbytes = p.c.lib.tq_hip_prefill_packed_ws_bytes(p.c.kv.h, 1, pos0.ctypes.data, start.ctypes.data)
        ws = p.c.up(np.full(nbytes, 0xFF, np.uint8))
        p.dev["out"].upload(blank)
        nat.check(p.c.lib.tq_hip_prefill_packed_async(p.c.kv.h, 1, seq.ctypes.data, pos0.ctypes.data, start.ctypes.data,
                                                      *ptrs, ws.ptr, nbytes, None), "packed")
        alone, at = p.results(), slice(int(start[0]), int(start[1]))
        assert (alone[:at.start] == 9.0).all() and (alone[at.stop:] == 9.0).all()
        got[at] = alone[at]
    at = slice(int(p.start[1]), int(p.start[2]))
    assert np.array_equal(got[at].view(np.uint32), out[at].view(np.uint32))
    qq = quantized(oracle, rotated(oracle, p.q, p.cos, p.sin))
    for i in (0, 2):
        n, b, at = lens[i], before[i], slice(int(p.start[i]), int(p.start[i + 1]))
        rows = p.c.rows(i, b + n)
        ref, bound, _, _ = attention(p.c, qq[at], rows, range(b, b + n), 2.0 ** -20)
        bound += (b + n) * 2.0 ** -28 * float(rows[:, :, 1]["d"].max())
        assert (np.abs(out[at] - ref) <= bound).all() and (np.abs(got[at] - ref) <= bound).all()


def test_two_calls_at_once(nat, oracle):
    """Other sequences of one cache on two streams, each call with its own workspace."""
    lens, before = [200, 90, 33, 150], [40, 0, 500, 7]
    p = Packed(nat, oracle, 15, 8, 2, 128, lens, before)
    a, b = Graphs(), Graphs()
    out = p.run()
    p.check(out)
    parts = []
    for order in ([0, 2], [1, 3]):
        # each part's rows stay where they are: the other sequences have none
        start = np.cumsum([0] + [lens[i] for i in range(4)]).astype(np.int32)
        calls = []
        for i in order:
            at, pos0, seq = start[i:i + 2].copy(), np.asarray([before[i]], np.int32), np.asarray([i], np.int32)
            nbytes = p.c.lib.tq_hip_prefill_packed_ws_bytes(p.c.kv.h, 1, pos0.ctypes.data, at.ctypes.data)
            calls.append((seq, pos0, at, nbytes, p.c.up(np.full(nbytes, 0xFF, np.uint8))))
        parts.append(calls)
    for _ in range(5):
        p.dev["out"].upload(np.full(p.q.shape, 9.0, np.float32))
        p.c.sync()
        for calls, s in ((parts[0], a.stream), (parts[1], b.stream)):
            for seq, pos0, at, nbytes, ws in calls:
                nat.check(p.c.lib.tq_hip_prefill_packed_async(
                    p.c.kv.h, 1, seq.ctypes.data, pos0.ctypes.data, at.ctypes.data, *(p.dev[k].ptr for k in (
                        "q", "k", "v", "cos", "sin", "out")), ws.ptr, nbytes, s), "packed")
        p.check(p.results())


def test_refusals(nat, oracle):
    c = Cache(nat, oracle, 12, 8, 2, 64, [50, 60, 70], room=20)
    lib, P = c.lib, 4096
    i32 = lambda *v: np.asarray(v, np.int32)  # noqa: E731
    pos0, start = i32(50, 60, 70), i32(0, 10, 20, 30)
    ws = lib.tq_hip_prefill_packed_ws_bytes
    nbytes = ws(c.kv.h, 3, pos0.ctypes.data, start.ctypes.data)
    good = dict(n=3, seq=None, pos0=pos0, start=start, q=P, k=P, v=P, cos=P, sin=P, out=P, ws=P, ws_bytes=nbytes)

    def call(**over):
        a = {**good, **over}
        arrays = [a[k] for k in ("seq", "pos0", "start")]
        ptrs = [None if x is None else x.ctypes.data for x in arrays]
        return lib.tq_hip_prefill_packed_async(c.kv.h, a["n"], *ptrs, *[a[k] for k in (
            "q", "k", "v", "cos", "sin", "out", "ws", "ws_bytes")], None)

    for over in (dict(n=-1), dict(n=4, start=i32(0, 1, 2, 3, 4), pos0=i32(0, 0, 0, 0)), dict(start=None),
                 dict(start=i32(-1, 10, 20, 30)), dict(start=i32(0, 20, 10, 30)), dict(pos0=i32(50, -1, 70)),
                 dict(pos0=i32(50, 60, 100)), dict(pos0=i32(50, 60, 2 ** 31 - 1)), dict(start=i32(0, 10, 20, 90)),
                 dict(seq=i32(0, 1, 3)), dict(seq=i32(0, -1, 2)), dict(seq=i32(0, 1, 1)), dict(q=None), dict(k=None),
                 dict(v=None), dict(out=None), dict(cos=None), dict(sin=None), dict(ws=None), dict(ws=P + 8),
                 dict(ws_bytes=nbytes - 1), dict(q=P + 2), dict(out=P + 1)):
        assert call(**over) == nat.EINVAL, over
    assert call(n=0) == 0
    assert call(start=i32(5, 5, 5, 5), q=None) == 0          # no rows
    assert ws(None, 3, None, start.ctypes.data) == ws(c.kv.h, 0, None, start.ctypes.data) == 0
    assert ws(c.kv.h, 3, None, None) == ws(c.kv.h, 3, None, i32(0, 2, 1, 3).ctypes.data) == 0
    # an unmapped page
    c.kv.set_pages(1, c.pages[1][:4])
    assert call() == nat.EINVAL

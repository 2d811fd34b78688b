"""tq_hip_decode_step_shared_async: queries whose sequences begin with common pages,
against attention on each sequence's tokens in 64 bits."""
from __future__ import annotations

import numpy as np
import pytest

from tests.hip_graphs import Graphs
from tests.serving import PAGE, Cache, attention, quantized, rope_rows, rotated

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nat():
    from tailorquantkernel_amd import native
    native.init(0)
    return native


def members(n):
    """Own tokens of n members of a group."""
    return [(7 * i) % 50 for i in range(n)]


def large_group(nq, nkv):
    """A group that makes a call attend to the common tokens of its groups of 4 and more together."""
    group = nq // nkv
    n = 120 // group
    saved = n * (1.5 if group > 4 else 1) - 6
    return PAGE * (int(400e3 / (saved * nkv)) // PAGE + 1), members(n)


class Shared:
    """Groups of (common tokens, [own tokens of each member]), `before` and `behind` lists of queries that share nothing.
    A query appends the token behind its own.  large: behind the others a group that makes the call attend to common
    tokens together."""

    def __init__(self, nat, oracle, seed, nq, nkv, hd, groups, before=(), behind=(), rope=True, order=None, room=1,
                 max_pos=None, large=True):
        self.checked = len(before) + sum(len(m) for _, m in groups)      # and the large group's last, and what is behind it
        if large:
            groups = [*groups, large_group(nq, nkv)]
        self.behind = len(behind)
        own = [*before, *(m for _, members in groups for m in members), *behind]
        base = [0] * len(before) + [p for p, members in groups for _ in members] + [0] * len(behind)
        lens = [b + m for b, m in zip(base, own)]
        self.order = list(range(len(own)))                                  # query i reads sequence order[i]
        self.order[:len(order or ())] = order or ()
        by_seq = [0] * len(own)
        for i, s in enumerate(self.order):
            by_seq[s] = own[i]                  # a group's first sequence holds its common tokens, and room for any own
        at = len(before)
        for p, rest in groups:
            if rest:
                by_seq[self.order[at]] = p + max(rest)
            at += len(rest)
        c = self.c = Cache(nat, oracle, seed, nq, nkv, hd, by_seq, room=room)
        at = len(before)
        self.start, self.prefix = [at], []
        for p, rest in groups:
            for i in range(at + 1, at + len(rest)):
                first, mine = self.order[at], self.order[i]
                c.pages[mine] = np.concatenate([c.pages[first][:p // PAGE], c.pages[mine]])
                c.kv.set_pages(mine, c.pages[mine])
            at += len(rest)
            self.start.append(at)
            self.prefix.append(p)
        self.host = np.asarray(self.start, np.int32), np.asarray(self.prefix, np.int32)
        self.n, self.base, r = len(own), base, c.r
        self.max_pos = max([*lens, *self.prefix]) if max_pos is None else max_pos
        self.q = r.standard_normal((self.n, nq, hd), dtype=np.float32)
        self.k = r.standard_normal((self.n, nkv, hd), dtype=np.float32)
        self.v = r.standard_normal((self.n, nkv, hd), dtype=np.float32)
        self.rope = rope
        self.dev = {"q": c.up(self.q), "k": c.up(self.k), "v": c.up(self.v), "seq": None,
                    "out": c.up(np.full(self.q.shape, 3.0, np.float32))}
        if order is not None:
            self.dev["seq"] = c.up(np.asarray(self.order, np.int32))
        self.at(lens)
        self.ws_bytes = c.lib.tq_hip_decode_step_shared_ws_bytes(c.kv.h, self.n, self.max_pos, len(self.prefix),
                                                                 self.host[0].ctypes.data, self.host[1].ctypes.data)
        assert self.ws_bytes > 0
        self.ws = c.up(np.full(self.ws_bytes, 0xFF, np.uint8))

    def at(self, pos):
        """The new tokens' positions."""
        self.pos = list(pos)
        self.cos, self.sin = rope_rows(self.c.oracle, self.c.hd, [max(p, 0) for p in pos]) if self.rope else (None, None)
        for k, a in (("pos", np.asarray(self.pos, np.int32)), ("cos", self.cos), ("sin", self.sin)):
            if a is None or k not in self.dev:
                self.dev[k] = None if a is None else self.c.up(a)
            else:
                self.dev[k].upload(a)

    def launch(self, stream=None):
        p = {k: None if b is None else b.ptr for k, b in self.dev.items()}
        self.c.nat.check(self.c.lib.tq_hip_decode_step_shared_async(
            self.c.kv.h, self.n, p["seq"], p["pos"], self.max_pos, len(self.prefix), self.host[0].ctypes.data,
            self.host[1].ctypes.data, p["q"], p["k"], p["v"], p["cos"], p["sin"], p["out"], self.ws.ptr, self.ws_bytes,
            stream), "step")

    def run(self):
        self.c.upload()
        self.launch()
        return self.results()

    def results(self):
        self.c.sync()
        return self.dev["out"].download(self.q.shape, np.float32)

    def check(self, out, finite=True):
        """Against the definition.  attention()'s bound with, per term, 2^-20 for the common tokens' products (two fp16
        parts each of weight and value) and 80 roundings for the weights of waves, splits, runs and their merge; and
        2^-28 of the largest V scale per common token, the weights too small for a part (as tests of the packed prefill)."""
        c = self.c
        kq = quantized(c.oracle, rotated(c.oracle, self.k, self.cos, self.sin))
        vq, qq = quantized(c.oracle, self.v), quantized(c.oracle, rotated(c.oracle, self.q, self.cos, self.sin))
        for i, p in enumerate(self.pos):
            s = self.order[i]
            if p < self.base[i] or p < 0:
                assert (out[i] == 3.0).all()
                continue
            c.put(s, [p], np.stack([kq[i], vq[i]], 1)[None])
            if not finite or self.checked <= i < len(self.pos) - self.behind - 1:
                continue
            rows = c.rows(s, p + 1)
            ref, bound, _, _ = attention(c, qq[i:i + 1], rows, [p], 2.0 ** -20 + 80 * 2.0 ** -24)
            top = np.abs(rows[:, :, 1]["d"]).max((0, 2)).astype(np.float64)
            bound += (p + 1) * 2.0 ** -28 * np.repeat(top, c.nq // c.nkv)[None, :, None]
            err = np.abs(out[i] - ref[0])
            assert (err <= bound[0]).all(), f"query {i} at {p} behind {self.base[i]}: {(err / bound[0]).max():.3g} of the bound"
        assert c.download().tobytes() == c.pool.tobytes(), "cache"


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 6, 7, 8])
def test_shapes(nat, oracle, hd, group):
    st = Shared(nat, oracle, hd + group, 2 * group, 2, hd, [(48, [0, 5, 40, 9]), (32, [7]), (320, [1, 2, 300, 16, 15])],
                before=[20], behind=[0, 33])
    st.check(st.run())


@pytest.mark.parametrize("prefix", [0, 16, 32, 48, 64, 496, 512, 528, 2000, 4096])
@pytest.mark.parametrize("n", [3, 4, 9, 33])
@pytest.mark.parametrize("nq", [2, 8])
def test_lengths(nat, oracle, prefix, n, nq):
    """Runs of one tile (1 head a kv head) and of several, a last tile that is half empty, rows in one block and in two."""
    st = Shared(nat, oracle, prefix + n, nq, 2, 64, [(prefix, members(n))])
    st.check(st.run())


@pytest.mark.parametrize("prefix", [0, 16, 64, 496, 2000])
@pytest.mark.parametrize("n", [2, 9])
def test_each_by_itself(nat, oracle, prefix, n):
    """Too few tokens to be attended to together."""
    st = Shared(nat, oracle, prefix + n, 8, 2, 64, [(prefix, members(n)), (16, [0, 3, 5, 7])], behind=[1200], large=False)
    st.check(st.run())


@pytest.mark.parametrize("nq,nkv,n", [(8, 8, 12), (32, 8, 12), (16, 2, 9)])
def test_worth_it_alone(nat, oracle, nq, nkv, n):
    """One group, with fewer common tokens than are attended to together, and with as many."""
    saved = n * (1.5 if nq > 4 * nkv else 1) - 6
    few = PAGE * (int(300e3 / (saved * nkv)) // PAGE)
    for prefix in (few, few + PAGE):
        st = Shared(nat, oracle, prefix, nq, nkv, 64, [(prefix, members(n))], large=False)
        st.check(st.run())


@pytest.mark.parametrize("n", [1, 4, 16, 17, 32, 64, 65])
def test_rows(nat, oracle, n):
    """Waves and blocks that the members' heads fill and do not."""
    st = Shared(nat, oracle, n, 16, 2, 128, [(208, [i % 20 for i in range(n)])])
    st.check(st.run())


def test_long_own_parts(nat, oracle):
    """What lies behind the common tokens in several splits, beside members that have none."""
    st = Shared(nat, oracle, 1, 8, 2, 64, [(160, [3000, 0, 1500, 1]), (64, [0, 0, 0, 0])], behind=[2500])
    st.check(st.run())


def test_a_long_prefix(nat, oracle):
    """As many runs as the merge takes."""
    st = Shared(nat, oracle, 2, 4, 1, 64, [(70000, members(12))], large=False)
    st.check(st.run())


def test_nothing_is_shared(nat, oracle):
    st = Shared(nat, oracle, 3, 8, 2, 64, [], before=[100, 0, 37], large=False)
    st.check(st.run())
    for large in (False, True):
        st = Shared(nat, oracle, 3, 8, 2, 64, [(0, [100, 5, 6, 7]), (32, [4])], large=large)
        st.check(st.run())
        st = Shared(nat, oracle, 3, 8, 2, 64, [(48, []), (32, [4, 5, 6, 7])], behind=[9], large=large)      # an empty group
        st.check(st.run())


def test_many_groups(nat, oracle):
    """More groups than one launch takes, and more queries than are ranked."""
    st = Shared(nat, oracle, 4, 2, 1, 64, [(16 * (1 + g % 5), [g % 7, g % 11, 2, 3][:2 + g % 3]) for g in range(70)],
                before=[3], behind=[4, 5])
    st.check(st.run())


def test_sequences_in_any_order_without_rope(nat, oracle):
    st = Shared(nat, oracle, 5, 8, 2, 128, [(96, [5, 6, 7, 8]), (32, [40, 1, 2, 3, 4])], before=[3], rope=False,
                order=[4, 0, 5, 9, 2, 1, 8, 3, 7, 6], max_pos=9500)
    st.check(st.run())


def test_queries_in_front_of_their_common_tokens_are_left_out(nat, oracle):
    for large in (False, True):
        st = Shared(nat, oracle, 6, 8, 2, 64, [(96, [5, 6, 7, 8, 9]), (32, [4])], behind=[10, 20], large=large)
        st.at([101, 95, -1, 96, 0, 31, *st.pos[6:-2], -1, 20])
        st.check(st.run())


@pytest.mark.parametrize("idle", [1, 3, 70])
def test_the_first_of_a_group_may_be_idle(nat, oracle, idle):
    """No sequence, or one that has not come to its common tokens: their pages are those of the first that has."""
    n = idle + 5
    st = Shared(nat, oracle, idle, 8, 2, 64, [(2064, members(n))], behind=[4], order=list(range(n)))
    st.at([-1] * idle + st.pos[idle:])
    seqs = np.asarray(st.order, np.int32)
    seqs[:idle] = -1
    if idle == 3:
        st.at([700, -1, 5000] + st.pos[idle:])
        seqs[:3] = 0, 10 ** 6, -7
    st.dev["seq"].upload(seqs)
    out = st.run()
    if idle == 3:
        st.pos[2], out[2] = -1, 3.0     # (a query of no sequence appends nothing, and its row says nothing)
    st.check(out)


def test_equal_results_every_time(nat, oracle):
    st = Shared(nat, oracle, 7, 32, 8, 128, [(1152, [i for i in range(40)])], large=False)
    first = st.run()
    assert np.array_equal(first, st.run())
    st.check(first)


def test_values_of_very_different_sizes(nat, oracle):
    """Scales of common tokens from 2^-60 to 2^60, in one tile and across tiles: each term keeps its bits."""
    st = Shared(nat, oracle, 8, 8, 2, 64, [(256, [3, 30, 0, 9])])
    c, page = st.c, st.c.pages[0]
    r = np.random.default_rng(1)
    sizes = np.float32(2.0) ** r.integers(-60, 60, (8, c.nkv, PAGE, c.nb)).astype(np.float32)
    c.pool["d"][page[:8], :, 1] *= sizes
    c.pool["d"][page[8:12], :, 1] *= np.float32(2.0 ** -40)
    c.pool["d"][page[12:16], :, 1] *= np.float32(2.0 ** 30)
    st.check(st.run())


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_a_block_that_is_no_number_stays_in_its_columns(nat, oracle, bad):
    st = Shared(nat, oracle, 9, 8, 2, 64, [(256, [3, 30, 7, 0])], behind=[40])
    clean = st.run()
    c = st.c
    c.pool["d"][c.pages[0][3], 1, 1, 5, 1] = bad       # token 53's value, kv head 1, second block
    c.pool["q"][c.pages[0][3], 1, 1, 5, 1] = 1
    out = st.run()
    st.check(out, finite=False)
    hit = np.zeros(out.shape, bool)
    hit[:4, 4:, 32:] = True
    if np.isnan(bad):
        assert np.isnan(out[hit]).all()
    else:
        assert (out[hit] == bad).all()
    assert np.abs(out[~hit] - clean[~hit]).max() <= 2.0 ** -18 * np.abs(clean).max()


def test_a_key_that_is_no_number_is_seen(nat, oracle):
    st = Shared(nat, oracle, 10, 8, 2, 64, [(64, [3, 30, 7, 0])], behind=[40])
    clean = st.run()
    st.c.pool["d"][st.c.pages[0][1], 0, 0, 2, 0] = np.nan
    out = st.run()
    assert np.isnan(out[:4, :4]).all()
    assert np.array_equal(out[:, 4:], clean[:, 4:]) and np.array_equal(out[4:], clean[4:])


def test_captured_and_two_at_once(nat, oracle):
    g, other = Graphs(), Graphs()
    a = Shared(nat, oracle, 11, 8, 2, 64, [(160, [5, 6, 60, 0])], room=20, max_pos=8500)
    b = Shared(nat, oracle, 12, 8, 2, 128, [(320, [i for i in range(20)])], room=20, max_pos=8500)
    for st in (a, b):
        st.c.upload()
    ga, gb = g.capture(a.launch), other.capture(b.launch)
    for turn in range(3):
        g.hip.launch_graph(ga, g.stream)
        other.hip.launch_graph(gb, other.stream)
        g.sync()
        for st in (a, b):
            st.check(st.results())
            st.at([p + 1 + turn for p in st.pos])
            # (a turn leaves gaps of rows that no step wrote: what the cache holds there counts)


def test_a_conversation_under_a_prompt(nat, oracle):
    """A prompt prefilled once, its pages mapped into every sequence, questions packed behind it, then steps together."""
    nq, nkv, hd, prompt, turns = 8, 2, 64, 96, [5, 17, 1, 9]
    st = Shared(nat, oracle, 13, nq, nkv, hd, [(prompt, turns)], room=8, max_pos=8500)
    c, r = st.c, st.c.r
    for pos0, lens, seqs in (([0], [prompt], [0]), ([prompt] * len(turns), turns, range(len(turns)))):
        rows = sum(lens)
        q, k, v = (r.standard_normal((rows, h, hd), dtype=np.float32) for h in (nq, nkv, nkv))
        at = [b + j for b, m in zip(pos0, lens) for j in range(m)]
        cos, sin = rope_rows(oracle, hd, at)
        start, first = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32), np.asarray(pos0, np.int32)
        ids = np.asarray(seqs, np.int32)
        d = [c.up(x) for x in (q, k, v, cos, sin, np.zeros_like(q))]
        nbytes = c.lib.tq_hip_prefill_packed_ws_bytes(c.kv.h, len(lens), first.ctypes.data, start.ctypes.data)
        ws = c.up(np.zeros(nbytes, np.uint8))
        nat.check(c.lib.tq_hip_prefill_packed_async(c.kv.h, len(lens), ids.ctypes.data, first.ctypes.data,
                                                    start.ctypes.data, *[x.ptr for x in d], ws.ptr, nbytes, None), "packed")
        c.sync()
        kq, vq = quantized(oracle, rotated(oracle, k, cos, sin)), quantized(oracle, v)
        for s, a, m, b in zip(seqs, start, lens, pos0):
            c.put(s, range(b, b + m), np.stack([kq[a:a + m], vq[a:a + m]], 2))
    for _ in range(6):
        st.launch()
        st.check(st.results())
        st.at([p + 1 for p in st.pos])

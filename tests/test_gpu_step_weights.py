"""tq_hip_decode_step_weights_async on the GPU: the step's output and cache
rows, and the totals that attention's weights are added to, against the
definition in 64 bits (bounds derived at tests.serving.attention)."""
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


class Step:
    """One step's inputs on the device: query i appends to sequence seqs[i] at slot pos[i]."""

    def __init__(self, cache, pos, seqs=None, stride=None, rope=True, at=None, max_pos=None, max_seqs=None):
        c, r = cache, cache.r
        self.c, self.pos, self.seqs, self.at = c, list(pos), seqs, at
        n = self.n = len(self.pos)
        self.max_pos = max(max(self.pos), 0) if max_pos is None else max_pos
        self.stride = stride or self.max_pos + 1
        self.q = r.standard_normal((n, c.nq, c.hd), dtype=np.float32)
        self.k = r.standard_normal((n, c.nkv, c.hd), dtype=np.float32)
        self.v = r.standard_normal((n, c.nkv, c.hd), dtype=np.float32)
        text = [max(p, 0) for p in (self.pos if at is None else at)]
        self.cos, self.sin = rope_rows(c.oracle, c.hd, text) if rope else (None, None)
        shape = (max_seqs or len(c.pages), c.nkv, self.stride)
        self.total = r.random(shape).astype(np.float32)
        self.where = np.full(shape, -4, np.int32)
        up = lambda a: None if a is None else c.up(a)  # noqa: E731
        self.dev = {k: up(a) for k, a in (
            ("q", self.q), ("k", self.k), ("v", self.v), ("cos", self.cos), ("sin", self.sin), ("total", self.total),
            ("where", self.where), ("pos", np.asarray(self.pos, np.int32)),
            ("seq", None if seqs is None else np.asarray(seqs, np.int32)),
            ("at", None if at is None else np.asarray(at, np.int32)),
            ("out", np.full((n, c.nq, c.hd), 3.0, np.float32)))}
        self.ws_bytes = c.lib.tq_hip_decode_step_weights_ws_bytes(c.kv.h, n, self.max_pos)
        assert self.ws_bytes > 0
        self.ws = c.up(np.full(self.ws_bytes, 0xFF, np.uint8))

    def p(self, k):
        return self.dev[k].ptr if self.dev[k] is not None else None

    def launch(self, stream=None, where=True):
        return self.c.lib.tq_hip_decode_step_weights_async(
            self.c.kv.h, self.n, self.p("seq"), self.p("pos"), self.max_pos, self.p("q"), self.p("k"), self.p("v"),
            self.p("cos"), self.p("sin"), self.p("out"), self.p("at"), self.p("total"),
            self.p("where") if where else None, self.stride, self.ws.ptr, self.ws_bytes, stream)

    def results(self):
        self.c.sync()
        get = lambda k, a, t: self.dev[k].download(a, t)  # noqa: E731
        return (get("out", self.q.shape, np.float32), get("total", self.total.shape, np.float32),
                get("where", self.where.shape, np.int32))

    def run(self, **kw):
        self.c.nat.check(self.launch(**kw), "step")
        return self.results()

    def check(self, got, total=None, where=None, stored=True):
        """Against the definition; total, where: the arrays before the step."""
        c = self.c
        out, got_total, got_where = got
        total, where = (self.total if total is None else total), (self.where if where is None else where)
        want_where = where.copy()
        same = np.ones(got_total.shape, bool)
        kq = quantized(c.oracle, rotated(c.oracle, self.k, self.cos, self.sin))
        vq, qq = quantized(c.oracle, self.v), quantized(c.oracle, rotated(c.oracle, self.q, self.cos, self.sin))
        for i, p in enumerate(self.pos):
            s = i if self.seqs is None else self.seqs[i]
            if p < 0:
                assert (out[i] == 3.0).all()
                continue
            c.put(s, [p], np.stack([kq[i], vq[i]], 1)[None])
            ref, bound, w, loose = attention(c, qq[i:i + 1], c.rows(s, p + 1), [p])
            assert (np.abs(out[i] - ref[0]) <= bound[0]).all(), f"query {i}: output"
            w, loose = w[0].reshape(c.nkv, -1, p + 1), loose[0].reshape(c.nkv, -1, 1)
            before = total[s, :, :p + 1].astype(np.float64)
            before[:, p] = 0.0
            want, off = before + w.sum(1), (w * loose).sum(1) + 2.0 ** -24 * (before + 10 * w.sum(1))
            assert (np.abs(got_total[s, :, :p + 1] - want) <= off).all(), f"query {i}: totals"
            same[s, :, :p + 1] = False
            want_where[s, :, p] = p if self.at is None else self.at[i]
        assert (got_total[same] == total[same]).all(), "totals past the step's tokens were written"
        assert (got_where == want_where).all()
        if stored:
            assert c.download().tobytes() == c.pool.tobytes(), "cache"


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 6, 7, 8])
def test_shapes(nat, oracle, hd, group):
    lens = [1, 31, 0, 33, 300, 700]
    c = Cache(nat, oracle, hd + group, 2 * group, 2, hd, lens, room=1)
    st = Step(c, lens, stride=705)
    st.check(st.run())


@pytest.mark.parametrize("length", [0, 1, 15, 16, 31, 32, 127, 255, 256, 1500, 9000])
@pytest.mark.parametrize("order", ["in order", "scattered"])
def test_one_sequence(nat, oracle, length, order):
    c = Cache(nat, oracle, length, 8, 2, 64, [length], room=1, pages_of=order)
    st = Step(c, [length])
    st.check(st.run())
    st = Step(c, [length], seqs=[0])
    st.check(st.run())


def test_without_rope_and_positions(nat, oracle):
    c = Cache(nat, oracle, 1, 4, 2, 128, [100, 40], room=1)
    st = Step(c, [100, 40], rope=False)
    out, total, where = st.run(where=False)
    assert (where == st.where).all()
    where[:, :, 100][0], where[:, :, 40][1] = 100, 40      # as if it had been given
    st.check((out, total, where))


def test_text_positions_past_the_slots(nat, oracle):
    """After an eviction a token's slot and its position in the text differ."""
    c = Cache(nat, oracle, 2, 8, 2, 64, [64, 200], room=1)
    st = Step(c, [64, 200], at=[1000, 4321])
    st.check(st.run())


def test_sequences_in_any_order(nat, oracle):
    c = Cache(nat, oracle, 3, 4, 2, 64, [50, 60, 70, 80], room=1)
    st = Step(c, [80, 50, 70], seqs=[3, 0, 2], stride=100, max_pos=99)
    st.check(st.run())


def test_idle_queries(nat, oracle):
    """A negative position: nothing of that query is read or written."""
    c = Cache(nat, oracle, 4, 4, 2, 64, [50, 60, 70], room=1)
    st = Step(c, [50, -1, 70])
    st.check(st.run())


def test_peaked_and_flat_rows(nat, oracle):
    """One key that takes nearly everything, and keys that are all alike."""
    c = Cache(nat, oracle, 5, 4, 1, 128, [900, 900], room=1)
    st = Step(c, [900, 900], rope=False)
    key = np.zeros((1, 1, 2, 128), np.float32)
    key[..., 0, :] = 6 * st.q[0, 0]
    key[..., 1, :] = st.v[0]
    c.put(0, [517], quantized(oracle, key))
    c.put(1, range(900), np.repeat(c.rows(1, 1), 900, 0))
    c.upload()
    st.check(st.run())


def test_steps_in_a_row(nat, oracle):
    c = Cache(nat, oracle, 6, 8, 2, 64, [40, 90], room=4)
    total = where = None
    for j in range(4):
        st = Step(c, [40 + j, 90 + j], stride=128, max_pos=100)
        if total is not None:
            st.dev["total"].upload(total)
            st.dev["where"].upload(where)
        got = st.run()
        st.check(got, total, where)
        total, where = got[1:]


def test_same_rows_as_the_plain_step(nat, oracle):
    """The cache bytes are the plain step's, the output within both kernels' bounds (twice the bound)."""
    lens = [500, 77]
    a, b = (Cache(nat, oracle, 7, 8, 2, 64, lens, room=1) for _ in range(2))
    x, y = Step(a, lens), Step(b, lens)
    got = x.run()
    nat.check(b.lib.tq_hip_decode_step_async(b.kv.h, 2, None, y.p("pos"), y.max_pos, y.p("q"), y.p("k"), y.p("v"),
                                             y.p("cos"), y.p("sin"), y.p("out"), None), "plain step")
    b.sync()
    assert a.download().tobytes() == b.download().tobytes()
    x.check(got)
    y.check((y.dev["out"].download(y.q.shape, np.float32),) + got[1:], stored=False)


def test_captured_and_replayed(nat, oracle):
    """Two graphs of different batches on one workspace, replayed in turn."""
    c = Cache(nat, oracle, 8, 8, 2, 64, [300, 200, 100], room=1)
    x, y = Step(c, [300, 200, 100]), Step(c, [200], seqs=[1], max_pos=300)
    y.ws = x.ws
    assert y.ws_bytes <= x.ws_bytes
    gr = Graphs()
    graphs = [gr.capture(lambda s, t=t: nat.check(t.launch(stream=s), "captured")) for t in (x, y)]
    for _ in range(3):
        for t, g in zip((x, y), graphs):
            t.dev["total"].upload(t.total)
            t.dev["where"].upload(t.where)
            gr.replay(g)
            t.check(t.results())


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 6, 7, 8])
def test_one_split(nat, oracle, hd, group):
    """One sequence of up to 256 keys is one split, which finishes the call itself."""
    length = 97 + 19 * group
    c = Cache(nat, oracle, 100 + hd + group, 3 * group, 3, hd, [length], room=1)
    st = Step(c, [length], at=[5 * length], stride=301)
    st.check(st.run())


def test_a_long_context(nat, oracle):
    c = Cache(nat, oracle, 21, 2, 1, 32, [70000, 12], room=1)
    st = Step(c, [70000, 12], seqs=[0, 1])
    st.check(st.run())


def test_a_sequence_named_twice(nat, oracle):
    """Against the contract: what its totals become is not said, the other sequences are as they should be."""
    lens = [300, 40, 700]
    c = Cache(nat, oracle, 22, 8, 2, 64, lens, room=2)
    st = Step(c, [300, 40, 301, 700], seqs=[0, 1, 0, 2], stride=800, max_seqs=3)
    out, total, where = st.run()
    kq = quantized(c.oracle, rotated(c.oracle, st.k, st.cos, st.sin))
    vq, qq = quantized(c.oracle, st.v), quantized(c.oracle, rotated(c.oracle, st.q, st.cos, st.sin))
    for i in (1, 3):
        s, p = st.seqs[i], st.pos[i]
        c.put(s, [p], np.stack([kq[i], vq[i]], 1)[None])
        ref, bound, w, loose = attention(c, qq[i:i + 1], c.rows(s, p + 1), [p])
        assert (np.abs(out[i] - ref[0]) <= bound[0]).all()
        w, loose = w[0].reshape(c.nkv, -1, p + 1), loose[0].reshape(c.nkv, -1, 1)
        before = st.total[s, :, :p + 1].astype(np.float64)
        before[:, p] = 0.0
        off = (w * loose).sum(1) + 2.0 ** -24 * (before + 10 * w.sum(1))
        assert (np.abs(total[s, :, :p + 1] - before - w.sum(1)) <= off).all()
        assert (total[s, :, p + 1:] == st.total[s, :, p + 1:]).all() and (where[s, :, p] == p).all()
    assert (total[0, :, 302:] == st.total[0, :, 302:]).all()


def test_one_split_batch(nat, oracle):
    """A batch with a work-group for each (sequence, kv head): lengths from nothing to many passes, idle queries."""
    r = np.random.default_rng(12)
    lens = [0, 1, 2100, 31, 32, 600] + [int(x) for x in r.integers(0, 90, 60)]
    c = Cache(nat, oracle, 13, 16, 8, 32, lens, room=1)
    seqs = [int(x) for x in r.permutation(len(lens))]
    pos = [lens[s] if i % 9 else -1 for i, s in enumerate(seqs)]
    st = Step(c, pos, seqs=seqs, at=[abs(p) + 7 for p in pos], stride=2200, max_pos=2150)
    out, total, where = st.run()
    st.check((out, total, where))
    st = Step(c, [lens[s] if i % 9 else -1 for i, s in enumerate(seqs)], seqs=seqs, stride=2200, max_pos=2150)
    out, total, where = st.run(where=False)
    assert (where == st.where).all()
    for s, p in zip(seqs, st.pos):
        if p >= 0:
            where[s, :, p] = p                             # as if it had been given
    st.check((out, total, where))


def test_refusals(nat, oracle):
    c = Cache(nat, oracle, 9, 8, 2, 64, [50, 60], room=1)
    lib, P = c.lib, 4096
    nbytes = lib.tq_hip_decode_step_weights_ws_bytes(c.kv.h, 2, 60)
    good = dict(n=2, seq=None, pos=P, max_pos=60, q=P, k=P, v=P, cos=P, sin=P, out=P, at=None, total=P, where=P,
                stride=61, ws=P, ws_bytes=nbytes)

    def call(kv=None, **over):
        return lib.tq_hip_decode_step_weights_async(kv or c.kv.h, *{**good, **over}.values(), None)

    for over in (dict(n=-1), dict(n=65536, seq=P), dict(n=3), dict(pos=None), dict(max_pos=-1), dict(max_pos=1 << 24),
                 dict(q=None), dict(k=None), dict(v=None), dict(cos=None), dict(sin=None), dict(out=None),
                 dict(total=None), dict(stride=60), dict(ws=None), dict(ws_bytes=nbytes - 1), dict(q=P + 4),
                 dict(k=P + 8), dict(v=P + 4), dict(cos=P + 4), dict(out=P + 4), dict(ws=P + 8), dict(total=P + 1),
                 dict(where=P + 2), dict(seq=P + 1), dict(at=P + 3), dict(pos=P + 2)):
        assert call(**over) == nat.EINVAL, over
    assert call(n=0) == 0
    ws = lib.tq_hip_decode_step_weights_ws_bytes
    assert ws(c.kv.h, 0, 5) == ws(c.kv.h, 1, -1) == ws(c.kv.h, 65536, 5) == ws(None, 1, 5) == 0
    wide = nat.PagedKV(4, 2, 256, 4, max_seqs=2)
    assert ws(wide.h, 1, 5) == 0
    assert call(kv=wide.h, ws_bytes=1 << 20) == nat.ETYPE

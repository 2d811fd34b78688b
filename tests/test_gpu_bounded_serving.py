"""A run of the serving operators as they are used together: several prompts in
one packed call, decode steps that gather attention weights, eviction to a
bounded cache, steps that go on behind it at their own text positions, and the
rules on the logits that come out.  Every part is checked against its definition
as it stands after the parts before it."""
from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest

from tests.hip_graphs import Graphs
from tests.test_gpu_evict import Caches
from tests.test_gpu_logits import Batch, best, check as check_logits
from tests.test_gpu_prefill_packed import Packed
from tests.test_gpu_step_weights import Step

pytestmark = pytest.mark.gpu

LENS, KEEP, SINKS, RECENT, STRIDE = [75, 1, 40], 32, 4, 8, 96


@pytest.fixture(scope="module")
def nat():
    from tailorquantkernel_amd import native
    native.init(0)
    return native


class Run:
    """Sequences with their slots, text positions and totals, kept between the calls on the device and on the host."""

    def __init__(self, nat, oracle, seed, nq, nkv, hd):
        self.nat, self.lib = nat, nat.load()
        p = Packed(nat, oracle, seed, nq, nkv, hd, LENS, [0] * len(LENS))
        p.check(p.run(), dense=hd in (64, 128))
        self.c = p.c
        self.n = len(LENS)
        self.slots, self.text = list(LENS), list(LENS)
        self.total = np.zeros((self.n, nkv, STRIDE), np.float32)
        self.where = np.tile(np.arange(STRIDE, dtype=np.int32), (self.n, nkv, 1))
        self.dev = {"total": self.c.up(self.total), "where": self.c.up(self.where)}

    def step(self):
        """Inputs of one step of every sequence, on the run's totals."""
        st = Step(self.c, self.slots, at=self.text, stride=STRIDE)
        st.total, st.where = self.total, self.where
        st.dev["total"], st.dev["where"] = self.dev["total"], self.dev["where"]
        return st

    def stepped(self, st):
        got = st.results()
        st.check(got)
        _, self.total, self.where = got
        self.slots = [s + 1 for s in self.slots]
        self.text = [t + 1 for t in self.text]
        return got[0]

    def evict_call(self):
        """(launch, what it leaves): eviction of every sequence, in place."""
        c, host = self.c, np.ascontiguousarray(self.c.pool).view(np.uint8).reshape(-1)
        shape = (-1, c.nkv, 2, 16, c.nb * 36)
        state = SimpleNamespace(pool=host, view=lambda a: a.reshape(shape), total=self.total, where=self.where,
                                next=np.asarray(self.text, np.int32), nkv=c.nkv, pages=c.pages)
        longest = max(self.slots)
        want = Caches.expect(state, KEEP, SINKS, RECENT, range(self.n), True, longest, self.slots, True, None, None)
        nbytes = self.lib.tq_hip_kv_evict_ws_bytes(c.kv.h, self.n, longest, KEEP)
        ws = c.up(np.full(nbytes, 0xA5, np.uint8))
        length, upto = c.up(np.asarray(self.slots, np.int32)), c.up(np.asarray(self.text, np.int32))
        total, where = self.dev["total"].ptr, self.dev["where"].ptr

        def launch(stream=None):
            self.nat.check(self.lib.tq_hip_kv_evict_async(
                c.kv.h, self.n, None, length.ptr, longest, upto.ptr, KEEP, SINKS, RECENT, total, where, total, where,
                STRIDE, ws.ptr, nbytes, stream), "evict")
        self.hold = ws, length, upto
        return launch, want

    def evicted(self, want):
        self.c.sync()
        pool, total, where = want
        assert self.c.download().tobytes() == pool.tobytes(), "cache"
        assert (self.dev["total"].download(total.shape, np.float32) == total).all()
        assert (self.dev["where"].download(where.shape, np.int32) == where).all()
        self.c.pool = pool.view(self.c.pool.dtype).reshape(self.c.pool.shape)
        self.total, self.where = total, where
        self.slots = [min(s, KEEP) for s in self.slots]


@pytest.mark.parametrize("nq,nkv,hd", [(8, 2, 64), (4, 4, 128), (6, 1, 128), (4, 2, 32)])
def test_prompts_steps_eviction_steps(nat, oracle, nq, nkv, hd):
    r = Run(nat, oracle, nq + hd, nq, nkv, hd)
    for _ in range(2):
        for _ in range(3):
            st = r.step()
            nat.check(st.launch(), "step")
            out = r.stepped(st)
        launch, want = r.evict_call()
        launch()
        r.evicted(want)
    # the text so far as the rules' history, the outputs as logits
    vocab = nq * hd
    g = np.random.default_rng(hd)
    b = {"vocab": vocab, "logits": out.reshape(r.n, vocab), "tokens": g.integers(0, vocab, (r.n, 90)).astype(np.int32),
         "tok_len": np.asarray(r.text, np.int32), "prompt_len": np.asarray(LENS, np.int32),
         "repetition": np.full(r.n, 1.2, np.float32), "frequency": np.full(r.n, 0.1, np.float32),
         "allowed": g.random((r.n, vocab)) < 0.5}
    batch = Batch(nat, b)
    new, tokens = batch.call()
    check_logits(b, new, tokens)
    assert tokens == best(new)


def test_step_and_eviction_in_one_graph(nat, oracle):
    """Captured once and replayed on a state put back each time: the same bytes as the eager calls'."""
    r = Run(nat, oracle, 3, 8, 2, 64)
    before = r.c.pool.copy(), r.total.copy(), r.where.copy()
    st = r.step()
    nat.check(st.launch(), "step")
    out = r.stepped(st)
    launch, want = r.evict_call()
    launch()
    r.evicted(want)
    after = r.c.pool.copy()

    def put_back():
        r.c.pool = before[0]
        r.c.upload()
        r.dev["total"].upload(before[1])
        r.dev["where"].upload(before[2])

    g = Graphs()

    def both(stream):
        nat.check(st.launch(stream), "step")
        launch(stream)

    graph = g.capture(both)
    for _ in range(3):
        put_back()
        g.replay(graph)
        assert st.dev["out"].download(out.shape, np.float32).tobytes() == out.tobytes()
        assert r.c.download().tobytes() == after.tobytes()
        assert r.dev["total"].download(r.total.shape, np.float32).tobytes() == r.total.tobytes()
        assert (r.dev["where"].download(r.where.shape, np.int32) == r.where).all()

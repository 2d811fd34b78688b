"""The operators for long contexts in turn, as a model's steps call them: heads of a fused projection normalized and turned
at scaled positions, a step over common tokens, bounds of what it appended, a choice of blocks, a step over those."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from tests.hip_graphs import Graphs
from tests.serving import Cache
from tests.test_gpu_blocks import Bounds, Select, Step, expected_bounds
from tests.test_gpu_rope import descriptor, turned
from tests.test_gpu_shared import Shared, members

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nat():
    from tailorquantkernel_amd import native
    native.init(0)
    return native


def project(nat, st, pos, layout):
    """A projection's rows [q | k | v], its q and k heads into st's arrays, v beside them; what they come to is checked."""
    c, r, n = st.c, st.c.r, len(pos)
    wide, eps = (c.nq + 2 * c.nkv) * c.hd, 1e-6
    x = r.standard_normal((n, wide), dtype=np.float32)
    weights = [r.standard_normal(c.hd, dtype=np.float32) for _ in range(2)]
    d_x, d_w, d_pos = c.up(x), [c.up(w) for w in weights], c.up(np.asarray(pos, np.int32))
    q = nat.Heads(d_x.ptr, c.nq, wide, d_w[0].ptr, st.dev["q"].ptr, c.nq * c.hd)
    k = nat.Heads(d_x.ptr + 4 * c.nq * c.hd, c.nkv, wide, d_w[1].ptr, st.dev["k"].ptr, c.nkv * c.hd)
    nat.check(c.lib.tq_hip_norm_rope(C.byref(descriptor(nat, c.hd, "yarn", layout)), c.hd, n, d_pos.ptr, C.byref(q), C.byref(k),
                                     eps, None), "norm_rope")
    st.v = np.ascontiguousarray(x[:, (c.nq + c.nkv) * c.hd:]).reshape(n, c.nkv, c.hd)
    st.dev["v"].upload(st.v)
    c.sync()
    heads = x.reshape(n, -1, c.hd)
    for name, at, weight in (("q", slice(0, c.nq), weights[0]), ("k", slice(c.nq, c.nq + c.nkv), weights[1])):
        got = st.dev[name].download(getattr(st, name).shape, np.float32)
        want, off = turned(heads[:, at], weight, eps, c.hd, "yarn", layout, pos)
        assert np.all(np.abs(got - want) <= off)
        setattr(st, name, got)


@pytest.mark.parametrize("layout", [0, 1])
def test_steps_of_a_batch(nat, oracle, layout):
    nq, nkv, hd, block, keep = 8, 2, 64, 32, 12
    st = Shared(nat, oracle, 21 + layout, nq, nkv, hd, [(1600, members(9))], behind=[2500], rope=False, room=16, max_pos=8500)
    c, n = st.c, st.n
    stride = 8500 // block + 1
    bounds = Bounds(c, block, stride)
    want = expected_bounds(c, bounds.host, block, range(n), [0] * n, st.pos, max(st.pos))
    assert np.array_equal(bounds.make(st.pos), want)
    bounds.host = want
    long_ones = [3, n - 2, n - 1]
    for _ in range(3):
        # every query, over all that it has
        project(nat, st, st.pos, layout)
        st.launch()
        st.check(st.results())
        bounds.host = bounds.make([p + 1 for p in st.pos], st.pos)
        assert np.array_equal(bounds.host, expected_bounds(c, want, block, range(n), st.pos, [p + 1 for p in st.pos],
                                                           max(st.pos) + 1))
        pos = [p + 1 for p in st.pos]
        # some, over the blocks that score highest
        part = Step(c, [pos[i] for i in long_ones], block, keep, seqs=long_ones, rope=False, max_pos=8500, bounds=False)
        project(nat, part, part.pos, layout)
        sel = Select(nat, oracle, 0, nq, nkv, hd, part.pos, block, keep, 1, 2, seqs=long_ones, rope=False, max_seqs=n,
                     max_pos=8500)
        sel.q = sel.turned = part.q
        sel.bounds, sel.stride = bounds.host, stride
        part.list = sel.run()
        assert np.array_equal(part.list, sel.expected())
        part.dev["list"].upload(part.list)
        part.bounds = bounds
        part.check(part.run())
        want = bounds.host
        for i in long_ones:
            pos[i] += 1
        st.at(pos)


def test_a_captured_step(nat, oracle):
    """Bounds of a block, heads, choice and step as one graph, replayed as the sequences grow."""
    nq, nkv, hd, block, keep, most = 8, 2, 64, 16, 20, 1200
    lens = [1100, 700, 30]
    g = Graphs()
    c = Cache(nat, oracle, 31, nq, nkv, hd, lens, room=most - min(lens))
    n, r, wide, eps, stride = len(lens), c.r, (nq + nkv) * hd, 1e-6, most // block + 1
    bounds = Bounds(c, block, stride)
    bounds.host = bounds.make(lens, max_len=most)
    st = Step(c, lens, block, keep, rope=False, max_pos=most, bounds=False)
    st.bounds = bounds
    weights = [r.standard_normal(hd, dtype=np.float32) for _ in range(2)]
    d_x, d_w, d_from = c.up(np.zeros((n, wide), np.float32)), [c.up(w) for w in weights], c.up(np.zeros(n, np.int32))
    q = nat.Heads(d_x.ptr, nq, wide, d_w[0].ptr, st.dev["q"].ptr, nq * hd)
    k = nat.Heads(d_x.ptr + 4 * nq * hd, nkv, wide, d_w[1].ptr, st.dev["k"].ptr, nkv * hd)
    rope = descriptor(nat, hd, "bands")
    ws_bytes = c.lib.tq_hip_kv_select_ws_bytes(c.kv.h, n, most, block, keep)
    ws = c.up(np.full(ws_bytes, 0xFF, np.uint8))

    def enqueue(stream):
        d = {name: None if b is None else b.ptr for name, b in st.dev.items()}
        nat.check(c.lib.tq_hip_kv_bounds_async(c.kv.h, n, None, d_from.ptr, d["pos"], most, block, bounds.dev.ptr, stride,
                                               stream), "bounds")
        nat.check(c.lib.tq_hip_norm_rope(C.byref(rope), hd, n, d["pos"], C.byref(q), C.byref(k), eps, stream), "norm_rope")
        nat.check(c.lib.tq_hip_kv_select_async(c.kv.h, n, None, d["pos"], most, block, keep, 1, 2, d["q"], None, None,
                                               bounds.dev.ptr, stride, d["list"], ws.ptr, ws_bytes, stream), "select")
        st.launch(stream)

    graph = g.capture(enqueue)
    for _ in range(4):
        x = r.standard_normal((n, wide), dtype=np.float32)
        st.v = r.standard_normal(st.v.shape, dtype=np.float32)
        # (the last block's bounds are made again, from the same tokens)
        for b, a in ((d_x, x), (st.dev["v"], st.v), (st.dev["pos"], np.asarray(st.pos, np.int32)),
                     (d_from, np.asarray(st.pos, np.int32) - 1)):
            b.upload(a)
        g.replay(graph)
        out = st.results()
        heads = x.reshape(n, -1, hd)
        for name, part, weight in (("q", heads[:, :nq], weights[0]), ("k", heads[:, nq:], weights[1])):
            got = st.dev[name].download(part.shape, np.float32)
            want, off = turned(part, weight, eps, hd, "bands", 0, st.pos)
            assert np.all(np.abs(got - want) <= off)
            setattr(st, name, got)
        sel = Select(nat, oracle, 0, nq, nkv, hd, st.pos, block, keep, 1, 2, rope=False, max_pos=most)
        sel.q = sel.turned = st.q
        sel.bounds, sel.stride = bounds.host, stride
        st.list = st.dev["list"].download(st.list.shape, np.int32)
        assert np.array_equal(st.list, sel.expected())
        st.check(out)
        bounds.host = bounds.dev.download(bounds.host.shape, np.uint16)
        st.pos = [p + 1 for p in st.pos]

"""The operators for long contexts in turn, as a model's steps call them: heads of a fused projection normalized and turned
at scaled positions, a step over common tokens, bounds of what it appended, a choice of blocks, a step over those."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

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

"""What the step with common tokens refuses of a real cache (nothing is launched)."""
from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
P = 4096   # an aligned address that no refused call looks behind


@pytest.fixture(scope="module")
def nat():
    from tailorquantkernel_amd import native
    native.init(0)
    return native


@pytest.fixture(scope="module")
def kv(nat):
    return nat.PagedKV(8, 2, 64, 4, 6, 100)


def call(nat, kv, **over):
    a = dict(n=6, seq=None, pos=P, max_pos=1000, start=[0, 2, 6], prefix=[32, 0], q=P, k=P, v=P, cos=P, sin=P, out=P, ws=P,
             ws_bytes=1 << 26)
    a.update(over)
    start, prefix = np.asarray(a["start"], np.int32), np.asarray(a["prefix"], np.int32)
    groups = over.get("groups", len(prefix))
    lib = nat.load()
    s, p = (None if over.get(k, 0) is None else x.ctypes.data for k, x in (("start_at", start), ("prefix_at", prefix)))
    rc = lib.tq_hip_decode_step_shared_async(kv.h, a["n"], a["seq"], a["pos"], a["max_pos"], groups, s, p, a["q"], a["k"],
                                             a["v"], a["cos"], a["sin"], a["out"], a["ws"], a["ws_bytes"], None)
    return rc, lib.tq_hip_decode_step_shared_ws_bytes(kv.h, a["n"], a["max_pos"], groups, s, p)


@pytest.mark.parametrize("over", [
    dict(n=-1), dict(n=65536), dict(max_pos=-1), dict(max_pos=1 << 30), dict(groups=-1), dict(start_at=None),
    dict(prefix_at=None), dict(start=[-1, 2, 6]), dict(start=[0, 3, 2]), dict(start=[0, 2, 7]), dict(prefix=[8, 0]),
    dict(prefix=[-16, 0]), dict(prefix=[32, 1008]), dict(prefix=[17, 0])])
def test_groups(nat, kv, over):
    assert call(nat, kv, **over) == (nat.EINVAL, 0)


@pytest.mark.parametrize("over", [
    dict(n=7), dict(pos=None), dict(q=None), dict(k=None), dict(v=None), dict(cos=None), dict(sin=None), dict(out=None),
    dict(ws=None), dict(ws_bytes=100), dict(q=P + 4), dict(k=P + 8), dict(v=P + 4), dict(cos=P + 4), dict(out=P + 8),
    dict(ws=P + 8), dict(pos=P + 2), dict(seq=P + 1)])
def test_arrays(nat, kv, over):
    assert call(nat, kv, **over)[0] == nat.EINVAL


def test_shapes_that_are_not_served(nat):
    for hd in (32, 256):
        assert call(nat, nat.PagedKV(8, 2, hd, 4, 6, 100)) == (nat.ETYPE, 0)


def test_nothing_to_do(nat, kv):
    assert call(nat, kv, n=0, start=[0], prefix=[], pos=None, q=None)[0] == nat.OK

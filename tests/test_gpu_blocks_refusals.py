"""What the calls over blocks refuse of a real cache (nothing is launched)."""
from __future__ import annotations

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
    return nat.PagedKV(8, 2, 64, 4, 2, 100)


BLOCKS = [dict(block=0), dict(block=8), dict(block=24), dict(block=1040), dict(block=-16)]


@pytest.mark.parametrize("over", BLOCKS + [
    dict(n=-1), dict(n=65536), dict(n=3), dict(len=None), dict(max_len=0), dict(max_len=1601), dict(bounds=None),
    dict(bounds=P + 8), dict(stride=0), dict(stride=99), dict(seq=P + 2), dict(start=P + 1), dict(len=P + 3)])
def test_bounds(nat, kv, over):
    a = dict(n=2, seq=None, start=P, len=P, max_len=1600, block=16, bounds=P, stride=100)
    a.update(over)
    assert nat.load().tq_hip_kv_bounds_async(kv.h, *a.values(), None) == nat.EINVAL


@pytest.mark.parametrize("over", BLOCKS + [
    dict(n=-1), dict(n=65536), dict(n=3), dict(pos=None), dict(max_pos=-1), dict(max_pos=1600), dict(keep=0),
    dict(sinks=-1), dict(recent=0), dict(sinks=4), dict(recent=5), dict(q=None), dict(cos=None), dict(sin=None),
    dict(bounds=None), dict(stride=99), dict(list=None), dict(ws=None), dict(ws_bytes=0), dict(q=P + 4), dict(cos=P + 4),
    dict(bounds=P + 2), dict(ws=P + 8), dict(list=P + 2), dict(pos=P + 1), dict(seq=P + 2)])
def test_select(nat, kv, over):
    a = dict(n=2, seq=None, pos=P, max_pos=1599, block=16, keep=4, sinks=1, recent=1, q=P, cos=P, sin=P, bounds=P,
             stride=100, list=P, ws=P, ws_bytes=1 << 20)
    a.update(over)
    assert nat.load().tq_hip_kv_select_async(kv.h, *a.values(), None) == nat.EINVAL


@pytest.mark.parametrize("over", BLOCKS + [
    dict(n=-1), dict(n=65536), dict(n=3), dict(pos=None), dict(max_pos=-1), dict(keep=0), dict(keep=1 << 19),
    dict(list=None), dict(q=None), dict(k=None), dict(v=None), dict(cos=None), dict(out=None), dict(stride=99),
    dict(ws=None), dict(ws_bytes=15), dict(q=P + 4), dict(k=P + 8), dict(v=P + 4), dict(out=P + 4), dict(bounds=P + 2),
    dict(ws=P + 8), dict(list=P + 2), dict(pos=P + 1)])
def test_step(nat, kv, over):
    a = dict(n=2, seq=None, pos=P, max_pos=1599, block=16, keep=40, list=P, q=P, k=P, v=P, cos=P, sin=P, out=P, bounds=P,
             stride=100, ws=P, ws_bytes=1 << 24)
    a.update(over)
    assert nat.load().tq_hip_decode_step_blocks_async(kv.h, *a.values(), None) == nat.EINVAL


def test_shapes_that_are_not_served(nat):
    lib = nat.load()
    wide = nat.PagedKV(4, 2, 256, 4, 2, 4)
    assert lib.tq_hip_kv_select_ws_bytes(wide.h, 1, 63, 16, 4) == lib.tq_hip_decode_step_blocks_ws_bytes(wide.h, 1, 63, 16, 4) == 0
    assert lib.tq_hip_kv_select_async(wide.h, 1, None, P, 63, 16, 4, 1, 1, P, P, P, P, 4, P, P, 1 << 20, None) == nat.ETYPE
    assert lib.tq_hip_decode_step_blocks_async(wide.h, 1, None, P, 63, 16, 4, P, P, P, P, P, P, P, P, 4, P, 1 << 20,
                                               None) == nat.ETYPE


def test_workspaces(nat, kv):
    lib = nat.load()
    for f in (lib.tq_hip_kv_select_ws_bytes, lib.tq_hip_decode_step_blocks_ws_bytes):
        assert f(kv.h, 0, 63, 16, 4) == f(kv.h, 65536, 63, 16, 4) == f(kv.h, 1, -1, 16, 4) == f(kv.h, 1, 63, 15, 4) == 0
        assert f(kv.h, 1, 63, 16, 0) == 0 < f(kv.h, 1, 63, 16, 4)
    assert lib.tq_hip_kv_select_ws_bytes(kv.h, 1, 1600, 16, 4) == 0


def test_nothing_to_do(nat, kv):
    lib = nat.load()
    assert lib.tq_hip_kv_bounds_async(kv.h, 0, None, None, None, 0, 16, None, 0, None) == nat.OK
    assert lib.tq_hip_kv_select_async(kv.h, 0, None, None, 63, 16, 4, 1, 1, *[None] * 4, 0, None, None, 0, None) == nat.OK
    assert lib.tq_hip_decode_step_blocks_async(kv.h, 0, None, None, 63, 16, 4, *[None] * 8, 0, None, 0, None) == nat.OK

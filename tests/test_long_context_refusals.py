"""What the operators for long contexts refuse, before any device call (CPU)."""
from __future__ import annotations

import ctypes as C
import math

import pytest


@pytest.fixture(scope="module")
def nat():
    from tailorquantkernel_amd import native
    native.load()
    return native


P = 4096   # an aligned address that no refused call looks behind


def rope(nat, **over):
    a = dict(rotary_dim=64, layout=0, scaling=0, trained_len=8192, theta=10000.0, factor=4.0, low=1.0, high=4.0,
             magnitude=0.0)
    a.update(over)
    return nat.Rope(*a.values())


BAD_ROPES = [
    dict(rotary_dim=0), dict(rotary_dim=63), dict(rotary_dim=-2), dict(rotary_dim=258), dict(layout=2), dict(layout=-1),
    dict(scaling=5), dict(scaling=-1), dict(theta=0.5), dict(theta=math.nan), dict(theta=math.inf),
    dict(scaling=1, factor=0.5), dict(scaling=2, factor=math.nan), dict(scaling=2, factor=math.inf),
    dict(scaling=3, trained_len=0), dict(scaling=3, low=4.0), dict(scaling=3, low=-1.0), dict(scaling=3, high=math.inf),
    dict(scaling=4, trained_len=-1), dict(scaling=4, low=0.0), dict(scaling=4, low=5.0), dict(scaling=4, theta=1.0),
    dict(scaling=4, magnitude=-1.0), dict(scaling=4, magnitude=math.nan), dict(scaling=2, theta=1e300, factor=1e300)]


@pytest.mark.parametrize("over", BAD_ROPES)
def test_rope_descriptors(nat, over):
    lib, r = nat.load(), rope(nat, **over)
    assert lib.tq_hip_rope_rows(C.byref(r), 0, P, P, P, None) == nat.EINVAL
    q = nat.Heads(P, 1, 256, None, P, 256)
    assert lib.tq_hip_norm_rope(C.byref(r), 256, 0, P, C.byref(q), None, 1e-6, None) == nat.EINVAL


def test_rope_rows_arguments(nat):
    lib, r = nat.load(), rope(nat)
    f = lambda *a: lib.tq_hip_rope_rows(*a, None)  # noqa: E731
    assert f(C.byref(r), 0, None, None, None) == nat.OK
    assert f(None, 1, P, P, P) == f(C.byref(r), -1, P, P, P) == f(C.byref(r), 1, P, None, P) == nat.EINVAL
    assert f(C.byref(r), 1, P, P, None) == f(C.byref(r), 1, P + 2, P, P) == f(C.byref(r), 1, P, P + 1, P) == nat.EINVAL
    wide = rope(nat, rotary_dim=256)
    assert f(C.byref(wide), 2 ** 31 - 1, P, P, P) == nat.EINVAL


@pytest.mark.parametrize("over", [
    dict(x=None), dict(out=None), dict(x=P + 2), dict(out=P + 1), dict(norm=P + 2), dict(heads=-1), dict(heads=65537),
    dict(stride=255), dict(out_stride=255), dict(out=P, out_stride=260)])
def test_norm_rope_heads(nat, over):
    a = dict(x=P, heads=4, stride=256, norm=P, out=2 * P, out_stride=256)
    a.update(over)
    h, r = nat.Heads(*a.values()), rope(nat)
    for q, k in ((C.byref(h), None), (None, C.byref(h))):
        assert nat.load().tq_hip_norm_rope(C.byref(r), 64, 1, P, q, k, 1e-6, None) == nat.EINVAL


def test_norm_rope_arguments(nat):
    lib, r, h = nat.load(), rope(nat), nat.Heads(P, 4, 1024, P, P, 1024)
    f = lambda hd, n, pos: lib.tq_hip_norm_rope(C.byref(r), hd, n, pos, C.byref(h), None, 1e-6, None)  # noqa: E731
    assert f(64, 0, P) == nat.OK
    assert f(62, 1, P) == f(0, 1, P) == f(260, 1, P) == f(64, -1, P) == f(64, 2 ** 23 + 1, P) == nat.EINVAL
    assert f(64, 1, P + 1) == f(60, 1, P) == nat.EINVAL     # more values turn than a head has
    assert lib.tq_hip_norm_rope(C.byref(r), 64, 1, P, None, None, 1e-6, None) == nat.OK


def test_blocks_without_a_cache(nat):
    lib = nat.load()
    assert lib.tq_hip_kv_bounds_async(None, 1, None, None, P, 64, 16, P, 4, None) == nat.EINVAL
    assert lib.tq_hip_kv_select_ws_bytes(None, 1, 63, 16, 4) == 0
    assert lib.tq_hip_kv_select_async(None, 1, None, P, 63, 16, 4, 1, 1, P, P, P, P, 4, P, P, 1 << 20, None) == nat.EINVAL
    assert lib.tq_hip_decode_step_blocks_ws_bytes(None, 1, 63, 16, 4) == 0
    assert lib.tq_hip_decode_step_blocks_async(None, 1, None, P, 63, 16, 4, P, P, P, P, P, P, P, P, 4, P, 1 << 20,
                                               None) == nat.EINVAL


def test_shared_without_a_cache(nat):
    lib, start, prefix = nat.load(), (C.c_int32 * 2)(0, 4), (C.c_int32 * 1)(16)
    a = 1, C.addressof(start), C.addressof(prefix)
    assert lib.tq_hip_decode_step_shared_ws_bytes(None, 4, 63, *a) == 0
    assert lib.tq_hip_decode_step_shared_async(None, 4, None, P, 63, *a, P, P, P, P, P, P, P, 1 << 20, None) == nat.EINVAL

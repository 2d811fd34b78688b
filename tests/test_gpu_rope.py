"""Rotary rows and the normalized, rotated heads against their formulas in 64 bits."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

THETA, FACTOR, TRAINED = 500000.0, 8.0, 8192
KINDS = ("plain", "linear", "ntk", "bands", "yarn")
EDGES = {"bands": (1.0, 4.0), "yarn": (1.0, 32.0)}
ULP = 2.0 ** -24      # half a step of fp32, relative


@pytest.fixture(scope="module")
def nat():
    from tailorquantkernel_amd import native
    native.init(0)
    return native


def descriptor(nat, rot, kind="plain", layout=0, magnitude=0.0):
    low, high = EDGES.get(kind, (0.0, 0.0))
    return nat.Rope(rot, layout, KINDS.index(kind), TRAINED, THETA, FACTOR, low, high, magnitude)


def frequencies(rot, kind, magnitude=0.0):
    i = np.arange(rot // 2, dtype=np.float64)
    theta = THETA * FACTOR ** (rot / (rot - 2)) if kind == "ntk" and rot > 2 else THETA
    f = theta ** (-2 * i / rot)
    if kind == "linear":
        return f / FACTOR, 1.0
    if kind == "bands":
        low, high = EDGES[kind]
        t = TRAINED * f / (2 * np.pi)
        s = (t - low) / (high - low)
        return np.where(t <= low, f / FACTOR, np.where(t >= high, f, s * f + (1 - s) * f / FACTOR)), 1.0
    if kind == "yarn":
        low, high = EDGES[kind]
        at = [rot * np.log(TRAINED / (2 * np.pi * b)) / (2 * np.log(theta)) for b in (high, low)]
        first, last = max(np.floor(at[0]), 0), min(np.ceil(at[1]), rot - 1)
        r = np.clip((i - first) / max(last - first, 0.001), 0, 1)
        return f * (1 - r) + f / FACTOR * r, magnitude or 0.1 * np.log(FACTOR) + 1
    return f, 1.0


def rows(rot, kind, pos, magnitude=0.0):
    """cos, sin and their bound: one rounding to fp32; a frequency off by two steps of fp64 (pow and the scaling), the
    angle by one more; the reduction and the series below 2^-32."""
    f, m = frequencies(rot, kind, magnitude)
    angle = np.asarray(pos, np.float64)[:, None] * f
    cos, sin = m * np.cos(angle), m * np.sin(angle)
    loose = m * (2.0 ** -32 + np.abs(angle) * 2.0 ** -50)
    return cos, sin, ULP * np.abs(cos) + loose, ULP * np.abs(sin) + loose


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,rot", [(1, 2), (1, 128), (3, 6), (64, 128), (77, 96), (5, 256), (1000, 64), (2, 254)])
def test_rows(nat, kind, n, rot):
    r = np.random.default_rng(n * 1000 + rot)
    pos = r.integers(0, 1 << 20, n).astype(np.int32)
    pos[0] = 0 if n == 3 else pos[0]
    half = rot // 2
    d_pos = nat.DeviceBuffer.from_numpy(pos)
    out = np.full((2, n * half + 8), 7.0, np.float32)       # something behind each array
    d = nat.DeviceBuffer.from_numpy(out)
    sin_at = d.ptr + out[0].nbytes
    nat.check(nat.load().tq_hip_rope_rows(C.byref(descriptor(nat, rot, kind)), n, d_pos.ptr, d.ptr, sin_at, None), "rows")
    got = d.download(out.shape, np.float32)
    cos, sin, cos_off, sin_off = rows(rot, kind, pos)
    assert np.all(got[:, n * half:] == 7.0)
    assert np.all(np.abs(got[0, :n * half].reshape(n, half) - cos) <= cos_off)
    assert np.all(np.abs(got[1, :n * half].reshape(n, half) - sin) <= sin_off)


def test_rows_far_negative_and_numbered(nat):
    pos = np.asarray([2 ** 31 - 1, -2 ** 31, -1, -70000, 2 ** 30 + 1], np.int32)
    d_pos, d = nat.DeviceBuffer.from_numpy(pos), nat.DeviceBuffer(2 * 5 * 64 * 4)
    for given in (pos, None):
        at = given if given is not None else np.arange(5)
        nat.check(nat.load().tq_hip_rope_rows(C.byref(descriptor(nat, 128)), 5, d_pos.ptr if given is not None else None,
                                              d.ptr, d.ptr + 5 * 64 * 4, None), "rows")
        got = d.download((2, 5, 64), np.float32)
        cos, sin, cos_off, sin_off = rows(128, "plain", at)
        assert np.all(np.abs(got[0] - cos) <= cos_off) and np.all(np.abs(got[1] - sin) <= sin_off)


def test_rows_magnitude(nat):
    pos = np.arange(0, 9000, 271, dtype=np.int32)
    n = len(pos)
    d_pos, d = nat.DeviceBuffer.from_numpy(pos), nat.DeviceBuffer(2 * n * 32 * 4)
    rope = descriptor(nat, 64, "yarn", magnitude=1.5)
    nat.check(nat.load().tq_hip_rope_rows(C.byref(rope), n, d_pos.ptr, d.ptr, d.ptr + n * 32 * 4, None), "rows")
    got = d.download((2, n, 32), np.float32)
    cos, sin, cos_off, sin_off = rows(64, "yarn", pos, 1.5)
    assert np.all(np.abs(got[0] - cos) <= cos_off) and np.all(np.abs(got[1] - sin) <= sin_off)


def turned(x, weight, eps, rot, kind, layout, pos):
    """Heads x [n][heads][hd] in 64 bits and the bound of what comes out.

    Roundings of fp32, each half a step: squares 1, their sum 2 in a lane and 6 over the lanes, of which the root halves
    9 to 4.5, as it halves those of the mean and of eps (1 together); the root and its inverse 2; times x, times the
    weight 2; cos or sin 1, its product 1, the pair's sum 1.  13 in all, of |a c| + |b s|."""
    x = x.astype(np.float64)
    if weight is not None:
        x = x / np.sqrt(eps + (x * x).mean(-1, keepdims=True)) * weight.astype(np.float64)
    cos, sin, cos_off, sin_off = (t[:, None] for t in rows(rot, kind, pos))
    i = np.arange(rot // 2)
    a, b = (i, i + rot // 2) if layout == 0 else (2 * i, 2 * i + 1)
    y, off = x.copy(), 13 * ULP * np.abs(x)
    y[..., a], y[..., b] = x[..., a] * cos - x[..., b] * sin, x[..., a] * sin + x[..., b] * cos
    for to, p, q in ((a, a, b), (b, b, a)):
        u, v = np.abs(x[..., p]), np.abs(x[..., q])
        off[..., to] = 13 * ULP * (u * np.abs(cos) + v * np.abs(sin)) + u * cos_off + v * sin_off
    return y, off


def run(nat, hd, x, q_heads, k_heads, weights, eps, rope, pos, shift=0, in_place=False, stream=None):
    """Rows x [n][wide] of q's heads, k's and more: q and k as they come out, and the whole buffer of the results."""
    n, wide = x.shape
    d_x = nat.DeviceBuffer(x.nbytes + 16)
    nat.check(nat.load().tq_hip_memcpy_h2d(d_x.ptr + shift, np.ascontiguousarray(x).ctypes.data, x.nbytes, None), "x")
    d_w = [None if w is None else nat.DeviceBuffer.from_numpy(w) for w in weights]
    d_pos = None if pos is None else nat.DeviceBuffer.from_numpy(pos)
    out_wide = wide if in_place else (q_heads + k_heads) * hd + 3
    out = np.full((n + 1, out_wide), 7.0, np.float32)
    d_out = nat.DeviceBuffer.from_numpy(out)
    base = d_x.ptr + shift if in_place else d_out.ptr
    ptr = lambda b: None if b is None else b.ptr  # noqa: E731
    q = nat.Heads(d_x.ptr + shift, q_heads, wide, ptr(d_w[0]), base, out_wide)
    k = nat.Heads(d_x.ptr + shift + 4 * q_heads * hd, k_heads, wide, ptr(d_w[1]), base + 4 * q_heads * hd, out_wide)
    nat.check(nat.load().tq_hip_norm_rope(C.byref(rope), hd, n, ptr(d_pos), C.byref(q) if q_heads else None,
                                          C.byref(k) if k_heads else None, eps, stream), "norm_rope")
    nat.check(nat.load().tq_hip_device_synchronize(), "sync")
    if in_place:
        got = np.empty((n, wide), np.float32)
        nat.check(nat.load().tq_hip_memcpy_d2h(got.ctypes.data, d_x.ptr + shift, got.nbytes, None), "out")
    else:
        got = d_out.download(out.shape, np.float32)
    heads = got[:n, :(q_heads + k_heads) * hd].reshape(n, q_heads + k_heads, hd)
    return heads, got


SHAPES = [(32, 8, 2, 32), (64, 8, 2, 64), (128, 32, 8, 128), (128, 16, 16, 64), (256, 4, 1, 256), (96, 3, 1, 96),
          (4, 5, 1, 4), (128, 8, 8, 2), (80, 6, 2, 20), (64, 24, 8, 62), (128, 1, 1, 126), (36, 2, 1, 18), (256, 2, 2, 10)]


@pytest.mark.parametrize("hd,nq,nk,rot", SHAPES)
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("norm", [True, False])
def test_heads(nat, hd, nq, nk, rot, layout, norm):
    r = np.random.default_rng(hd * 7 + rot)
    n, kind = 9, KINDS[(hd + rot) % 5]
    x = (3 * r.standard_normal((n, (nq + 2 * nk) * hd))).astype(np.float32)
    weights = [r.standard_normal(hd).astype(np.float32) if norm else None for _ in range(2)]
    pos = r.integers(0, 200000, n).astype(np.int32)
    got, whole = run(nat, hd, x, nq, nk, weights, 1e-6, descriptor(nat, rot, kind, layout), pos)
    heads = x[:, :(nq + nk) * hd].reshape(n, nq + nk, hd)
    for part, weight in ((slice(0, nq), weights[0]), (slice(nq, None), weights[1])):
        want, off = turned(heads[:, part], weight, 1e-6, rot, kind, layout, pos)
        assert np.all(np.abs(got[:, part] - want) <= off)
    assert np.all(whole[n:] == 7.0) and np.all(whole[:, (nq + nk) * hd:] == 7.0)


@pytest.mark.parametrize("hd,nq,nk,rot", [(128, 32, 8, 128), (64, 8, 2, 32), (128, 4, 1, 66), (96, 3, 1, 96)])
@pytest.mark.parametrize("layout", [0, 1])
def test_in_place_and_unaligned_give_the_same(nat, hd, nq, nk, rot, layout):
    r = np.random.default_rng(5)
    n = 300                            # enough work-groups for four heads a lane at 32 + 8 heads
    x = r.standard_normal((n, (nq + 2 * nk) * hd + 1)).astype(np.float32)     # an odd stride
    weights = [r.standard_normal(hd).astype(np.float32) for _ in range(2)]
    rope = descriptor(nat, rot, "bands", layout)
    got, _ = run(nat, hd, x, nq, nk, weights, 1e-5, rope, None)
    want, off = turned(x[:, :nq * hd].reshape(n, nq, hd), weights[0], 1e-5, rot, "bands", layout, np.arange(n))
    assert np.all(np.abs(got[:, :nq] - want) <= off)
    for shift, in_place in ((4, False), (0, True), (12, True)):
        other, whole = run(nat, hd, x, nq, nk, weights, 1e-5, rope, None, shift, in_place)
        assert np.array_equal(other, got)
        if in_place:
            assert np.array_equal(whole[:, (nq + nk) * hd:], x[:, (nq + nk) * hd:])


@pytest.mark.parametrize("n,nq,nk", [(1, 32, 8), (511, 32, 8), (513, 32, 8), (3001, 32, 8), (1030, 6, 1), (1030, 9, 2),
                                     (1030, 20, 1), (1030, 28, 4), (400, 64, 8)])
def test_many_rows(nat, n, nq, nk):
    """Every number of heads that a lane takes, and rows either side of where it changes."""
    r = np.random.default_rng(n)
    hd = 128
    x = r.standard_normal((n, (nq + nk) * hd)).astype(np.float32)
    weights = [r.standard_normal(hd).astype(np.float32) for _ in range(2)]
    pos = r.integers(0, 100000, n).astype(np.int32)
    got, _ = run(nat, hd, x, nq, nk, weights, 1e-6, descriptor(nat, hd, "yarn"), pos)
    for part, weight in ((slice(0, nq), weights[0]), (slice(nq, None), weights[1])):
        want, off = turned(x.reshape(n, nq + nk, hd)[:, part], weight, 1e-6, hd, "yarn", 0, pos)
        assert np.all(np.abs(got[:, part] - want) <= off)


def test_only_queries_or_only_keys(nat):
    r = np.random.default_rng(2)
    x = r.standard_normal((4, 6 * 64)).astype(np.float32)
    rope = descriptor(nat, 64)
    both, _ = run(nat, 64, x, 4, 2, [None, None], 0.0, rope, None)
    queries, _ = run(nat, 64, x, 4, 0, [None, None], 0.0, rope, None)
    keys, _ = run(nat, 64, np.ascontiguousarray(x[:, 4 * 64:]), 0, 2, [None, None], 0.0, rope, None)
    assert np.array_equal(both[:, :4], queries) and np.array_equal(both[:, 4:], keys)


def test_a_head_that_is_no_number_or_nothing(nat):
    """Infinities and NaN stay in their head; a head of zeros comes out as zeros."""
    r = np.random.default_rng(3)
    x = r.standard_normal((3, 4 * 64)).astype(np.float32)
    clean, _ = run(nat, 64, x, 4, 0, [np.ones(64, np.float32), None], 1e-6, descriptor(nat, 64), None)
    x[0, 5], x[1, 64 + 9], x[2, 128:192] = np.nan, np.inf, 0.0
    got, _ = run(nat, 64, x, 4, 0, [np.ones(64, np.float32), None], 1e-6, descriptor(nat, 64), None)
    assert np.all(np.isnan(got[0, 0])) and np.isnan(got[1, 1]).any() and np.all(got[2, 2] == 0)
    same = np.ones((3, 4), bool)
    same[0, 0] = same[1, 1] = same[2, 2] = False
    assert np.array_equal(got[same], clean[same])


def test_position_zero_leaves_a_head_as_it_is(nat):
    x = np.random.default_rng(4).standard_normal((1, 128)).astype(np.float32)
    got, _ = run(nat, 128, x, 1, 0, [None, None], 0.0, descriptor(nat, 128), np.zeros(1, np.int32))
    assert np.array_equal(got.reshape(-1), x.reshape(-1))


def test_captured_and_replayed(nat):
    from tests.hip_graphs import Graphs
    g, r = Graphs(), np.random.default_rng(6)
    n, hd = 5, 128
    d_pos, d_x = nat.DeviceBuffer.from_numpy(np.zeros(n, np.int32)), nat.DeviceBuffer(n * 4 * hd * 4)
    d_out, d_rows = nat.DeviceBuffer(n * 4 * hd * 4), nat.DeviceBuffer(2 * n * 64 * 4)
    rope, q = descriptor(nat, hd, "bands"), nat.Heads(d_x.ptr, 4, 4 * hd, None, d_out.ptr, 4 * hd)

    def calls(stream):
        nat.check(nat.load().tq_hip_rope_rows(C.byref(rope), n, d_pos.ptr, d_rows.ptr, d_rows.ptr + n * 256, stream), "r")
        nat.check(nat.load().tq_hip_norm_rope(C.byref(rope), hd, n, d_pos.ptr, C.byref(q), None, 0.0, stream), "n")

    graph = g.capture(calls)
    for _ in range(3):
        pos = r.integers(0, 50000, n).astype(np.int32)
        x = r.standard_normal((n, 4, hd)).astype(np.float32)
        d_pos.upload(pos)
        d_x.upload(x)
        g.replay(graph)
        cos, sin, cos_off, sin_off = rows(hd, "bands", pos)
        got = d_rows.download((2, n, 64), np.float32)
        assert np.all(np.abs(got[0] - cos) <= cos_off) and np.all(np.abs(got[1] - sin) <= sin_off)
        want, off = turned(x, None, 0.0, hd, "bands", 0, pos)
        assert np.all(np.abs(d_out.download((n, 4, hd), np.float32) - want) <= off)

"""What tq_hip_kv_select_async ranks blocks by: the sum over heads and channels of max(q M, q m) while a block's bounds are
finite, and what infinite bounds make of the sum that stands in the header."""
from __future__ import annotations

import numpy as np
import pytest

from tests.serving import PAGE, Cache
from tests.test_gpu_blocks import Bounds, Select, value

pytestmark = pytest.mark.gpu
INF = np.inf


@pytest.fixture(scope="module")
def nat():
    from tailorquantkernel_amd import native
    native.init(0)
    return native


def bf16(x):
    """Bits of values that bf16 holds as they are."""
    bits = np.ascontiguousarray(x, np.float32).view(np.uint32)
    assert not (bits & 0xFFFF).any()
    return (bits >> 16).astype(np.uint16)


def listed(scores, keep, sinks, recent):
    """The rules over scores that need no rounding; None ranks lowest."""
    count = len(scores)
    free = range(sinks, count - recent)
    best = sorted(free, key=lambda b: (scores[b] is None, -scores[b] if scores[b] is not None else 0, b))
    return sorted([*range(sinks), *best[:keep - sinks - recent], *range(count - recent, count)])


@pytest.mark.parametrize("nq,nkv,hd", [(2, 2, 32), (8, 2, 64), (8, 1, 128), (3, 1, 64)])
@pytest.mark.parametrize("blocks", [40, 700])
def test_finite_bounds_score_what_a_key_can(nat, oracle, nq, nkv, hd, blocks):
    """Products of quarters and sixteenths, of which 64 bits lose nothing in any order; heads of both signs and zeros."""
    s = Select(nat, oracle, blocks, nq, nkv, hd, [16 * blocks - 1], 16, blocks // 3, 1, 2, rope=False)
    r = np.random.default_rng(blocks)
    s.q = s.turned = (r.integers(-8, 9, s.q.shape) / 4).astype(np.float32)
    least = r.integers(-100, 101, s.bounds.shape[:3] + (hd,))
    m = np.stack([least + r.integers(0, 101, least.shape), least], 3) / 16
    s.bounds = bf16(m)
    got = s.run()
    for h in range(nkv):
        q = s.q[0, h * nq // nkv:(h + 1) * nq // nkv].astype(np.float64)
        per = np.maximum(q[:, None] * m[0, h, :blocks, 0], q[:, None] * m[0, h, :blocks, 1])       # [head][block][channel]
        assert got[0, h].tolist() == listed([float(x) for x in per.sum((0, 2))], *s.rules[1:]), f"kv head {h}"


# the group's q in two channels, a block's bounds there, and its score: a number, an infinity, or None (NaN)
INFINITE = [
    ([(1, -2)], (3, INF), (-1, -4), None),               # infinity times the sum of no positive q
    ([(1, -2)], (3, 1), (-INF, -4), None),
    ([(1, -2)], (-INF, 1), (INF, -4), None),             # a channel without a number, as the bounds have it
    ([(1, -2)], (3, 1), (-1, -INF), INF),
    ([(1, 2)], (3, INF), (-1, -4), INF),
    ([(1, -2), (1, 3)], (3, INF), (-1, -4), INF),        # heads of both signs: nothing times infinity
    ([(1, -2), (1, 3)], (3, 1), (-1, -INF), INF),
    ([(1, -2), (1, 3)], (3, -INF), (-1, INF), -INF),     # without a number
    ([(1, -2), (-3, 3)], (INF, -INF), (-1, INF), None),
    ([(0, 0)], (INF, 1), (-1, -4), None),
    ([(1, -2)], (3, 1), (-1, -4), 11)]


@pytest.mark.parametrize("q,most,least,score", INFINITE)
def test_infinite_bounds(nat, oracle, q, most, least, score):
    """Block 7 has them; the others score 2^100 downwards, below 0 too, and every one's place is known."""
    g, blocks = len(q), 60
    sizes = [0] * blocks
    for h in (0, 1):
        s = Select(nat, oracle, 1, 2 * g, 2, 32, [16 * blocks - 1], 16, 2, 0, 1, rope=False)
        s.q[:] = 0
        s.q[0, h * g:(h + 1) * g, 4], s.q[0, h * g:(h + 1) * g, 30] = np.asarray(q, np.float32).T
        s.turned = s.q
        up, down = (f(s.q[0, h * g:(h + 1) * g].astype(np.float64), 0).sum(0) for f in (np.maximum, np.minimum))
        m = np.zeros((blocks, 2, 32), np.float32)
        for c in (4, 30):                                # bounds that are no interval score any size
            k = np.arange(blocks) - 30
            x = np.sign(k) * np.exp2(np.abs(k)) / 2
            m[:, 0, c] = x if up[c] else 0
            m[:, 1, c] = -x if down[c] else 0
        m[7, :, 4], m[7, :, 30] = (most[0], least[0]), (most[1], least[1])
        s.bounds[:, h, :blocks] = bf16(m)
        sizes = [float((up[[4, 30]] * m[b, 0, [4, 30]] + down[[4, 30]] * m[b, 1, [4, 30]]).sum()) if b != 7 else score
                 for b in range(blocks)]
        for keep in (2, 30, 31, 32, 58, 59):
            s.rules = (16, keep, 0, 1)
            assert s.run()[0, h].tolist() == listed(sizes, keep, 0, 1), keep


def test_blocks_without_pages_come_last(nat, oracle):
    """Of a sequence that lost pages: the bounds as made, and no list that has another choice names them."""
    c = Cache(nat, oracle, 3, 8, 2, 64, [640])
    lost = [3, 11, 12, 30]
    c.kv.set_pages(0, np.where(np.isin(np.arange(40), lost), -1, c.pages[0]).astype(np.int32))
    b = Bounds(c, PAGE, 40)
    b.host = b.make([640])
    assert (value(b.host[0, :, lost, 0]) == -INF).all() and (value(b.host[0, :, lost, 1]) == INF).all()
    for keep in (9, 36, 38):
        s = Select(nat, oracle, keep, 8, 2, 64, [639], PAGE, keep, 0, 1, rope=False)
        s.bounds, s.stride = b.host, 40
        got = s.run()
        for h in range(2):
            assert len(set(got[0, h]) & set(lost)) == max(0, keep - 36)

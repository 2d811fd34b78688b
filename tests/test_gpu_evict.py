"""tq_hip_kv_evict_async on the GPU: the kept tokens, the rows that move, the
totals and positions, against the definition on the host.  Nothing is computed
that could round: every comparison is exact, and bytes that the call does not
write are those from before."""
from __future__ import annotations

import numpy as np
import pytest

from tests.hip_graphs import Graphs

pytestmark = pytest.mark.gpu

PAGE = 16


@pytest.fixture(scope="module")
def nat():
    from tailorquantkernel_amd import native
    native.init(0)
    return native


class Caches:
    """A cache of random bytes on scattered pages, with totals and positions."""

    def __init__(self, nat, seed, nkv, hd, lens, stride=None, nq=None):
        r = self.r = np.random.default_rng(seed)
        self.nat, self.lens, self.nkv, self.hd = nat, list(lens), nkv, hd
        n, longest = len(lens), max(1, max(lens))
        self.stride = stride or longest
        need = [-(-max(1, m) // PAGE) for m in lens]
        extra = 3                                             # pages of nobody
        ids = r.permutation(sum(need) + extra).astype(np.int32)
        self.kv = nat.PagedKV(nq or nkv, nkv, hd, sum(need) + extra, n, max(need) + 1)
        self.pages, at = [], 0
        for i, p in enumerate(need):
            self.pages.append(ids[at:at + p])
            self.kv.set_pages(i, ids[at:at + p])
            at += p
        self.base, self.nbytes, _ = self.kv.pool()
        self.pool = r.integers(0, 256, self.nbytes).astype(np.uint8)
        self.total = r.random((n, nkv, self.stride)).astype(np.float32)
        self.where = np.tile(np.arange(self.stride, dtype=np.int32), (n, nkv, 1))
        self.next = np.asarray(lens, np.int32)

    def view(self, pool):
        return pool.reshape(-1, self.nkv, 2, PAGE, self.hd // 32 * 36)

    def up(self, a):
        return self.nat.DeviceBuffer.from_numpy(np.ascontiguousarray(a))

    def run(self, keep, sinks=0, recent=0, order=None, in_place=False, max_len=None, lens=None, use_next=True):
        nat, lib = self.nat, self.nat.load()
        order = list(range(len(self.lens))) if order is None else order
        lens = self.lens if lens is None else lens
        nat.check(lib.tq_hip_memcpy_h2d(self.base, self.pool.ctypes.data, self.nbytes, None), "pool")
        total, where = self.up(self.total), self.up(self.where)
        fill_t, fill_w = np.full_like(self.total, -5.0), np.full_like(self.where, -6)
        total_out = total if in_place else self.up(fill_t)
        where_out = where if in_place else self.up(fill_w)
        seq = self.up(np.asarray(order, np.int32))
        length = self.up(np.asarray([lens[i] if 0 <= i < len(lens) else 9 for i in order], np.int32))
        upto = self.up(np.asarray([self.next[i] if 0 <= i < len(lens) else 9 for i in order], np.int32))
        max_len = max(1, max(self.lens)) if max_len is None else max_len
        nbytes = lib.tq_hip_kv_evict_ws_bytes(self.kv.h, len(order), max_len, keep)
        ws = self.up(np.full(nbytes, 0xAB, np.uint8))
        nat.check(lib.tq_hip_kv_evict_async(self.kv.h, len(order), seq.ptr, length.ptr, max_len,
                                            upto.ptr if use_next else None, keep, sinks, recent, total.ptr, where.ptr,
                                            total_out.ptr, where_out.ptr, self.stride, ws.ptr, nbytes, None), "evict")
        nat.check(lib.tq_hip_device_synchronize(), "sync")
        pool = np.empty(self.nbytes, np.uint8)
        nat.check(lib.tq_hip_memcpy_d2h(pool.ctypes.data, self.base, self.nbytes, None), "pool")
        got = (pool, total_out.download(self.total.shape, np.float32), where_out.download(self.where.shape, np.int32))
        want = self.expect(keep, sinks, recent, order, in_place, max_len, lens, use_next, fill_t, fill_w)
        for g, w, what in zip(got, want, ("cache", "totals", "positions")):
            assert g.tobytes() == w.tobytes(), what
        return got

    def expect(self, keep, sinks, recent, order, in_place, max_len, lens, use_next, fill_t, fill_w):
        pool = self.pool.copy()
        old, new = self.view(self.pool), self.view(pool)
        total, where = (self.total.copy(), self.where.copy()) if in_place else (fill_t.copy(), fill_w.copy())
        for i in order:
            if not 0 <= i < len(lens):
                continue
            m = min(lens[i], max_len)
            upto = int(self.next[i]) if use_next else lens[i]
            for h in range(self.nkv):
                p = self.where[i, h, :max(0, m)]
                t = self.total[i, h, :max(0, m)]
                safe = (p < sinks) | (p >= upto - recent)
                # rank: safe, then the total, NaN last; the lower slot first
                rank = sorted(range(max(0, m)), key=lambda s: (not safe[s], bool(np.isnan(t[s])) and not safe[s],
                                                               0.0 if safe[s] or np.isnan(t[s]) else -float(t[s]), s))
                stay = set(rank[:keep])
                holes = [s for s in range(min(m, keep)) if s not in stay]
                movers = [s for s in sorted(stay) if s >= keep]
                assert len(holes) == len(movers)
                for s in stay:
                    if s < keep:
                        total[i, h, s], where[i, h, s] = self.total[i, h, s], self.where[i, h, s]
                for a, b in zip(holes, movers):
                    total[i, h, a], where[i, h, a] = self.total[i, h, b], self.where[i, h, b]
                    pa, pb = self.pages[i][a // PAGE], self.pages[i][b // PAGE]
                    new[pa, h, :, a % PAGE] = old[pb, h, :, b % PAGE]
        return pool, total, where


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("in_place", [False, True])
def test_kept_and_moved(nat, hd, in_place):
    c = Caches(nat, hd, 2, hd, [200, 0, 1, 64, 65, 17, 131], stride=211)
    c.run(64, 2, 10, in_place=in_place)
    c.run(1, 0, 0, in_place=in_place)
    c.run(1, 0, 1, in_place=in_place)
    c.run(199, 4, 100, in_place=in_place)
    c.run(200, in_place=in_place)                # nothing to drop
    c.run(5000, 100, 300, in_place=in_place)


@pytest.mark.parametrize("keep", [1, 63, 64, 1023, 1024, 2047, 2048, 3000])
def test_lengths_around_the_waves(nat, keep):
    c = Caches(nat, keep, 3, 64, [keep + 1, keep + 64, 3333, 1024, 1025])
    c.run(keep, min(2, keep), min(5, keep - min(2, keep)))


def test_long(nat):
    c = Caches(nat, 1, 1, 32, [70001])
    c.run(30000, 4, 5000)
    c.run(69999, 0, 1)


def test_equal_totals_keep_the_lower_slots(nat):
    c = Caches(nat, 2, 2, 64, [500, 300])
    c.total[:] = 0.25
    c.run(100)
    c.total[0, :, ::2] = 0.0
    c.total[0, :, 1::4] = -0.0
    c.run(300)
    c.run(100, 3, 20)


def test_totals_that_are_no_numbers(nat):
    c = Caches(nat, 3, 1, 64, [256])
    c.total[0, 0, ::3] = np.nan
    c.total[0, 0, 1::9] = np.inf
    c.total[0, 0, 2::9] = -np.inf
    c.total[0, 0, 5] = np.finfo(np.float32).max
    for keep in (10, 60, 150, 200, 255):
        c.run(keep, 2, 5)
    c.total[:] = np.nan
    c.run(100, 0, 7)


def test_positions_decide_not_slots(nat):
    """After earlier evictions the slots are out of order: the window goes by text position."""
    c = Caches(nat, 4, 2, 128, [400])
    for h in range(2):
        c.where[0, h] = c.r.permutation(1000)[:400]
    c.next[:] = 1000
    c.run(150, 40, 100)
    c.run(390, 0, 300)
    # more tokens are safe than kept: the lower slots
    c.where[:] = 0
    c.run(100, 1, 0)


def test_order_subset_and_strangers(nat):
    """Sequences in any order, some not in the call, some that the cache does not have; the length as the next position."""
    c = Caches(nat, 5, 2, 64, [90, 70, 40, 110])
    c.run(32, 1, 8, order=[3, 1])
    c.run(32, 1, 8, order=[2, -1, 0, 4])
    c.run(32, 1, 8, use_next=False)
    c.run(32, 1, 8, max_len=64)                  # longer ones are cut
    c.run(32, 1, 8, lens=[90, -4, 0, 110])


def test_twice_in_a_row(nat):
    """In place, then more tokens, then again: the first call's state is the second's input."""
    c = Caches(nat, 6, 2, 64, [300])
    pool, total, where = c.run(200, 4, 50, in_place=True)
    c.pool, c.total, c.where = pool, total, where
    c.lens, c.next = [240], np.asarray([340], np.int32)
    c.where[:, :, 200:240] = np.arange(300, 340)
    c.run(200, 4, 50, in_place=True)


def test_captured_and_replayed(nat):
    lib, gr = nat.load(), Graphs()
    c = Caches(nat, 7, 2, 64, [300, 500])
    total, where = c.up(c.total), c.up(c.where)
    total_out, where_out = c.up(np.full_like(c.total, -5.0)), c.up(np.full_like(c.where, -6))
    length = c.up(np.asarray(c.lens, np.int32))
    nbytes = lib.tq_hip_kv_evict_ws_bytes(c.kv.h, 2, 500, 128)
    ws = nat.DeviceBuffer(nbytes)
    g = gr.capture(lambda s: nat.check(lib.tq_hip_kv_evict_async(
        c.kv.h, 2, None, length.ptr, 500, None, 128, 2, 30, total.ptr, where.ptr, total_out.ptr, where_out.ptr,
        c.stride, ws.ptr, nbytes, s), "captured"))
    fills = np.full_like(c.total, -5.0), np.full_like(c.where, -6)
    for seed in range(4):
        c.total = np.random.default_rng(seed).random(c.total.shape).astype(np.float32)
        total.upload(c.total)
        total_out.upload(fills[0])
        where_out.upload(fills[1])
        nat.check(lib.tq_hip_memcpy_h2d(c.base, c.pool.ctypes.data, c.nbytes, None), "pool")
        gr.replay(g)
        pool = np.empty(c.nbytes, np.uint8)
        nat.check(lib.tq_hip_memcpy_d2h(pool.ctypes.data, c.base, c.nbytes, None), "pool")
        want = c.expect(128, 2, 30, [0, 1], False, 500, c.lens, False, *fills)
        assert pool.tobytes() == want[0].tobytes()
        assert total_out.download(c.total.shape, np.float32).tobytes() == want[1].tobytes()


@pytest.mark.parametrize("length,keep", [(300, 150), (40000, 10000), (40000, 39950)])
def test_a_sequence_named_twice(nat, length, keep):
    """Against the contract: what becomes of that sequence is not said, everything else is as it should be."""
    lib = nat.load()
    c = Caches(nat, length, 2, 32, [length, 700, 90], stride=length + 3)
    pages, guard = [p for i in (1, 2) for p in c.pages[i]], 4096
    total, where = c.up(c.total), c.up(c.where)
    order = np.asarray([0, 1, 0, 0], np.int32)
    seq, length_of = c.up(order), c.up(np.asarray([c.lens[i] for i in order], np.int32))
    nbytes = lib.tq_hip_kv_evict_ws_bytes(c.kv.h, 4, length, keep)
    ws = c.up(np.full(nbytes + guard, 0xAB, np.uint8))
    nat.check(lib.tq_hip_memcpy_h2d(c.base, c.pool.ctypes.data, c.nbytes, None), "pool")
    nat.check(lib.tq_hip_kv_evict_async(c.kv.h, 4, seq.ptr, length_of.ptr, length, None, keep, 2, 10, total.ptr, where.ptr,
                                        total.ptr, where.ptr, c.stride, ws.ptr, nbytes, None), "evict")
    nat.check(lib.tq_hip_device_synchronize(), "sync")
    pool = np.empty(c.nbytes, np.uint8)
    nat.check(lib.tq_hip_memcpy_d2h(pool.ctypes.data, c.base, c.nbytes, None), "pool")
    want = c.expect(keep, 2, 10, [1], True, length, c.lens, False, None, None)
    nobody = sorted(set(range(c.view(pool).shape[0])) - set(c.pages[0]))
    assert set(pages) <= set(nobody)
    assert c.view(pool)[nobody].tobytes() == c.view(want[0])[nobody].tobytes()
    got = total.download(c.total.shape, np.float32), where.download(c.where.shape, np.int32)
    for g, w in zip(got, want[1:]):
        assert g[1:].tobytes() == w[1:].tobytes() and g[0, :, length:].tobytes() == w[0, :, length:].tobytes()
    assert (ws.download((nbytes + guard,), np.uint8)[nbytes:] == 0xAB).all()


def test_refusals(nat):
    lib, P = nat.load(), 4096
    c = Caches(nat, 8, 2, 64, [100, 50])
    nbytes = lib.tq_hip_kv_evict_ws_bytes(c.kv.h, 2, 100, 32)
    good = dict(n=2, seq=None, len=P, max_len=100, next=None, keep=32, sinks=1, recent=8, total=P, where=P, total_out=P,
                where_out=P, stride=100, ws=P, ws_bytes=nbytes)

    def call(**over):
        a = {**good, **over}
        return lib.tq_hip_kv_evict_async(c.kv.h, *a.values(), None)

    for over in (dict(n=-1), dict(n=65536), dict(n=3), dict(len=None), dict(max_len=0), dict(max_len=10 ** 6),
                 dict(stride=99), dict(keep=0), dict(keep=-1), dict(sinks=-1), dict(recent=-1), dict(sinks=33),
                 dict(recent=32), dict(recent=2 ** 31 - 1), dict(total=None), dict(where=None), dict(total_out=None),
                 dict(where_out=None), dict(total_out=8192), dict(where_out=8192), dict(ws=None), dict(ws=P + 4),
                 dict(ws_bytes=nbytes - 1), dict(total=P + 2, total_out=P + 2), dict(len=P + 1), dict(next=P + 2)):
        assert call(**over) == nat.EINVAL, over
    assert call(n=0) == 0
    assert lib.tq_hip_kv_evict_ws_bytes(c.kv.h, 0, 100, 32) == 0
    assert lib.tq_hip_kv_evict_ws_bytes(c.kv.h, 2, 0, 32) == 0 == lib.tq_hip_kv_evict_ws_bytes(c.kv.h, 2, 100, 0)

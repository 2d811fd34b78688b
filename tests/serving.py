"""What the tests of the serving operators share: a paged cache with known
contents, and attention on its codes in 64 bits."""
from __future__ import annotations

import numpy as np

from oracle.binding import BLOCK_Q8, QK

PAGE = 16


def values(blocks):
    """What block_q8 rows [..., nb] stand for, in 64 bits: [..., nb * 32]."""
    x = blocks["q"].astype(np.float64) * blocks["d"].astype(np.float64)[..., None]
    return x.reshape(*blocks.shape[:-1], -1)


def quantized(oracle, x):
    """block_q8 rows of fp32 rows x [..., hd]."""
    return oracle.quantize_row_q8(x.reshape(-1)).reshape(*x.shape[:-1], x.shape[-1] // QK)


def rotated(oracle, x, cos, sin):
    """RoPE of x [rows][heads][hd] with rows cos, sin (None: as it is)."""
    if cos is None:
        return x
    out = np.empty_like(x)
    for r in range(x.shape[0]):
        for h in range(x.shape[1]):
            out[r, h] = oracle.rope_apply(x[r, h], cos[r], sin[r])
    return out


def rope_rows(oracle, hd, positions, theta=10000.0):
    t = [oracle.rope_table(hd, int(p), theta) for p in positions]
    return np.stack([c for c, _ in t]), np.stack([s for _, s in t])


class Cache:
    """Sequences of quantized random rows on scattered pages of a PagedKV; what holds no row is random bytes (finite scales)."""

    def __init__(self, nat, oracle, seed, nq, nkv, hd, lens, room=0, pages_of=None):
        self.nat, self.lib, self.oracle = nat, nat.load(), oracle
        self.nq, self.nkv, self.hd, self.nb = nq, nkv, hd, hd // QK
        self.r = np.random.default_rng(seed)
        need = [max(1, -(-(m + room) // PAGE)) for m in lens]
        ids = self.r.permutation(sum(need) + 2).astype(np.int32)
        self.kv = nat.PagedKV(nq, nkv, hd, len(ids), len(lens), max(need))
        self.pages, at = [], 0
        for i, p in enumerate(need):
            self.pages.append(np.arange(at, at + p, dtype=np.int32) if pages_of == "in order" else ids[at:at + p])
            self.kv.set_pages(i, self.pages[i])
            at += p
        self.base, self.nbytes, _ = self.kv.pool()
        pool = np.empty((len(ids), nkv, 2, PAGE, self.nb), BLOCK_Q8)
        pool["q"] = self.r.integers(-128, 128, pool["q"].shape)
        pool["d"] = self.r.random(pool["d"].shape)
        self.pool = pool
        for i, m in enumerate(lens):
            if m > 0:
                rows = self.r.standard_normal((m, nkv, 2, hd), dtype=np.float32)
                self.put(i, range(m), quantized(oracle, rows))
        self.upload()

    def put(self, i, slots, rows):
        """rows [n][nkv][2][nb] into sequence i's slots, on the host."""
        for t, row in zip(slots, rows):
            self.pool[self.pages[i][t // PAGE], :, :, t % PAGE] = row

    def rows(self, i, n):
        """Sequence i's first n rows [n][nkv][2][nb], from the host's pool."""
        t = np.arange(n)
        return self.pool[self.pages[i][t // PAGE], :, :, t % PAGE]

    def upload(self):
        p = np.ascontiguousarray(self.pool)
        self.nat.check(self.lib.tq_hip_memcpy_h2d(self.base, p.ctypes.data, self.nbytes, None), "pool")

    def download(self):
        p = np.empty(self.pool.shape, BLOCK_Q8)
        self.nat.check(self.lib.tq_hip_memcpy_d2h(p.ctypes.data, self.base, self.nbytes, None), "pool")
        return p

    def up(self, a):
        return self.nat.DeviceBuffer.from_numpy(np.ascontiguousarray(a))

    def sync(self):
        self.nat.check(self.lib.tq_hip_device_synchronize(), "sync")


def attention(cache, q_blocks, rows, last, term=2.0 ** -17):
    """Query rows q_blocks [m][nq][nb], row r over keys rows[0..last[r]] ([n][nkv][2][nb]): outputs [m][nq][hd], their
    error bound in fp32, weights [m][nq][n] and theirs (relative).

    The bound.  A score (base 2, scaled) is nb products of an exact integer dot with two scales, added up and taken
    against a running maximum: 3 nb + 6 roundings of numbers no larger than S, the largest sum of magnitudes in the
    row, so it is off by (3 nb + 6) 2^-24 S and the weight by ln 2 times that; exp2 and its argument's subtraction add
    2^-23 and ln 2 * 126 * 2^-24 (beyond 126 the weight is nothing).  A sum of n non-negative terms in any order of
    partial sums is off by at most n 2^-24 of itself.  A weight is such a term over such a sum.  An output is such a
    sum of weights times values, each product kept to `term` (2^-17 where they are split in two bf16 parts).
    """
    nq, nkv, hd, nb = cache.nq, cache.nkv, cache.hd, cache.nb
    group, n, m = nq // nkv, rows.shape[0], q_blocks.shape[0]
    k, v = values(rows[:, :, 0]), values(rows[:, :, 1])             # [n][nkv][hd]
    q = values(q_blocks)
    out, bound = np.empty((m, nq, hd)), np.empty((m, nq, hd))
    weights, loose = np.empty((m, nq, n)), np.empty((m, nq))
    hidden = np.arange(n)[None, :] > np.asarray(last)[:, None]
    for h in range(nq):
        kh, vh = k[:, h // group], v[:, h // group]
        per_block = np.abs(np.einsum("mbj,nbj->mnb", q[:, h].reshape(m, nb, QK), kh.reshape(n, nb, QK)))
        s = q[:, h] @ kh.T / np.sqrt(hd)
        size = np.where(hidden, 0.0, per_block.sum(-1)).max(1) / np.sqrt(hd) * np.log2(np.e)
        s[hidden] = -np.inf
        w = np.exp(s - s.max(1, keepdims=True))
        w /= w.sum(1, keepdims=True)
        one = 2.0 ** -24 * (2 * np.log(2) * ((3 * nb + 6) * size + 126) + 4 + n)
        weights[:, h], loose[:, h] = w, one
        out[:, h] = w @ vh
        bound[:, h] = (w @ np.abs(vh)) * (one + 2.0 ** -24 * n + term)[:, None]
    return out, bound, weights, loose

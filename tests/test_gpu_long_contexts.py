"""The longest contexts of the packed prefill and of the step with weights, with
values that mark each key tile: one column of 64 is 1 in a tile's rows, the
others 0, so that an output is the share of the attention weight that its tiles
have.  The general bound grows with the context (a sum of n terms in any order,
n 2^-24 of itself: 0.8 % here), a tile of 32 keys is about 3 % of its column.
Two arrangements, tile % 64 and tile // 32, tell every tile of 2,048 apart, so
that one left out, taken twice or read in another's place shows; that one left
out does is tested on the reference itself, on the CPU."""
from __future__ import annotations

from types import SimpleNamespace

import numpy as np
import pytest

from tests.serving import Cache, attention, quantized

HD, TILE, N = 64, 32, 65536


@pytest.fixture(scope="module")
def nat():
    from tailorquantkernel_amd import native
    native.init(0)
    return native


def column(arrangement, t):
    tile = np.asarray(t) // TILE
    return tile % HD if arrangement == "by turns" else tile // 32 % HD


def marks(arrangement, t):
    """fp32 value rows [len(t)][HD]."""
    v = np.zeros((len(t), HD), np.float32)
    v[np.arange(len(t)), column(arrangement, t)] = 1.0
    return v


ARRANGEMENTS = pytest.mark.parametrize("arrangement", ["by turns", "in a row"])


@ARRANGEMENTS
def test_the_bound_sees_a_tile(oracle, arrangement):
    """Reference outputs without one tile (the first, some in the middle, the last) are outside the bound."""
    c = SimpleNamespace(nq=2, nkv=1, hd=HD, nb=2)
    r = np.random.default_rng(1)
    rows = np.stack([quantized(oracle, r.standard_normal((N, 1, HD), dtype=np.float32)),
                     quantized(oracle, marks(arrangement, range(N))[:, None])], 2)
    q = quantized(oracle, r.standard_normal((2, 2, HD), dtype=np.float32))
    last = [N - 2, N - 1]
    ref, bound, _, _ = attention(c, q, rows, last, 2.0 ** -17)
    bound += N * 2.0 ** -28 / 127
    for tile in (0, 1, 31, 32, 777, 1024, 1999, 2046, 2047):
        less = rows.copy()
        less["d"][TILE * tile:TILE * tile + TILE, :, 1] = 0.0
        out = attention(c, q, less, last, 2.0 ** -17)[0]
        assert (np.abs(out - ref) > 2 * bound).any(2).all(), tile


@pytest.mark.gpu
@ARRANGEMENTS
@pytest.mark.parametrize("form,new,before", [
    ("dense", 40, N - 40), ("dense", 200, N - 200), ("dense", 129, 30001), ("rows", 3, N - 3), ("rows", 20, N - 16)])
def test_packed(nat, oracle, arrangement, form, new, before):
    from tests.test_gpu_prefill_packed import Packed

    def change(p):
        c = p.c
        rows = c.rows(0, before)
        rows[:, :, 1] = quantized(oracle, marks(arrangement, range(before))[:, None])
        c.put(0, range(before), rows)
        c.upload()
        p.v[:new] = marks(arrangement, range(before, before + new))[:, None]
    p = Packed(nat, oracle, new, 2, 1, HD, [new, 7], [before, 3], change=change)
    p.check(p.run(), dense=form == "dense")


@pytest.mark.gpu
@ARRANGEMENTS
@pytest.mark.parametrize("length", [N, 70000])
def test_step_with_weights(nat, oracle, arrangement, length):
    from tests.test_gpu_step_weights import Step
    c = Cache(nat, oracle, 3, 2, 1, HD, [length, 12], room=1)
    rows = c.rows(0, length)
    rows[:, :, 1] = quantized(oracle, marks(arrangement, range(length))[:, None])
    c.put(0, range(length), rows)
    c.upload()
    st = Step(c, [length, 12], seqs=[0, 1])
    st.check(st.run())

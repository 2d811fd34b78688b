"""Values beside much larger ones where key tiles are attended to by many rows at once: each product of a weight and a value
keeps 2^-20 of itself, and nothing past 2^-28 of the row's largest V scale is lost.

A row's q is the sign pattern of one key, whose score is 200 and more above every other's in base 2, so its weight is 1
and what the others add is below 2^-180: the output is that key's value.  Of the term stay the 2^-20, some 16 roundings of
2^-24 (the row's sum, divisions, units, splits and their merge) and the 2^-28."""
from __future__ import annotations

import numpy as np
import pytest

from tests.serving import values
from tests.test_gpu_prefill_packed import Packed
from tests.test_gpu_shared import Shared

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nat():
    from tailorquantkernel_amd import native
    native.init(0)
    return native


def patterns(r, rows, wild):
    """Keys of sign patterns into block_q8 rows [n][nkv][2][nb], V scales 2^-4 .. 2^-24 apart within a key; wild: keys far
    below their tile's largest, too."""
    n, nkv, _, nb = rows.shape
    sign = r.choice(np.asarray([-1, 1], np.int8), (n, nkv, nb, 32))
    rows["q"][:, :, 0], rows["d"][:, :, 0] = 100 * sign, 0.5
    size = np.exp2(-r.uniform(0, 24, (n, nkv, nb)))
    size[np.arange(n)[:, None], np.arange(nkv), r.integers(0, nb, (n, nkv))] = 1.0     # a large block in every key
    if wild:
        size *= np.exp2(-r.integers(0, 2, (n, nkv, 1)) * 20.0)
    rows["q"][:, :, 1] = r.integers(-127, 128, (n, nkv, nb, 32))
    small = r.random((n, nkv, nb, 1)) < 0.5
    rows["q"][:, :, 1] = np.where(small, np.sign(rows["q"][:, :, 1]) * (np.abs(rows["q"][:, :, 1]) % 4), rows["q"][:, :, 1])
    rows["d"][:, :, 1] = size * r.uniform(0.5, 1.0, (n, nkv, 1))
    return sign.reshape(n, nkv, -1)


def compare(out, want, top):
    bound = np.abs(want) * (2.0 ** -20 + 16 * 2.0 ** -24) + 2.0 ** -28 * top
    far = np.abs(out - want) / bound
    assert (far <= 1).all(), f"{(far > 1).sum()} of {far.size} values, up to {far.max():.3g} of the bound"


@pytest.mark.parametrize("wild", [False, True])
@pytest.mark.parametrize("nq,nkv,hd,n", [(8, 2, 64, 40), (8, 2, 128, 40), (4, 4, 128, 100)])
def test_behind_common_tokens(nat, oracle, nq, nkv, hd, n, wild):
    prefix = 272
    st = Shared(nat, oracle, hd + n, nq, nkv, hd, [(prefix, [i % 9 for i in range(n)])], rope=False)
    c, r, g = st.c, st.c.r, nq // nkv
    rows = np.array(c.rows(0, prefix))
    sign = patterns(r, rows, wild)
    c.put(0, range(prefix), rows)
    at = r.integers(0, prefix, (st.n, nq))
    st.q = sign[at, np.arange(nq) // g].astype(np.float32)
    st.dev["q"].upload(st.q)
    out = st.run()[:n]
    v = values(rows[:, :, 1])
    top = max(rows["d"][:, :, 1].max(), *(c.rows(i, p + 1)["d"][prefix:, :, 1].max() for i, p in enumerate(st.pos[:n])))
    compare(out, v[at[:n], np.arange(nq) // g], float(top))


@pytest.mark.parametrize("wild", [False, True])
@pytest.mark.parametrize("nq,nkv,hd,n", [(8, 2, 64, 200), (8, 2, 128, 100), (2, 2, 128, 300)])
def test_packed_prompts(nat, oracle, nq, nkv, hd, n, wild):
    before, g = 250, nq // nkv

    def change(p):
        p.rows_of = np.array(p.c.rows(0, before))
        p.sign = patterns(p.c.r, p.rows_of, wild)
        p.c.put(0, range(before), p.rows_of)
        p.c.upload()
        p.at = p.c.r.integers(0, before, (p.q.shape[0], nq))
        p.q = p.sign[p.at, np.arange(nq) // g].astype(np.float32)
    p = Packed(nat, oracle, hd + n, nq, nkv, hd, [n], [before], rope=False, change=change, spare=0)
    out = p.run()
    v = values(p.rows_of[:, :, 1])
    compare(out, v[p.at, np.arange(nq) // g], max(1.0, float(np.abs(p.v).max()) / 127))

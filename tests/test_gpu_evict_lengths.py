"""tq_hip_kv_evict_async at the lengths where another form of its selection
begins (1,024, 4,096, 16,384 and 32,768 tokens, then any), with few moves, made
by the selecting work-groups, and many, made by a second launch: exact, as in
tests/test_gpu_evict.py."""
from __future__ import annotations

import numpy as np
import pytest

from tests.test_gpu_evict import Caches

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nat():
    from tailorquantkernel_amd import native
    native.init(0)
    return native


@pytest.mark.parametrize("length", [1023, 1024, 1025, 4095, 4096, 4097, 16383, 16384, 16385, 32767, 32768, 32769])
@pytest.mark.parametrize("in_place", [False, True])
def test_lengths_around_the_forms(nat, length, in_place):
    c = Caches(nat, length, 1, 32, [length, length // 2 + 1, 0, length - 1], stride=length + 3)
    c.run(length - 128, 4, 100, in_place=in_place)       # at most 128 moves: few
    c.run(length - 129, 4, 100, in_place=in_place)       # one more: listed
    c.run(128, 2, 60, in_place=in_place)                 # few stay
    c.run(length // 2, 3, length // 8, in_place=in_place)


@pytest.mark.parametrize("length,few", [(9000, True), (9000, False), (30000, True), (30000, False)])
def test_equal_and_odd_totals(nat, length, few):
    """Ties over the waves' runs of slots, and totals that are no numbers."""
    c = Caches(nat, length, 2, 32, [length, length - 777])
    keep = length - 60 if few else length // 3
    c.total[:] = 0.25
    c.run(keep, 2, 50)
    c.total[:, :, ::2] = 0.0
    c.total[:, :, 1::4] = -0.0
    c.run(keep, 2, 50, in_place=True)
    c.total[:] = c.r.random(c.total.shape).astype(np.float32)
    c.total[:, :, ::3], c.total[:, :, 1::9], c.total[:, :, 2::9] = np.nan, np.inf, -np.inf
    c.run(keep, 2, 50, in_place=True)
    c.where[:, 0] = c.r.permutation(length)[None, :]     # the window by text position
    c.run(keep, 20, length // 4)

"""Steps whose new token has no page."""
from __future__ import annotations

import numpy as np
import pytest

from tests.serving import PAGE, Cache
from tests.test_gpu_blocks import Bounds, Step, value

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nat():
    from tailorquantkernel_amd import native
    native.init(0)
    return native


@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("block", [16, 64])
@pytest.mark.parametrize("keep", [3, 40])
def test_a_key_that_is_not_cached_enters_no_bounds(nat, oracle, hd, block, keep):
    """The new token first of a block, at a page's start within one, and (its page taken away) in the middle of a page: the
    bounds that the step keeps are those that are made of what the cache holds."""
    lens = [640, 656, 700, 333]
    c = Cache(nat, oracle, hd + block, 8, 2, hd, lens, room=1)
    for i, p in enumerate(lens[:3]):
        c.kv.set_pages(i, np.where(np.arange(len(c.pages[i])) == p // PAGE, -1, c.pages[i]).astype(np.int32))
    st = Step(c, lens, block, keep)
    made = Bounds(c, block, st.bounds.stride, seed=1)
    made.make(lens)
    st.bounds.dev.upload(made.dev.download(made.host.shape, np.uint16))
    before = c.download()
    st.run()
    kept = st.bounds.dev.download(made.host.shape, np.uint16)
    again = made.make([p + 1 for p in lens])
    for i, p in enumerate(lens):
        assert np.array_equal(kept[i, :, :p // block + 1], again[i, :, :p // block + 1]), f"sequence {i}"
    if block == 16:
        assert (value(kept[0, :, 40, 0]) == -np.inf).all() and (value(kept[0, :, 40, 1]) == np.inf).all()
    after = c.download()
    assert [s for s in range(len(before)) if before[s].tobytes() != after[s].tobytes()] == [c.pages[3][333 // PAGE]]

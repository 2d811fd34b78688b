"""Steps with queries whose sequence is none of the cache's."""
from __future__ import annotations

import numpy as np
import pytest

from tests.serving import Cache
from tests.test_gpu_blocks import Step
from tests.test_gpu_shared import Shared, members

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nat():
    from tailorquantkernel_amd import native
    native.init(0)
    return native


@pytest.mark.parametrize("length,keep", [(20, 2), (300, 6), (5000, 300)])
def test_a_step_over_blocks_leaves_queries_of_no_sequence_out(nat, oracle, length, keep):
    """In one split and in several; whatever stands in their lists."""
    lens = [length, length // 2, length]
    c = Cache(nat, oracle, length, 8, 2, 64, lens, room=1)
    seqs = np.asarray([1, -1, 3, 0, 10 ** 6], np.int32)
    pos = [length // 2, length, length, length, 7]
    st = Step(c, pos, 16, keep, seqs=[1, 2, 2, 0, 2])
    st.list[1:3:2] = -1
    st.dev["list"].upload(st.list)
    st.dev["seq"].upload(seqs)
    out = st.run()
    st.seqs, st.pos = seqs.tolist(), [pos[0], -1, -1, pos[3], -1]
    st.check(out)


@pytest.mark.parametrize("large", [False, True])
@pytest.mark.parametrize("own", [30, 2500])
def test_a_shared_step_leaves_queries_of_no_sequence_out(nat, oracle, large, own):
    """Some of a group, all of a group, and one that shares nothing."""
    st = Shared(nat, oracle, own, 8, 2, 64, [(96, [5, own, 7, 8]), (4112, members(20)), (64, members(40)), (32, [4])],
                behind=[10, 20], order=[], large=large)
    seqs = np.asarray(st.order, np.int32)
    away = [0, 2, *range(24, 64), st.n - 2]
    seqs[away] = [(-1, st.n, -7, 10 ** 6)[i % 4] for i in range(len(away))]
    st.dev["seq"].upload(seqs)
    out = st.run()
    for i in away:
        st.pos[i] = -1
    st.check(out)


def test_a_step_by_itself_leaves_queries_of_no_sequence_out(nat, oracle):
    st = Shared(nat, oracle, 5, 8, 2, 64, [(0, [900, 5, 6, 7]), (32, [4])], behind=[3], order=[], large=False)
    seqs = np.asarray(st.order, np.int32)
    seqs[[1, 4, 5]] = -1, 6, 100
    st.dev["seq"].upload(seqs)
    out = st.run()
    for i in (1, 4, 5):
        st.pos[i] = -1
    st.check(out)


@pytest.mark.parametrize("length,keep", [(40, 3), (5000, 300)])
@pytest.mark.parametrize("seq", [-1, 2])
def test_one_query_of_no_sequence(nat, oracle, length, keep, seq):
    """Alone in the call, over blocks and behind common tokens: nothing is written."""
    c = Cache(nat, oracle, length, 8, 2, 64, [length, 5], room=1)
    st = Step(c, [length], 16, keep, seqs=[0])
    st.dev["seq"].upload(np.asarray([seq], np.int32))
    out = st.run()
    st.pos = [-1]
    st.check(out)
    st = Shared(nat, oracle, length, 8, 2, 64, [], behind=[length], order=[], large=False)
    st.dev["seq"].upload(np.asarray([seq - 1], np.int32) if seq > 0 else np.asarray([seq], np.int32))
    out = st.run()
    st.pos = [-1]
    st.check(out)


def test_many_queries_some_of_no_sequence(nat, oracle):
    """More than are ranked by length, over blocks."""
    lens = [int(x) for x in np.random.default_rng(3).integers(0, 200, 140)]
    st = Step(Cache(nat, oracle, 6, 4, 2, 64, lens, room=1), lens, 16, 4, seqs=list(range(140)))
    seqs = np.arange(140, dtype=np.int32)
    seqs[::9] = 140 + seqs[::9]
    seqs[4::9] = -1 - seqs[4::9]
    st.dev["seq"].upload(seqs)
    out = st.run()
    st.pos = [p if 0 <= s < 140 else -1 for p, s in zip(lens, seqs)]
    st.check(out)

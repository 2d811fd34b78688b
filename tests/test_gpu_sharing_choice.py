"""Which groups of a step attend to their common tokens together: a group by what it gains itself, whatever stands beside
it.  A member's page table is changed under a group's common tokens: read together these are the first member's, by itself
its own."""
from __future__ import annotations

import numpy as np
import pytest

from tests.serving import PAGE
from tests.test_gpu_shared import Shared, members

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def nat():
    from tailorquantkernel_amd import native
    native.init(0)
    return native


def other_pages(st, group, together):
    """The last member of `group` gets the group's first page over and over; the expected rows follow what is read."""
    c, last, pages = st.c, st.start[group + 1] - 1, st.prefix[group] // PAGE
    table = np.array(c.pages[last])
    table[:pages] = table[0]
    c.kv.set_pages(last, table)
    if not together:
        c.pages[last] = table


@pytest.mark.parametrize("rest", [[], [(768, members(4))], [(480, members(4))] * 12, [(768, members(2)), (1600, members(5))]])
def test_a_group_that_gains_is_not_held_back(nat, oracle, rest):
    """64 queries of 8 heads each save 58 x 672 tokens' reads per head, 4 % more than it takes; 4 with their block of rows
    lose."""
    st = Shared(nat, oracle, len(rest), 8, 8, 64, [(672, members(64)), *rest], large=False, max_pos=7000)
    other_pages(st, 0, True)
    st.check(st.run())


def test_a_group_that_loses_goes_by_itself(nat, oracle):
    """Beside one that gains much: 5 queries of 8 heads each save less than their block of rows takes."""
    st = Shared(nat, oracle, 1, 8, 8, 64, [(1600, members(64)), (768, members(4)), (768, members(5))], large=False, max_pos=7000)
    for group in (1, 2):
        other_pages(st, group, False)
    st.check(st.run())


def test_small_groups_together_where_few_others_have_as_much(nat, oracle):
    """Far more common tokens than each work-group has of the others: two members are enough."""
    st = Shared(nat, oracle, 2, 8, 8, 64, [(1600, members(64)), (6400, members(2)), (6400, members(4))], large=False)
    for group in (0, 1, 2):
        other_pages(st, group, True)
    st.check(st.run())


def test_too_little_to_gain(nat, oracle):
    st = Shared(nat, oracle, 3, 8, 8, 64, [(640, members(64))], large=False, max_pos=7000)
    other_pages(st, 0, False)
    st.check(st.run())


@pytest.mark.parametrize("nq,nkv", [(8, 8), (24, 8), (32, 8), (64, 8), (16, 16), (4, 1)])
@pytest.mark.parametrize("n,prefix", [(12, 8192), (32, 2048)])
def test_as_many_as_the_header_says(nat, oracle, nq, nkv, n, prefix):
    """With fewer kv heads as many times more common tokens; a small group beside them changes nothing."""
    prefix *= max(1, 8 // nkv)
    st = Shared(nat, oracle, n, nq, nkv, 64, [(64, members(4)), (prefix, [0] * n)], large=False)
    other_pages(st, 1, True)
    st.checked = 0                   # the last query alone: the one whose table is another
    st.check(st.run())

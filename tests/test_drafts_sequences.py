"""Placed trees and their sequences: what became another sequence, or other tokens of it, since place() is neither committed nor cut."""
import pytest

from sabrewing_amd.attention import PagedCache
from sabrewing_amd.drafts import DraftTrees
from test_drafts_host import Fake
from test_paged_cache import invariants


def closed_and_another_opened(c, s):
    c.close(s)
    assert c.open() == s
    c.rows([(s, 7)])


def cut_and_filled_again(c, s):
    c.truncate(s, 3)
    c.rows([(s, 4)])


def the_tree_cut_and_filled_again(c, s):
    c.truncate(s, 6)
    c.rows([s])


def closed_and_a_fork_in_its_place(c, s):
    other = c.open()
    c.rows([(other, 7)])
    c.close(s)
    assert c.fork(other) == s


@pytest.mark.parametrize("how", [closed_and_another_opened, cut_and_filled_again, the_tree_cut_and_filled_again, closed_and_a_fork_in_its_place])
def test_as_long_as_before_but_not_the_same(how):
    be = Fake()
    c = PagedCache(be, 1, 12, 8, 2, 32, max_seqs=3, max_rows=16)
    s = c.open()
    c.rows([(s, 5)])
    t = DraftTrees(c, max_trees=2, max_nodes=4)
    t.place([(s, [-1, 0], [1, 2])])
    how(c, s)
    assert c.length(s) == 7
    be.accept = [[0]]
    with pytest.raises(ValueError):
        t.commit(0)
    assert c.length(s) == 7
    t.drop()
    assert c.length(s) == 7
    invariants(c)
    t.place([(s, [-1, 0, 0], [1, 2, 3])])              # and the trees can be used again
    be.accept = [[0, 2]]
    assert t.commit(0) == [([0, 2], 7)]
    assert c.length(s) == 9
    invariants(c)


def test_what_leaves_a_sequence_as_it_is():
    """a truncation to its own length, its pages moved, other sequences' steps, a fork that is gone again: still the tree's"""
    be = Fake()
    c = PagedCache(be, 1, 12, 8, 2, 32, max_seqs=4, max_rows=16)
    x, s = c.open(), c.open()
    c.rows([(x, 9), (s, 5)])
    t = DraftTrees(c, max_trees=2, max_nodes=4)
    t.place([(s, [-1, 0], [1, 2])])
    c.truncate(s, 7)
    c.rows([x])
    c.close(c.fork(s))
    c.close(x)
    c.compact()
    be.accept = [[0, 1]]
    assert t.commit(0) == [([0, 1], 7)]
    assert c.length(s) == 7
    invariants(c)

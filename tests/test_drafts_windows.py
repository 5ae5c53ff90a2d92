"""Trees as deep as a layer's window: a node would attend to ancestors that the same token in a plain step does not see, so they are refused."""
import pytest

from sabrewing_amd.attention import AttnConfig, PagedCache
from sabrewing_amd.backend import Backend
from sabrewing_amd.drafts import DraftTrees
from test_attention_stack_host import Recorder, stack


class R(Recorder):
    trees = staticmethod(Backend.trees)


CHAIN = lambda n: ([-1] + list(range(n - 1)), list(range(n)))


def step(be, st, cache, rows, S, trees):
    be.calls.clear()
    st.step(be.alloc(4), be.alloc(4), be.alloc(4), be.alloc(4), S, cache=cache, rows=rows, trees=trees)


@pytest.mark.parametrize("windows", [(0, 4), (4, 0), (9, 4), (4, 4)])
def test_trees_as_deep_as_a_window(windows):
    be = R()
    configs = [AttnConfig(4, 2, 32, 32, window=w) for w in windows]
    st = stack(be, configs)
    cache = PagedCache(be, 2, 16, 8, 2, 32, max_seqs=3, max_rows=16)
    t = DraftTrees(cache, max_nodes=8)
    s = cache.open()
    rows, S = t.place([(s, *CHAIN(4))])                # 3 deep: its last node sees its first
    step(be, st, cache, rows, S, t)
    assert be.calls.count("attn_tree") == 2
    t.drop()
    with pytest.raises(ValueError):                    # what a recorded step would replay over
        t.place([(s, *CHAIN(5))])
    assert cache.length(s) == 0
    rows, S = t.place([(s, [-1, 0, 0, 1, 1, 0, 0, 0], list(range(8)))])      # many nodes, 2 deep
    step(be, st, cache, rows, S, t)
    t.drop()
    other = DraftTrees(cache, max_nodes=8)             # deep trees, placed before any layer was run over them
    rows, S = other.place([(s, *CHAIN(5))])
    with pytest.raises(ValueError):
        step(be, st, cache, rows, S, other)
    assert not be.calls
    with pytest.raises(ValueError):
        st.attn[windows.index(4)].forward(be.alloc(4), be.alloc(4), S, cache.layers[0], rows, st.scratch, other)
    assert not be.calls


def test_windows_as_long_as_any_tree():
    be = R()
    st = stack(be, [AttnConfig(4, 2, 32, 32, window=64)])
    cache = PagedCache(be, 1, 16, 8, 2, 32, max_seqs=3, max_rows=64)
    t = DraftTrees(cache, max_nodes=64)
    rows, S = t.place([(cache.open(), *CHAIN(64))])
    step(be, st, cache, rows, S, t)
    assert be.calls.count("attn_tree") == 1

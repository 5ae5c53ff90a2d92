"""Calls of placed trees that nothing can answer, refused before anything runs on the device."""
import pytest

from sabrewing_amd.attention import AttnConfig, PagedCache
from sabrewing_amd.backend import Backend
from sabrewing_amd.drafts import DraftTrees
from sabrewing_amd.latent import LatentCache
from sabrewing_amd.stack import DeviceStack
from test_attention_stack_host import Recorder, stack


class R(Recorder):
    trees, latent_cache = staticmethod(Backend.trees), staticmethod(Backend.latent_cache)


A = AttnConfig(4, 2, 32, 32)


def step(be, st, cache, rows, S, trees=None):
    be.calls.clear()
    st.step(be.alloc(4), be.alloc(4), be.alloc(4), be.alloc(4), S, cache=cache, rows=rows, trees=trees)


def test_trees_and_a_stack_without_attention():
    be = R()
    like = stack(be, [A])
    st = DeviceStack(be, like.cfg, 1000)
    st.layers, st.norms, st.final_norm, st.head = like.layers, like.norms, like.final_norm, like.head
    cache = PagedCache(be, 1, 8, 8, 2, 32, max_seqs=3)
    t = DraftTrees(cache)
    rows, S = t.place([(cache.open(), [-1, 0], [1, 2])])
    with pytest.raises(ValueError):
        step(be, st, cache, rows, S, t)
    assert not be.calls
    step(be, st, None, None, S)


def test_places_for_no_rows():
    be = R()
    cache = PagedCache(be, 1, 8, 8, 2, 32, max_seqs=3)
    t = DraftTrees(cache)
    s = cache.open()
    for rows in (0, 1, -1):
        with pytest.raises(ValueError):
            t.place([(s, [-1, 0], [1, 2])], rows=rows)
    with pytest.raises(TypeError):
        t.place([(s, [-1, 0], [1, 2])], rows=2.0)
    assert cache.length(s) == 0
    assert t.place([(s, [-1, 0], [1, 2])], rows=2)[1] == 2


def test_trees_over_latents():
    """at their making: place() would take cells that no step may fill and no commit can move"""
    be = R()
    with pytest.raises(ValueError):
        DraftTrees(LatentCache(be, 1, 8, 8, 128, 16, max_seqs=3))

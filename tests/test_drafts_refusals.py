"""Calls of placed trees that nothing can answer, refused before anything runs on the device."""
import numpy as np
import pytest

from sabrewing_amd.attention import AttnConfig, PagedCache, Rope
from sabrewing_amd.backend import Backend
from sabrewing_amd.drafts import DraftTrees
from sabrewing_amd.latent import DeviceLatentAttention, LatentCache, LatentConfig
from sabrewing_amd.stack import DeviceStack
from test_attention_stack_host import Recorder, stack


class R(Recorder):
    trees, latent_cache, heads = (staticmethod(getattr(Backend, n)) for n in ("trees", "latent_cache", "heads"))


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


def test_steps_behind_other_rows():
    """a cache's row arrays hold its last rows(): trees or a prompt placed before would be appended to other sequences' cells"""
    be = R()
    st = stack(be, [A])
    cache = PagedCache(be, 1, 16, 8, 2, 32, max_seqs=4, max_rows=8)
    a, b = cache.open(), cache.open()
    first, second = DraftTrees(cache), DraftTrees(cache)
    rows, S = first.place([(a, [-1, 0], [1, 2])])
    with pytest.raises(ValueError):
        cache.rows([(b, 9)])                           # more than it has rows for: nothing was made
    step(be, st, cache, rows, S, first)
    second.place([(b, [-1, 0], [3, 4])])
    with pytest.raises(ValueError):
        step(be, st, cache, rows, S, first)
    assert not be.calls
    step(be, st, cache, rows, S, second)
    cache.rows([cache.open(), None])
    with pytest.raises(ValueError):
        step(be, st, cache, rows, S, second)
    assert not be.calls


def test_prompts_behind_other_rows():
    be = R()
    like, L = stack(be, [A]), LatentConfig(4, 128, 32, 16, 32)
    D, u16, f32 = like.cfg.D, (lambda *s: np.zeros(s, np.uint16)), (lambda *s: np.ones(s, np.float32))
    st = DeviceStack(be, like.cfg, 1000)
    st.layers, st.norms, st.final_norm, st.head = like.layers, like.norms, like.final_norm, like.head
    st.add_attention(L, [DeviceLatentAttention.from_host(be, L, D, f32(D), u16(L.cell, D), f32(L.rank), None, None, u16(L.n_heads * L.q_dim, D),
                                                         u16(L.n_heads, L.nope, L.rank), u16(L.n_heads, L.v_dim, L.rank), u16(D, L.n_heads * L.v_dim), Rope(be, L))])
    cache, other = (LatentCache(be, 1, 8, 8, 128, 16, max_seqs=3, max_rows=16) for _ in range(2))
    a, b = cache.open(), cache.open()
    other.open()
    rows, S = cache.prompt(a, 5)
    step(be, st, cache, rows, S)
    far, _ = other.prompt(0, 5)
    late, _ = cache.prompt(b, 5)
    for c, r in ((cache, rows), (cache, far)):
        with pytest.raises(ValueError):
            step(be, st, c, r, 5)
        assert not be.calls
    step(be, st, cache, late, 5)

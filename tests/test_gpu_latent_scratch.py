"""The scratch of latent prompts: recordings that do not use it do not keep it, recordings that do go on replaying over theirs."""
import ctypes as C

import numpy as np
import pytest

from paged import from_bits
from test_gpu_latent import Case
from test_gpu_prompt import Case as Prompt

pytestmark = pytest.mark.gpu


def held(be, f):
    """(bytes that f's results hold on the device, the results)"""
    free, total = C.c_size_t(), C.c_size_t()

    def left():
        be.sync()
        assert be.lib.hipMemGetInfo(C.byref(free), C.byref(total)) == 0
        return free.value
    before = left()
    r = f()
    return before - left(), r


def recorded(be, call):
    be.graph_begin()
    call()
    return be.graph_end()


def test_steps_recorded_after_a_long_prompt(be):
    """two recordings of a decode step before a prompt with half a GiB of keys and values, and two behind it, hold as much"""
    d = Case(be, 1, "bf16", 16, 128, 32, 64, [700, 40], poison=False)
    want = d.run()
    step = lambda: be.attn_latent(d.cache.c, d.rows, d.bufs[2], d.H, d.scale, d.bufs[3], d.S)
    graphs = [recorded(be, step)]                      # (the arena's size from here on)
    first, more = held(be, lambda: [recorded(be, step) for _ in range(2)])
    graphs += more
    p = Prompt(be, 2, "bf16", 32, 128, 32, 256, 256, 64, 16000, 2)
    p.run()
    behind, more = held(be, lambda: [recorded(be, step) for _ in range(2)])
    graphs += more
    assert behind <= first + (64 << 20)
    p.run()
    for g in graphs:
        be.h2d(d.bufs[3], np.zeros(want.size, np.uint16))
        be.graph_launch(g)
        be.sync()
        assert np.array_equal(from_bits(be.d2h(d.bufs[3], want.shape, np.uint16)), want)
        be.graph_destroy(g)
    d.free()
    p.free()


def test_prompts_recorded_back_to_back(be):
    """two recordings of prompts without an eager call between, replayed with larger and smaller eager prompts between them"""
    a, b, big = Prompt(be, 3, "bf16", 4, 128, 32, 64, 64, 16, 30, 40), Prompt(be, 4, "f16", 3, 256, 16, 96, 32, 16, 0, 33), Prompt(be, 5, "bf16", 8, 128, 32, 64, 64, 16, 900, 100)
    want = [a.check(), b.check()]
    graphs = [recorded(be, x.call) for x in (a, b)]
    alone = big.run()
    for _ in range(3):
        for x, g, w in zip((a, b), graphs, want):
            be.h2d(x.bufs[4], x.out)
            be.graph_launch(g)
            be.sync()
            assert np.array_equal(x.read(), w)
            assert np.array_equal(big.run(), alone)
            assert np.array_equal(x.run(), w)
    be.graph_destroy(graphs[0])
    be.h2d(b.bufs[4], b.out)
    be.graph_launch(graphs[1])
    be.sync()
    assert np.array_equal(b.read(), want[1])
    be.graph_destroy(graphs[1])
    for x in (a, b, big):
        x.free()

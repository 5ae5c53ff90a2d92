"""Latent attention where its lists and values are at the ends of their ranges, against the definitions in 64 bits (tolerances: latents.py)."""
import numpy as np
import pytest

from test_gpu_latent import Case

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ free places ----

@pytest.mark.parametrize("free", [-1, -32, -33, -64, -2 ** 31])
@pytest.mark.parametrize("named", [False, True])
@pytest.mark.parametrize("S,at", [(1, [0]), (3, [0]), (3, [1]), (3, [2]), (70, [0, 33, 69]), (256, [255]), (257, [0, 200]), (300, [299])])
def test_every_negative_position_is_a_free_place(be, free, named, S, at):
    """zeros there, all other rows as they are without it"""
    lens = [int(n) for n in np.random.default_rng(S).integers(0, 140, S)]
    c = Case(be, 12, "bf16", 8, 128, 32, 16, lens, poison=False, seq=list(np.random.default_rng(1).permutation(S)) if named else None)
    c.table[:] = np.maximum(c.table, 0)                                # (a row's sequence may be shorter than the row: page 0)
    be.h2d(c.bufs[0], c.table)
    c.pos[at] = free
    be.h2d(c.bufs[1], c.pos)
    got = c.check()
    assert not np.any(got[at])
    c.free()

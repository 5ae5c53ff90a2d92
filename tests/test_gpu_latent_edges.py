"""Latent attention where its lists and values are at the ends of their ranges, against the definitions in 64 bits (tolerances: latents.py)."""
import numpy as np
import pytest

from latents import Latents, NAN, normal
from paged import from_bits, to_type
from test_gpu_latent import Case
from test_gpu_prompt import Case as Prompt

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


# ------------------------------------------------------------------ the expanded form's range ----

@pytest.mark.parametrize("kind,wsigma,csigma", [("bf16", 1.0, 1e-30), ("bf16", 1e-30, 1.0), ("bf16", 1e10, 1e-33), ("bf16", 1.0, 1e25), ("bf16", 1e25, 1.0), ("bf16", 1e-15, 1e33),
                                                ("bf16", 1e-33, 1e33), ("f16", 1.0, 1e-6), ("f16", 1.0, 1e4)])
@pytest.mark.parametrize("rope", [0, 32])
def test_norms_whose_squares_pass_32_bits(be, kind, wsigma, csigma, rope):
    """latents and matrices whose squares' sum is 0 or infinite in 32 bits"""
    c = Prompt(be, 3, kind, 2, 128, rope, 64, 64, 16, 40, 60, wsigma=wsigma, csigma=csigma, f32=True)
    if rope:                                                           # (rotary keys of a size with the others)
        rng = np.random.default_rng(4)
        stored, _ = normal(rng, kind, *c.cells.shape[:2], rope, sigma=min(wsigma * csigma, 1e4))
        live = np.isfinite(from_bits(c.cells[..., :1]))
        c.cells[..., 128:] = np.where(live, stored, NAN[kind])
        c.cache.free()
        c.cache = Latents(be, kind, c.cells, 128)
    c.check()
    c.free()


@pytest.mark.parametrize("size", [1.0, 1e12, 1e30])
def test_rotary_keys_beside_none(be, size):
    """Wk of zeros: the scores are the rotary part's alone, of any size"""
    c = Prompt(be, 5, "bf16", 2, 128, 32, 64, 64, 16, 40, 60, f32=True)
    c.wk[...], c.wk64[...] = 0, 0.0
    live = np.isfinite(from_bits(c.cells[..., :1]))
    c.cells[..., 128:] = np.where(live, normal(np.random.default_rng(6), "bf16", *c.cells.shape[:2], 32, sigma=size)[0], NAN["bf16"])
    c.scale = float(np.float32(c.scale / size))
    c.cache.free()
    c.cache = Latents(be, "bf16", c.cells, 128)
    be.h2d(c.bufs[1], c.wk)
    c.check()
    c.free()


@pytest.mark.parametrize("by", [2.0 ** 15, 1e20])
def test_one_large_latent_behind(be, by):
    """a token whose latent is so many times the others': rows before it stay within the bound (which counts 2^-31 of the largest key and value),
    and finite"""
    c = Prompt(be, 7, "bf16", 2, 128, 32, 64, 64, 16, 40, 60, f32=True)
    at = c.pages[99 // 16], 99 % 16
    c.cells[at[0], at[1], :128] = to_type(from_bits(c.cells[at[0], at[1], :128]) * by, "bf16")[0]
    c.cache.free()
    c.cache = Latents(be, "bf16", c.cells, 128)
    got, (want, bound) = c.run(), c.want()
    assert np.all(np.isfinite(got))
    assert np.all(np.abs(got - want) <= bound)
    c.free()


# ------------------------------------------------------------------ appended without a turn ----

@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("inter", [False, True])
def test_what_is_not_turned_passes_as_it_is(be, kind, inter):
    """without a rope a rotary part is rounded and no more: infinities and NaN stay beside their partners, -0 keeps its sign"""
    S, H, rank, rope, nope, P = 3, 2, 128, 32, 16, 8
    rng = np.random.default_rng(2)
    ckv, q = rng.standard_normal((S, rank + rope)).astype(np.float32), rng.standard_normal((S, H, nope + rope)).astype(np.float32)
    odd = np.array([np.inf, -0.0, np.nan, 0.0, -np.inf, -0.0], np.float32)
    for x, at in ((ckv, rank), (q, nope)):
        x[..., at:at + 6], x[..., at + rope // 2 + 3:at + rope // 2 + 9] = odd, odd[::-1]
    cache = Latents(be, kind, normal(rng, kind, 1, P, rank + rope)[0], rank)
    one = np.zeros(S * H * (nope + rope), np.uint16)
    b = [be.upload(np.ascontiguousarray(a)) for a in (np.arange(S, dtype=np.int32), np.zeros(S, np.int32), np.zeros(1, np.int32), ckv, q, one)]
    pd, sd, td, cd, qd, od = b
    width = nope + rope
    be.latent_append(cache.c, be.kv_rows(pd, td, 1, 1, sd), None, cd, rank + rope, None, 1e-6, qd, H * width, H, nope,
                     be.heads(od, H * width, width), be.heads(int(od) + 2 * nope, H * width, width), S)
    nan = lambda a: np.where(np.isnan(from_bits(a)), np.uint16(0xFFFF), np.uint16(0))              # (any NaN is one)
    same = lambda a, f: np.array_equal(a.view(np.uint16) | nan(a), to_type(f, kind)[0].view(np.uint16) | nan(to_type(f, kind)[0]))
    assert same(cache.read()[0, :S], ckv)
    assert same(be.d2h(od, (S, H, width), np.float16 if kind == "f16" else np.uint16), q)
    for x in b + [cache]:
        x.free()


@pytest.mark.parametrize("H,start,S", [(3, 40, 60), (130, 0, 129)])
@pytest.mark.parametrize("nope,vd", [(64, 64), (192, 96)])
def test_rows_whose_rotary_part_outweighs_the_other(be, H, start, S, nope, vd):
    """f16: every third row's other part is 2^-14 of the rotary one, so that its rotary scores are lifted, beside rows where they are not; and all cells at
    1e-6, where every row's are"""
    c = Prompt(be, 8, "f16", H, 128, 32, nope, vd, 16, start, S)
    c.q[::3, :, :nope], c.q64[::3, :, :nope] = to_type(c.q64[::3, :, :nope] * 2.0 ** -14, "f16")
    be.h2d(c.bufs[3], c.q)
    c.check()
    c.free()
    c = Prompt(be, 9, "f16", H, 128, 32, nope, vd, 16, start, S, csigma=1e-6, f32=True)
    c.check()
    c.free()

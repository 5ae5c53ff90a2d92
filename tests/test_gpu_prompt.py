"""The expanded form of latent attention against its definition in 64 bits.

Tolerance, value by value: keys, values, queries and weights are each rounded to 11 bits (2^-11 of their own size at most, and 2^-20 of
2^-11 of the head's largest), sums are in 32 bits, and the output is rounded once to its type.  A score is off by d <= 2 * 2^-11 * sum |q k|
scale, which moves an output by at most 2 d of sum p |v|.  The errors' norm: each rounding is 0.41 of its half step in the
mean, a score's spread is at most 1.5 here; in bf16 the output's alone counts, in f16 it, the weights', the values' and the keys' do:
0.41 sqrt(3 + 1.5^2) = 0.94 of 2^-11, held to 1.5."""
import numpy as np
import pytest

from latents import DTYPE, HALF, Latents, NAN, normal
from paged import from_bits

pytestmark = pytest.mark.gpu

KINDS = ["bf16", "f16"]
R = 2.0 ** -11


def exact(cells, rank, pages, P, start, wk, wv, q, scale, S):
    H, vd = wk.shape[0], wv.shape[1]
    T = start + S
    t = np.arange(T)
    page = np.full(T, -1)
    has = t // P < len(pages)
    page[has] = pages[t[has] // P]
    ok = (page >= 0) & (page < cells.shape[0])
    c = cells[np.where(ok, page, 0), t % P]
    out, bound = np.zeros((S, H, vd)), np.zeros((S, H, vd))
    for h in range(H):
        k = np.concatenate([c[:, :rank] @ wk[h].T, c[:, rank:]], 1)
        v = c[:, :rank] @ wv[h].T
        nope = wk.shape[1]
        small = R * 2.0 ** -20
        for s in range(S):
            see = ok & (t <= start + s)
            if not see.any():
                continue
            x = k[see] @ q[s, h] * scale
            p = np.exp(x - x.max())
            l = p.sum()
            out[s, h] = p @ v[see] / l
            d = 2 * R * np.max(np.abs(k[see]) @ np.abs(q[s, h])) + small * (np.max(np.abs(k)) * np.sum(np.abs(q[s, h])))
            d = abs(scale) * d + 2.0 ** -23 * (np.max(np.abs(x - x.max())) + 4)
            av = p @ np.abs(v[see]) / l
            bound[s, h] = (2 * d + 2 * R + 2.0 ** -20) * av + small * np.max(np.abs(v)) + 2.0 ** -32 * np.sum(np.abs(v[see]), 0) / l
    return out, bound


class Case:
    def __init__(self, be, seed, kind, H, rank, rope, nope, vd, P, start, S, gap=0, f32=False, sharp=1.5, wsigma=1.0, csigma=1.0):
        rng = np.random.default_rng(seed)
        self.be, self.kind, self.args, self.f32 = be, kind, (H, rank, rope, nope, vd, P, start, S), f32
        T = start + S
        n = -(-T // P)
        self.pages = rng.permutation(n + 3)[:n].astype(np.int32)
        self.cells = normal(rng, kind, n + 3, P, rank + rope, sigma=csigma)[0]
        live = np.zeros((n + 3, P), bool)
        live[self.pages[np.arange(T) // P], np.arange(T) % P] = True
        self.cells[~live] = NAN[kind]
        self.wk, self.wk64 = normal(rng, kind, H, nope, rank, sigma=wsigma * rank ** -0.5)
        self.wv, self.wv64 = normal(rng, kind, H, vd, rank, sigma=wsigma * rank ** -0.5)
        self.q, self.q64 = normal(rng, kind, S, H, nope + rope, sigma=sharp)
        self.scale = float(np.float32((nope + rope) ** -0.5 / (wsigma * csigma)))
        self.cache = Latents(be, kind, self.cells, rank, gap)
        self.out = np.full(S * H * vd + 64, 7, np.float32 if f32 else DTYPE[kind])
        self.bufs = [be.upload(np.ascontiguousarray(a)) for a in (self.pages, self.wk, self.wv, self.q, self.out)]

    def call(self):
        H, rank, rope, nope, vd, P, start, S = self.args
        p, wk, wv, q, out = self.bufs
        self.be.attn_latent_prompt(self.cache.c, p, len(self.pages), start, wk, wv, nope, vd, q, H, self.scale, out, self.f32, S)

    def run(self):
        self.call()
        return self.read()

    def read(self):
        H, S, vd = self.args[0], self.args[7], self.args[4]
        got = self.be.d2h(self.bufs[4], self.out.shape, self.out.dtype)
        assert np.all(got[S * H * vd:] == 7)
        got = got[:S * H * vd]
        return (got.astype(np.float64) if self.f32 else from_bits(got)).reshape(S, H, vd)

    def want(self):
        H, rank, rope, nope, vd, P, start, S = self.args
        cells = np.nan_to_num(from_bits(self.cells))
        out, bound = exact(cells, rank, self.pages, P, start, self.wk64, self.wv64, self.q64, self.scale, S)
        if not self.f32:
            bound = bound + HALF[self.kind] * (np.abs(out) + bound) + 2.0 ** -25
        return out, bound

    def check(self):
        got, (want, bound) = self.run(), self.want()
        assert np.all(np.isfinite(got))
        assert np.all(np.abs(got - want) <= bound), np.max(np.abs(got - want) / np.maximum(bound, 1e-300))
        norm = 0.6 * HALF["bf16"] if self.kind == "bf16" and not self.f32 else 1.5 * R
        assert np.linalg.norm(got - want) <= norm * np.linalg.norm(want)
        return got

    def free(self):
        for b in self.bufs + [self.cache]:
            b.free()


def one(be, *a, **k):
    c = Case(be, *a, **k)
    got = c.check()
    c.free()
    return got


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rank,rope", [(128, 0), (256, 16), (384, 48), (512, 64)])
@pytest.mark.parametrize("nope,vd", [(32, 32), (64, 96), (128, 128), (96, 256), (192, 64), (256, 160)])
def test_sizes(be, kind, rank, rope, nope, vd):
    one(be, rank + nope, kind, 3, rank, rope, nope, vd, 16, 37, 50)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("start,S", [(0, 1), (0, 2), (0, 31), (0, 32), (0, 33), (0, 129), (1, 1), (31, 1), (300, 1), (300, 70), (64, 128), (5, 257)])
@pytest.mark.parametrize("f32", [False, True])
def test_lengths(be, kind, start, S, f32):
    one(be, S, kind, 2, 128, 32, 64, 64, 16, start, S, f32=f32)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("start,S", [(0, 300), (100, 129)])
@pytest.mark.parametrize("nope,vd", [(64, 64), (128, 128), (192, 256)])
def test_many_heads(be, kind, start, S, nope, vd):
    """enough heads for the form with 128 rows a block"""
    one(be, S, kind, 130, 128, 64, nope, vd, 64, start, S)


@pytest.mark.parametrize("P", [8, 16, 32, 4096])
@pytest.mark.parametrize("gap", [0, 8])
def test_pages_and_strides(be, P, gap):
    one(be, P, "bf16", 2, 128, 16, 64, 64, P, 50, 60, gap=gap)


@pytest.mark.parametrize("kind,wsigma,csigma", [("bf16", 1e4, 1e3), ("bf16", 1e-6, 1e-4), ("bf16", 1e15, 1.0), ("f16", 30.0, 50.0), ("f16", 1e-2, 1e-2)])
def test_any_size_of_values(be, kind, wsigma, csigma):
    """keys and values far from 1: the scale of each head keeps them in f16's range"""
    one(be, 3, kind, 2, 128, 0, 64, 64, 16, 40, 60, wsigma=wsigma, csigma=csigma, f32=True)


def test_sharp_softmax(be):
    c = Case(be, 4, "bf16", 4, 256, 64, 128, 128, 64, 400, 100, sharp=40.0)
    got, (want, bound) = c.run(), c.want()
    assert np.all(np.abs(got - want) <= bound)
    c.free()


@pytest.mark.parametrize("H", [4, 130])
def test_no_numbers(be, H):
    c = Case(be, 5, "bf16", H, 128, 32, 64, 64, 16, 70, 90)
    clean = c.check()
    t = 100
    for at in (3, 127, 140):
        cells = c.cells.copy()
        cells[c.pages[t // 16], t % 16, at] = NAN["bf16"]
        c.cache.free()
        c.cache = Latents(be, "bf16", cells, 128)
        got = c.run()
        assert not np.any(np.isfinite(got[t - 70:]))
        assert np.linalg.norm(got[:t - 70] - clean[:t - 70]) <= HALF["bf16"] * np.linalg.norm(clean[:t - 70])
    c.free()


def test_pages_that_lead_nowhere(be):
    c = Case(be, 6, "bf16", 3, 128, 32, 64, 64, 16, 70, 90)
    c.pages[[0, 5]] = -1, 10 ** 6
    c.pages = c.pages[:8]                                              # and tokens behind the list
    c.bufs[0].free()
    c.bufs[0] = be.upload(c.pages)
    c.check()
    c.pages[:] = -1
    be.h2d(c.bufs[0], c.pages)
    assert not np.any(c.run())
    c.free()


def test_same_bits_again_and_recorded(be):
    c = Case(be, 7, "bf16", 16, 512, 64, 128, 128, 64, 300, 200)
    want = c.run()
    be.graph_begin()
    c.call()
    g = be.graph_end()
    for _ in range(3):
        be.h2d(c.bufs[4], np.full(want.size, 9, np.uint16))
        be.graph_launch(g)
        be.sync()
        assert np.array_equal(c.read(), want)
        assert np.array_equal(c.run(), want)
    be.graph_destroy(g)
    c.free()

"""Paged caches of latents for the tests, and latent attention in 64 bits from its definitions."""
import numpy as np

from paged import from_bits, to_type

DTYPE = {"bf16": np.uint16, "f16": np.float16}
HALF = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}                          # a rounding to nearest, relative
NAN = {"bf16": np.uint16(0x7FC0), "f16": np.float16(np.nan)}


class Latents:
    """a pool [n_pages, P, rank + rope] (as stored) on the device, `gap` elements behind every cell and page"""

    def __init__(self, be, kind, cells, rank, gap=0):
        self.be, self.kind, (n, P, w), self.gap = be, kind, cells.shape, gap
        self.strides = (P * (w + gap) + gap, w + gap)
        self.shape = cells.shape
        img = np.full(n * self.strides[0], NAN[kind], DTYPE[kind])
        self._view(img)[...] = cells
        self.buf, self.n = be.upload(img), img.size
        self.c = be.latent_cache(self.buf, kind, n, P, rank, w - rank, self.strides)

    def _view(self, img):
        return np.lib.stride_tricks.as_strided(img, self.shape, (2 * self.strides[0], 2 * self.strides[1], 2))

    def read(self):
        img = self.be.d2h(self.buf, (self.n,), DTYPE[self.kind])
        mark = img.copy()
        self._view(mark)[...] = NAN[self.kind]
        assert np.array_equal(mark.view(np.uint16), np.full(self.n, NAN[self.kind], DTYPE[self.kind]).view(np.uint16))     # nothing between cells
        return self._view(img).copy()

    def free(self):
        self.buf.free()


def normal(rng, kind, *shape, sigma=1.0):
    """(stored, in 64 bits)"""
    return to_type(sigma * rng.standard_normal(shape), kind)


def exact_absorbed(cells, rank, table, P, pos, seq, q, scale, kind):
    """cells [pages, P, rank + rope], q [S, H, rank + rope] in 64 bits -> (out [S, H, rank], bound).

    The bound: 32-bit sums as paged.exact_attention's; besides, each weight is rounded to the cache's type (HALF of it; f16 weights
    far below the largest are rounded to 2^-25 of 2^7 times it, i.e. 2^-32 of the largest's sum, in the sums' share below) and so
    is the output."""
    S, H, w = q.shape
    out, bound, eps = np.zeros((S, H, rank)), np.zeros((S, H, rank)), 2.0 ** -24
    for s in range(S):
        if pos[s] < 0 or not 0 <= seq[s] < table.shape[0]:
            continue
        t = np.arange(min(int(pos[s]) + 1, table.shape[1] * P))
        page = table[seq[s]][t // P]
        ok = (page >= 0) & (page < cells.shape[0])
        t, page = t[ok], page[ok]
        if not len(t):
            continue
        c = cells[page, t % P]
        x = q[s] @ c.T * scale
        x0 = x.max(1, keepdims=True)
        p = np.exp(x - x0)
        l = p.sum(1, keepdims=True)
        v = c[:, :rank]
        out[s] = p @ v / l
        score = (w + 2) * eps * np.max(np.abs(q[s]) @ np.abs(c).T, 1, keepdims=True) * abs(scale) + 4 * eps * (np.max(np.abs(x - x0), 1, keepdims=True) + 4)
        bound[s] = (2 * score + (2 * len(t) + 16) * eps + HALF[kind]) * (p @ np.abs(v)) / l
        if kind == "f16":
            bound[s] += 2.0 ** -32 * np.abs(v).sum(0) / l
        bound[s] += HALF[kind] * (np.abs(out[s]) + bound[s]) + 2.0 ** -25 * (kind == "f16")
    return out, bound

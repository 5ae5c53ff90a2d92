"""Paged caches on host and device for the attention tests, and the operators in 64 bits from their
definitions."""
import numpy as np

LAYOUTS = ("head", "token", "apart")


def to_type(x, kind):
    """f32 values as the cache stores them: (stored bits, their values in 64 bits)"""
    x = np.asarray(x, np.float32)
    if kind == "f32":
        return x, x.astype(np.float64)
    if kind == "f16":
        h = x.astype(np.float16)
        return h, h.astype(np.float64)
    u = x.view(np.uint32)
    b = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    b = np.where(np.isnan(x), np.uint16(0x7FC0), b)
    return b, from_bits(b)


def from_bits(b):
    """stored bits to 64-bit values"""
    if b.dtype == np.uint16:
        return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return b.astype(np.float64)


class Cache:
    """pools k, v [n_pages, Hkv, P, dh] on the host (as stored), laid out on the device as `layout`:
    head [page][head][token], token [page][token][head], apart: k and v in one allocation, a gap
    behind every cell row, head and page"""

    def __init__(self, be, kind, n_pages, P, Hkv, dh, k, v, layout="head"):
        self.be, self.kind, self.shape, self.layout = be, kind, (n_pages, Hkv, P, dh), layout
        per = 4 if kind == "f32" else 8
        if layout == "head":
            ts, hs, ps = dh, P * dh, Hkv * P * dh
        elif layout == "token":
            hs, ts, ps = dh, Hkv * dh, Hkv * P * dh
        else:
            ts = dh + per
            hs = P * ts + per
            ps = 2 * (Hkv * hs + per)
        self.strides, self.item = (ps, hs, ts), 4 if kind == "f32" else 2
        self.n = n_pages * ps
        self.vat = ps // 2 if layout == "apart" else self.n
        total = self.n if layout == "apart" else 2 * self.n
        self.dtype = np.float32 if kind == "f32" else np.float16 if kind == "f16" else np.uint16
        img = np.full(total, 0x7FC0 if kind == "bf16" else np.nan, self.dtype)
        self._view(img, 0)[...] = k
        self._view(img, self.vat)[...] = v
        self.buf, self.total = be.upload(img), total
        self.c = be.kv_cache(int(self.buf), int(self.buf) + self.vat * self.item, kind, n_pages, P, Hkv, dh, self.strides)

    def _view(self, img, at):
        n, H, P, dh = self.shape
        ps, hs, ts = (x * self.item for x in self.strides)
        return np.lib.stride_tricks.as_strided(img[at:], (n, H, P, dh), (ps, hs, ts, self.item))

    def image(self):
        return self.be.d2h(self.buf, (self.total,), self.dtype)

    def read(self):
        """(k, v) as stored, from the device"""
        img = self.image()
        return self._view(img, 0).copy(), self._view(img, self.vat).copy()

    def free(self):
        self.buf.free()


def exact_attention(k, v, table, P, pos, seq, q, scale, window=0):
    """k, v [pages, Hkv, P, dh] and q [S, Hq, dh] in 64 bits -> (out, bound): bound[s, h, d] holds what the
    errors of 32-bit sums can come to (a derivation stands with the tests)"""
    S, Hq, dh = q.shape
    n_pages, Hkv = k.shape[:2]
    G = Hq // Hkv
    out, bound = np.zeros((S, Hq, dh)), np.zeros((S, Hq, dh))
    eps = 2.0 ** -24
    for s in range(S):
        if pos[s] < 0 or not 0 <= seq[s] < table.shape[0]:
            continue
        t = np.arange(max(0, pos[s] - window + 1) if window else 0, pos[s] + 1)
        t = t[t // P < table.shape[1]]
        page = table[seq[s]][t // P]
        ok = (page >= 0) & (page < n_pages)
        t, page = t[ok], page[ok]
        if not len(t):
            continue
        for h in range(Hq):
            kk, vv = k[page, h // G, t % P], v[page, h // G, t % P]
            x = kk @ q[s, h] * scale
            p = np.exp(x - x.max())
            l = p.sum()
            out[s, h] = (p @ vv) / l
            # score: dh products summed in 32 bits, the scale, the exponential's argument and result
            score = (dh + 2) * eps * np.max(np.abs(kk) @ np.abs(q[s, h])) * abs(scale) + 4 * eps * (np.max(np.abs(x - x.max())) + 4)
            bound[s, h] = (2 * score + (2 * len(t) + 16) * eps) * (p @ np.abs(vv)) / l
    return out, bound


def exact_rope(x, pos, freq, dims, interleaved, factor, w, eps):
    """x [S, H, dh] in 64 bits, normalised (w not None) and turned"""
    x = x.copy()
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    if dims:
        half = dims // 2
        a = pos[:, None].astype(np.float64) * freq
        z = np.exp(1j * a)[:, None] * factor
        i = np.arange(half)
        f, g = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        y = (x[..., f] + 1j * x[..., g]) * z
        x[..., f], x[..., g] = y.real, y.imag
    return x


def exact_pick(l, u, temp=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """a row's pick in 64 bits from the definition"""
    l = np.asarray(l, np.float32)
    if np.isnan(l[0]) and (not temp > 0):
        return 0
    x = np.where(np.isnan(l), -np.inf, l.astype(np.float64))
    order = np.lexsort((np.arange(len(x)), -x))
    top = x[order[0]]
    if top == -np.inf:
        return 0
    if not temp > 0:
        return int(order[0])
    if 0 < top_k < len(x):
        order = order[:top_k]
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / np.float64(np.float32(temp))))
    w[x[order] == -np.inf] = 0.0                       # (at an infinite temperature the quotient is none)
    if top_p < 1:
        want = float(np.float32(top_p)) * w.sum()
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        n = max(1, int((before < want).sum()))
        order, w = order[:n], w[:n]
    if min_p > 0:
        n = max(1, int((w >= min(1.0, float(np.float32(min_p)))).sum()))
        order, w = order[:n], w[:n]
    by = np.argsort(order)
    run = np.cumsum(w[by])
    i = int(np.searchsorted(run, float(np.float32(u)) * run[-1], side="right"))
    return int(order[by][min(i, len(run) - 1)])

"""Latent attention against its definitions in 64 bits: cells and queries of new tokens, products for each head, the absorbed form.

Tolerances: latents.exact_absorbed derives the attention's.  The errors' norm is held to 2.5 roundings' worth of the outputs' (a
rounding of the weights and one of the output, each uniform: 0.41 of HALF a value, 0.58 together, and room for the tails)."""
import numpy as np
import pytest

from latents import DTYPE, HALF, Latents, NAN, exact_absorbed, normal
from paged import exact_rope, from_bits, to_type

pytestmark = pytest.mark.gpu

KINDS = ["bf16", "f16"]


def random_pages(rng, lens, P, spare=2):
    need = [-(-max(0, n) // P) for n in lens]
    ids = rng.permutation(sum(need) + spare)
    table = np.full((len(lens), max(1, max(need))), -7, np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    return table, len(ids)


# ------------------------------------------------------------------ the absorbed form ----

class Case:
    def __init__(self, be, seed, kind, H, rank, rope, P, lens, gap=0, sharp=1.5, poison=True, seq=None):
        rng = np.random.default_rng(seed)
        self.be, self.kind, self.H, self.rank, self.P = be, kind, H, rank, P
        self.table, n = random_pages(rng, lens, P)
        self.pos = np.asarray(lens, np.int32) - 1
        self.seq = np.arange(len(lens)) if seq is None else np.asarray(seq)
        self.S = len(self.pos)
        self.cells = normal(rng, kind, n, P, rank + rope)[0]
        if poison:                                                     # cells that no row attends to
            live = np.zeros((n, P), bool)
            for s in range(self.S):
                for t in range(self.pos[s] + 1):
                    live[self.table[self.seq[s], t // P], t % P] = True
            self.cells[~live] = NAN[kind]
        self.q, self.q64 = normal(rng, kind, self.S, H, rank + rope, sigma=sharp)
        self.scale = float(np.float32((rank + rope) ** -0.5))
        self.cache = Latents(be, kind, self.cells, rank, gap)
        self.bufs = [be.upload(np.ascontiguousarray(a)) for a in (self.table, self.pos, self.q, np.full(self.S * H * rank + 64, 7, DTYPE[kind]))]
        self.sd = None if seq is None else be.upload(np.asarray(seq, np.int32))
        self.rows = be.kv_rows(self.bufs[1], self.bufs[0], self.table.shape[0], self.table.shape[1], self.sd)

    def run(self):
        self.be.attn_latent(self.cache.c, self.rows, self.bufs[2], self.H, self.scale, self.bufs[3], self.S)
        n = self.S * self.H * self.rank
        got = self.be.d2h(self.bufs[3], (n + 64,), DTYPE[self.kind])
        assert np.all(got[n:] == 7)
        return from_bits(got[:n]).reshape(self.S, self.H, self.rank)

    def check(self):
        got = self.run()
        want, bound = exact_absorbed(from_bits(self.cells), self.rank, self.table, self.P, self.pos, self.seq, self.q64, self.scale, self.kind)
        assert np.all(np.isfinite(got))
        assert np.all(np.abs(got - want) <= bound), np.max(np.abs(got - want) / np.maximum(bound, 1e-300))
        assert np.linalg.norm(got - want) <= HALF[self.kind] * np.linalg.norm(want)
        return got

    def free(self):
        for b in self.bufs + [self.cache] + ([self.sd] if self.sd else []):
            b.free()


def one(be, *a, **k):
    c = Case(be, *a, **k)
    got = c.check()
    c.free()
    return got


LENS = [0, 1, 2, 31, 32, 33, 64, 65, 129, 300]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rank", [128, 256, 384, 512])
@pytest.mark.parametrize("rope", [0, 16, 48, 64])
@pytest.mark.parametrize("H", [5, 40, 128])
def test_ranks_ropes_and_heads(be, kind, rank, rope, H):
    one(be, rank + rope, kind, H, rank, rope, 16, LENS)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H", [1, 32, 33, 64, 65, 100, 129, 300])
def test_heads(be, kind, H):
    one(be, H, kind, H, 256, 32, 64, [100, 0, 7])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("P", [8, 16, 32, 64, 4096])
@pytest.mark.parametrize("gap", [0, 8])
def test_pages_and_strides(be, kind, P, gap):
    one(be, P, kind, 16, 512, 64, P, [1, 70, 0, 300, 8], gap=gap)


@pytest.mark.parametrize("kind,H,lens", [("bf16", 16, [5000]), ("f16", 128, [9000, 40]), ("bf16", 64, [3000, 1, 9999]), ("bf16", 4, [40000])])
def test_long(be, kind, H, lens):
    one(be, 1, kind, H, 512, 64, 64, lens, poison=False)


@pytest.mark.parametrize("H", [16, 100])
def test_blocks_that_take_several_rows(be, H):
    rng = np.random.default_rng(H)
    one(be, H, "bf16", H, 512, 64, 64, list(rng.integers(500, 3000, 60)), poison=False)


@pytest.mark.parametrize("S", [100, 256, 257, 400])
def test_many_rows(be, S):
    rng = np.random.default_rng(S)
    one(be, S, "bf16", 8, 128, 32, 16, list(rng.integers(0, 150, S)))


def test_rows_of_one_sequence(be):
    """a prompt's chunk: rows at consecutive positions each see what is theirs to see"""
    c = Case(be, 3, "bf16", 16, 512, 64, 16, [90], poison=False)
    c.free()
    rng = np.random.default_rng(3)
    c = Case(be, 4, "bf16", 16, 256, 64, 16, [90], poison=False)
    S = 12
    q, q64 = normal(rng, "bf16", S, 16, 320, sigma=1.5)
    pos, seq = np.arange(78, 90, dtype=np.int32), np.zeros(S, np.int32)
    b = [be.upload(a) for a in (pos, seq, q, np.zeros(S * 16 * 256, np.uint16))]
    be.attn_latent(c.cache.c, be.kv_rows(b[0], c.bufs[0], 1, c.table.shape[1], b[1]), b[2], 16, c.scale, b[3], S)
    got = from_bits(be.d2h(b[3], (S, 16, 256), np.uint16))
    want, bound = exact_absorbed(from_bits(c.cells), 256, c.table, 16, pos, seq, q64, c.scale, "bf16")
    assert np.all(np.abs(got - want) <= bound)
    for x in b:
        x.free()
    c.free()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H", [16, 128])
def test_sharp_softmax(be, kind, H):
    """one token weighs nearly all: the weights' range and a maximum that grows late"""
    c = Case(be, 6, kind, H, 512, 64, 64, [700, 33, 1000], sharp=40.0, poison=False)
    got = c.run()
    want, bound = exact_absorbed(from_bits(c.cells), 512, c.table, 64, c.pos, c.seq, c.q64, c.scale, kind)
    assert np.all(np.abs(got - want) <= bound)
    c.free()


@pytest.mark.parametrize("kind", KINDS)
def test_no_numbers(be, kind):
    """a cell that is no number reaches the rows that attend to it alone"""
    c = Case(be, 7, kind, 16, 256, 64, 16, [40, 90, 20, 90], seq=[0, 1, 2, 1], poison=False)
    c.pos[3] = 49                                                      # rows 1 and 3 are of one sequence; token 50 is bad
    be.h2d(c.bufs[1], c.pos)
    clean = c.check()
    for at in (3, 255, 300):                                           # in the latent and in the rotary part
        cells = c.cells.copy()
        cells[c.table[1, 50 // 16], 50 % 16, at] = NAN[kind]
        c.cache.free()
        c.cache = Latents(be, kind, cells, 256)
        got = c.run()
        assert not np.any(np.isfinite(got[1][:, min(at, 255)]))
        assert np.array_equal(got[[0, 2, 3]], clean[[0, 2, 3]])
    c.free()


def test_lists_that_lead_nowhere(be):
    c = Case(be, 8, "bf16", 16, 512, 64, 16, [100, 70, 50], poison=False)
    c.table[0, 2], c.table[1, 0], c.table[1, 3] = -1, 10 ** 6, -2 ** 31
    be.h2d(c.bufs[0], c.table)
    c.check()
    c.pos[:] = [2 ** 31 - 1, -5, 3]                                    # beyond the table; a free place
    be.h2d(c.bufs[1], c.pos)
    c.check()
    c.free()


def test_same_bits_again_and_recorded(be):
    c = Case(be, 9, "bf16", 128, 512, 64, 64, [3000, 100, 900], poison=False)
    want = c.run()
    be.graph_begin()
    be.attn_latent(c.cache.c, c.rows, c.bufs[2], c.H, c.scale, c.bufs[3], c.S)
    g = be.graph_end()
    for _ in range(3):
        be.h2d(c.bufs[3], np.zeros(want.size, np.uint16))
        be.graph_launch(g)
        be.sync()
        assert np.array_equal(from_bits(be.d2h(c.bufs[3], want.shape, np.uint16)), want)
        assert np.array_equal(c.run(), want)
    be.graph_destroy(g)
    c.free()


# ------------------------------------------------------------------ cells and queries of new tokens ----

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rank,rope,nope,H,inter,norm,turn", [
    (512, 64, 128, 16, True, True, True), (512, 64, 128, 128, False, True, True), (128, 16, 16, 1, True, False, True),
    (256, 48, 96, 5, False, True, True), (384, 0, 64, 3, False, True, True), (256, 32, 256, 7, True, True, False), (128, 64, 192, 0, True, True, True)])
@pytest.mark.parametrize("S", [1, 9, 130])
def test_append(be, kind, rank, rope, nope, H, inter, norm, turn, S):
    rng = np.random.default_rng(rank + rope + S)
    P, n = 16, 12
    pos, seq = np.zeros(S, np.int32), rng.integers(0, 3, S).astype(np.int32)
    for i in range(3):
        k = np.flatnonzero(seq == i)
        pos[k] = rng.permutation(4 * P)[:len(k)] if len(k) <= 4 * P else np.arange(len(k))
    pos[rng.random(S) < 0.1] = -1
    pos[pos >= 4 * P] = 10 ** 6                                        # beyond the table
    table = rng.permutation(n).astype(np.int32).reshape(3, 4)
    table[2, 1] = -1
    ldc, ldq, width = rank + rope + 4, H * (nope + rope) + 8, rank + rope
    ckv, q = rng.standard_normal((S, ldc)).astype(np.float32), rng.standard_normal((S, ldq)).astype(np.float32)
    w = (1 + 0.1 * rng.standard_normal(rank)).astype(np.float32)
    freq = 1e4 ** (-2.0 * np.arange(rope // 2) / max(1, rope))
    before = normal(rng, kind, n, P, width)[0]
    cache = Latents(be, kind, before, rank, gap=8)
    up = lambda a: be.upload(np.ascontiguousarray(a))
    one = np.full(S * max(1, H) * (nope + width) + 64, 7, DTYPE[kind])
    b = [up(a) for a in (pos, seq, table, ckv, q, w, freq if rope else np.zeros(1), one, one)]
    pd, sd, td, cd, qd, wd, fd, nd, rd = b
    rows = be.kv_rows(pd, td, 3, 4, sd)
    be.latent_append(cache.c, rows, be.rope(fd if rope else None, rope, inter) if turn else None, cd, ldc, wd if norm else None, 1e-6, qd if H else None, ldq, H, nope,
                     be.heads(nd, H * nope, nope) if H else None, be.heads(int(rd) + 2 * rank, H * width, width) if H else None, S)
    c64, q64 = ckv[:, :width].astype(np.float64), q[:, :H * (nope + rope)].astype(np.float64).reshape(S, H, nope + rope)
    lat, dims = c64[:, :rank], rope if turn else 0
    if norm:
        lat = lat / np.sqrt((lat * lat).mean(1, keepdims=True) + 1e-6) * w.astype(np.float64)
    kr = exact_rope(c64[:, None, rank:], pos, freq, dims, inter, 1.0, None, 0)[:, 0]
    qr = exact_rope(q64[..., nope:], pos, freq, dims, inter, 1.0, None, 0)
    want = before.copy()
    got = cache.read()
    live = np.zeros((n, P), bool)
    # a value and then one rounding: the norm's sum (rank terms), root, quotient and products; the turn's angle, cos, sin, products and sum
    near = lambda x, y, big: np.all(np.abs(from_bits(x) - y) <= (HALF[kind] + (rank + 24) * 2.0 ** -23) * np.abs(y) + 24 * 2.0 ** -24 * big + 2.0 ** -25)
    for s in range(S):
        if pos[s] < 0 or pos[s] >= 4 * P or table[seq[s], pos[s] // P] < 0:
            continue
        at = table[seq[s], pos[s] // P], pos[s] % P
        live[at] = True
        assert near(got[at], np.concatenate([lat[s], kr[s]]), np.max(np.abs(c64[s])))
    assert np.array_equal(got[~live].view(np.uint16), before[~live].view(np.uint16))
    qn, qa = (be.d2h(x, one.shape, DTYPE[kind]) for x in (nd, rd))
    full = qa[:S * H * width].reshape(S, H, width)
    assert np.all(full[..., :rank] == 7) and np.all(qa[S * H * width:] == 7) and np.all(qn[S * H * nope:] == 7)
    qn = qn[:S * H * nope].reshape(S, H, nope)
    for s in range(S):
        if pos[s] < 0:
            assert np.all(qn[s] == 7) and np.all(full[s] == 7)
        else:
            assert near(qn[s], q64[s, :, :nope], 0.0) and near(full[s, :, rank:], qr[s], 8.0)
    for x in b + [cache]:
        x.free()


# ------------------------------------------------------------------ a product for each head ----

@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("S,H,n_in,n_out", [(1, 128, 128, 512), (1, 3, 32, 32), (31, 5, 96, 160), (33, 2, 512, 128), (64, 16, 512, 96), (65, 4, 64, 32),
                                            (300, 3, 1024, 1024), (129, 7, 192, 96)])
@pytest.mark.parametrize("shared", [False, True])
def test_products(be, kind, f32, S, H, n_in, n_out, shared):
    rng = np.random.default_rng(S + n_in)
    x, x64 = normal(rng, kind, S, 1 if shared else H, n_in + 8)
    w, w64 = normal(rng, kind, H, n_out, n_in, sigma=n_in ** -0.5)
    pad = n_out + 16
    y = np.full(S * H * pad + 64, 7, np.float32 if f32 else DTYPE[kind])
    xd, wd, yd = be.upload(x), be.upload(w), be.upload(y)
    be.latent_heads(kind, be.heads(xd, x.shape[1] * (n_in + 8), 0 if shared else n_in + 8), wd, H, n_in, n_out, be.heads(yd, H * pad, pad), f32, S)
    got = be.d2h(yd, y.shape, y.dtype)
    assert np.all(got[S * H * pad:] == 7)
    got = got[:S * H * pad].reshape(S, H, pad)
    assert np.all(got[..., n_out:] == 7)
    got = got[..., :n_out].astype(np.float64) if f32 else from_bits(np.ascontiguousarray(got[..., :n_out]))
    for h in range(H):
        xs = x64[:, 0 if shared else h, :n_in]
        want, size = xs @ w64[h].T, np.abs(xs) @ np.abs(w64[h]).T
        bound = n_in * 2.0 ** -24 * size
        if not f32:
            bound = bound + HALF[kind] * (np.abs(want) + bound) + 2.0 ** -25
        assert np.all(np.abs(got[:, h] - want) <= bound)
    for b in (xd, wd, yd):
        b.free()


def test_a_token_from_end_to_end(be):
    """append, into the latent space, attention, out of it: the attention of expanded keys and values"""
    rng = np.random.default_rng(11)
    kind, H, rank, rope, nope, vd, P, T = "bf16", 8, 256, 32, 64, 96, 16, 50
    S, width = 3, rank + rope
    wk, wk64 = normal(rng, kind, H, nope, rank, sigma=rank ** -0.5)
    wv, wv64 = normal(rng, kind, H, vd, rank, sigma=rank ** -0.5)
    table = rng.permutation(12).astype(np.int32).reshape(S, 4)
    cache = Latents(be, kind, normal(rng, kind, 12, P, width)[0], rank)
    pos = np.array([T, 20, 63], np.int32)
    ckv, q = rng.standard_normal((S, width)).astype(np.float32), rng.standard_normal((S, H, nope + rope)).astype(np.float32)
    freq = 1e4 ** (-2.0 * np.arange(rope // 2) / rope)
    up = lambda a: be.upload(np.ascontiguousarray(a))
    b = [up(a) for a in (pos, table, ckv, q, freq, wk.transpose(0, 2, 1), wv, np.zeros(S * H * nope, np.uint16), np.zeros(S * H * width, np.uint16),
                         np.zeros(S * H * rank, np.uint16), np.zeros(S * H * vd, np.float32))]
    pd, td, cd, qd, fd, kd, vd_, nd, ad, od, yd = b
    rows, scale = be.kv_rows(pd, td, S, 4), (nope + rope) ** -0.5
    be.latent_append(cache.c, rows, be.rope(fd, rope, True), cd, width, None, 1e-6, qd, H * (nope + rope), H, nope, be.heads(nd, H * nope, nope),
                     be.heads(int(ad) + 2 * rank, H * width, width), S)
    be.latent_heads(kind, be.heads(nd, H * nope, nope), kd, H, nope, rank, be.heads(ad, H * width, width), False, S)
    be.attn_latent(cache.c, rows, ad, H, scale, od, S)
    be.latent_heads(kind, be.heads(od, H * rank, rank), vd_, H, rank, vd, be.heads(yd, H * vd, vd), True, S)
    got = be.d2h(yd, (S, H, vd), np.float32)
    cells = from_bits(cache.read())
    q64 = to_type(q, kind)[1]
    qr = exact_rope(q.astype(np.float64)[..., nope:], pos, freq, rope, True, 1.0, None, 0)
    want = np.zeros((S, H, vd))
    for s in range(S):
        t = np.arange(pos[s] + 1)
        c = cells[table[s, t // P], t % P]
        for h in range(H):
            x = (c[:, :rank] @ wk64[h].T @ q64[s, h, :nope] + c[:, rank:] @ qr[s, h]) * scale
            p = np.exp(x - x.max())
            want[s, h] = (p / p.sum()) @ (c[:, :rank] @ wv64[h].T)
    # roundings to bf16 on the way: q's two parts, the absorbed query, the weights, the latent output: each 2^-8 at most of its own size
    assert np.linalg.norm(got - want) <= 4 * HALF[kind] * np.linalg.norm(want)
    for x in b + [cache]:
        x.free()

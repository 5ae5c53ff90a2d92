"""Rotary positions, head norms and the append to a paged cache, and page copies, against their
definitions in 64 bits.

Tolerances, e = 2^-24: a head's sum of dh squares in 32 bits is at most dh e off, half of that in its
root; with the division, the root, two products and the turn (products, their sum, cos and sin: 2 e
each, the angle 2 e pi) a value is at most (dh / 2 + 16) e of the pair's size off.  What the cache
holds is rounded once more, by half a step of its type (2^-9 and 2^-12 of the value's binade: at most
2^-8 and 2^-11 of the value; below f16's least normal number 2^-25)."""
import numpy as np
import pytest

from paged import Cache, LAYOUTS, exact_rope, from_bits, to_type

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
HALF_STEP = {"f32": E, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def freqs(dims, theta=1e4):
    return theta ** (-2.0 * np.arange(dims // 2) / max(1, dims))


def pair_size(x, dims, interleaved):
    """for each value the size of the pair it turns in"""
    p = np.abs(x)
    half = dims // 2
    if half:
        i = np.arange(half)
        f, g = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        r = np.hypot(x[..., f], x[..., g])
        p[..., f] = p[..., g] = r
    return p


def case(be, seed, kind, S, Hq, Hkv, dh, P, dims, interleaved=False, norm=True, layout="head", factor=1.0, pos=None, seq=None,
         seqs=None, ld_more=0, max_pages=None, table=None, theta=1e4):
    rng = np.random.default_rng(seed)
    pos = np.asarray(pos if pos is not None else rng.integers(0, 500, S))
    seqs = seqs or S
    sq = np.asarray(seq) if seq is not None else np.arange(S)
    n_pages = 0
    if table is None:
        width = max(1, int(max(pos.max(), 0)) // P + 1)
        # the rows' pages alone are real ones
        table = np.full((seqs, width), -1, np.int32)
        want = sorted({(int(b), int(p) // P) for b, p in zip(sq, pos) if p >= 0})
        ids = rng.permutation(len(want) + 2)
        for (b, j), i in zip(want, ids):
            table[b, j] = i
        n_pages = len(want) + 2
    else:
        n_pages = 6
    old = [to_type(rng.standard_normal((n_pages, Hkv, P, dh)), kind)[0] for _ in range(2)]
    c = Cache(be, kind, n_pages, P, Hkv, dh, *old, layout)
    before = c.image()
    ld = (Hq + 2 * Hkv) * dh + ld_more
    qkv = (rng.standard_normal((S, ld)) * np.exp(rng.standard_normal((S, 1)))).astype(np.float32)
    wq, wk = ((1 + 0.1 * rng.standard_normal(dh)).astype(np.float32) for _ in range(2))
    f = freqs(dims, theta)
    bufs = [be.upload(a) for a in (qkv, wq, wk, np.full(S * Hq * dh + 64, 9.0, np.float32), pos.astype(np.int32),
                                   table.astype(np.int32), sq.astype(np.int32))]
    fd = be.upload(f) if dims else None
    rows = be.kv_rows(bufs[4], bufs[5], table.shape[0], table.shape[1], bufs[6] if seq is not None else None)
    be.qk_rope_append(c.c, rows, be.rope(fd, dims, interleaved, factor), bufs[0], ld, bufs[1] if norm else None,
                      bufs[2] if norm else None, 1e-6, Hq, bufs[3], S)
    q = be.d2h(bufs[3], (S * Hq * dh + 64,), np.float32)
    k, v = c.read()
    after = c.image()
    for b in bufs + ([fd] if dims else []):
        b.free()
    c.free()
    assert np.all(q[S * Hq * dh:] == 9.0)
    q = q[:S * Hq * dh].reshape(S, Hq, dh)
    x = qkv[:, :(Hq + 2 * Hkv) * dh].astype(np.float64).reshape(S, -1, dh)
    tol = (dh / 2 + 16) * E
    live = pos >= 0
    normed = [exact_rope(h, pos, f, 0, 0, 1, w if norm else None, 1e-6) for h, w in ((x[:, :Hq], wq), (x[:, Hq:Hq + Hkv], wk))]
    eq, ek = (exact_rope(h, pos, f, dims, interleaved, factor, None, 0) for h in normed)
    sq_, sk = (pair_size(h, dims, interleaved) * max(1.0, factor) for h in normed)
    assert np.all(np.abs(q - eq)[live] <= tol * sq_[live])
    assert np.all(q[~live] == 9.0)
    hk, hv = (from_bits(a).copy() for a in old)
    bk = np.zeros_like(hk)
    touched = np.zeros((n_pages, P), bool)
    for s in range(S):
        if pos[s] < 0 or not 0 <= sq[s] < table.shape[0] or pos[s] // P >= table.shape[1]:
            continue
        p = table[sq[s], pos[s] // P]
        if not 0 <= p < n_pages:
            continue
        hk[p, :, pos[s] % P] = ek[s]
        bk[p, :, pos[s] % P] = tol * sk[s] * (1 + HALF_STEP[kind]) + HALF_STEP[kind] * np.abs(ek[s]) + (2.0 ** -25 if kind == "f16" else 0)
        hv[p, :, pos[s] % P] = to_type(x[s, Hq + Hkv:], kind)[1]
        touched[p, pos[s] % P] = True
    assert np.all(np.abs(from_bits(k) - hk) <= bk)
    assert np.array_equal(from_bits(v), hv)
    # nothing but the rows' cells changed: gaps, other pages, the cells beside them
    if not touched.any():
        assert np.array_equal(before.view(np.uint8), after.view(np.uint8))
    same = ~touched
    for new, was in ((k, old[0]), (v, old[1])):
        assert np.array_equal(new.transpose(0, 2, 1, 3)[same], was.transpose(0, 2, 1, 3)[same])
    changed = (before.view(np.uint32 if kind == "f32" else np.uint16) != after.view(np.uint32 if kind == "f32" else np.uint16)).sum()
    assert changed <= touched.sum() * 2 * Hkv * dh


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dh", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("interleaved", [False, True])
def test_head_sizes(be, kind, dh, interleaved):
    case(be, dh, kind, 5, 6, 2, dh, 16, dh, interleaved)


@pytest.mark.parametrize("dims", [0, 2, 6, 50, 64, 126, 128, 130, 254])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_part_of_the_head(be, dims, interleaved, norm):
    case(be, dims, "bf16", 4, 4, 2, 256, 32, dims, interleaved, norm)
    if dims <= 128:
        case(be, dims + 1, "f16", 4, 4, 2, 128, 32, dims, interleaved, norm, factor=1.3)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("P", [8, 64, 1024])
def test_layouts(be, kind, layout, P):
    case(be, P, kind, 7, 4, 4, 64, P, 32, layout=layout, ld_more=20)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (17, 1), (40, 8), (128, 2), (5, 5)])
def test_head_counts(be, Hq, Hkv):
    case(be, Hq, "bf16", 3, Hq, Hkv, 64, 16, 64)


@pytest.mark.parametrize("S", [1, 2, 63, 256, 1000])
def test_row_counts(be, S):
    case(be, S, "bf16", S, 8, 2, 128, 16, 128)


def test_chunks_of_sequences(be):
    """rows of a few sequences, free places among them"""
    seq = np.array([1] * 40 + [0] * 3 + [2] * 21)
    pos = np.concatenate([np.arange(13, 53), np.arange(3), np.arange(100, 121)])
    pos[[5, 41, 63]] = -1
    case(be, 1, "bf16", 64, 4, 2, 64, 16, 64, pos=pos, seq=seq, seqs=3)


def test_no_place_for_a_row(be):
    """rows without a place and cells that lead nowhere leave the cache as it was"""
    table = np.array([[0, -1, 6], [2 ** 31 - 1, -2 ** 31, 3], [1, 2, 4]], np.int32)
    pos = np.array([-1, 17, 33, 5, 20, 48, 10 ** 9, 2 ** 31 - 1, -2 ** 31, 3, 4, 40])
    seq = np.array([0, 0, 0, 1, 1, 2, 2, 2, 2, -1, 3, 1])
    case(be, 2, "bf16", 12, 4, 2, 64, 16, 0, pos=pos, seq=seq, table=table, norm=False)
    case(be, 2, "f32", 9, 4, 2, 64, 16, 0, pos=[-1] * 9, seq=[0] * 9, table=table)


@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions(be, interleaved):
    """angles in the millions of radians: a 32-bit product would be 0.06 off at 10^6"""
    pos = np.array([0, 1, 4095, 131071, 1000003, 16777217, 268435455, 99999999])
    case(be, 4, "f32", 8, 4, 2, 128, 4096, 128, interleaved, pos=pos, norm=False)
    case(be, 4, "f32", 8, 4, 2, 128, 4096, 128, interleaved, pos=pos, norm=True, theta=5e6)


def test_rows_of_zeros_and_large_values(be):
    """a head of zeros stays one (eps alone under the root); values beyond f16 become its infinities"""
    be_rows = np.zeros((2, 3 * 64), np.float32)
    be_rows[1] = 1e5
    c = Cache(be, "f16", 2, 8, 1, 64, *[np.zeros((2, 1, 8, 64), np.float16)] * 2)
    bufs = [be.upload(a) for a in (be_rows, np.full(2 * 64, 5.0, np.float32), np.array([0, 1], np.int32), np.zeros((2, 1), np.int32),
                                   np.ones(64, np.float32))]
    rows = be.kv_rows(bufs[2], bufs[3], 2, 1)
    be.qk_rope_append(c.c, rows, be.rope(None, 0), bufs[0], 192, bufs[4], bufs[4], 1e-6, 1, bufs[1], 2)
    q = be.d2h(bufs[1], (2, 64), np.float32)
    k, v = c.read()
    assert not np.any(q[0]) and np.allclose(q[1], 1.0, rtol=1e-5) and not np.any(k[0, 0, 0])
    assert np.all(np.isinf(v[0, 0, 1])) and not np.any(v[0, 0, 0])
    for b in bufs:
        b.free()
    c.free()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dims", [2, 6, 10, 16, 50])
def test_values_behind_the_turned_part(be, dims, interleaved):
    """they pass through bit for bit, whatever stands beside them: infinities, NaN, zeros of either sign"""
    S, Hq, Hkv, dh, P = 3, 2, 1, 64, 8
    rng = np.random.default_rng(dims)
    qkv = rng.standard_normal((S, (Hq + 2 * Hkv) * dh)).astype(np.float32)
    x = qkv.reshape(S, Hq + 2 * Hkv, dh)
    x[:, :, dims] = [[np.inf], [-0.0], [np.nan]]
    x[:, :, dims + 3] = -0.0
    c = Cache(be, "f32", S, P, Hkv, dh, *[np.zeros((S, Hkv, P, dh), np.float32)] * 2)
    f = freqs(dims)
    bufs = [be.upload(a) for a in (qkv, np.zeros(S * Hq * dh, np.float32), np.full(S, 5, np.int32),
                                   np.arange(S, dtype=np.int32)[:, None].copy(), f)]
    rows = be.kv_rows(bufs[2], bufs[3], S, 1)
    be.qk_rope_append(c.c, rows, be.rope(bufs[4], dims, interleaved), bufs[0], qkv.shape[1], None, None, 1e-6, Hq, bufs[1], S)
    q = be.d2h(bufs[1], (S, Hq, dh), np.float32)
    k, v = c.read()
    for b in bufs:
        b.free()
    c.free()
    bits = lambda a: np.ascontiguousarray(a).view(np.uint32)
    assert np.array_equal(bits(q[..., dims:]), bits(x[:, :Hq, dims:]))
    assert np.array_equal(bits(k[np.arange(S), 0, 5, dims:]), bits(x[:, Hq, dims:]))
    assert np.array_equal(bits(v[np.arange(S), 0, 5]), bits(x[:, Hq + 1]))
    assert np.all(np.isfinite(q[..., :dims])) and np.all(np.isfinite(k[np.arange(S), 0, 5, :dims]))


# ------------------------------------------------------------- page copies ----

@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("layers,n_pages,P,Hkv,dh", [(1, 5, 8, 1, 32), (3, 9, 16, 2, 96), (2, 300, 8, 3, 64)])
def test_copies(be, kind, layout, layers, n_pages, P, Hkv, dh):
    rng = np.random.default_rng(layers)
    host = [[to_type(rng.standard_normal((n_pages, Hkv, P, dh)), kind)[0] for _ in range(2)] for _ in range(layers)]
    cs = [Cache(be, kind, n_pages, P, Hkv, dh, k, v, layout) for k, v in host]
    was = [c.image() for c in cs]
    ids = rng.permutation(n_pages)
    half = n_pages // 2
    dst = ids[:half]
    src = ids[half + rng.integers(0, n_pages - half, half)]       # a source may be named often
    be.kv_copy_pages(be.kv_caches([c.c for c in cs]), src, dst)
    be.kv_copy_pages(be.kv_caches([c.c for c in cs]), [], [])
    for c, (k, v), img in zip(cs, host, was):
        gk, gv = c.read()
        k[dst], v[dst] = k[src], v[src]
        assert np.array_equal(gk, k) and np.array_equal(gv, v)
        if layout == "apart":                                     # the gaps between cells as they were
            new = c.image()
            c._view(img, 0)[...], c._view(img, c.vat)[...] = k, v
            assert np.array_equal(new.view(np.uint8), img.view(np.uint8))
        c.free()


def test_copies_of_many_layers_and_pages(be):
    """more layers and pages than one launch takes"""
    rng = np.random.default_rng(2)
    layers, n_pages, P, Hkv, dh = 70, 600, 8, 1, 32
    host = to_type(rng.standard_normal((2, layers, n_pages, Hkv, P, dh)), "f16")[0]
    buf = be.upload(host)
    one = n_pages * P * dh * 2
    cs = be.kv_caches([be.kv_cache(int(buf) + i * one, int(buf) + (layers + i) * one, "f16", n_pages, P, Hkv, dh) for i in range(layers)])
    ids = rng.permutation(n_pages)
    src, dst = ids[:290], ids[290:580]
    be.kv_copy_pages(cs, src, dst)
    got = be.d2h(buf, host.shape, np.float16)
    buf.free()
    host[:, :, dst] = host[:, :, src]
    assert np.array_equal(got, host)


def test_recorded_copies_and_appends(be):
    """a recording keeps its page list; an append in it reads positions at each replay"""
    rng = np.random.default_rng(3)
    P, Hkv, dh, Hq = 8, 2, 64, 4
    pool = [to_type(rng.standard_normal((6, Hkv, P, dh)), "bf16")[0] for _ in range(2)]
    c = Cache(be, "bf16", 6, P, Hkv, dh, *pool)
    qkv = rng.standard_normal((2, (Hq + 2 * Hkv) * dh)).astype(np.float32)
    bufs = [be.upload(a) for a in (qkv, np.zeros(2 * Hq * dh, np.float32), np.array([0, 0], np.int32),
                                   np.array([[0, 1], [2, 3]], np.int32), freqs(dh))]
    rows, rope = be.kv_rows(bufs[2], bufs[3], 2, 2), be.rope(bufs[4], dh)
    src, dst = np.array([0], np.int32), np.array([5], np.int32)
    be.graph_begin()
    be.qk_rope_append(c.c, rows, rope, bufs[0], qkv.shape[1], None, None, 1e-6, Hq, bufs[1], 2)
    be.kv_copy_pages(be.kv_caches([c.c]), src, dst)
    src[0] = dst[0] = 4                                           # the lists are the caller's again
    g = be.graph_end()
    for step in range(4):
        be.h2d(bufs[2], np.array([3 * step, step + 8], np.int32))
        be.graph_launch(g)
        be.sync()
        gk, gv = c.read()
        gq = be.d2h(bufs[1], (2 * Hq * dh,), np.float32)
        be.qk_rope_append(c.c, rows, rope, bufs[0], qkv.shape[1], None, None, 1e-6, Hq, bufs[1], 2)
        assert np.array_equal(gq, be.d2h(bufs[1], (2 * Hq * dh,), np.float32))
        k, v = c.read()
        assert np.array_equal(gk, k) and np.array_equal(gv, v)
        assert np.array_equal(k[5], k[0]) and np.array_equal(v[5], v[0])
    be.graph_destroy(g)
    for b in bufs:
        b.free()
    c.free()


@pytest.mark.parametrize("n,off", [(1, 0), (3, 0), (4, 0), (1023, 0), (5000, 4), (4097, 8)])
def test_add(be, n, off):
    rng = np.random.default_rng(n)
    x, t = (rng.standard_normal(n + 8).astype(np.float32) for _ in range(2))
    xd, td = be.upload(x), be.upload(t)
    be.add(int(xd) + off, int(td), n)
    got = be.d2h(xd, (n + 8,), np.float32)
    i = off // 4
    x[i:i + n] += t[:n]
    assert np.array_equal(got, x)
    xd.free()
    td.free()


@pytest.mark.parametrize("n,off", [(4096, 0), (1021, 0), (777, 4)])
def test_add_to_itself(be, n, off):
    x = np.random.default_rng(n).standard_normal(n + 8).astype(np.float32)
    xd = be.upload(x)
    be.add(int(xd) + off, int(xd) + off, n)
    x[off // 4:off // 4 + n] *= 2
    assert np.array_equal(be.d2h(xd, (n + 8,), np.float32), x)
    xd.free()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dims", [0, 24, 50, 128])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_norm_weights_anywhere(be, interleaved, dims, kind):
    """norm weights that do not begin on 16 bytes give what aligned ones give, to the errors of two orders of summing and of
    one more rounding into the cache; one of the two may be left out"""
    S, Hq, Hkv, dh, P = 3, 6, 2, 128, 8
    rng = np.random.default_rng(dims)
    qkv = rng.standard_normal((S, (Hq + 2 * Hkv) * dh)).astype(np.float32)
    w = (1 + 0.1 * rng.standard_normal((2, dh))).astype(np.float32)
    f = freqs(dims)
    host = [qkv, np.array([5, 70, 0], np.int32), np.arange(27, dtype=np.int32).reshape(3, 9), np.concatenate([[0], w.ravel()]).astype(np.float32),
            w]
    bufs = [be.upload(np.ascontiguousarray(a)) for a in host]
    fd = be.upload(f) if dims else None
    rows = be.kv_rows(bufs[1], bufs[2], 3, 9)

    def call(qn, kn):
        c = Cache(be, kind, 27, P, Hkv, dh, *[np.zeros((27, Hkv, P, dh), np.float32 if kind == "f32" else np.uint16)] * 2)
        out = be.upload(np.zeros(S * Hq * dh, np.float32))
        be.qk_rope_append(c.c, rows, be.rope(fd, dims, interleaved, 1.2), bufs[0], qkv.shape[1], qn, kn, 1e-6, Hq, out, S)
        q = be.d2h(out, (S, Hq, dh), np.float32)
        k, v = (from_bits(a)[[0, 17, 18], :, [5, 6, 0]] for a in c.read())
        out.free()
        c.free()
        return q, k, v
    even, odd = int(bufs[4]), int(bufs[3]) + 4
    q, k, v = call(even, even + 4 * dh)
    q2, k2, v2 = call(odd, odd + 4 * dh)
    x = qkv.astype(np.float64).reshape(S, -1, dh)
    sq, sk = (pair_size(exact_rope(h, np.zeros(S), f, 0, 0, 1, g, 1e-6), dims, interleaved) * 1.2 for h, g in
              ((x[:, :Hq], w[0]), (x[:, Hq:Hq + Hkv], w[1])))
    tol = 2 * (dh / 2 + 16) * E
    assert np.all(np.abs(q - q2) <= tol * sq)
    assert np.all(np.abs(k - k2) <= tol * sk + 2 * HALF_STEP[kind] * (1 + tol) * sk)
    assert np.array_equal(v, v2) and np.array_equal(v, to_type(x[:, Hq + Hkv:], kind)[1])
    plain = call(None, None)
    for a, b in ((call(even, None), (q, plain[1])), (call(None, even + 4 * dh), (plain[0], k))):
        assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    for b in bufs + ([fd] if dims else []):
        b.free()

"""Attention of one new token over a paged cache against its definition in 64 bits.

Tolerance: an output is sum_t p_t v_t / sum_t p_t.  With e = 2^-24: a score is dh products summed in
32 bits (at most (dh + 2) e sum |q k| with the scale), its distance to the maximum and the exponential
take 4 e (|x| + 4) more; a score off by d moves each p by a factor of at most exp(d), numerator and
denominator both, so an output by 2 d of sum p |v|; the sums over n cells, and the joins of parts,
are at most (2 n + 16) e of it.  paged.exact_attention gives that bound for every value.  It is
the worst case: the errors' norm over a whole output is far smaller.  There a rounding of q or
p to 16 bits would show (2^-9); two 8-bit parts of them leave 2^-17, so the norm of the errors is
held to 2^-18 of the output's where scores are of ordinary size."""
import numpy as np
import pytest

from paged import Cache, LAYOUTS, exact_attention, from_bits, to_type

pytestmark = pytest.mark.gpu

LENS = [0, 1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 129, 257, 520]


def random_pages(rng, lens, P, spare=2):
    need = [-(-n // P) for n in lens]
    ids = rng.permutation(sum(need) + spare)
    table = np.full((len(lens), max(1, max(need))), -7, np.int32)      # unused entries lead nowhere
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    return table, len(ids)


def pools(rng, kind, n_pages, P, Hkv, dh):
    return [to_type(rng.standard_normal((n_pages, Hkv, P, dh)), kind)[0] for _ in range(2)]


def poison(k, v, table, pos, seq, P, window):
    """every cell that no row attends to becomes NaN"""
    live = np.zeros((k.shape[0], P), bool)
    for p, q in zip(pos, seq):
        for t in range(max(0, p - window + 1) if window else 0, p + 1):
            if 0 <= table[q, t // P] < k.shape[0]:
                live[table[q, t // P], t % P] = True
    nan = np.uint16(0x7FC0) if k.dtype == np.uint16 else np.nan
    for a in (k, v):
        a.transpose(0, 2, 1, 3)[~live] = nan


def run(be, cache, table, pos, q, Hq, scale, window=0, seq=None, fill=7.0):
    S, dh = q.shape[0], q.shape[2]
    bufs = [be.upload(np.ascontiguousarray(a)) for a in (table.astype(np.int32), np.asarray(pos, np.int32), q.astype(np.float32),
                                                         np.full(S * Hq * dh + 64, fill, np.float32))]
    sd = be.upload(np.asarray(seq, np.int32)) if seq is not None else None
    rows = be.kv_rows(bufs[1], bufs[0], table.shape[0], table.shape[1], sd)
    be.attn_paged(cache.c, rows, bufs[2], Hq, scale, window, bufs[3], S)
    out = be.d2h(bufs[3], (S * Hq * dh + 64,), np.float32)
    for b in bufs + ([sd] if sd else []):
        b.free()
    assert np.array_equal(out[S * Hq * dh:], np.full(64, fill, np.float32))           # nothing behind the last row
    return out[:S * Hq * dh].reshape(S, Hq, dh)


def check(got, want, bound, norm=2.0 ** -18):
    assert np.all(np.isfinite(got))
    assert np.all(np.abs(got - want) <= bound), np.max(np.abs(got - want) / np.maximum(bound, 1e-300))
    if np.linalg.norm(want):
        assert np.linalg.norm(got - want) <= norm * np.linalg.norm(want)


def one(be, seed, kind, Hq, Hkv, dh, P, lens, layout="head", window=0, sharp=1.5):
    rng = np.random.default_rng(seed)
    table, n_pages = random_pages(rng, lens, P)
    k, v = pools(rng, kind, n_pages, P, Hkv, dh)
    pos, seq = np.asarray(lens) - 1, np.arange(len(lens))
    poison(k, v, table, pos, seq, P, window)
    q = (sharp * rng.standard_normal((len(lens), Hq, dh))).astype(np.float32)
    scale = float(np.float32(1 / np.sqrt(dh)))
    c = Cache(be, kind, n_pages, P, Hkv, dh, k, v, layout)
    got = run(be, c, table, pos, q, Hq, scale, window)
    c.free()
    want, bound = exact_attention(from_bits(k), from_bits(v), table, P, pos, seq, q.astype(np.float64), scale, window)
    check(got, want, bound)
    assert not np.any(got[np.asarray(lens) == 0])
    return got


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dh", [32, 64, 96, 128, 160, 192, 224, 256])
def test_types_and_head_sizes(be, kind, dh):
    one(be, dh, kind, 8, 2, dh, 16, LENS)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 1), (16, 1), (17, 1), (40, 1), (64, 2), (6, 3), (5, 5), (16, 16)])
def test_shared_heads(be, kind, Hq, Hkv):
    one(be, Hq, kind, Hq, Hkv, 64, 32, [33, 0, 1, 200, 95])


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("P", [8, 16, 32, 64, 256, 4096])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_pages_and_layouts(be, kind, P, layout):
    one(be, P, kind, 4, 2, 64, P, [1, 70, 0, 300, 8, 40], layout)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 33, 100, 256, 5000])
def test_windows(be, kind, window):
    one(be, window, kind, 8, 2, 64, 16, LENS, window=window)


@pytest.mark.parametrize("kind,Hq,Hkv,dh,P,lens", [
    ("bf16", 8, 2, 128, 16, [5000]), ("f16", 4, 1, 64, 64, [40001]), ("f32", 4, 4, 128, 128, [3001, 17]),
    ("bf16", 4, 1, 256, 32, [20000, 1, 9999]), ("bf16", 20, 1, 96, 8, [7777])])
def test_long(be, kind, Hq, Hkv, dh, P, lens):
    one(be, 1, kind, Hq, Hkv, dh, P, lens)


def test_many_rows(be):
    rng = np.random.default_rng(3)
    one(be, 2, "bf16", 4, 2, 64, 16, list(rng.integers(0, 300, 200)))


@pytest.mark.parametrize("S", [63, 64, 65, 128, 129, 255, 256, 257, 700])
@pytest.mark.parametrize("most,Hq,Hkv", [(40, 4, 2), (700, 2, 1)])
def test_row_counts(be, S, most, Hq, Hkv):
    """rows of any number, long ones and free places among them: the positions are counted in rounds of 64 rows, and
    beyond 256 rows not at all"""
    rng = np.random.default_rng(S)
    lens = rng.integers(0, most, S)
    lens[rng.integers(0, S, 3)] = [0, 3000, 1]
    one(be, S, "bf16", Hq, Hkv, 32, 16, [int(n) for n in lens])


@pytest.mark.parametrize("kind,Hq,Hkv,dh,P,lens", [
    ("bf16", 1, 1, 32, 32, [7900, 7900]), ("bf16", 1, 1, 32, 32, [7936, 5, 7936]), ("f16", 2, 1, 64, 16, [4000, 0, 3999, 17]),
    ("f32", 3, 3, 32, 64, [1500] * 7), ("bf16", 4, 2, 96, 128, [600, 1, 599, 300] * 9), ("f16", 5, 1, 128, 256, [3100, 2000]),
    ("bf16", 5, 5, 64, 8, [3, 90, 400] * 30), ("bf16", 8, 1, 128, 64, [2500, 1, 900, 40, 0] * 8), ("f16", 12, 1, 256, 16, [370, 31] * 16)])
def test_joins_over_more_blocks(be, kind, Hq, Hkv, dh, P, lens):
    """few cache heads: more than 64 blocks for each, whose parts are joined in the same launch where no row has many"""
    one(be, 11, kind, Hq, Hkv, dh, P, lens)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_a_chunk_of_one_sequence(be, kind):
    """rows of the same sequences in any order: each sees the cells up to its own position"""
    rng = np.random.default_rng(4)
    P, Hkv, dh, Hq = 16, 2, 64, 6
    table, n_pages = random_pages(rng, [90, 40, 200], P)
    k, v = pools(rng, kind, n_pages, P, Hkv, dh)
    seq = np.array([2, 0, 0, 0, 2, 1, 2, 0, 1, 2])
    pos = np.array([199, 3, 4, 5, 0, 39, -1, 89, 12, 150])
    q = rng.standard_normal((10, Hq, dh)).astype(np.float32)
    c = Cache(be, kind, n_pages, P, Hkv, dh, k, v)
    got = run(be, c, table, pos, q, Hq, 0.125, seq=seq)
    c.free()
    check(got, *exact_attention(from_bits(k), from_bits(v), table, P, pos, seq, q.astype(np.float64), 0.125))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_cells_that_lead_nowhere(be, kind):
    """pages outside the pool, sequences and positions outside the table: left out, never read"""
    rng = np.random.default_rng(5)
    P, Hkv, dh, Hq = 16, 2, 64, 4
    table, n_pages = random_pages(rng, [200, 200, 200, 200, 200, 200], P)
    k, v = pools(rng, kind, n_pages, P, Hkv, dh)
    table[0, 3] = -1
    table[1, 0] = n_pages
    table[2, 5:9] = [2 ** 31 - 1, -2 ** 31, 0x40000000, n_pages + 3]
    table[3, :] = -1
    seq, pos = np.array([0, 1, 2, 3, -1, 6, 4, 5]), np.array([199, 150, 180, 199, 20, 20, 2 ** 31 - 1, 13 * P + 4])
    q = rng.standard_normal((8, Hq, dh)).astype(np.float32)
    c = Cache(be, kind, n_pages, P, Hkv, dh, k, v)
    got = run(be, c, table, pos, q, Hq, 0.125, seq=seq)
    c.free()
    live = pos.copy()
    live[6] = 13 * P + 500                             # beyond the table: the table's cells are all there are
    want, bound = exact_attention(from_bits(k), from_bits(v), table, P, live, seq, q.astype(np.float64), 0.125)
    check(got, want, bound)
    assert not np.any(got[[3, 4, 5]])


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_scores_of_any_size(be, kind):
    """scores in the hundreds (one cell takes all), and tiny values whose weights spread evenly: the bound alone"""
    rng = np.random.default_rng(6)
    P, Hkv, dh, Hq = 32, 1, 128, 4
    lens = [300, 65, 1]
    table, n_pages = random_pages(rng, lens, P)
    k, v = pools(rng, kind, n_pages, P, Hkv, dh)
    pos, seq = np.asarray(lens) - 1, np.arange(3)
    c = Cache(be, kind, n_pages, P, Hkv, dh, k, v)
    for sharp in (60.0, 1e-6, 1e-30, 0.0, 3e4):
        q = (sharp * rng.standard_normal((3, Hq, dh))).astype(np.float32)
        got = run(be, c, table, pos, q, Hq, 0.0883883461, seq=seq)
        want, bound = exact_attention(from_bits(k), from_bits(v), table, P, pos, seq, q.astype(np.float64), 0.0883883461)
        assert np.all(np.isfinite(got)) and np.all(np.abs(got - want) <= bound + 1e-300), sharp
    c.free()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_a_cell_without_value(be, kind):
    """a NaN in a key reaches the heads that read it in the row that attends to it, and nothing else"""
    rng = np.random.default_rng(7)
    P, Hkv, dh, Hq = 16, 2, 64, 4
    lens = [120, 50, 64]
    table, n_pages = random_pages(rng, lens, P)
    k, v = pools(rng, kind, n_pages, P, Hkv, dh)
    k[table[1, 1], 1, 7, 3] = np.uint16(0x7FC0) if kind == "bf16" else np.nan
    q = rng.standard_normal((3, Hq, dh)).astype(np.float32)
    pos, seq = np.asarray(lens) - 1, np.arange(3)
    c = Cache(be, kind, n_pages, P, Hkv, dh, k, v)
    got = run(be, c, table, pos, q, Hq, 0.125)
    c.free()
    assert np.all(np.isnan(got[1, 2:]))
    k[table[1, 1], 1, 7, 3] = 0
    want, bound = exact_attention(from_bits(k), from_bits(v), table, P, pos, seq, q.astype(np.float64), 0.125)
    got[1, 2:], want[1, 2:] = 0, 0
    check(got, want, bound)


def test_offsets_past_32_bits(be):
    """pages more than 2^32 elements apart"""
    rng = np.random.default_rng(8)
    P, Hkv, dh, Hq, far = 16, 2, 64, 4, (1 << 31) + 1024
    n_pages = 4
    item = 2
    buf = be.alloc((n_pages * far + Hkv * P * dh) * item)
    table = np.array([[3, 1, 2]], np.int32)
    k, v = pools(rng, "f16", n_pages, P, Hkv, dh)
    page = Hkv * P * dh
    for p in range(n_pages):
        for off, a in ((0, k), (page, v)):
            arr = np.ascontiguousarray(a[p])
            be.check(be.lib.lag_hip_h2d(int(buf) + (p * far + off) * item, arr.ctypes.data, arr.nbytes), "h2d")

    class C:
        c = be.kv_cache(int(buf), int(buf) + page * item, "f16", n_pages, P, Hkv, dh, (far, P * dh, dh))
    q = rng.standard_normal((1, Hq, dh)).astype(np.float32)
    pos = np.array([41])
    got = run(be, C, table, pos, q, Hq, 0.125)
    buf.free()
    check(got, *exact_attention(from_bits(k), from_bits(v), table, P, pos, np.zeros(1, int), q.astype(np.float64), 0.125))


@pytest.mark.parametrize("lens,Hq,Hkv", [([700, 40, 3], 8, 2), ([9000], 4, 1)])
def test_recorded_and_replayed(be, lens, Hq, Hkv):
    """two recordings of different shapes, replayed in turn with other positions and queries, against eager calls, bit for bit"""
    rng = np.random.default_rng(9)
    P, dh = 16, 64
    table, n_pages = random_pages(rng, lens, P)
    k, v = pools(rng, "bf16", n_pages, P, Hkv, dh)
    c = Cache(be, "bf16", n_pages, P, Hkv, dh, k, v)
    S, n = len(lens), len(lens) * Hq * dh
    td, pd, qd = be.upload(table), be.upload(np.asarray(lens, np.int32) - 1), be.upload(np.zeros(n, np.float32))
    outs = [be.upload(np.zeros(n, np.float32)) for _ in range(3)]
    rows = be.kv_rows(pd, td, table.shape[0], table.shape[1])
    calls = [lambda o: be.attn_paged(c.c, rows, qd, Hq, 0.125, 0, o, S), lambda o: be.attn_paged(c.c, rows, qd, Hq, 0.125, 100, o, 1)]
    for f in calls:
        f(outs[0])
    graphs = []
    for i, f in enumerate(calls):
        be.graph_begin()
        f(outs[i])
        graphs.append(be.graph_end())
    for step in range(4):
        be.h2d(qd, rng.standard_normal(n).astype(np.float32))
        be.h2d(pd, (rng.integers(0, np.asarray(lens)) if step else np.asarray(lens) - 1).astype(np.int32))
        for i in (0, 1, 0):
            be.h2d(outs[i], np.full(n, 3.0, np.float32))
            be.graph_launch(graphs[i])
        be.sync()
        for i, f in enumerate(calls):
            be.h2d(outs[2], np.full(n, 3.0, np.float32))
            f(outs[2])
            assert np.array_equal(be.d2h(outs[i], (n,), np.uint32), be.d2h(outs[2], (n,), np.uint32))
    for g in graphs:
        be.graph_destroy(g)
    for b in [td, pd, qd] + outs:
        b.free()
    c.free()


def test_same_bits_every_time(be):
    """the same call gives the same bits, and a row's bits do not change with the other rows' contents"""
    a = one(be, 11, "bf16", 8, 2, 128, 16, [3000, 10, 700])
    b = one(be, 11, "bf16", 8, 2, 128, 16, [3000, 10, 700])
    assert np.array_equal(a.view(np.uint32), b.view(np.uint32))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_queries_near_the_largest_float(be, kind):
    """queries whose largest values lie between 2^119 and 2^123: the scores are finite in 32 bits, and so far apart that
    one cell takes everything, so each output is that cell's v, exactly.  (That the two largest scores are further
    apart than the errors of 32-bit sums, 2 (dh + 2) e sum |q k|, and than 200, is asserted of the inputs.)"""
    rng = np.random.default_rng(12)
    P, Hkv, dh, Hq, scale = 16, 2, 128, 6, 0.0883883461
    lens = [300, 65, 1, 1000]
    table, n_pages = random_pages(rng, lens, P)
    k, v = pools(rng, kind, n_pages, P, Hkv, dh)
    pos, seq = np.asarray(lens) - 1, np.arange(4)
    q = (1e36 * rng.standard_normal((4, Hq, dh))).astype(np.float32)
    want = np.zeros(q.shape)
    for s, n in enumerate(lens):
        t = np.arange(n)
        for h in range(Hq):
            kk, vv = (from_bits(a)[table[s, t // P], h // 3, t % P] for a in (k, v))
            x, size = kk @ q[s, h].astype(np.float64) * scale, np.abs(kk) @ np.abs(q[s, h].astype(np.float64)) * scale
            top = np.argmax(x)
            gap = x[top] - np.delete(x, top)
            assert np.all(gap > 2 * (dh + 2) * 2.0 ** -24 * size.max() + 200) and np.abs(x).max() < 1e38
            want[s, h] = vv[top]
    c = Cache(be, kind, n_pages, P, Hkv, dh, k, v)
    got = run(be, c, table, pos, q, Hq, scale, seq=seq)
    c.free()
    assert np.array_equal(got, want.astype(np.float32))


@pytest.mark.parametrize("size", [1e-30, 1e-36])
def test_tiny_queries_and_a_large_scale(be, size):
    """an f16 cache's queries are scaled to f16's range whatever their size: with a scale that makes up for it the
    scores are ordinary ones, in the same bounds"""
    rng = np.random.default_rng(13)
    P, Hkv, dh, Hq = 16, 2, 64, 4
    lens = [200, 33, 700]
    table, n_pages = random_pages(rng, lens, P)
    k, v = pools(rng, "f16", n_pages, P, Hkv, dh)
    pos, seq = np.asarray(lens) - 1, np.arange(3)
    q = (1.5 * size * rng.standard_normal((3, Hq, dh))).astype(np.float32)
    scale = float(np.float32(0.125 / size))
    c = Cache(be, "f16", n_pages, P, Hkv, dh, k, v)
    got = run(be, c, table, pos, q, Hq, scale, seq=seq)
    c.free()
    check(got, *exact_attention(from_bits(k), from_bits(v), table, P, pos, seq, q.astype(np.float64), scale))


@pytest.mark.parametrize("kind,Hq,Hkv,dh,lens,window", [
    ("bf16", 8, 2, 128, [3000, 10, 700, 0, 61], 0), ("f16", 32, 8, 64, [900, 40, 2000, 333], 512), ("f32", 4, 4, 64, [600, 1, 77, 1500], 0),
    ("bf16", 1, 1, 32, [7900, 60, 7900], 0), ("f16", 20, 1, 128, [20000, 333, 9000], 0), ("bf16", 4, 1, 64, [130, 9, 1] * 100, 0)])
def test_bits_do_not_depend_on_other_rows_contents(be, kind, Hq, Hkv, dh, lens, window):
    """one row's cells and query stay, all others change: whole rows, parts joined in the launch and behind it"""
    rng = np.random.default_rng(14)
    P = 16
    table, n_pages = random_pages(rng, lens, P)
    pos, S = np.asarray(lens) - 1, len(lens)
    k, v = pools(rng, kind, n_pages, P, Hkv, dh)
    q = rng.standard_normal((S, Hq, dh)).astype(np.float32)
    c = Cache(be, kind, n_pages, P, Hkv, dh, k, v)
    first = run(be, c, table, pos, q, Hq, 0.125, window)
    c.free()
    for keep in range(min(S, 5)):
        k2, v2 = pools(rng, kind, n_pages, P, Hkv, dh)
        q2 = (30 * rng.standard_normal((S, Hq, dh))).astype(np.float32)
        own = table[keep][table[keep] >= 0]
        k2[own], v2[own], q2[keep] = k[own], v[own], q[keep]
        c = Cache(be, kind, n_pages, P, Hkv, dh, k2, v2)
        again = run(be, c, table, pos, q2, Hq, 0.125, window)
        c.free()
        assert np.array_equal(first[keep].view(np.uint32), again[keep].view(np.uint32)), keep
        assert not np.array_equal(np.delete(first, keep, 0), np.delete(again, keep, 0))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("sign", [1, -1])
def test_infinities(be, kind, sign):
    """in cells that no row attends to they change nothing; in one that a row attends to (as an append into f16 gives for
    values beyond its largest) they reach that row's heads that read it alone"""
    rng = np.random.default_rng(15)
    P, Hkv, dh, Hq, window = 16, 2, 64, 6, 90
    lens = [120, 50, 64, 0, 700]
    table, n_pages = random_pages(rng, lens, P)
    k, v = pools(rng, kind, n_pages, P, Hkv, dh)
    pos, seq = np.asarray(lens) - 1, np.arange(5)
    q = rng.standard_normal((5, Hq, dh)).astype(np.float32)
    inf = sign * np.inf if kind != "bf16" else np.uint16(0x7F80 if sign > 0 else 0xFF80)

    def attend(k, v):
        c = Cache(be, kind, n_pages, P, Hkv, dh, k, v)
        got = run(be, c, table, pos, q, Hq, 0.125, window)
        c.free()
        return got
    clean = attend(k, v)
    live = np.zeros((n_pages, P), bool)
    for s, p in enumerate(pos):
        for t in range(max(0, p - window + 1), p + 1):
            live[table[s, t // P], t % P] = True
    k2, v2 = k.copy(), v.copy()
    for a in (k2, v2):
        a.transpose(0, 2, 1, 3)[~live] = inf
    assert np.array_equal(clean.view(np.uint32), attend(k2, v2).view(np.uint32))
    for which in (0, 1):
        a = [k2.copy(), v2.copy()]
        a[which][table[0, 5], 1, 3] = inf              # token 83 of row 0, heads 3 to 5
        got = attend(*a)
        others = np.ones((5, Hq), bool)
        others[0, 3:] = False
        assert np.array_equal(got[others].view(np.uint32), clean[others].view(np.uint32))
        assert not np.any(np.isfinite(got[0, 3:]))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("window", [0, 40])
def test_a_prompt_of_more_than_256_rows(be, kind, window):
    """a chunk of 230 rows of one sequence beside 70 of others, free places and places that lead nowhere among them"""
    rng = np.random.default_rng(16)
    P, Hkv, dh, Hq = 8, 2, 96, 8
    lens = [260] + [int(n) for n in rng.integers(1, 120, 70)]
    table, n_pages = random_pages(rng, lens, P)
    k, v = pools(rng, kind, n_pages, P, Hkv, dh)
    seq = np.concatenate([np.zeros(230, int), np.arange(1, 71)])
    pos = np.concatenate([np.arange(30, 260), np.asarray(lens[1:]) - 1])
    at = rng.permutation(300)
    seq, pos = seq[at], pos[at]
    pos[[3, 250, 299]], seq[[7, 280]] = -1, [71, -1]
    q = rng.standard_normal((300, Hq, dh)).astype(np.float32)
    c = Cache(be, kind, n_pages, P, Hkv, dh, k, v)
    got = run(be, c, table, pos, q, Hq, 0.102, window, seq=seq)
    c.free()
    scale = float(np.float32(0.102))
    check(got, *exact_attention(from_bits(k), from_bits(v), table, P, pos, seq, q.astype(np.float64), scale, window))
    assert not np.any(got[[3, 250, 299, 7, 280]])

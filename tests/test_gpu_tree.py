"""Attention of trees of drafted tokens, their positions' turn and their acceptance, against the definitions in 64 bits.

Tolerances as in test_gpu_attention.py: every output within the worst case of 32-bit sums, the errors' norm within 2^-18 of the
outputs' (a rounding of q or of a weight to 16 bits would show)."""
import numpy as np
import pytest

from paged import Cache, LAYOUTS, exact_rope, from_bits, to_type
from trees import exact_path, exact_tree, sees_of, tree

pytestmark = pytest.mark.gpu

NAN = {"f32": np.float32(np.nan), "f16": np.float16(np.nan), "bf16": np.uint16(0x7FC0)}


class Case:
    """trees over a cache: prefixes `base`, nodes `sizes`; cells that nobody attends to are NaN"""

    def __init__(self, be, seed, kind, Hq, Hkv, dh, P, base, sizes, layout="head", window=0, sharp=1.5, spare_rows=0, poison=True, sees=None):
        rng = np.random.default_rng(seed)
        self.be, self.kind, self.Hq, self.window, self.P = be, kind, Hq, window, P
        self.base, n = np.asarray(base, np.int32), len(base)
        self.first = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
        self.S = int(self.first[-1]) + spare_rows
        self.parents = [tree(rng, s) if s else np.zeros(0, np.int32) for s in sizes]
        self.sees, self.pos = np.zeros(self.S, np.uint64), np.zeros(self.S, np.int32)
        for i, p in enumerate(self.parents):
            a, b = self.first[i], self.first[i + 1]
            self.sees[a:b], depth = sees_of(p)
            self.pos[a:b] = max(0, base[i]) + depth
        if sees is not None:
            self.sees = sees(self)
        self.seq = rng.permutation(n).astype(np.int32)
        need = np.zeros(n, np.int64)
        need[self.seq] = [max(0, b) + s if b >= 0 else 0 for b, s in zip(base, sizes)]
        pages = -(-need // P)
        ids = rng.permutation(int(pages.sum()) + 2)
        self.table = np.full((n, max(1, int(pages.max()))), -7, np.int32)
        at = 0
        for i, c in enumerate(pages):
            self.table[i, :c] = ids[at:at + c]
            at += c
        self.k, self.v = (to_type(rng.standard_normal((len(ids), Hkv, P, dh)), kind)[0] for _ in range(2))
        if poison:
            live = np.zeros((len(ids), P), bool)
            for i in range(n):
                for s in range(self.first[i], self.first[i + 1]):
                    if base[i] < 0:
                        continue
                    lo = max(0, max(self.pos[s], base[i]) - window + 1) if window else 0
                    for t in list(range(lo, base[i])) + [base[i] + j for j in range(sizes[i]) if int(self.sees[s]) >> j & 1]:
                        live[self.table[self.seq[i], t // P], t % P] = True
            for a in (self.k, self.v):
                a.transpose(0, 2, 1, 3)[~live] = NAN[kind]
        self.q = (sharp * rng.standard_normal((self.S, Hq, dh))).astype(np.float32)
        self.scale = float(np.float32(1 / np.sqrt(dh)))
        self.cache = Cache(be, kind, len(ids), P, Hkv, dh, self.k, self.v, layout)
        up = lambda a: be.upload(np.ascontiguousarray(a))
        self.max_nodes = max(1, max(sizes))
        self.bufs = [up(a) for a in (self.first, self.base, self.sees, self.table, self.seq, self.pos, self.q)]
        f, b, s, t, sq, ps, self.qd = self.bufs
        self.trees = be.trees(f, b, s, t, n, n, self.table.shape[1], self.max_nodes, sq, ps)
        self.out = up(np.full(self.q.size + 64, 7.0, np.float32))

    def run(self):
        self.be.attn_tree(self.cache.c, self.trees, self.qd, self.Hq, self.scale, self.window, self.out, self.S)
        got = self.be.d2h(self.out, (self.q.size + 64,), np.float32)
        assert np.all(got[self.q.size:] == 7.0)
        return got[:self.q.size].reshape(self.q.shape)

    def want(self):
        return exact_tree(from_bits(self.k), from_bits(self.v), self.table, self.P, self.first, self.base, self.seq, self.sees, self.pos,
                          self.q.astype(np.float64), self.scale, self.window, np.full(self.q.shape, 7.0))

    def check(self):
        got, (want, bound) = self.run(), self.want()
        assert np.all(np.isfinite(got))
        assert np.all(np.abs(got - want) <= bound), np.max(np.abs(got - want) / np.maximum(bound, 1e-300))
        live = slice(0, self.first[-1])
        assert np.linalg.norm((got - want)[live]) <= 2.0 ** -18 * np.linalg.norm(want[live])
        return got

    def free(self):
        for b in self.bufs + [self.out, self.cache]:
            b.free()


def one(be, *a, **k):
    c = Case(be, *a, **k)
    got = c.check()
    c.free()
    return got


BASES, SIZES = [0, 1, 5, 31, 32, 33, 64, 100, 257], [1, 7, 2, 1, 32, 3, 17, 9, 5]


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dh", [32, 64, 96, 128, 160, 192, 224, 256])
def test_types_and_head_sizes(be, kind, dh):
    one(be, dh, kind, 4, 2, dh, 16, BASES, SIZES)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dh", [32, 96, 128, 256])
def test_few_columns(be, kind, dh):
    one(be, dh + 1, kind, 4, 2, dh, 16, BASES, [1, 2, 3, 1, 4, 5, 2, 7, 6])


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("Hq,Hkv,top", [(1, 1, 64), (3, 1, 64), (16, 1, 9), (40, 2, 30), (6, 3, 33), (5, 5, 12), (128, 8, 4)])
def test_heads_and_trees(be, kind, Hq, Hkv, top):
    one(be, Hq, kind, Hq, Hkv, 64, 32, [33, 0, 90], [top, 1, max(1, top // 2)])


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("P", [8, 16, 32, 64, 4096])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_pages_and_layouts(be, kind, P, layout):
    one(be, P, kind, 4, 2, 64, P, [1, 70, 0, 300, 8], [3, 12, 20, 1, 9], layout)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("window", [1, 2, 15, 33, 100, 5000])
def test_windows(be, kind, window):
    one(be, window, kind, 4, 2, 64, 16, BASES, SIZES, window=window)


@pytest.mark.parametrize("kind,Hq,Hkv,dh,P,base,sizes", [
    ("bf16", 8, 2, 128, 16, [5000], [20]), ("f16", 4, 1, 64, 64, [40001], [3]), ("f32", 4, 4, 128, 128, [3001, 17], [5, 60]),
    ("bf16", 4, 1, 256, 32, [20000, 1, 9999], [2, 30, 64]), ("bf16", 20, 1, 96, 8, [7777], [40])])
def test_long(be, kind, Hq, Hkv, dh, P, base, sizes):
    one(be, 1, kind, Hq, Hkv, dh, P, base, sizes, poison=False)


@pytest.mark.parametrize("top", [8, 30])
def test_blocks_that_take_several_trees(be, top):
    """more tiles than blocks: a block ends one tree and begins the next"""
    rng = np.random.default_rng(top)
    one(be, 5, "bf16", 8, 2, 64, 64, list(rng.integers(1500, 6000, 40)), list(rng.integers(1, top + 1, 40)), poison=False)


def test_many_trees(be):
    rng = np.random.default_rng(3)
    one(be, 2, "bf16", 4, 2, 64, 16, list(rng.integers(0, 200, 150)), list(rng.integers(1, 9, 150)))


def test_free_places_and_rows_of_no_tree(be):
    c = Case(be, 4, "bf16", 4, 2, 64, 16, [10, -1, 0, 40, -1], [3, 2, 0, 4, 1], spare_rows=5)
    got = c.check()
    assert not np.any(got[3:5]) and np.all(got[-5:] == 7.0)
    c.free()


def test_masks_of_any_kind(be):
    """rows that see nothing, themselves alone, all nodes, bits behind the tree"""
    def sees(c):
        s = c.sees.copy()
        s[0::4], s[1::4], s[2::4] = 0, np.uint64(0xFFFFFFFFFFFFFFFF), np.uint64(1 << 63)
        return s
    c = Case(be, 5, "bf16", 4, 2, 64, 16, [0, 0, 20], [13, 33, 64], poison=False, sees=sees)
    c.sees_all = c.sees.copy()
    for i in range(3):                                                 # bits behind the tree name no node
        n = c.first[i + 1] - c.first[i]
        if n < 64:
            c.sees[c.first[i]:c.first[i + 1]] &= np.uint64((1 << int(n)) - 1)
    got = c.check()
    assert not np.any(got[0]) and not np.any(got[13 + 3])
    c.free()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("what", ["nan", "inf"])
def test_infinities_reach_who_attends(be, kind, what):
    """a node's cell that is no number: rows that attend to it have no finite output somewhere, all others are right"""
    c = Case(be, 6, kind, 4, 2, 64, 16, [40], [20], poison=False)
    t = 40 + 5
    bad = NAN[kind] if what == "nan" else {"f32": np.float32(np.inf), "f16": np.float16(np.inf), "bf16": np.uint16(0x7F80)}[kind]
    clean, bound = c.want()
    c.v[c.table[c.seq[0], t // 16], :, t % 16, 3] = bad
    c.cache.free()
    c.cache = Cache(be, kind, len(c.k), 16, 2, 64, c.k, c.v)
    got = c.run()
    hit = np.array([int(s) >> 5 & 1 for s in c.sees], bool)
    assert hit.any() and not hit.all()
    assert not np.any(np.isfinite(got[hit][..., 3]))
    assert np.all(np.abs(got[~hit] - clean[~hit]) <= bound[~hit])
    c.free()


def test_pages_that_lead_nowhere(be):
    c = Case(be, 7, "bf16", 4, 2, 64, 16, [100, 70], [9, 12], poison=False)
    c.table[:, 2], c.table[0, 4], c.table[1, 0] = -1, 10 ** 6, -2 ** 31
    be.h2d(c.bufs[3], c.table)
    c.check()
    c.free()


def test_bad_row_lists_stay_in_bounds(be):
    """lists that name rows outside the batch, too many nodes or none: whatever is computed, nothing else is written"""
    c = Case(be, 8, "bf16", 4, 2, 64, 16, [10, 20, 30], [3, 4, 5], poison=False)
    for first in ([-5, 3, 7, 12], [0, 100, 7, 12], [7, 3, 0, 2 ** 31 - 1], [2 ** 31 - 1, -2 ** 31, 5, 6]):
        be.h2d(c.bufs[0], np.asarray(first, np.int32))
        c.run()
    be.h2d(c.bufs[0], c.first)
    be.h2d(c.bufs[1], np.asarray([2 ** 31 - 1, 2 ** 30, -2 ** 31], np.int32))
    c.run()
    c.free()


def test_same_bits_again_and_recorded(be):
    c = Case(be, 9, "bf16", 8, 2, 128, 64, [3000, 100, 900], [16, 3, 30], poison=False)
    want = c.run()
    be.graph_begin()
    be.attn_tree(c.cache.c, c.trees, c.qd, c.Hq, c.scale, 0, c.out, c.S)
    g = be.graph_end()
    for _ in range(3):
        be.h2d(c.out, np.zeros(c.q.size, np.float32))
        be.graph_launch(g)
        be.sync()
        assert np.array_equal(be.d2h(c.out, c.q.shape, np.float32), want)
        assert np.array_equal(c.run(), want)
    be.graph_destroy(g)
    c.free()


def test_a_chain_is_a_prompt(be):
    """a tree without branches attends like rows of a prompt at consecutive positions"""
    c = Case(be, 10, "bf16", 8, 2, 128, 16, [77], [12], poison=False,
             sees=lambda c: np.array([(1 << (j + 1)) - 1 for j in range(12)], np.uint64))
    got = c.check()
    pos, seq = be.upload(np.arange(77, 89, dtype=np.int32)), be.upload(np.zeros(12, np.int32))
    be.attn_paged(c.cache.c, be.kv_rows(pos, c.bufs[3], 1, c.table.shape[1], seq), c.qd, 8, c.scale, 0, c.out, 12)
    other = be.d2h(c.out, c.q.shape, np.float32)
    assert np.linalg.norm(got - other) <= 2.0 ** -18 * np.linalg.norm(got)
    for b in (pos, seq):
        b.free()
    c.free()


# ------------------------------------------------------------------ append at positions of their own ----

@pytest.mark.parametrize("rd,interleaved,norm", [(64, False, True), (64, True, False), (30, False, True), (0, False, False)])
def test_turned_by_other_positions(be, rd, interleaved, norm):
    rng = np.random.default_rng(rd)
    S, Hq, Hkv, dh, P = 9, 4, 2, 64, 16
    cell, at = rng.permutation(48)[:S].astype(np.int32), rng.integers(0, 5000, S).astype(np.int32)
    qkv = rng.standard_normal((S, Hq + 2 * Hkv, dh)).astype(np.float32)
    w = [(1 + 0.1 * rng.standard_normal(dh)).astype(np.float32) for _ in range(2)] if norm else [None, None]
    freq = 1e4 ** (-2.0 * np.arange(rd // 2) / max(1, rd))
    c = Cache(be, "f32", 3, P, Hkv, dh, np.zeros((3, Hkv, P, dh), np.float32), np.zeros((3, Hkv, P, dh), np.float32))
    up = lambda a: be.upload(np.ascontiguousarray(a)) if a is not None else None
    pd, ad, sd, td, xd, qd, fd, wq, wk = map(up, (cell, at, np.zeros(S, np.int32), np.arange(3, dtype=np.int32), qkv, np.zeros((S, Hq, dh), np.float32),
                                                  freq if rd else None, *w))
    be.qk_rope_append_at(c.c, be.kv_rows(pd, td, 1, 3, sd), ad, be.rope(fd, rd, interleaved), xd, (Hq + 2 * Hkv) * dh, wq, wk, 1e-6, Hq, qd, S)
    k, v = c.read()
    q = be.d2h(qd, (S, Hq, dh), np.float32)
    x = qkv.astype(np.float64)
    for got, h, ww in ((q, x[:, :Hq], w[0]), (np.stack([k[t // P, :, t % P] for t in cell]), x[:, Hq:Hq + Hkv], w[1])):
        want = exact_rope(h, at, freq, rd, interleaved, 1.0, None if ww is None else ww.astype(np.float64), 1e-6)
        # norm: sum of squares, root, quotient, two products; the turn: angle to 2^-24 of a turn's pi, cos, sin, two products, a sum
        assert np.max(np.abs(got - want)) <= (dh + 24) * 2.0 ** -24 * np.max(np.abs(h)) * 2
    assert np.array_equal(np.stack([v[t // P, :, t % P] for t in cell]), qkv[:, Hq + Hkv:])
    for b in (pd, ad, sd, td, xd, qd, fd, wq, wk, c):
        if b is not None:
            b.free()


# ------------------------------------------------------------------ acceptance ----

def commit(be, seed, kind, P, Hkv, dh, base, sizes, layers=2, layout="head", accept=0.8, max_nodes=None, vocab=3, parents=None, hole=False):
    rng = np.random.default_rng(seed)
    n, first = len(base), np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    S, top = int(first[-1]), max_nodes or max(sizes)
    parents = parents or [tree(rng, s) if s else np.zeros(0, np.int32) for s in sizes]
    draft, tok = rng.integers(0, vocab, S).astype(np.int32), rng.integers(0, vocab, S).astype(np.int32)
    seq = rng.permutation(n).astype(np.int32)
    for i, p in enumerate(parents):                                    # a long path is usual
        for j in range(1, len(p)):
            if rng.random() < accept:
                tok[first[i] + p[j]] = draft[first[i] + j]
    pages = np.array([-(-(max(0, b) + s) // P) for b, s in zip(base, sizes)])
    ids = rng.permutation(int(pages.sum()) + 1)
    table, at = np.full((n, max(1, int(pages.max()))), -1, np.int32), 0
    for i in range(n):
        table[seq[i], :pages[i]] = ids[at:at + pages[i]]
        at += pages[i]
    if hole:
        table[seq[0], pages[0] - 1] = -1
    kv = [[to_type(rng.standard_normal((len(ids), Hkv, P, dh)), kind)[0] for _ in range(2)] for _ in range(layers)]
    caches = [Cache(be, kind, len(ids), P, Hkv, dh, k, v, layout) for k, v in kv]
    up = lambda a: be.upload(np.ascontiguousarray(a))
    bufs = [up(a) for a in (first, np.asarray(base, np.int32), table, seq, np.concatenate(parents).astype(np.int32), draft, tok,
                            np.full(n * top + 8, -5, np.int32), np.full(n + 8, -5, np.int32), np.full(n + 8, -5, np.int32))]
    f, b, t, sq, pa, dr, tk, path, count, nxt = bufs
    be.tree_commit(be.kv_caches([c.c for c in caches]), be.trees(f, b, None, t, n, n, table.shape[1], top, sq), pa, dr, tk, path, count, nxt, S)
    got = [be.d2h(x, (m + 8,), np.int32) for x, m in ((path, n * top), (count, n), (nxt, n))]
    for x in got:
        assert np.all(x[-8:] == -5)
    wp, wc, wn = np.full((n, top), -1), np.zeros(n, np.int64), np.full(n, -1)
    want = [[a.copy() for a in l] for l in kv]
    for i in range(n):
        a, e = first[i], min(first[i + 1], first[i] + top)
        if base[i] < 0 or e == a:
            continue
        way, wn[i] = exact_path(parents[i][:e - a], draft[a:e], tok[a:e])
        wp[i, :len(way)], wc[i] = way, len(way)
        for l in want:
            for x in l:
                for to, fr in enumerate(way):
                    u, w = base[i] + to, base[i] + fr
                    pu, pw = table[seq[i], u // P], table[seq[i], w // P]
                    if pu >= 0 and pw >= 0:
                        x[pu, :, u % P] = x[pw, :, w % P]
    assert np.array_equal(got[0][:-8].reshape(n, top), wp) and np.array_equal(got[1][:-8], wc) and np.array_equal(got[2][:-8], wn)
    for c, l in zip(caches, want):
        for x, y in zip(c.read(), l):
            assert np.array_equal(x, y)
    for x in bufs + caches:
        x.free()
    return wc


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("P", [8, 64])
def test_commit(be, kind, layout, P):
    assert commit(be, P, kind, P, 2, 64, [0, 5, 17, -1, 31, 0], [7, 64, 1, 4, 30, 0], layout=layout).max() > 3


def test_commit_chains_and_stars(be):
    chain = lambda n: np.arange(-1, n - 1, dtype=np.int32)
    assert list(commit(be, 1, "bf16", 16, 3, 96, [3, 9], [64, 20], accept=1.0, vocab=1, parents=[chain(64), chain(20)])) == [64, 20]
    star = np.array([-1] + [0] * 40, np.int32)
    commit(be, 2, "bf16", 16, 1, 256, [3], [41], vocab=50, parents=[star])
    # every other node of a chain: places that are read just before they are written
    commit(be, 3, "f16", 8, 2, 32, [6], [63], accept=1.0, vocab=1, parents=[np.array([-1] + [0 if j < 3 else j - 2 for j in range(1, 63)], np.int32)])


def test_commit_many_layers_and_trees(be):
    commit(be, 4, "bf16", 8, 1, 32, list(range(40)), [9] * 40, layers=70)


def test_commit_odd_parents(be):
    """parents behind their node, outside the tree or themselves name no path; more nodes than max_nodes are not looked at"""
    commit(be, 5, "bf16", 8, 1, 32, [2], [6], accept=0.0, vocab=1, parents=[np.array([3, 2, 1, 0, 3, 900], np.int32)])
    commit(be, 6, "bf16", 8, 1, 32, [2, 9], [12, 12], max_nodes=5, vocab=1, accept=1.0)


def test_commit_leaves_out_cells_that_lead_nowhere(be):
    commit(be, 7, "bf16", 8, 1, 32, [2, 9], [20, 12], vocab=1, accept=1.0, hole=True)

"""Trees of drafted tokens through a stack's layers: nodes against a dense computation of each node's own path in 64 bits, sequences after
their commits, recorded steps, and a stack that accepts what it would have picked.

Tolerances as in the layers' own tests over the same sums: 2e-4 of an update's size with f32 caches; with bf16 and f16 caches 2e-3, for
keys and values that are rounded to another neighbour."""
import numpy as np
import pytest

from sabrewing_amd.attention import AttnConfig, AttnScratch, PagedCache
from sabrewing_amd.drafts import DraftTrees
from test_gpu_attn_stack import Dense, stack_of

pytestmark = pytest.mark.gpu

CHAIN3, BUSH = [-1, 0, 1], [-1, 0, 0, 1, 1, 2, 3, 6, 5]


def path_of(parents, i):
    p = []
    while i >= 0:
        p.append(i)
        i = parents[i]
    return p[::-1]


@pytest.mark.parametrize("kind,tol", [("f32", 2e-4), ("bf16", 2e-3), ("f16", 2e-3)])
@pytest.mark.parametrize("acfg", [AttnConfig(8, 2, 32, 32), AttnConfig(4, 4, 64, 32, interleaved=True, qk_norm=False, window=7), AttnConfig(2, 1, 128, 64)], ids=str)
def test_nodes_and_what_follows(be, acfg, kind, tol):
    """two steps of trees over prompts of 19 and 6 tokens and none, commits of different lengths between, and a plain step behind"""
    D, rng = 256, np.random.default_rng(8)
    dense = Dense(be, acfg, D, 2, 5)
    cache = PagedCache(be, 2, 40, 8, acfg.n_kv, acfg.head_dim, kind, max_seqs=5, max_len=64, max_rows=40)
    trees = DraftTrees(cache, max_trees=5, max_nodes=10)
    scratch = AttnScratch(be, acfg, D, 40)
    hd, xn, tokd = be.alloc(40 * D * 4), be.alloc(40 * D * 4), be.alloc(40 * 4)
    row = lambda n: rng.standard_normal((n, D)).astype(np.float32)

    def run(x, rows, t=None):
        be.h2d(hd, x)
        for l, layer in enumerate(dense.layers):
            layer.forward(hd, xn, len(x), cache.layers[l], rows, scratch, t)
        return be.d2h(hd, x.shape, np.float32)

    def near(got, have, x):
        want = dense.run(np.concatenate([have, x]), kind)[-len(x):] - x
        assert np.linalg.norm(got - x - want) <= tol * np.linalg.norm(want)
    cache.open()                                       # (sequence 0 stays empty)
    seqs = [cache.open() for _ in range(3)]
    have = [row(n) for n in (19, 6, 0)]
    rows, S = cache.rows([(s, len(x)) for s, x in zip(seqs, have) if len(x)])
    run(np.concatenate(have), rows)
    for shapes, accept in (((BUSH, CHAIN3, [-1]), ([0, 1, 3, 6, 7], [0], [0])), ((CHAIN3, BUSH, CHAIN3), ([0, 1], [0, 2, 5, 8], [0, 1, 2]))):
        xs = [row(len(p)) for p in shapes]
        # drafted tokens and picks that accept those paths: node i's token is 10 + i, and every other pick is none of them
        rows, S = trees.place([(s, p, [10 + i for i in range(len(p))]) for s, p in zip(seqs, shapes)], rows=31)
        tok = np.full(31, 99, np.int32)
        at = 0
        for p, a in zip(shapes, accept):
            tok[at + np.array(a[:-1], int)] = 10 + np.array(a[1:], int)
            at += len(p)
        x = np.concatenate(xs + [np.full((31 - at, D), 3.0, np.float32)])
        got = run(x, rows, trees)
        assert np.all(got[at:] == 3.0)                 # free places: nothing attended, nothing added
        at = 0
        for p, mine, had in zip(shapes, xs, have):
            for i in range(len(p)):
                path = path_of(p, i)
                near(got[at + i:at + i + 1], np.concatenate([had, mine[path[:-1]]]), mine[i:i + 1])
            at += len(p)
        be.h2d(tokd, tok)
        assert trees.commit(tokd) == [(a, 99) for a in accept]
        have = [np.concatenate([had, mine[a]]) for had, mine, a in zip(have, xs, accept)]
        assert [cache.length(s) for s in seqs] == [len(x) for x in have]
        cache.compact()
    x = row(3)
    rows, S = cache.rows(seqs)
    got = run(x, rows)
    for i in range(3):
        near(got[i:i + 1], have[i], x[i:i + 1])
    for b in (hd, xn, tokd):
        b.free()
    for b in (trees, scratch, cache, dense):
        b.free()


def test_a_recorded_step_of_trees(be, orc):
    """a stack's step over trees, recorded once and replayed over what place() puts there, against eager steps: the same bits, picks and
    accepted paths, with the stack's own eager work and commits between"""
    acfg = AttnConfig(8, 2, 64, 64)
    cfg, st = stack_of(be, orc, acfg)
    D, V, S = cfg.D, 1000, 12
    caches = [PagedCache(be, 2, 40, 8, 2, 64, "bf16", max_seqs=4, max_len=96, max_rows=S) for _ in range(2)]
    trees = [DraftTrees(c, max_trees=4, max_nodes=8) for c in caches]
    seqs = [[c.open() for _ in range(3)] for c in caches]
    hd, xn = [be.alloc(S * D * 4) for _ in range(2)], be.alloc(S * D * 4)
    lg, tok = [be.alloc(S * V * 4) for _ in range(2)], [be.alloc(S * 4) for _ in range(2)]
    rng, graph = np.random.default_rng(4), None
    st.reserve(S)
    for step in range(7):
        live = [0, 1, 2] if step % 2 == 0 else [2, 0]
        shape = [([-1] + [int(rng.integers(0, i)) for i in range(1, int(rng.integers(1, 5)))]) for _ in live]
        toks = [[int(t) for t in rng.integers(0, V, len(p))] for p in shape]
        x = rng.standard_normal((S, D)).astype(np.float32)
        for k in range(2):
            rows, n = trees[k].place([(seqs[k][i], p, t) for i, p, t in zip(live, shape, toks)], rows=S if sum(map(len, shape)) >= S - 8 else None)
            be.h2d(hd[k], x)
            if k == 1 and n == S and graph is None and step > 0:
                be.graph_begin()
                st.step(hd[1], xn, lg[1], tok[1], S, cache=caches[1], rows=rows, trees=trees[1])
                graph = be.graph_end()
            if k == 1 and n == S and graph:
                be.graph_launch(graph)
            else:
                st.step(hd[k], xn, lg[k], tok[k], n, cache=caches[k], rows=rows, trees=trees[k])
        a, b = (be.d2h(t, (S, V), np.uint32)[:n] for t in lg)
        assert np.array_equal(a, b)
        kept = [t.commit(p) for t, p in zip(trees, tok)]
        assert kept[0] == kept[1] and all(p[0] == 0 for p, _ in kept[0])
    assert graph
    be.graph_destroy(graph)
    st.free()
    for b in trees + caches + hd + lg + tok + [xn]:
        b.free()


def test_drafts_that_are_the_picks(be, orc):
    """greedy decoding of 12 tokens, then the same tokens as drafts beside wrong ones: all of them are accepted, and the sequence holds as
    many tokens.  (An f32 cache: both runs' logits differ by 32-bit sums alone.)"""
    acfg = AttnConfig(4, 2, 64, 64)
    cfg, st = stack_of(be, orc, acfg)
    D, V = cfg.D, 1000
    cache = PagedCache(be, 2, 20, 8, 2, 64, "f32", max_seqs=2, max_len=64, max_rows=16)
    trees = DraftTrees(cache, max_trees=1, max_nodes=16)
    emb = np.random.default_rng(6).standard_normal((V, D)).astype(np.float32)
    hd, xn, lg, tok = be.alloc(16 * D * 4), be.alloc(16 * D * 4), be.alloc(16 * V * 4), be.alloc(16 * 4)
    plain, drafted = cache.open(), cache.open()
    t, greedy = 17, []
    for _ in range(12):
        greedy.append(t)
        rows, S = cache.rows([plain])
        be.h2d(hd, emb[[t]])
        st.step(hd, xn, lg, tok, S, cache=cache, rows=rows)
        t = int(be.d2h(tok, (1,), np.int32)[0])
    greedy.append(t)
    at = 0
    while at < 12:
        n = min(4, 12 - at)
        # node 0, the right drafts at the odd nodes, a wrong one beside each
        parents, tokens, last = [-1], [greedy[at]], 0
        for k in range(1, n):
            parents += [last, last]
            tokens += [greedy[at + k], (greedy[at + k] + 1) % V]
            last = len(parents) - 2
        rows, S = trees.place([(drafted, parents, tokens)])
        be.h2d(hd, emb[tokens])
        st.step(hd, xn, lg, tok, S, cache=cache, rows=rows, trees=trees)
        (path, nxt), = trees.commit(tok)
        assert path == [0] + [2 * k - 1 for k in range(1, n)] and nxt == greedy[at + n]
        at += n
        assert cache.length(drafted) == at
    st.free()
    for b in (trees, cache, hd, xn, lg, tok):
        b.free()

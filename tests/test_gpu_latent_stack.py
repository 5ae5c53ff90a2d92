"""Latent attention through a stack's layers over a LatentCache: prompts in the expanded form and token by token in the absorbed one against a
dense computation in 64 bits, forks and compaction, recorded steps.

The dense side rounds to the cache's type where the layer does (cells, queries, absorbed queries, mixed latents), but not the softmax's weights and not
what the expanded form rounds to 11 bits.  What is left, per output value, with u half a step of the cache's type (bf16 2^-8, f16 2^-11) and A = |Wo| |Wv|
sum_t p_t |c_t| the size of the sums' terms: a weight's rounding, u A; where 32 bits fell on the other side of a rounding's middle, a
whole step of a value, 2 u of it: of the mixed latents 2 u A at most, of a cell 2 u A and of a query or key 2 u times the size of a score's terms, X, in a score, which
doubles in a softmax: 4 u X A at most, if all of them did.  Those are few of many, so that u A (1 + 2 + 2) and a quarter of the last are a wide bound; keys
and values in 11 bits give 2^-11 (2 X + 1) A.  The rest, 32-bit sums, is below 2^-12 of them for f16 and less for bf16."""
import numpy as np
import pytest

from paged import exact_rope, to_type
from sabrewing_amd.attention import AttnConfig, Rope, rope_frequencies
from sabrewing_amd.latent import DeviceLatentAttention, LatentCache, LatentConfig, LatentScratch
from sabrewing_amd.stack import DeviceStack
from test_gpu_attn_stack import stack_of

pytestmark = pytest.mark.gpu

HALF = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11}


class Dense:
    def __init__(self, be, a, D, kind, seed):
        rng = np.random.default_rng(seed)
        self.a, self.D, self.kind, self.rope = a, D, kind, Rope(be, a)
        self.f, self.m = rope_frequencies(a.rope_dims, a.theta, a.factor, a.trained)
        bits = lambda k, sigma, *s: to_type(sigma * rng.standard_normal(s), k)
        one = lambda n: (1 + 0.1 * rng.standard_normal(n)).astype(np.float32)
        r, H = a.q_rank or D, a.n_heads
        self.norm, self.kvn, self.qn = one(D), one(a.rank), one(a.q_rank) if a.q_rank else None
        w = dict(wkv=bits("bf16", 0.06, a.cell, D), wqa=bits("bf16", 0.06, a.q_rank, D) if a.q_rank else (None, None), wq=bits("bf16", 1 / np.sqrt(r), H * a.q_dim, r),
                 wk=bits(kind, 1 / np.sqrt(a.rank), H, a.nope, a.rank), wv=bits(kind, 1 / np.sqrt(a.rank), H, a.v_dim, a.rank), wo=bits("bf16", 0.06, D, H * a.v_dim))
        self.w = {k: v[1] for k, v in w.items()}
        s = {k: v[0] for k, v in w.items()}
        self.layer = DeviceLatentAttention.from_host(be, a, D, self.norm, s["wkv"], self.kvn, s["wqa"], self.qn, s["wq"], s["wk"], s["wv"], s["wo"], self.rope, kind)

    def run(self, h, absorbed):
        """h [T, D], one sequence from position 0; absorbed [T]: rows of that form -> (update, bound)"""
        a, w, T, H, u = self.a, self.w, len(h), self.a.n_heads, HALF[self.kind]
        rms = lambda x, g: x / np.sqrt((x * x).mean(-1, keepdims=True) + a.eps) * g
        r = lambda x: to_type(x, self.kind)[1]
        turn = lambda x: r(exact_rope(x, np.arange(T), self.f, a.rope_dims, a.interleaved, self.m, None, 0)) if a.rope_dims else x
        x = rms(h.astype(np.float64), self.norm)
        ckv = x @ w["wkv"].T
        c, kr = r(rms(ckv[:, :a.rank], self.kvn)), turn(ckv[:, None, a.rank:])[:, 0]
        q = (rms(x @ w["wqa"].T, self.qn) if a.q_rank else x) @ w["wq"].T
        q = q.reshape(T, H, a.q_dim)
        qn, qr = r(q[..., :a.nope]), turn(q[..., a.nope:])
        out, bound = np.zeros((T, self.D)), np.zeros((T, self.D))
        for t in range(T):
            o, A, X = np.zeros((H, a.v_dim)), np.zeros((H, a.v_dim)), 0.0
            for j in range(H):
                ql = w["wk"][j].T @ qn[t, j]
                ql = r(ql) if absorbed[t] else ql
                s = (c[:t + 1] @ ql + kr[:t + 1] @ qr[t, j]) / np.sqrt(a.q_dim)
                X = max(X, np.max(np.abs(c[:t + 1]) @ (np.abs(ql) if absorbed[t] else np.abs(w["wk"][j]).T @ np.abs(qn[t, j])) + np.abs(kr[:t + 1]) @ np.abs(qr[t, j])) / np.sqrt(a.q_dim))
                p = np.exp(s - s.max())
                p /= p.sum()
                mix = p @ c[:t + 1]
                o[j] = w["wv"][j] @ (r(mix) if absorbed[t] else mix)
                A[j] = np.abs(w["wv"][j]) @ (p @ np.abs(c[:t + 1]))
            out[t] = w["wo"] @ o.ravel()
            bound[t] = (u * (5 + X) + (2.0 ** -11 * (2 * X + 1) if not absorbed[t] else 0)) * 1.01 * (np.abs(w["wo"]) @ A.ravel())
        return out, bound

    def free(self):
        self.layer.free()
        self.rope.free()


CONFIGS = [LatentConfig(8, 128, 32, 16, 32), LatentConfig(4, 512, 128, 64, 64, q_rank=128), LatentConfig(6, 256, 64, 32, 64, interleaved=True), LatentConfig(4, 384, 96, 0, 32)]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("a", CONFIGS, ids=str)
def test_prompts_then_tokens(be, a, kind):
    """two sequences: a prompt in one piece, one in two pieces (the second behind the first's cells), then tokens of both, a fork of one that goes on
    by itself, pages moved in between"""
    D, rng = 256, np.random.default_rng(a.rank)
    dense = Dense(be, a, D, kind, 3)
    cache = LatentCache(be, 1, 20, 16, a.rank, a.rope_dims, kind, max_seqs=3, max_len=96, max_rows=64)
    scratch = LatentScratch(be, a, D, 64)
    hd, xn = be.alloc(64 * D * 4), be.alloc(64 * D * 4)
    x = [rng.standard_normal((60, D)).astype(np.float32), rng.standard_normal((45, D)).astype(np.float32)]
    got, form, done = [np.zeros_like(v) for v in x], [np.ones(len(v), bool) for v in x], [0, 0]
    seqs = [cache.open(), cache.open()]

    def run(h, rows):
        be.h2d(hd, h)
        dense.layer.forward(hd, xn, len(h), cache.layers[0], rows, scratch)
        return be.d2h(hd, h.shape, np.float32) - h
    for i, pieces in ((0, [51]), (1, [7, 33])):
        for n in pieces:
            rows, S = cache.prompt(seqs[i], n)
            got[i][done[i]:done[i] + n] = run(x[i][done[i]:done[i] + n], rows)
            form[i][done[i]:done[i] + n] = False
            done[i] += n
    for step in range(5):
        rows, S = cache.rows([seqs[0], None, seqs[1]])
        out = run(np.stack([x[0][done[0]], np.full(D, 2.0, np.float32), x[1][done[1]]]), rows)
        got[0][done[0]], got[1][done[1]] = out[0], out[2]
        assert not out[1].any()
        done = [d + 1 for d in done]
        if step == 1:
            fork = cache.fork(seqs[0])
            rows, S = cache.rows([fork])               # (its own copy of the shared last page)
            run(x[1][:1], rows)
            cache.compact()
        if step == 2:
            cache.close(fork)
    rows, S = cache.rows([(seqs[0], 4)])               # a chunk of a sequence's next rows in the absorbed form
    got[0][done[0]:] = run(x[0][done[0]:], rows)
    assert done[0] + 4 == 60 and done[1] == 45
    for v, g, f in zip(x, got, form):
        want, bound = dense.run(v, f)
        # (h + update and its difference from h: two roundings of their sizes)
        worst = np.max(np.abs(g - want) / (bound + 2.0 ** -23 * (np.abs(v) + np.abs(want))))
        assert worst <= 1.0, worst
    for b in (hd, xn):
        b.free()
    for b in (scratch, cache, dense):
        b.free()


def test_a_stack_of_latent_layers(be, orc):
    """a seeded stack: its step is its layers' entries, a recorded step gives the eager one's bits at every replay, over rows that move on"""
    a = LatentConfig(16, 256, 64, 32, 64, q_rank=128)
    cfg, _ = stack_of(be, orc, AttnConfig(8, 2, 64, 64))
    _.free()
    D, V, S = cfg.D, 1000, 3
    st = DeviceStack.generate(be, cfg, 2, V, 5).add_attention(a, seed=5)
    caches = [LatentCache(be, 2, 24, 8, a.rank, a.rope_dims, max_seqs=4, max_len=64, max_rows=40) for _ in range(2)]
    seqs = [[c.open() for _ in range(S)] for c in caches]
    hd, xn, lg, tok = [be.alloc(40 * D * 4) for _ in range(2)], be.alloc(40 * D * 4), [be.alloc(40 * V * 4) for _ in range(2)], [be.alloc(40 * 4) for _ in range(2)]
    rng, graph = np.random.default_rng(1), None
    st.reserve(40)
    x = rng.standard_normal((20, D)).astype(np.float32)
    for k in range(2):
        rows, n = caches[k].prompt(seqs[k][1], 20)
        be.h2d(hd[k], x)
        st.step(hd[k], xn, lg[k], tok[k], n, cache=caches[k], rows=rows)
    for step in range(10):                             # over a page's end
        x = rng.standard_normal((S, D)).astype(np.float32)
        for k in range(2):
            rows = caches[k].rows(seqs[k])[0]
            be.h2d(hd[k], x)
            if k and graph is None and step == 1:
                be.graph_begin()
                st.step(hd[1], xn, lg[1], tok[1], S, cache=caches[1], rows=rows)
                graph = be.graph_end()
            if k and graph:
                be.graph_launch(graph)
            else:
                st.step(hd[k], xn, lg[k], tok[k], S, cache=caches[k], rows=rows)
        h, lo, t = ([be.d2h(b, (S, n), np.uint32) for b in bufs] for bufs, n in ((hd, D), (lg, V), (tok, 1)))
        assert np.array_equal(h[0], h[1]) and np.array_equal(lo[0], lo[1]) and np.array_equal(t[0], t[1])
        assert np.all(np.isfinite(h[0].view(np.float32)))
    be.graph_destroy(graph)
    st.free()
    for b in caches + hd + lg + tok + [xn]:
        b.free()

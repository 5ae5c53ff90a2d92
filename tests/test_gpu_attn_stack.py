"""Attention layers over a paged cache as a stack uses them: prompts in chunks and decoding token by
token, forks, compaction, sampling and recorded steps, against a dense computation in 64 bits and against
the entries called one by one.

Tolerance of the dense comparison: the longest sums are D and n_q * head_dim products in 32 bits (at
most 256 x 2^-24 of their terms' sizes), a norm, the head's dot product and the softmax over at most 60
cells, which doubles a score's error: below 1,000 x 2^-24 = 6e-5 of the update's size a layer, and what a
layer is off goes through the next: 2e-4 for two.  A bf16 cache rounds k and v of both sides alike but for
values near the middle of two, which land one step (2^-8) apart: seldom, and one cell's share of a sum
of many, 2e-3."""
import numpy as np
import pytest

from oracle import synth
from paged import exact_rope, from_bits, to_type
from sabrewing_amd import configs as cf
from sabrewing_amd.attention import AttnConfig, AttnScratch, DeviceAttention, PagedCache, Rope, rope_frequencies
from sabrewing_amd.stack import DeviceStack, head_bf16, norm_weights

pytestmark = pytest.mark.gpu


class Dense:
    """the layers' weights on the host, their computation in 64 bits over whole sequences"""

    def __init__(self, be, acfg, D, n_layers, seed):
        rng = np.random.default_rng(seed)
        self.a, self.D = acfg, D
        self.rope = Rope(be, acfg)
        self.f, self.m = rope_frequencies(acfg.rope_dims, acfg.theta, acfg.factor, acfg.trained)
        bf = lambda *s: to_type(0.06 * rng.standard_normal(s), "bf16")[0]
        one = lambda n: (1 + 0.1 * rng.standard_normal(n)).astype(np.float32)
        head = lambda: one(acfg.head_dim) if acfg.qk_norm else None
        self.w = [(one(D), bf(acfg.qkv_rows, D), bf(D, acfg.n_q * acfg.head_dim), head(), head()) for _ in range(n_layers)]
        self.layers = [DeviceAttention.from_host(be, acfg, D, *w, self.rope) for w in self.w]

    def run(self, h, kind):
        """h [T, D], one sequence's rows from position 0: what the layers make of them"""
        a, h, T = self.a, h.astype(np.float64), len(h)
        for norm, wqkv, wo, qn, kn in self.w:
            x = h / np.sqrt((h * h).mean(1, keepdims=True) + a.eps) * norm
            p = (x @ from_bits(wqkv).T).reshape(T, -1, a.head_dim)
            q, k, v = p[:, :a.n_q], p[:, a.n_q:a.n_q + a.n_kv], p[:, a.n_q + a.n_kv:]
            pos = np.arange(T)
            q, k = ([exact_rope(exact_rope(t, pos, self.f, 0, 0, 1, w, a.eps), pos, self.f, a.rope_dims,
                                a.interleaved, self.m, None, 0) for t, w in ((q, qn), (k, kn))])
            k, v = to_type(k, kind)[1], to_type(v, kind)[1]
            ctx = np.zeros((T, a.n_q, a.head_dim))
            for t in range(T):
                lo = max(0, t - a.window + 1) if a.window else 0
                for j in range(a.n_q):
                    kk, vv = k[lo:t + 1, j * a.n_kv // a.n_q], v[lo:t + 1, j * a.n_kv // a.n_q]
                    s = kk @ q[t, j] / np.sqrt(a.head_dim)
                    e = np.exp(s - s.max())
                    ctx[t, j] = e @ vv / e.sum()
            h = h + ctx.reshape(T, -1) @ from_bits(wo).T
        return h

    def free(self):
        for l in self.layers:
            l.free()
        self.rope.free()


CONFIGS = [AttnConfig(8, 2, 32, 32), AttnConfig(4, 4, 64, 32, interleaved=True, qk_norm=False, window=7),
           AttnConfig(2, 1, 128, 64, factor=4.0, trained=32)]


@pytest.mark.parametrize("kind,tol", [("f32", 2e-4), ("bf16", 2e-3), ("f16", 2e-3)])
@pytest.mark.parametrize("acfg", CONFIGS, ids=str)
def test_prompts_then_tokens(be, acfg, kind, tol):
    """three sequences of different lengths, prompts in chunks beside each other and beside decoding rows, a free
    place among them"""
    D, n_layers, lens = 256, 2, (60, 23, 9)
    rng = np.random.default_rng(3)
    dense = Dense(be, acfg, D, n_layers, 5)
    cache = PagedCache(be, n_layers, 20, 8, acfg.n_kv, acfg.head_dim, kind, max_seqs=4, max_len=80, max_rows=64)
    seqs = [cache.open() for _ in lens]
    x = [rng.standard_normal((n, D)).astype(np.float32) for n in lens]
    got = [np.zeros_like(a) for a in x]
    done, scratch = [0, 0, 0], AttnScratch(be, acfg, D, 64)
    hd, xn = be.alloc(64 * D * 4), be.alloc(64 * D * 4)
    step = 0
    while any(d < n for d, n in zip(done, lens)):
        take = [min(n - d, (11, 1, 4)[i] if step < 3 else 1) for i, (d, n) in enumerate(zip(done, lens))]
        batch = [(s, t) for s, t in zip(seqs, take) if t]
        batch.insert(1, None)
        rows, S = cache.rows(batch)
        h = np.concatenate([x[i][done[i]:done[i] + t] for i, t in enumerate(take) if t])
        first = take[0] if take[0] else take[1] if take[1] else take[2]
        h = np.insert(h, first, 7.0, axis=0)
        assert len(h) == S
        be.h2d(hd, h)
        for l, layer in enumerate(dense.layers):
            layer.forward(hd, xn, S, cache.layers[l], rows, scratch)
        out = be.d2h(hd, (S, D), np.float32)
        assert np.all(out[first] == 7.0)               # the free place: nothing attended, nothing added
        out = np.delete(out, first, axis=0)
        at = 0
        for i, t in enumerate(take):
            got[i][done[i]:done[i] + t] = out[at:at + t]
            done[i] += t
            at += t
        if step == 4:                                  # pages move in between: nothing may change
            cache.close(seqs[2]) if done[2] == lens[2] else None
            cache.compact()
            if done[2] == lens[2]:
                seqs[2] = cache.open()
        step += 1
    for a, g in zip(x, got):
        want = dense.run(a, kind) - a
        assert np.linalg.norm(g - a - want) <= tol * np.linalg.norm(want)
    for b in (hd, xn):
        b.free()
    scratch.free()
    cache.free()
    dense.free()


def stack_of(be, orc, acfg, n_layers=2, V=1000, seed=77):
    cfg = cf.scaled(cf.C5_LAYER, D=512, E=32, K=8, I=384)
    layers = [synth.make_layer(orc, cfg, seed, layer=l) for l in range(n_layers)]
    nw = norm_weights(orc, cfg, seed, n_layers)
    st = DeviceStack.from_host(be, cfg, layers, nw[:n_layers], nw[n_layers], head_bf16(orc, cfg, seed, V))
    return cfg, st.add_attention(acfg, seed=seed)


def test_step_is_its_entries(be, orc):
    """a stack's step with attention and a drawn token against the entries called one by one: the same bits, and the
    greedy step's logits; a recorded step replayed over the cache's rows against eager steps"""
    acfg = AttnConfig(8, 2, 64, 64)
    cfg, st = stack_of(be, orc, acfg)
    D, V, S = cfg.D, 1000, 3
    from sabrewing_amd.backend import desc_of
    caches = [PagedCache(be, 2, 24, 8, 2, 64, "bf16", max_seqs=4, max_len=64) for _ in range(3)]
    seqs = [[c.open() for _ in range(S)] for c in caches]
    hd = [be.alloc(S * D * 4) for _ in range(3)]
    xn, lg, tok = be.alloc(S * D * 4), [be.alloc(S * V * 4) for _ in range(3)], [be.alloc(S * 4) for _ in range(3)]
    temp, u = be.upload(np.array([0.8, 1.0, 0.0], np.float32)), be.upload(np.zeros(S, np.float32))
    params = be.sample_params(temp)
    rng = np.random.default_rng(1)
    st.reserve(S)
    graph = None
    for step in range(11):                             # over a page's end
        x, uu = rng.standard_normal((S, D)).astype(np.float32), rng.random(S, dtype=np.float32)
        be.h2d(u, uu)
        for b in hd:
            be.h2d(b, x)
        rows = [c.rows(s)[0] for c, s in zip(caches, seqs)]
        st.step(hd[0], xn, lg[0], tok[0], S, cache=caches[0], rows=rows[0], draw=(params, u))
        for l, dl in enumerate(st.layers):
            st.attn[l].forward(hd[1], xn, S, caches[1].layers[l], rows[1], st.scratch)
            be.rmsnorm(hd[1], st.norms[l], xn, S, D, 1e-6)
            be.moe_forward(desc_of(cfg), dl.weights(), xn, hd[1], S)
        be.rmsnorm(hd[1], st.final_norm, xn, S, D, 1e-6)
        be.head_argmax(st.head, True, xn, S, D, V, lg[1], tok[1])
        greedy = be.d2h(tok[1], (S,), np.int32)
        be.sample(lg[1], S, V, params, u, tok[1])
        if graph is None and step == 1:                # the same shapes were issued at step 0
            be.graph_begin()
            st.step(hd[2], xn, lg[2], tok[2], S, cache=caches[2], rows=rows[2], draw=(params, u))
            graph = be.graph_end()
        if graph:
            be.graph_launch(graph)
        else:
            st.step(hd[2], xn, lg[2], tok[2], S, cache=caches[2], rows=rows[2], draw=(params, u))
        h = [be.d2h(b, (S, D), np.uint32) for b in hd]
        lo = [be.d2h(b, (S, V), np.uint32) for b in lg]
        t = [be.d2h(b, (S,), np.int32) for b in tok]
        for i in (1, 2):
            assert np.array_equal(h[0], h[i]) and np.array_equal(lo[0], lo[i]) and np.array_equal(t[0], t[i])
        assert t[0][2] == greedy[2]                    # temperature 0
    be.graph_destroy(graph)
    with pytest.raises(ValueError):
        st.step(hd[0], xn, lg[0], tok[0], S)           # no cache
    st.free()
    for c in caches:
        c.free()
    for b in hd + lg + tok + [xn, temp, u]:
        b.free()


def test_forked_streams_agree(be, orc):
    """two branches of one prompt that take the same tokens stay equal, bit for bit, whoever copies the shared page; a
    truncated stream that takes its tokens again ends where it was"""
    acfg = AttnConfig(8, 2, 64, 32, window=9)
    cfg, st = stack_of(be, orc, acfg)
    D, V = cfg.D, 1000
    cache = PagedCache(be, 2, 30, 8, 2, 64, "f16", max_seqs=4, max_rows=16)
    hd, xn, lg, tok = be.alloc(16 * D * 4), be.alloc(16 * D * 4), be.alloc(16 * V * 4), be.alloc(16 * 4)
    rng = np.random.default_rng(2)

    def run(batch, x):
        rows, S = cache.rows(batch)
        be.h2d(hd, x)
        st.step(hd, xn, lg, tok, S, cache=cache, rows=rows)
        return be.d2h(hd, (S, D), np.float32)
    a = cache.open()
    run([(a, 13)], rng.standard_normal((13, D)).astype(np.float32))
    b = cache.fork(a)
    x = rng.standard_normal((6, D)).astype(np.float32)
    for t in range(6):
        h = run([a, b], np.stack([x[t], x[t]]))
        assert np.array_equal(h[0], h[1])
        last = h[0]
    cache.truncate(a, 13)
    for t in range(6):
        h = run([a, b] if t == 5 else [a], np.stack([x[t], x[t]])[:2 if t == 5 else 1])
    assert cache.length(a) == 19 and cache.length(b) == 20
    err = np.linalg.norm(h[0] - last) / np.linalg.norm(last)
    assert err <= 1e-5                                 # (another batch: sums cut elsewhere)
    cache.close(b)
    assert cache.pages_free() == 30 - 3
    st.free()
    cache.free()
    for q in (hd, xn, lg, tok):
        q.free()


def test_groups_after_attention(be, orc):
    """lag_hip_last_groups tells of the last forward until another call takes the scratch its lists lie in, or makes it grow:
    an attention whose rows have parts, a matmul of host arrays, a routing of more tokens; then there are none.
    What takes no scratch, or other scratch than the lists lie in, leaves them, a routing of the same tokens among it."""
    from paged import Cache
    from sabrewing_amd.backend import DeviceLayer, desc_of
    cfg = cf.scaled(cf.C5_LAYER, D=512, E=32, K=8, I=384)
    layer = synth.make_layer(orc, cfg, 91)
    dl, S = DeviceLayer.from_host(be, cfg, layer), 5
    x = synth.make_x(orc, cfg, 92, S)
    xd, od = be.upload(x), be.upload(np.zeros_like(x))
    P, dh, far = 16, 64, 20000                         # one row of 20,000 tokens: split, and more scratch than the forward
    n_pages = -(-far // P)
    c = Cache(be, "bf16", n_pages, P, 1, dh, *[np.zeros((n_pages, 1, P, dh), np.uint16)] * 2)
    bufs = [be.upload(a) for a in (np.array([far - 1], np.int32), np.arange(n_pages, dtype=np.int32)[None].copy(),
                                   np.ones((1, 16, dh), np.float32), np.ones((1, 16, dh), np.float32))]
    rows, head = be.kv_rows(bufs[0], bufs[1], 1, n_pages), be.upload(np.zeros((8, cfg.D), np.uint16))
    many = be.upload(np.tile(x, (120, 1)))
    attend = lambda: be.attn_paged(c.c, rows, bufs[2], 16, 0.125, 0, bufs[3], 1)
    forward = lambda: be.moe_forward(desc_of(cfg), dl.weights(), xd, od, S)
    _, sel, _ = be.route(desc_of(cfg), dl.weights(), xd, S)
    want = orc.bucket(sel, S, cfg.K, cfg.E)

    def same():
        got = be.last_groups()
        assert got[0] == want[0] and all(np.array_equal(a, b) for a, b in zip(got[1:], want[1:4]))
    forward()
    same()
    be.add(od, xd, x.size)                             # no scratch
    same()
    attend()
    assert be.last_groups()[0] == 0
    forward()
    same()
    be.route(desc_of(cfg), dl.weights(), xd, S)
    same()
    be.route(desc_of(cfg), dl.weights(), many, 600)    # its scores reach further than the lists
    assert be.last_groups()[0] == 0
    forward()
    be.matmul_bf16(x[:1, :128], head, 1)               # 516 bytes: the lists lie behind 5 rows' scores
    same()
    be.matmul_bf16(x, head, 8)
    assert be.last_groups()[0] == 0
    be.moe_forward_noalloc(desc_of(cfg), dl.weights(), xd, od, S)
    same()
    attend()                                           # its lists lie in the static region
    same()
    for b in [xd, od, head, many] + bufs:
        b.free()
    c.free()
    dl.free()

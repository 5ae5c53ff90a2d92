"""Trees of drafted tokens and caches of latents on the host: the arrays that place() gives the device, what commit() and drop() leave of
the sequences, and what is refused, over the paged cache's stand-in for a device."""
import numpy as np
import pytest

from sabrewing_amd.attention import AttnConfig, CacheFull, PagedCache, Rope
from sabrewing_amd.backend import Backend, BackendError
from sabrewing_amd.drafts import DraftTrees, tree_of
from sabrewing_amd.latent import DeviceLatentAttention, LatentCache, LatentConfig, LatentPrompt, LatentScratch
from sabrewing_amd.stack import DeviceStack
from test_attention_stack_host import Recorder, stack
from test_paged_cache import FakeBackend, invariants


class Fake(FakeBackend):
    trees, latent_cache = staticmethod(Backend.trees), staticmethod(Backend.latent_cache)
    accept = None                                      # paths that the next commit keeps

    def ints(self, addr, n):
        return self.read(int(addr), n)

    def tree_commit(self, layers, desc, parent, draft, tok, path, count, nxt, S):
        T, N = desc.n_trees, desc.max_nodes
        out = np.full((T, N), -1, np.int32)
        for i, p in enumerate(self.accept):
            out[i, :len(p)] = p
        self.mem[int(path) - 8 * T] = bytearray(np.concatenate(
            [[len(p) for p in self.accept] + [0] * (T - len(self.accept)), [7 + i for i in range(T)], out.ravel()]).astype(np.int32).tobytes())

    def d2h(self, buf, shape, dtype):
        return np.frombuffer(bytes(self.mem[int(buf)]), dtype)[:shape[0]].copy()


def test_trees_of_parents():
    depth, sees = tree_of([-1, 0, 0, 1, 3, 2])
    assert list(depth) == [0, 1, 1, 2, 3, 2]
    assert [int(s) for s in sees] == [1, 3, 5, 11, 27, 37]
    assert tree_of([-1] + list(range(63)))[1][63] == (1 << 64) - 1
    for bad in ([], [0], [-1, -1], [-1, 1], [-1, 0, 2], [-1] + [0] * 64):
        with pytest.raises(ValueError):
            tree_of(bad)
    with pytest.raises(ValueError):
        tree_of([-1, 0, 0], 2)


def arrays(be, t):
    d, T, R = t.desc, t.max_trees, t.cache.max_rows
    return dict(first=be.ints(d.first, T + 1), base=be.ints(d.base, T), seq=be.ints(d.seq, T), at=be.ints(t.at, R),
                sees=be.ints(d.sees, 2 * R).view(np.uint64), parent=be.ints(t._parent, R), draft=be.ints(t._draft, R))


def test_place_and_commit():
    be = Fake()
    c = PagedCache(be, 2, 24, 8, 2, 32, max_seqs=4, max_rows=24)
    a, b = c.open(), c.open()
    c.rows([(a, 13), (b, 3)])
    t = DraftTrees(c, max_trees=4, max_nodes=8)
    assert t.desc.sees % 8 == 0
    desc, S = t.place([(b, [-1, 0, 1], [5, 6, 7]), (a, [-1, 0, 0, 2], [1, 2, 3, 4])])
    assert S == 7 and c.length(a) == 17 and c.length(b) == 6
    x = arrays(be, t)
    assert list(x["first"]) == [0, 3, 7, 7, 7] and list(x["base"]) == [3, 13, -1, -1] and list(x["seq"]) == [b, a, -1, -1]
    assert list(x["at"][:8]) == [3, 4, 5, 13, 14, 14, 15, -1] and list(x["sees"][:8]) == [1, 3, 7, 1, 3, 5, 13, 0]
    assert list(x["parent"][:7]) == [-1, 0, 1, -1, 0, 0, 2] and list(x["draft"][:7]) == [5, 6, 7, 1, 2, 3, 4]
    assert list(be.ints(desc.pos, 24)[:8]) == [3, 4, 5, 13, 14, 15, 16, -1]
    assert list(be.ints(desc.seq, 24)[:8]) == [b, b, b, a, a, a, a, -1]
    with pytest.raises(ValueError):
        t.place([(a, [-1], [1])])                      # the trees before are open
    be.accept = [[0], [0, 2, 3]]
    assert t.commit(0) == [([0], 7), ([0, 2, 3], 8)]
    assert c.length(b) == 4 and c.length(a) == 16
    invariants(c)
    with pytest.raises(ValueError):
        t.commit(0)
    # free places behind the trees, and a tree dropped
    desc, S = t.place([(a, [-1, 0], [1, 2])], rows=20)
    x = arrays(be, t)
    assert S == 20 and list(x["first"]) == [0, 2, 10, 18, 20] and list(x["base"]) == [16, -1, -1, -1]
    t.drop()
    assert c.length(a) == 16
    invariants(c)


def test_what_place_refuses_changes_nothing():
    be = Fake()
    c = PagedCache(be, 1, 5, 8, 2, 32, max_seqs=4, max_rows=24)
    a, b = c.open(), c.open()
    c.rows([(a, 14), (b, 7)])
    t = DraftTrees(c, max_trees=2, max_nodes=8)
    chain = lambda n: ([-1] + list(range(n - 1)), list(range(n)))
    for batch, kw in [([], {}), ([(a, [-1, 0], [1])], {}), ([(a, *chain(9))], {}), ([(a, *chain(2)), (a, *chain(2))], {}), ([(3, *chain(2))], {}),
                      ([(a, *chain(2))], dict(rows=1)), ([(a, *chain(2))], dict(rows=11)), ([(a, *chain(1))] * 3, {}),
                      ([(a, *chain(8)), (b, *chain(8))], dict(rows=17))]:
        with pytest.raises(ValueError):
            t.place(batch, **kw)
        assert c.length(a) == 14 and c.length(b) == 7 and t._placed is None
    c.rows([(a, 2), (b, 8)])
    with pytest.raises(CacheFull):
        t.place([(a, *chain(8)), (b, *chain(8))])
    h2d = be.h2d
    be.h2d = lambda dst, arr: (_ for _ in ()).throw(BackendError("no")) if int(dst) == int(t.dev) else h2d(dst, arr)
    with pytest.raises(BackendError):
        t.place([(a, *chain(2))])
    assert c.length(a) == 16
    be.h2d = h2d
    invariants(c)
    t.place([(a, *chain(2))])
    c.fork(a)
    with pytest.raises(ValueError):
        t.commit(0)                                    # the fork holds the tree's cells
    c2 = PagedCache(be, 1, 4, 8, 2, 32, max_seqs=2, max_rows=8)
    t2 = DraftTrees(c2)
    s = c2.open()
    t2.place([(s, [-1], [1])])
    c2.rows([s])
    with pytest.raises(ValueError):
        t2.commit(0)
    t2.drop()
    assert c2.length(s) == 2                           # (it went on: left as it is)
    r = c2.open()
    t2.place([(s, [-1], [1]), (r, [-1, 0], [1, 2])])
    c2.close(r)
    with pytest.raises(ValueError):
        t2.commit(0)
    t2.drop()
    assert c2.length(s) == 2
    with pytest.raises(OverflowError):
        t2.place([(s, [-1], [1 << 31])])
    assert c2.length(s) == 2 and t2._placed is None
    invariants(c2)
    for kw in (dict(max_nodes=0), dict(max_nodes=65), dict(max_trees=65536)):
        with pytest.raises(ValueError):
            DraftTrees(c, **kw)


L = LatentConfig(4, 128, 32, 16, 32)


def test_caches_of_latents():
    be = Fake()
    for kw in (dict(rank=64), dict(rope_dims=8), dict(rope_dims=80), dict(kind="f32"), dict(page_size=24), dict(page_size=4), dict(n_pages=0)):
        with pytest.raises(ValueError):
            LatentCache(be, **{**dict(n_layers=2, n_pages=8, page_size=8, rank=128, rope_dims=16), **kw})
    c = LatentCache(be, 2, 8, 8, 128, 16, max_seqs=3, max_rows=20)
    x, y = c.layers[1], c.copied[1]
    assert (x.token_stride, x.page_stride, x.rank, x.rope_dims) == (192, 1536, 128, 16)
    # the halves of a cell, 3 heads of 32 values each, are all of it
    assert y.k == x.c and y.v == x.c + 192 and (y.n_heads, y.head_dim, y.head_stride, y.token_stride, y.page_stride) == (3, 32, 32, 192, 1536)
    s = c.open()
    p, n = c.prompt(s, 11)
    assert n == 11 and isinstance(p, LatentPrompt) and (p.start, p.n_pages) == (0, 2) and p.pages == int(c.dev_table) + 4 * s * c.max_pages
    p, n = c.prompt(s, 9)
    assert (p.start, p.n_pages, c.length(s)) == (11, 3, 20)
    f = c.fork(s)
    c.rows([s, f])
    assert be.copies == [1]
    invariants(c)


def test_stacks_of_latents_and_trees_refuse_each_other():
    class R(Recorder):
        trees, latent_cache, heads = (staticmethod(getattr(Backend, n)) for n in ("trees", "latent_cache", "heads"))
    be = R()
    A = AttnConfig(4, 2, 32, 32)
    st = stack(be, [A])
    cache, other = (PagedCache(be, 1, 8, 8, 2, 32, max_seqs=3) for _ in range(2))
    lat = LatentCache(be, 1, 8, 8, 128, 16, max_seqs=3)
    t = DraftTrees(cache)

    def step(s, c, rows, trees=None):
        be.calls.clear()
        s.step(be.alloc(4), be.alloc(4), be.alloc(4), be.alloc(4), 2, cache=c, rows=rows, trees=trees)
    t.place([(cache.open(), [-1, 0], [3, 4])])
    step(st, cache, cache.desc, t)
    assert "attn_tree" in be.calls and "attn_paged" not in be.calls and "qk_rope_append_at" in be.calls
    one = DraftTrees(cache, 1)
    one.place([(cache.open(), [-1], [3])])
    for c, tr in ((lat, None), (other, t), (cache, one), (cache, DraftTrees(cache))):
        with pytest.raises(ValueError):
            step(st, c, c.desc, tr)
        assert not be.calls
    # latents
    u16, f32 = (lambda *s: np.zeros(s, np.uint16)), (lambda *s: np.ones(s, np.float32))
    D = st.cfg.D
    make = lambda a, q=None: DeviceLatentAttention.from_host(be, a, D, f32(D), u16(a.cell, D), f32(a.rank), None, q, u16(a.n_heads * a.q_dim, D),
                                                             u16(a.n_heads, a.nope, a.rank), u16(a.n_heads, a.v_dim, a.rank), u16(D, a.n_heads * a.v_dim), Rope(be, a))
    ls = DeviceStack(be, st.cfg, 1000)
    ls.layers, ls.norms, ls.final_norm, ls.head = st.layers, st.norms, st.final_norm, st.head
    ls.add_attention(L, [make(L)])
    step(ls, lat, lat.desc)
    assert isinstance(ls.scratch, LatentScratch) and be.calls.count("latent_heads") == 2 and "attn_latent" in be.calls
    step(ls, lat, LatentPrompt(lat.desc, 4096, 2, 0, 2))
    assert "latent_heads" not in be.calls and "attn_latent" not in be.calls and "attn_latent_prompt" in be.calls
    for n in (1, 3):
        with pytest.raises(ValueError):
            step(ls, lat, LatentPrompt(lat.desc, 4096, 2, 0, n))
        assert not be.calls
    for c, tr in ((cache, None), (LatentCache(be, 1, 8, 8, 256, 16, max_seqs=3), None), (LatentCache(be, 1, 8, 8, 128, 16, "f16", max_seqs=3), None), (lat, t)):
        with pytest.raises(ValueError):
            step(ls, c, c.desc, tr)
        assert not be.calls
    for bad in (LatentConfig(4, 128, 48, 16, 32), LatentConfig(2, 128, 32, 16, 32), LatentConfig(4, 128, 32, 16, 32, q_rank=64)):
        with pytest.raises(ValueError):
            make(bad)
    with pytest.raises(ValueError):
        make(L, f32(128))

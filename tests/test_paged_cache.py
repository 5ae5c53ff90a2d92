"""The paged cache's host side against a plain model (lists of tokens), with a stand-in for the device:
cells that hold a token's number, copied and addressed as the kernels copy and address them."""
import numpy as np
import pytest

from sabrewing_amd.attention import AttnConfig, CacheFull, PagedCache, rope_frequencies
from sabrewing_amd.backend import Backend, BackendError


class Buf:
    def __init__(self, addr):
        self.addr = addr

    def __int__(self):
        return self.addr

    def free(self):
        self.addr = None


class FakeBackend:
    """device memory as byte arrays by address; one cell of a layer's pools as one number"""
    kv_cache, kv_caches, kv_rows = (staticmethod(getattr(Backend, n)) for n in ("kv_cache", "kv_caches", "kv_rows"))

    def __init__(self):
        self.next, self.mem, self.cells, self.copies = 4096, {}, {}, []

    def alloc(self, n):
        b = Buf(self.next)
        self.next += (n + 4095) // 4096 * 4096
        return b

    def upload(self, arr):
        b = self.alloc(arr.nbytes)
        self.mem[b.addr] = bytearray(arr.tobytes())
        return b

    def h2d(self, dst, arr):
        at = int(dst)
        base = max(a for a in self.mem if a <= at)
        assert at - base + arr.nbytes <= len(self.mem[base])
        self.mem[base][at - base:at - base + arr.nbytes] = np.ascontiguousarray(arr).tobytes()

    def read(self, addr, n):
        base = max(a for a in self.mem if a <= addr)
        return np.frombuffer(bytes(self.mem[base][addr - base:addr - base + 4 * n]), np.int32)

    def kv_copy_pages(self, layers, src, dst):
        src, dst = list(map(int, src)), list(map(int, dst))
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        self.copies.append(len(src))
        P = layers[0].page_size
        for a, b in zip(src, dst):
            for i in range(P):
                self.cells[b, i] = self.cells.get((a, i))


def append(be, desc, S, P, tokens):
    """what qk_rope_append does with a batch's rows"""
    pos, seq = be.read(desc.pos, S), be.read(desc.seq, S)
    for s in range(S):
        if pos[s] < 0:
            continue
        page = be.read(desc.table + 4 * (int(seq[s]) * desc.max_pages + int(pos[s]) // P), 1)[0]
        assert page >= 0
        be.cells[int(page), int(pos[s]) % P] = tokens[s]
    return pos, seq


def contents(be, c, seq):
    """a sequence's tokens through the device's table"""
    out = []
    for t in range(c.length(seq)):
        page = be.read(c.desc.table + 4 * (seq * c.max_pages + t // c.page_size), 1)[0]
        out.append(be.cells[int(page), t % c.page_size])
    return out


def invariants(c):
    held = [p for pages in c._pages if pages for p in pages]
    users = np.bincount(held, minlength=c.n_pages) if held else np.zeros(c.n_pages, int)
    assert np.array_equal(users, c._users)
    assert sorted(c._free) == list(np.flatnonzero(users == 0))
    for s, pages in enumerate(c._pages):
        if pages is not None:
            assert len(pages) == -(-c._len[s] // c.page_size)
            assert list(c._table[s, :len(pages)]) == pages and np.all(c._table[s, len(pages):] == -1)


@pytest.mark.parametrize("seed", range(12))
@pytest.mark.parametrize("P", [8, 16])
def test_against_lists(seed, P):
    rng = np.random.default_rng(seed)
    be = FakeBackend()
    c = PagedCache(be, 2, 24, P, 2, 32, "bf16", max_seqs=7, max_len=10 * P, max_rows=40)
    model, token = {}, 0
    for step in range(250):
        op = rng.choice(["open", "fork", "close", "truncate", "compact", "rows", "rows", "rows", "rows"])
        live = list(model)
        try:
            if op == "open":
                model[c.open()] = []
            elif op == "fork" and live:
                s = int(rng.choice(live))
                model[c.fork(s)] = list(model[s])
            elif op == "close" and live:
                s = int(rng.choice(live))
                c.close(s)
                del model[s]
            elif op == "truncate" and live:
                s = int(rng.choice(live))
                n = int(rng.integers(0, len(model[s]) + 1))
                c.truncate(s, n)
                model[s] = model[s][:n]
            elif op == "compact":
                n = c.compact()
                assert n == (c._users > 0).sum() and np.all(c._users[:n] > 0)
            elif op == "rows" and live:
                pick = rng.permutation(live)[:rng.integers(1, len(live) + 1)]
                batch = [(int(s), int(rng.integers(1, 9))) if rng.random() < 0.4 else int(s) for s in pick]
                if rng.random() < 0.3:
                    batch.insert(int(rng.integers(0, len(batch) + 1)), None)
                total = sum(1 if e is None or np.isscalar(e) else e[1] for e in batch)
                if total > 40:
                    continue
                before = (c._users.copy(), list(c._free), list(c._len), [list(p) if p is not None else None for p in c._pages])
                try:
                    desc, S = c.rows(batch)
                except CacheFull:
                    assert np.array_equal(before[0], c._users) and before[1] == c._free and before[2] == c._len and before[3] == c._pages
                    continue
                assert S == total
                tokens = list(range(token, token + S))
                token += S
                append(be, desc, S, P, tokens)
                at = 0
                for e in batch:
                    if e is None:
                        at += 1
                        continue
                    s, n = (e, 1) if np.isscalar(e) else e
                    model[s] = model[s] + tokens[at:at + n]
                    at += n
                rest = be.read(desc.pos, c.max_rows)[S:]
                assert np.all(rest == -1)
        except CacheFull:
            assert len(model) == 7
        invariants(c)
        c._upload()
        for s in model:
            assert c.length(s) == len(model[s]) and contents(be, c, s) == model[s]


def test_a_fork_copies_one_page():
    be = FakeBackend()
    c = PagedCache(be, 3, 10, 8, 1, 32, max_seqs=4)
    a = c.open()
    desc, S = c.rows([(a, 2)])
    append(be, desc, S, 8, [0, 1])
    b, d = c.fork(a), c.fork(a)
    assert c.pages_free() == 9
    desc, S = c.rows([a, b, d])                        # two copies; the last holder keeps the page
    assert be.copies == [2] and c.pages_free() == 7
    append(be, desc, S, 8, [10, 11, 12])
    assert [contents(be, c, s) for s in (a, b, d)] == [[0, 1, 10], [0, 1, 11], [0, 1, 12]]
    c.close(a)
    c.close(d)
    assert c.compact() == 1 and contents(be, c, b) == [0, 1, 11]


def test_a_failed_copy_changes_nothing():
    be = FakeBackend()
    c = PagedCache(be, 1, 8, 8, 1, 32, max_seqs=4, max_rows=9)
    a = c.open()
    desc, S = c.rows([(a, 2)])
    append(be, desc, S, 8, [0, 1])
    b, d = c.fork(a), c.fork(a)

    def state():
        return c._users.tolist(), list(c._free), list(c._len), [list(p) if p is not None else None for p in c._pages], c._table.tolist()
    before = state()

    def broken(*_):
        raise BackendError("injected fault")
    be.kv_copy_pages = broken
    with pytest.raises(BackendError):
        c.rows([a, (b, 7), d])
    assert state() == before
    del be.kv_copy_pages
    desc, S = c.rows([a, (b, 7), d])
    append(be, desc, S, 8, list(range(10, 19)))
    invariants(c)
    assert [contents(be, c, s) for s in (a, b, d)] == [[0, 1, 10], [0, 1] + list(range(11, 18)), [0, 1, 18]]


@pytest.mark.parametrize("nth", range(5))
def test_a_failed_upload_changes_nothing(nth):
    """the nth upload of a step fails (a changed sequence's table, or the rows): the call again gives the same step, and
    what lies on the device afterwards is right"""
    be = FakeBackend()
    c = PagedCache(be, 1, 12, 8, 1, 32, max_seqs=5, max_rows=30)
    a, e = c.open(), c.open()
    desc, S = c.rows([(a, 10), (e, 8)])
    append(be, desc, S, 8, list(range(18)))
    b, d = c.fork(a), c.fork(a)

    def state():
        return c._users.tolist(), list(c._free), list(c._len), [list(p) if p is not None else None for p in c._pages], c._table.tolist()
    before, batch, h2d, left = state(), [a, (b, 9), None, d, (e, 2)], be.h2d, [nth]

    def broken(*args):
        if not left[0]:
            raise BackendError("injected fault")
        left[0] -= 1
        h2d(*args)
    be.h2d = broken
    with pytest.raises(BackendError):
        c.rows(batch)
    assert state() == before
    invariants(c)
    be.h2d = h2d
    desc, S = c.rows(batch)
    assert S == 14
    append(be, desc, S, 8, list(range(100, 114)))
    invariants(c)
    ten = list(range(10))
    assert [contents(be, c, s) for s in (a, b, d, e)] == [ten + [100], ten + list(range(101, 110)), ten + [111],
                                                         list(range(10, 18)) + [112, 113]]


def test_free_places():
    be = FakeBackend()
    c = PagedCache(be, 1, 4, 8, 1, 32, max_seqs=3, max_rows=9)
    a, b = c.open(), c.open()
    desc, S = c.rows([(None, 2), (a, 3), None, b])
    assert S == 7
    assert list(be.read(desc.pos, 9)) == [-1, -1, 0, 1, 2, -1, 0, -1, -1]
    assert list(be.read(desc.seq, 9)) == [-1, -1, a, a, a, -1, b, -1, -1]


def test_refusals():
    be = FakeBackend()
    c = PagedCache(be, 1, 4, 8, 1, 32, max_seqs=2, max_len=16, max_rows=20)
    a = c.open()
    for bad in ([a, a], [(a, 0)], [(a, -1)], [1], [7], [-1], [], [(a, 21)]):
        with pytest.raises(ValueError):
            c.rows(bad)
    with pytest.raises(CacheFull):
        c.rows([(a, 17)])                              # beyond its table
    c.open()
    with pytest.raises(CacheFull):
        c.open()
    with pytest.raises(CacheFull):
        c.fork(a)
    with pytest.raises(ValueError):
        c.truncate(a, 1)
    c.close(a)
    for f in (c.close, c.fork, c.length):
        with pytest.raises(ValueError):
            f(a)
    with pytest.raises(TypeError):
        c.rows([(c.open(), 2.0)])                      # before anything changes
    assert c.pages_free() == 4 and not c._table[c._table >= 0].size
    for kw in (dict(page_size=12), dict(n_pages=0), dict(max_seqs=0), dict(page_size=4), dict(page_size=8192), dict(head_dim=48),
               dict(head_dim=288), dict(n_heads=1025), dict(kind="f64"), dict(max_len=(1 << 30) + 1)):
        d = dict(n_layers=1, n_pages=4, page_size=8, n_heads=1, head_dim=32)
        d.update(kw)
        with pytest.raises(ValueError):
            PagedCache(be, **d)


def test_rope_frequencies():
    f, m = rope_frequencies(64, 1e4)
    assert m == 1.0 and np.allclose(f, [1e4 ** (-i / 32) for i in range(32)], rtol=1e-15)
    f2, m = rope_frequencies(64, 1e4, factor=4.0)
    assert m == 1.0 and np.allclose(f2, f / 4, rtol=1e-15)
    f3, m = rope_frequencies(64, 1e4, factor=4.0, trained=4096)
    assert np.isclose(m, 1 + 0.1 * np.log(4.0))
    turns = 4096 * f / (2 * np.pi)
    assert np.allclose(f3[turns >= 32], f[turns >= 32]) and np.allclose(f3[turns <= 1], f[turns <= 1] / 4)
    between = (turns < 32) & (turns > 1)
    assert between.any() and np.all((f3 < f)[between]) and np.all((f3 > f / 4)[between])
    assert rope_frequencies(0)[0].size == 0
    for bad in (dict(dims=3), dict(dims=-2), dict(dims=4, factor=0.0)):
        with pytest.raises(ValueError):
            rope_frequencies(**bad)
    assert AttnConfig(8, 2, 64, 64).qkv_rows == 12 * 64

"""The attention half of a stack's layers: a paged cache of keys and values with its host-side
bookkeeping, rotary frequencies, and a layer's weights.

    h += Wo . attention(rope(norm(Wqkv . rmsnorm(h))))

runs as rmsnorm, the bf16 projection, `qk_rope_append`, `attn_paged`, the output projection and
`add` (the projections are the head's kernels: any [rows, inputs] matrix of bf16).  The reference's
engines keep this half on the CPU (SDPA over their own caches).
"""
import math
from dataclasses import dataclass
from operator import index

import numpy as np

from . import synth
from .backend import BackendError, DevBuf, KV_TYPES
from .configs import WEIGHT_SIGMA

T_QKV, T_O, T_ATTN_NORM, T_Q_NORM, T_K_NORM = range(11, 16)


# ------------------------------------------------------------------ rotary ----

def rope_frequencies(dims, theta=10000.0, factor=1.0, trained=0, fast=32.0, slow=1.0):
    """Radians per position of each pair, [dims/2] doubles, and the factor that cos and sin take.

    factor > 1 stretches a model trained on `trained` positions: pairs that turn more than `fast`
    times over them keep their frequency, pairs that turn less than `slow` times are slowed by
    `factor`, those between along a ramp, and cos and sin grow by 0.1 ln(factor) + 1 (the "by
    parts" interpolation of the YaRN paper).  trained = 0: every pair slowed alike, factor 1.  A model with
    another ramp or factor gives Backend.rope frequencies of its own."""
    if dims % 2 or dims < 0 or factor <= 0:
        raise ValueError("rope_frequencies: dims must be even, factor positive")
    f = float(theta) ** (-2.0 * np.arange(dims // 2, dtype=np.float64) / max(1, dims))
    if factor == 1.0:
        return f, 1.0
    if not trained:
        return f / factor, 1.0
    turns = trained * f / (2 * math.pi)
    keep = np.clip((turns - slow) / (fast - slow), 0.0, 1.0)
    return f * keep + f / factor * (1.0 - keep), 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0


# ------------------------------------------------------------------- cache ----

class CacheFull(BackendError):
    """no page left: the call changed nothing; free a sequence and call again"""


class PagedCache:
    """Keys and values of many sequences, in pages of `page_size` tokens that every layer shares
    the numbering of.  Sequences hold pages and pages count the sequences that hold them: a fork
    shares them all, and whoever appends first to a shared last page gets a copy of it.

    rows() is the step of a decode loop: it gives the next positions of the named sequences
    their cells and says where they are.  The row arrays are the cache's own and stay where they are,
    so that a recorded step replays over what the next rows() put there."""

    def __init__(self, be, n_layers, n_pages, page_size, n_heads, head_dim, kind="bf16", max_seqs=64, max_len=None, max_rows=None):
        self.be, self.n_layers, self.n_pages, self.page_size = be, n_layers, n_pages, page_size
        self.n_heads, self.head_dim, self.kind = n_heads, head_dim, kind
        if min(n_layers, n_pages, page_size, n_heads, head_dim, max_seqs) < 1 or page_size & (page_size - 1):
            raise ValueError("PagedCache: sizes must be positive, page_size a power of two")
        if not 8 <= page_size <= 4096 or head_dim % 32 or head_dim > 256 or n_heads > 1024 or kind not in KV_TYPES:
            raise ValueError("PagedCache: page_size 8 to 4096, head_dim a multiple of 32 up to 256, at most 1024 heads, f32, bf16 or f16")
        item = 4 if KV_TYPES[kind] == 0 else 2
        self.max_seqs, self.max_rows = max_seqs, max_rows or max_seqs
        self.max_pages = -(-(max_len or n_pages * page_size) // page_size)
        if self.max_pages * page_size > 1 << 30:
            raise ValueError("PagedCache: sequences of more than 2^30 tokens (max_len)")
        one = n_pages * n_heads * page_size * head_dim * item              # one layer's keys or values
        self.pool = be.alloc(2 * n_layers * one)
        base = int(self.pool)
        self.layers = be.kv_caches([be.kv_cache(base + 2 * l * one, base + (2 * l + 1) * one, kind, n_pages, page_size, n_heads,
                                                head_dim) for l in range(n_layers)])
        self._users = np.zeros(n_pages, np.int32)
        self._free = list(range(n_pages - 1, -1, -1))                      # the lowest last
        self._pages = [None] * max_seqs
        self._len = [0] * max_seqs
        self._table = np.full((max_seqs, self.max_pages), -1, np.int32)
        self._dirty = set()
        self._rows = np.full((2, self.max_rows), -1, np.int32)             # positions, sequences
        self.dev_rows, self.dev_table = be.upload(self._rows), be.upload(self._table)
        self.desc = be.kv_rows(self.dev_rows, self.dev_table, max_seqs, self.max_pages, int(self.dev_rows) + 4 * self.max_rows)

    # ---- sequences ----
    def _check(self, seq):
        if not 0 <= seq < self.max_seqs or self._pages[seq] is None:
            raise ValueError(f"PagedCache: no sequence {seq}")

    def _slot(self):
        for i, p in enumerate(self._pages):
            if p is None:
                return i
        raise CacheFull(f"all {self.max_seqs} sequences are in use")

    def open(self):
        """a new, empty sequence"""
        seq = self._slot()
        self._pages[seq], self._len[seq] = [], 0
        return seq

    def fork(self, seq):
        """a sequence that goes on from where `seq` is; their pages are shared until written"""
        self._check(seq)
        new = self._slot()
        self._pages[new], self._len[new] = list(self._pages[seq]), self._len[seq]
        self._users[self._pages[new]] += 1
        self._table[new] = self._table[seq]
        self._dirty.add(new)
        return new

    def close(self, seq):
        """the sequence's pages that no other holds are free again"""
        self._check(seq)
        self._drop(self._pages[seq])
        self._pages[seq], self._len[seq] = None, 0
        self._table[seq] = -1
        self._dirty.add(seq)

    def truncate(self, seq, length):
        """forget the tokens from position `length` on"""
        self._check(seq)
        if not 0 <= length <= self._len[seq]:
            raise ValueError(f"PagedCache: sequence {seq} has {self._len[seq]} tokens, not {length}")
        keep = -(-length // self.page_size)
        gone, self._pages[seq], self._len[seq] = self._pages[seq][keep:], self._pages[seq][:keep], length
        if gone:
            self._drop(gone)
            self._table[seq, keep:] = -1
            self._dirty.add(seq)

    def _drop(self, pages):
        for p in reversed(pages):
            self._users[p] -= 1
            if not self._users[p]:
                self._free.append(p)

    def _take(self, took):
        p = self._free.pop()
        self._users[p] = 1
        took.append(p)
        return p

    def length(self, seq):
        self._check(seq)
        return self._len[seq]

    def pages_free(self):
        return len(self._free)

    # ---- a step ----
    def rows(self, batch):
        """The next tokens of a batch: entries are a sequence (one token), (sequence, n) (its next
        n tokens, rows in order), None or (None, n) (free places).  Returns (rows descriptor, number
        of rows); appending through them is the caller's next calls, for every layer.  CacheFull,
        or a copy or an upload that fails, leaves everything as it was."""
        batch = [(e, 1) if e is None or np.isscalar(e) else tuple(e) for e in batch]
        batch = [(s if s is None else index(s), index(n)) for s, n in batch]
        named = [s for s, _ in batch if s is not None]
        total = sum(n for _, n in batch)
        if len(set(named)) != len(named) or any(n < 1 for _, n in batch):
            raise ValueError("PagedCache.rows: a sequence named twice, or no tokens for one")
        for s in named:
            self._check(s)
        if not 1 <= total <= self.max_rows:
            raise ValueError(f"PagedCache.rows: {total} rows (at most {self.max_rows})")
        # what it takes: copies of shared last pages, then new ones
        P, users, need, old = self.page_size, {}, 0, {}                    # (old: the lengths before)
        for s, n in batch:
            if s is None:
                continue
            pages, ln = self._pages[s], self._len[s]
            old[s] = ln
            if ln + n > self.max_pages * P:
                raise CacheFull(f"sequence {s}: {ln + n} tokens, at most {self.max_pages * P}")
            if ln % P:
                last = pages[-1]
                if users.setdefault(last, int(self._users[last])) > 1:
                    users[last] -= 1
                    need += 1
            need += -(-(ln + n) // P) - len(pages)
        if need > len(self._free):
            raise CacheFull(f"{need} pages needed, {len(self._free)} free")
        took, src, of = [], [], {}                                         # pages taken, shared ones left, and those in their place
        try:
            for s, ln in old.items():                                      # the shared last pages are copied first
                if ln % P and self._users[self._pages[s][-1]] > 1:
                    src.append(self._pages[s][-1])
                    of[s] = self._take(took)
                    self._users[src[-1]] -= 1
            if src:
                self.be.kv_copy_pages(self.layers, src, list(of.values()))
            at = 0
            for s, n in batch:
                if s is None:
                    self._rows[:, at:at + n] = -1
                    at += n
                    continue
                pages, ln = self._pages[s], self._len[s]
                if s in of:
                    pages[-1] = of[s]
                    self._table[s, len(pages) - 1] = of[s]
                    self._dirty.add(s)
                while len(pages) * P < ln + n:
                    p = self._take(took)
                    self._table[s, len(pages)] = p
                    pages.append(p)
                    self._dirty.add(s)
                self._rows[0, at:at + n] = np.arange(ln, ln + n)
                self._rows[1, at:at + n] = s
                self._len[s] = ln + n
                at += n
            self._rows[:, at:] = -1
            self._upload()
            self.be.h2d(self.dev_rows, self._rows)
        except BaseException:
            for s, ln in old.items():                                      # as it was
                n = -(-ln // P)
                del self._pages[s][n:]
                self._table[s, n:], self._len[s] = -1, ln
                self._dirty.add(s)
            for s, p in zip(of, src):
                self._pages[s][-1] = self._table[s, len(self._pages[s]) - 1] = p
                self._users[p] += 1
            for p in reversed(took):
                self._users[p] = 0
                self._free.append(p)
            raise
        return self.desc, total

    def _upload(self):
        for s in sorted(self._dirty):
            self.be.h2d(int(self.dev_table) + s * self.max_pages * 4, self._table[s])
        self._dirty.clear()

    def compact(self):
        """Move the pages in use to the pool's beginning; returns how many they are."""
        used = np.flatnonzero(self._users > 0)
        n = used.size
        src = used[used >= n]
        dst = np.flatnonzero(self._users[:n] == 0)
        if src.size:
            self.be.kv_copy_pages(self.layers, src, dst)
            to = np.arange(self.n_pages)
            to[src] = dst
            for s, pages in enumerate(self._pages):
                if pages:
                    self._pages[s] = [int(to[p]) for p in pages]
                    self._table[s, :len(pages)] = self._pages[s]
                    self._dirty.add(s)
            self._users[dst] = self._users[src]
            self._users[src] = 0
        self._free = list(range(self.n_pages - 1, n - 1, -1))
        self._upload()
        return int(n)

    def free(self):
        for b in (self.pool, self.dev_rows, self.dev_table):
            b.free()


# ------------------------------------------------------------------ layers ----

@dataclass(frozen=True)
class AttnConfig:
    n_q: int
    n_kv: int
    head_dim: int
    rope_dims: int
    interleaved: bool = False
    qk_norm: bool = True
    window: int = 0
    theta: float = 10000.0
    factor: float = 1.0            # rope_frequencies' stretch of a model trained on `trained` positions
    trained: int = 0
    eps: float = 1e-6

    @property
    def qkv_rows(self):
        return (self.n_q + 2 * self.n_kv) * self.head_dim


class DeviceAttention:
    """One layer's attention weights in HBM: norm [D], wqkv bf16 [qkv_rows, D] (q heads, k heads, v
    heads), wo bf16 [D, n_q * head_dim], q_norm and k_norm [head_dim]."""

    def __init__(self, be, acfg, D, norm, wqkv, wo, q_norm, k_norm, rope):
        if D % 128 or acfg.n_q * acfg.head_dim % 128 or acfg.n_q % acfg.n_kv:
            raise ValueError("DeviceAttention: D and n_q * head_dim must be multiples of 128, n_q of n_kv")
        if (q_norm is None or k_norm is None) == acfg.qk_norm:
            raise ValueError("DeviceAttention: q_norm and k_norm belong to a config with qk_norm, and to no other")
        self.be, self.acfg, self.D, self.shape = be, acfg, D, (acfg.n_q, acfg.n_kv, acfg.head_dim, D)
        self.norm, self.wqkv, self.wo, self.q_norm, self.k_norm, self.rope = norm, wqkv, wo, q_norm, k_norm, rope
        self.bufs = [b for b in (norm, wqkv, wo, q_norm, k_norm) if isinstance(b, DevBuf)]

    @classmethod
    def from_host(cls, be, acfg, D, norm, wqkv_bf16, wo_bf16, q_norm, k_norm, rope):
        """norm, q_norm, k_norm f32; wqkv_bf16, wo_bf16: u16; rope: from rope_of"""
        f32 = lambda a: be.upload(np.ascontiguousarray(a, np.float32)) if a is not None else None
        return cls(be, acfg, D, f32(norm), be.router_upload(wqkv_bf16, True), be.router_upload(wo_bf16, True), f32(q_norm),
                   f32(k_norm), rope)

    @classmethod
    def generate(cls, be, acfg, D, seed, layer, rope):
        """seeded weights made on the device: projections N(0, 0.02), norm weights 1 + N(0, 0.02)"""
        def ones(n, tid):
            g = be.alloc(n * 4)
            be.gen_normal(g, n, synth.tensor_seed(seed, layer, tid), WEIGHT_SIGMA)
            w = (np.float32(1.0) + be.d2h(g, (n,), np.float32)).astype(np.float32)
            g.free()
            return be.upload(w)

        def matrix(rows, cols, tid):
            tmp = be.alloc(rows * cols * 2)
            be.gen_bf16(tmp, rows * cols, synth.tensor_seed(seed, layer, tid), WEIGHT_SIGMA)
            out = be.alloc((rows + 3) // 4 * 4 * cols * 2)
            be.check(be.lib.lag_hip_router_chain(int(tmp), int(out), rows, cols, 1), "projection chain")
            be.sync()
            tmp.free()
            return out
        qn, kn = (ones(acfg.head_dim, T_Q_NORM), ones(acfg.head_dim, T_K_NORM)) if acfg.qk_norm else (None, None)
        return cls(be, acfg, D, ones(D, T_ATTN_NORM), matrix(acfg.qkv_rows, D, T_QKV),
                   matrix(D, acfg.n_q * acfg.head_dim, T_O), qn, kn, rope)

    def forward(self, h, xn, S, cache_layer, rows, scratch):
        """h [S, D] += attention of its normalised rows (device; xn [S, D] scratch)"""
        be, a, D = self.be, self.acfg, self.D
        if (cache_layer.n_heads, cache_layer.head_dim) != (a.n_kv, a.head_dim):
            raise ValueError("DeviceAttention: a cache of other heads")
        if S > scratch.S or scratch.shape != self.shape:
            raise ValueError("DeviceAttention: scratch for fewer rows or other heads")
        be.rmsnorm(h, self.norm, xn, S, D, a.eps)
        be.head_argmax(self.wqkv, True, xn, S, D, a.qkv_rows, scratch.qkv)
        be.qk_rope_append(cache_layer, rows, self.rope.desc, scratch.qkv, a.qkv_rows, self.q_norm, self.k_norm, a.eps, a.n_q,
                          scratch.q, S)
        be.attn_paged(cache_layer, rows, scratch.q, a.n_q, 1.0 / math.sqrt(a.head_dim), a.window, scratch.ctx, S)
        be.head_argmax(self.wo, True, scratch.ctx, S, a.n_q * a.head_dim, D, scratch.out)
        be.add(h, scratch.out, S * D)

    def free(self):
        for b in self.bufs:
            b.free()
        self.bufs = []


class Rope:
    """the rotary descriptor of a config, its frequencies on the device"""

    def __init__(self, be, acfg):
        f, factor = rope_frequencies(acfg.rope_dims, acfg.theta, acfg.factor, acfg.trained)
        self.freq = be.upload(f) if acfg.rope_dims else None
        self.desc = be.rope(self.freq, acfg.rope_dims, acfg.interleaved, factor)

    def free(self):
        if self.freq:
            self.freq.free()
            self.freq = None


class AttnScratch:
    """what a layer's attention keeps between its calls, for up to S rows (the layers of a stack share it)"""

    def __init__(self, be, acfg, D, S):
        self.S, self.shape = S, (acfg.n_q, acfg.n_kv, acfg.head_dim, D)
        heads = acfg.n_q * acfg.head_dim
        self.qkv, self.q, self.ctx, self.out = (be.alloc(4 * S * n) for n in (acfg.qkv_rows, heads, heads, D))

    def free(self):
        for b in (self.qkv, self.q, self.ctx, self.out):
            b.free()

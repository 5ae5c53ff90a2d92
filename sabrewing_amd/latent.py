"""Latent attention as a stack's layers use it: a token's keys and values of all heads come from one vector
of `rank` values, the cell of a paged cache, and one rotary part that the heads share.

    ckv = Wkv . x                        cell: (norm(c), turned r)
    q   = Wq . x, or Wqb . norm(Wqa . x)
    k_t[h] = (Wk[h] c_t, r_t), v_t[h] = Wv[h] c_t, h += Wo . attention

New tokens run in the latent space (`latent_append`, `latent_heads` in, `attn_latent`, `latent_heads` out); a prompt, where that would
cost each of its rows products of `rank` values a token, with keys and values made from its latents once
(`attn_latent_prompt`).  Parity unpinned: the reference's engines keep this half on the CPU.
"""
import math
from dataclasses import dataclass

import numpy as np

from . import synth
from .attention import PagedCache
from .backend import DevBuf, KV_TYPES
from .configs import WEIGHT_SIGMA

T_L_NORM, T_L_KV, T_L_KV_NORM, T_L_QA, T_L_Q_NORM, T_L_Q, T_L_K, T_L_V, T_L_O = range(21, 30)


@dataclass(frozen=True)
class LatentConfig:
    n_heads: int
    rank: int                      # values of a latent
    nope: int                      # values of a head's query and key that are not turned
    rope_dims: int
    v_dim: int                     # values of a head's output
    q_rank: int = 0                # queries come through so many values (0: straight from the row)
    interleaved: bool = False
    theta: float = 10000.0
    factor: float = 1.0            # rope_frequencies' stretch of a model trained on `trained` positions
    trained: int = 0
    eps: float = 1e-6

    @property
    def q_dim(self):
        return self.nope + self.rope_dims

    @property
    def cell(self):
        return self.rank + self.rope_dims


class LatentPrompt:
    """the n rows of a prompt: `rows` for appending, where its sequence's pages are listed, its first position; of a cache's
    prompt(), the cache and its rows_made"""

    def __init__(self, rows, pages, n_pages, start, n, cache=None):
        self.rows, self.pages, self.n_pages, self.start, self.n, self.cache = rows, pages, n_pages, start, n, cache
        self.rows_made = cache.rows_made if cache is not None else 0


class LatentCache(PagedCache):
    """Latents of many sequences in pages, with PagedCache's sequences (open, fork, truncate, rows, ...).  A cell is `rank + rope_dims`
    16-bit values, its room whole 128 bytes."""

    def __init__(self, be, n_layers, n_pages, page_size, rank, rope_dims, kind="bf16", max_seqs=64, max_len=None, max_rows=None):
        self.rank, self.rope_dims, self.kind = rank, rope_dims, kind
        if min(n_layers, n_pages, page_size, max_seqs) < 1 or page_size & (page_size - 1) or not 8 <= page_size <= 4096:
            raise ValueError("LatentCache: sizes must be positive, page_size a power of two from 8 to 4096")
        if rank not in (128, 256, 384, 512) or rope_dims not in (0, 16, 32, 48, 64) or kind not in ("bf16", "f16"):
            raise ValueError("LatentCache: rank 128, 256, 384 or 512, rope_dims a multiple of 16 up to 64, bf16 or f16")
        self._sizes(be, n_layers, n_pages, page_size, max_seqs, max_len, max_rows)
        cell = (rank + rope_dims + 63) // 64 * 64
        one = n_pages * page_size * cell * 2
        self.pool = be.alloc(n_layers * one)
        base = int(self.pool)
        self.layers = [be.latent_cache(base + l * one, kind, n_pages, page_size, rank, rope_dims, (page_size * cell, cell)) for l in range(n_layers)]
        # pages are copied as those of a cache whose k and v are the cells' halves
        self.copied = be.kv_caches([be.kv_cache(base + l * one, base + l * one + cell, kind, n_pages, page_size, cell // 64, 32,
                                                (page_size * cell, 32, cell)) for l in range(n_layers)])
        self._sequences()

    def prompt(self, seq, n):
        """rows((seq, n)) for a step that takes a prompt's keys and values from its latents once: (LatentPrompt, n)"""
        start = self.length(seq)
        rows, total = self.rows([(seq, n)])
        return LatentPrompt(rows, int(self.dev_table) + 4 * seq * self.max_pages, len(self._pages[seq]), start, n, self), total


class DeviceLatentAttention:
    """One layer's weights in HBM: norm [D], wkv bf16 [rank + rope_dims, D], kv_norm [rank], wq bf16 [n_heads * (nope + rope_dims), D] or, with
    q_rank, wqa [q_rank, D], q_norm [q_rank] and wq [.., q_rank]; wk [n_heads][nope][rank] and its transposed heads wkt, wv [n_heads][v_dim][rank] in the
    cache's type; wo bf16 [D, n_heads * v_dim]."""

    def __init__(self, be, acfg, D, norm, wkv, kv_norm, wqa, q_norm, wq, wk, wkt, wv, wo, rope, kind="bf16"):
        if D % 128 or acfg.n_heads * acfg.v_dim % 128 or acfg.q_rank % 128 or acfg.nope % 32 or acfg.v_dim % 32:
            raise ValueError("DeviceLatentAttention: D, q_rank and n_heads * v_dim must be multiples of 128, nope and v_dim of 32")
        if any((w is not None) != bool(acfg.q_rank) for w in (wqa, q_norm)):
            raise ValueError("DeviceLatentAttention: wqa and q_norm belong to a config with q_rank, and to no other")
        self.be, self.acfg, self.D, self.kind, self.rope, self.shape = be, acfg, D, kind, rope, (acfg, D)
        self.norm, self.wkv, self.kv_norm, self.wqa, self.q_norm, self.wq = norm, wkv, kv_norm, wqa, q_norm, wq
        self.wk, self.wkt, self.wv, self.wo = wk, wkt, wv, wo
        self.bufs = [b for b in (norm, wkv, kv_norm, wqa, q_norm, wq, wk, wkt, wv, wo) if isinstance(b, DevBuf)]

    @classmethod
    def from_host(cls, be, acfg, D, norm, wkv, kv_norm, wqa, q_norm, wq, wk, wv, wo, rope, kind="bf16"):
        """norm, kv_norm, q_norm f32; the rest u16: bf16, but wk [n_heads, nope, rank] and wv [n_heads, v_dim, rank] of `kind`"""
        f32 = lambda a: be.upload(np.ascontiguousarray(a, np.float32)) if a is not None else None
        m = lambda a: be.router_upload(a, True) if a is not None else None
        return cls(be, acfg, D, f32(norm), m(wkv), f32(kv_norm), m(wqa), f32(q_norm), m(wq), be.upload(np.ascontiguousarray(wk)),
                   be.upload(np.ascontiguousarray(wk.transpose(0, 2, 1))), be.upload(np.ascontiguousarray(wv)), m(wo), rope, kind)

    @classmethod
    def generate(cls, be, acfg, D, seed, layer, rope):
        """seeded weights (for a bf16 cache): matrices N(0, 0.02), norm weights 1 + N(0, 0.02)"""
        def ones(n, tid):
            g = be.alloc(n * 4)
            be.gen_normal(g, n, synth.tensor_seed(seed, layer, tid), WEIGHT_SIGMA)
            w = (np.float32(1.0) + be.d2h(g, (n,), np.float32)).astype(np.float32)
            g.free()
            return w

        def matrix(shape, tid):
            n = int(np.prod(shape))
            tmp = be.alloc(n * 2)
            be.gen_bf16(tmp, n, synth.tensor_seed(seed, layer, tid), WEIGHT_SIGMA)
            w = be.d2h(tmp, shape, np.uint16)
            tmp.free()
            return w
        a, q = acfg, acfg.q_rank
        return cls.from_host(be, a, D, ones(D, T_L_NORM), matrix((a.cell, D), T_L_KV), ones(a.rank, T_L_KV_NORM), matrix((q, D), T_L_QA) if q else None,
                             ones(q, T_L_Q_NORM) if q else None, matrix((a.n_heads * a.q_dim, q or D), T_L_Q), matrix((a.n_heads, a.nope, a.rank), T_L_K),
                             matrix((a.n_heads, a.v_dim, a.rank), T_L_V), matrix((D, a.n_heads * a.v_dim), T_L_O), rope)

    def forward(self, h, xn, S, cache_layer, rows, scratch):
        """h [S, D] += attention of its normalised rows (device; xn [S, D] scratch); rows: a cache's rows(), or its prompt()"""
        be, a, D, t, H = self.be, self.acfg, self.D, scratch, self.acfg.n_heads
        if (cache_layer.rank, cache_layer.rope_dims, cache_layer.type) != (a.rank, a.rope_dims, KV_TYPES[self.kind]):
            raise ValueError("DeviceLatentAttention: a cache of other latents")
        if S > t.S or t.shape != self.shape:
            raise ValueError("DeviceLatentAttention: scratch for fewer rows or other heads")
        if isinstance(rows, LatentPrompt) and S != rows.n:
            raise ValueError("DeviceLatentAttention: a prompt of another number of rows")
        be.rmsnorm(h, self.norm, xn, S, D, a.eps)
        be.head_argmax(self.wkv, True, xn, S, D, a.cell, t.ckv)
        if a.q_rank:
            be.head_argmax(self.wqa, True, xn, S, D, a.q_rank, t.qa)
            be.rmsnorm(t.qa, self.q_norm, t.qn, S, a.q_rank, a.eps)
        be.head_argmax(self.wq, True, t.qn if a.q_rank else xn, S, a.q_rank or D, H * a.q_dim, t.q)
        prompt = rows if isinstance(rows, LatentPrompt) else None
        # heads of queries: (nope, rope) of the expanded form, (latent, rope) of the absorbed one
        n = a.q_dim if prompt else a.cell
        nope = be.heads(t.heads, H * a.q_dim, a.q_dim) if prompt else be.heads(t.plain, H * a.nope, a.nope)
        turned = be.heads(int(t.heads) + 2 * (n - a.rope_dims), H * n, n)
        be.latent_append(cache_layer, prompt.rows if prompt else rows, self.rope.desc if a.rope_dims else None, t.ckv, a.cell, self.kv_norm, a.eps, t.q,
                         H * a.q_dim, H, a.nope, nope, turned, S)
        scale = 1.0 / math.sqrt(a.q_dim)
        if prompt:
            be.attn_latent_prompt(cache_layer, prompt.pages, prompt.n_pages, prompt.start, self.wk, self.wv, a.nope, a.v_dim, t.heads, H, scale, t.ctx,
                                  True, S)
        else:
            be.latent_heads(self.kind, nope, self.wkt, H, a.nope, a.rank, be.heads(t.heads, H * n, n), False, S)
            be.attn_latent(cache_layer, rows, t.heads, H, scale, t.mixed, S)
            be.latent_heads(self.kind, be.heads(t.mixed, H * a.rank, a.rank), self.wv, H, a.rank, a.v_dim, be.heads(t.ctx, H * a.v_dim, a.v_dim), True, S)
        be.head_argmax(self.wo, True, t.ctx, S, H * a.v_dim, D, t.out)
        be.add(h, t.out, S * D)

    def free(self):
        for b in self.bufs:
            b.free()
        self.bufs = []


class LatentScratch:
    """what a layer's latent attention keeps between its calls, for up to S rows (the layers of a stack share it)"""

    def __init__(self, be, acfg, D, S):
        a, H = acfg, acfg.n_heads
        self.S, self.shape = S, (acfg, D)
        self.ckv, self.q, self.ctx, self.out = (be.alloc(4 * S * n) for n in (a.cell, H * a.q_dim, H * a.v_dim, D))
        self.plain, self.heads, self.mixed = (be.alloc(2 * S * H * n) for n in (a.nope, max(a.cell, a.q_dim), a.rank))
        self.qa, self.qn = (be.alloc(4 * S * a.q_rank) if a.q_rank else None for _ in range(2))

    def free(self):
        for b in (self.ckv, self.q, self.ctx, self.out, self.plain, self.heads, self.mixed, self.qa, self.qn):
            if b:
                b.free()

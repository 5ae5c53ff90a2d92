"""Attention over trees of drafted tokens and over caches of latent vectors, as timed cases.

A case is a dict of plain values.  `op` says which operator it is:

  tree     `Backend.attn_tree`: the nodes of each sequence's tree of drafted tokens against its cells
           and their ancestors'
  commit   `Backend.tree_commit`: the accepted path of each tree found, its cells moved together in every
           layer's cache
  append   `Backend.latent_append`: a token's latent vector normalised, its rotary part turned, both
           written into the paged cache of latents, its query heads turned
  heads    `Backend.latent_heads`: a product for each head, into the latent space or out of it
  latent   `Backend.attn_latent`: one new token of each row against its sequence's latents (the absorbed form)
  prompt   `Backend.attn_latent_prompt`: a chunk of a prompt against keys and values expanded from the
           latents

`run` computes the operator in plain torch where `own` is false, and calls the framework where it is
true.  Both leave their results in the state's own buffers.
"""
import math

import numpy as np
import torch

own = False
_backend = []

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6


def _be():
    if not _backend:
        from sabrewing_amd.backend import Backend
        _backend.append(Backend(0))
    return _backend[0]


# ------------------------------------------------------------------ cases ----

def listed():
    return [
        # one stream with eight drafted tokens, a short context: the smallest call
        dict(name="tree_1x700", op="tree", trees=1, nodes=8, Hq=32, Hkv=8, dh=128, type="bf16", page=16, ctx=700, short=700,
             window=0, ragged=False),
        # a server's batch, every stream at another length and with a tree of its own
        dict(name="tree_16x12000", op="tree", trees=16, nodes=26, Hq=32, Hkv=8, dh=128, type="bf16", page=64, ctx=12000,
             short=500, window=0, ragged=True),
        # one stream's accepted tokens, 48 layers
        dict(name="commit_1", op="commit", trees=1, nodes=16, layers=48, Hkv=8, dh=128, type="bf16", page=16),
        # a batch's
        dict(name="commit_32", op="commit", trees=32, nodes=64, layers=48, Hkv=8, dh=128, type="bf16", page=64),
        # a decode step of one stream, heads as one of eight cards would hold them
        dict(name="append_1", op="append", S=1, seqs=1, H=16, nope=128, rank=512, rope=64, interleaved=True, norm=True,
             type="bf16", page=64, ctx=32768, pad=0),
        # a chunk of two streams' prompts, all heads
        dict(name="append_1024", op="append", S=1024, seqs=2, H=128, nope=128, rank=512, rope=64, interleaved=True, norm=True,
             type="bf16", page=64, ctx=65536, pad=0),
        # queries of one token into the latent space
        dict(name="heads_1", op="heads", S=1, H=128, n_in=128, n_out=512, type="bf16", f32=False),
        # a batch's latents back to value heads, for the output projection
        dict(name="heads_64", op="heads", S=64, H=128, n_in=512, n_out=128, type="bf16", f32=True),
        # one stream, few heads, a short context
        dict(name="latent_1x1500", op="latent", S=1, H=16, rank=512, rope=64, type="bf16", page=64, ctx=1500, short=1500, pad=0),
        # a server's batch with a free place, all heads, every stream at another length
        dict(name="latent_32x16384", op="latent", S=32, H=128, rank=512, rope=64, type="bf16", page=64, ctx=16384, short=100, pad=1),
        # a short prompt from its beginning
        dict(name="prompt_300", op="prompt", S=300, start=0, H=16, nope=128, v=128, rank=512, rope=64, type="bf16", page=64, f32=False),
        # a chunk far into a document
        dict(name="prompt_2048", op="prompt", S=2048, start=6000, H=32, nope=128, v=128, rank=512, rope=64, type="bf16", page=64,
             f32=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    op = rng.choice(["tree"] * 4 + ["commit"] * 2 + ["append"] * 2 + ["heads"] * 2 + ["latent"] * 4 + ["prompt"] * 3)
    kind, page = rng.choice(["bf16", "bf16", "f16"]), 1 << rng.randint(3, 8)
    if op in ("tree", "commit"):
        Hkv, dh = rng.choice([1, 2, 3, 4, 8, 8, 8, 12]), rng.choice([32, 64, 96, 128, 128, 128, 160, 192, 256])
        kind = rng.choice(["bf16", "bf16", "bf16", "f16", "f16", "f32"])
        nodes = _log_int(rng, 1, 64)
        if op == "commit":
            layers = _log_int(rng, 1, 60)
            trees = _log_int(rng, 1, max(1, min(64, 48 * 32 * 64 * 2048 // (layers * (nodes + page) * Hkv * dh * (4 if kind == "f32" else 2)))))
            return dict(op="commit", trees=trees, nodes=nodes, layers=layers, Hkv=Hkv, dh=dh, type=kind, page=page)
        G = rng.choice([1, 2, 3, 4, 4, 5, 6, 7, 8, 8, 12, 16])
        G = min(G, 64 // Hkv)
        trees = _log_int(rng, 1, 48)
        # no more cells than the batch's, and no more work
        cells = min(100000 * 1024 * 2 // (Hkv * dh * (4 if kind == "f32" else 2)),
                    100000 * 26 * 32 * 128 // (nodes * Hkv * G * dh * (6 if kind == "f32" else 1)))
        ctx = _log_int(rng, 1, max(2, min(60000, cells // trees)))
        return dict(op="tree", trees=trees, nodes=nodes, Hq=Hkv * G, Hkv=Hkv, dh=dh, type=kind, page=page, ctx=ctx,
                    short=rng.randint(0, ctx), window=0 if rng.random() < 0.75 else rng.randint(1, 2 * ctx + 8), ragged=rng.random() < 0.7)
    if op == "heads":
        H, n_in, n_out = _log_int(rng, 1, 128), 32 * rng.randint(1, 16), 32 * rng.randint(1, 16)
        return dict(op="heads", S=_log_int(rng, 1, 300), H=H, n_in=n_in, n_out=n_out, type=kind, f32=rng.random() < 0.5)
    H, rank, rope = _log_int(rng, 1, 128), rng.choice([128, 256, 384, 512, 512, 512]), rng.choice([32, 64, 64, 64])
    if op == "append":
        S = _log_int(rng, 1, 1024)
        return dict(op="append", S=S, seqs=rng.randint(1, 4) if S > 4 and rng.random() < 0.5 else S, H=H, nope=rng.choice([64, 96, 128, 128, 192]),
                    rank=rank, rope=rope, interleaved=rng.random() < 0.6, norm=rng.random() < 0.8, type=kind, page=page,
                    ctx=max(_log_int(rng, 64, 65536), 2 * S), pad=rng.randint(0, min(2, S - 1)))
    if op == "latent":
        S = _log_int(rng, 1, 96)
        ctx = _log_int(rng, 1, max(2, min(65536, 260000 // S)))
        return dict(op="latent", S=S, H=H, rank=rank, rope=rope, type=kind, page=page, ctx=ctx, short=rng.randint(1, ctx),
                    pad=rng.randint(0, min(2, S - 1)))
    S, H = _log_int(rng, 1, 2048), _log_int(rng, 1, 32)
    start = 0 if rng.random() < 0.4 else rng.randint(0, 6000)
    return dict(op="prompt", S=S, start=start, H=H, nope=rng.choice([64, 128, 128, 96]), v=rng.choice([64, 128, 128, 96]), rank=rank,
                rope=rope, type=kind, page=page, f32=False)


# ----------------------------------------------------------------- inputs ----

class _Dev:
    """A torch tensor handed to the framework as device memory."""

    def __init__(self, t, at=0):
        self.t, self.at = t, at * t.element_size()

    def __int__(self):
        return self.t.data_ptr() + self.at


class _State:
    def __init__(self, **kw):
        self.__dict__.update(kw)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _pool(g, *shape, dtype):
    """N(0, 1) in the cache's type"""
    t = torch.empty(*shape, dtype=dtype, device="cuda")
    for part in t.view(-1).split(1 << 27):
        part.copy_(_randn(g, part.numel()))
    return t


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


def _tables(r, need, page):
    """page tables of streams of `need` tokens, their pages in no order: table [streams, pages of the longest], all pages"""
    pages = [-(-int(n) // page) for n in need]
    ids = r.permutation(sum(pages) + 2)
    table = np.zeros((len(need), max(1, max(pages))), np.int32)
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = ids[at:at + n]
        at += n
    return table, sum(pages) + 2


def _tree(r, n):
    """parents of a drafted tree's n nodes in order of depth: a few likely chains with branches"""
    parent = np.full(n, -1)
    width = int(r.integers(1, 5))
    for j in range(1, n):
        parent[j] = max(0, (j - 1) // 2 if r.random() < 0.3 else j - int(r.integers(1, width + 1)))
    return np.maximum.accumulate(parent)


def prepare(case, seed):
    c, g, r = case, _gen(seed), np.random.default_rng([int(seed), 29])
    s = _State(op=c["op"], c=c)
    if c["op"] in ("tree", "commit"):
        n, top = c["trees"], c["nodes"]
        # (the trees' sizes are the case's own: outputs of one shape whatever the seed)
        count = np.random.default_rng([n, top]).integers(max(1, top // 3), top + 1, n) if c.get("ragged", True) else np.full(n, top)
        count[0] = top
        first = np.concatenate([[0], np.cumsum(count)])
        parents = [_tree(r, int(k)) for k in count]
        s.rows, s.first, s.parent = int(first[-1]), _i32(first), _i32(np.concatenate(parents))
        s.owner, s.index = _i32(np.repeat(np.arange(n), count)), _i32(np.arange(s.rows) - np.repeat(first[:-1], count))
    if c["op"] == "tree":
        base = r.integers(c["short"], c["ctx"] + 1, n)
        base[r.integers(0, n)] = c["ctx"]
        sees, depth = np.zeros(s.rows, np.uint64), np.zeros(s.rows, np.int64)
        for f, p in zip(first, parents):
            for j in range(len(p)):
                sees[f + j] = np.uint64(1 << j) | (sees[f + p[j]] if j else np.uint64(0))
                depth[f + j] = depth[f + p[j]] + 1 if j else 0
        table, s.n_pages = _tables(r, base + count, c["page"])
        s.kv = [_pool(g, s.n_pages, c["Hkv"], c["page"], c["dh"], dtype=TYPES[c["type"]]) for _ in range(2)]
        s.q = 1.5 * _randn(g, s.rows, c["Hq"], c["dh"])
        s.out = torch.zeros_like(s.q)
        s.base, s.table, s.pos = _i32(base), _i32(table), _i32(np.repeat(base, count) + depth)
        s.sees = torch.from_numpy(sees.view(np.int64)).cuda()
        s.scale = 1.0 / math.sqrt(c["dh"])
    elif c["op"] == "commit":
        base = r.integers(0, c["page"], n)
        table, _ = _tables(r, base + count, c["page"])
        s.n_pages = int(sum(-(-(count + c["page"] - 1) // c["page"]))) + 2         # (as many wherever the trees begin)
        s.kv = _pool(g, 2, c["layers"], s.n_pages, c["Hkv"], c["page"], c["dh"], dtype=TYPES[c["type"]])
        # every node drafts its own index; along one path from the root the pick is the next node, else one nobody drafted.
        # The path ends before a cell of it would be written over, so that a pass can be repeated.
        draft, tok = np.arange(s.rows) - np.repeat(first[:-1], count), np.full(s.rows, 1000)
        for f, p in zip(first, parents):
            path = [0]
            while True:
                kids = np.flatnonzero((p == path[-1]) & (np.arange(len(p)) > path[-1]))
                if not len(kids):
                    break
                path.append(int(r.choice(kids)))
                moved = [x for i, x in enumerate(path) if x != i]
                if set(moved) & set(range(len(path))):
                    path.pop()
                    break
            for a, b in zip(path, path[1:]):
                tok[f + a] = b
        s.base, s.table, s.draft, s.tok = _i32(base), _i32(table), _i32(draft), _i32(tok)
        s.sees = torch.zeros(s.rows, dtype=torch.int64, device="cuda")
        s.path, s.count, s.next = (torch.full(k, -5, dtype=torch.int32, device="cuda") for k in ((n, top), (n,), (n,)))
    elif c["op"] == "append":
        S, width = c["S"], c["rank"] + c["rope"]
        if c["seqs"] == S:                        # a decode step: one row of each stream
            pos, seq = r.integers(0, c["ctx"], S), np.arange(S)
        else:                                     # chunks: consecutive positions of a few streams
            seq = np.sort(r.integers(0, c["seqs"], S))
            begin = r.integers(0, c["ctx"] - S + 1, c["seqs"])
            pos = begin[seq] + np.arange(S) - np.searchsorted(seq, seq)
        # the positions before a stream's rows share page 0, so that the cache holds about what is written
        table, at = np.zeros((c["seqs"], -(-c["ctx"] // c["page"])), np.int32), 1
        for q in np.unique(seq):
            a, b = pos[seq == q].min() // c["page"], pos[seq == q].max() // c["page"] + 1
            table[q, a:b] = np.arange(at, at + b - a)
            at += b - a
        s.n_pages = S // c["page"] + 2 * c["seqs"] + 2
        pos[S - c["pad"]:] = -1
        s.ckv, s.qin = _randn(g, S, width), _randn(g, S, c["H"], c["nope"] + c["rope"])
        s.pool = _pool(g, s.n_pages, c["page"], width, dtype=TYPES[c["type"]])
        s.q_nope = torch.zeros(S, c["H"], c["nope"], dtype=TYPES[c["type"]], device="cuda")
        s.q_abs = torch.zeros(S, c["H"], width, dtype=TYPES[c["type"]], device="cuda")        # its first `rank` values are another product's
        s.norm = 1.0 + 0.1 * _randn(g, c["rank"])
        s.freq = torch.from_numpy(1e4 ** (-2.0 * np.arange(c["rope"] // 2) / c["rope"])).cuda()
        s.pos, s.seq, s.table = _i32(pos), _i32(seq), _i32(table)
    elif c["op"] == "heads":
        S, H, t = c["S"], c["H"], TYPES[c["type"]]
        s.x = _randn(g, S, H, c["n_in"]).to(t)
        s.w = (_randn(g, H, c["n_out"], c["n_in"]) / math.sqrt(c["n_in"])).to(t)
        s.y = torch.zeros(S, H, c["n_out"], dtype=torch.float32 if c["f32"] else t, device="cuda")
    elif c["op"] == "latent":
        S, width, t = c["S"], c["rank"] + c["rope"], TYPES[c["type"]]
        length = r.integers(c["short"], c["ctx"] + 1, S)
        length[r.integers(0, S - c["pad"])] = c["ctx"]
        length[S - c["pad"]:] = 0
        table, s.n_pages = _tables(r, length, c["page"])
        s.pool = _pool(g, s.n_pages, c["page"], width, dtype=t)
        s.q = (1.5 * _randn(g, S, c["H"], width)).to(t)
        s.out = torch.zeros(S, c["H"], c["rank"], dtype=t, device="cuda")
        s.pos, s.table = _i32(length - 1), _i32(table)
        s.scale = 1.0 / math.sqrt(width)
    else:
        S, H, T, t = c["S"], c["H"], c["S"] + c["start"], TYPES[c["type"]]
        table, s.n_pages = _tables(r, [T], c["page"])
        s.pool = _pool(g, s.n_pages, c["page"], c["rank"] + c["rope"], dtype=t)
        s.pages = _i32(table[0])
        s.wk, s.wv = ((_randn(g, H, n, c["rank"]) / math.sqrt(c["rank"])).to(t) for n in (c["nope"], c["v"]))
        s.q = (1.5 * _randn(g, S, H, c["nope"] + c["rope"])).to(t)
        s.out = torch.zeros(S, H, c["v"], dtype=torch.float32 if c["f32"] else t, device="cuda")
        s.scale = 1.0 / math.sqrt(c["nope"] + c["rope"])
    if own:
        _handles(s)
    torch.cuda.synchronize()
    return s


def _handles(s):
    """what a program keeps: the caches' and rows' descriptors"""
    be, c = _be(), s.c
    s.be = be
    if s.op in ("tree", "commit"):
        s.trees = be.trees(_Dev(s.first), _Dev(s.base), _Dev(s.sees), _Dev(s.table), c["trees"], c["trees"], s.table.shape[1], c["nodes"],
                           pos_dev=_Dev(s.pos) if s.op == "tree" else None)
    if s.op == "tree":
        s.cache = be.kv_cache(s.kv[0].data_ptr(), s.kv[1].data_ptr(), c["type"], s.n_pages, c["page"], c["Hkv"], c["dh"])
        s.d = _Dev(s.q), _Dev(s.out)
    elif s.op == "commit":
        s.caches = be.kv_caches([be.kv_cache(s.kv[0, i].data_ptr(), s.kv[1, i].data_ptr(), c["type"], s.n_pages, c["page"], c["Hkv"], c["dh"])
                                 for i in range(c["layers"])])
        s.d = tuple(_Dev(t) for t in (s.parent, s.draft, s.tok, s.path, s.count, s.next))
    elif s.op in ("append", "latent"):
        s.cache = be.latent_cache(_Dev(s.pool), c["type"], s.n_pages, c["page"], c["rank"], c["rope"])
        s.rowsd = be.kv_rows(_Dev(s.pos), _Dev(s.table), s.table.shape[0], s.table.shape[1], _Dev(s.seq) if s.op == "append" else None)
        if s.op == "latent":
            s.d = _Dev(s.q), _Dev(s.out)
        else:
            H, width = c["H"], c["rank"] + c["rope"]
            s.rope = be.rope(_Dev(s.freq), c["rope"], c["interleaved"])
            s.to = be.heads(_Dev(s.q_nope), H * c["nope"], c["nope"]), be.heads(_Dev(s.q_abs, c["rank"]), H * width, width)
            s.d = _Dev(s.ckv), _Dev(s.norm) if c["norm"] else None, _Dev(s.qin)
    elif s.op == "heads":
        s.d = (be.heads(_Dev(s.x), c["H"] * c["n_in"], c["n_in"]), _Dev(s.w), be.heads(_Dev(s.y), c["H"] * c["n_out"], c["n_out"]))
    else:
        s.cache = be.latent_cache(_Dev(s.pool), c["type"], s.n_pages, c["page"], c["rank"], c["rope"])
        s.d = tuple(_Dev(t) for t in (s.pages, s.wk, s.wv, s.q, s.out))


# -------------------------------------------------------------------- run ----

def run(s):
    c = s.c
    if s.op == "tree":
        if own:
            s.be.attn_tree(s.cache, s.trees, s.d[0], c["Hq"], s.scale, c["window"], s.d[1], s.rows)
        else:
            _plain_tree(s)
        return s.out
    if s.op == "commit":
        if own:
            s.be.tree_commit(s.caches, s.trees, *s.d, s.rows)
        else:
            _plain_commit(s)
        return {"kv": s.kv, "path": s.path, "count": s.count, "next": s.next}
    if s.op == "append":
        if own:
            s.be.latent_append(s.cache, s.rowsd, s.rope, s.d[0], c["rank"] + c["rope"], s.d[1], EPS, s.d[2], c["H"] * (c["nope"] + c["rope"]),
                               c["H"], c["nope"], s.to[0], s.to[1], c["S"])
        else:
            _plain_append(s)
        return {"cells": s.pool, "q_nope": s.q_nope, "q_abs": s.q_abs}
    if s.op == "heads":
        if own:
            s.be.latent_heads(c["type"], s.d[0], s.d[1], c["H"], c["n_in"], c["n_out"], s.d[2], c["f32"], c["S"])
        else:
            x, w = s.x.float().transpose(0, 1).contiguous(), s.w.float().transpose(1, 2).contiguous()
            s.y.copy_(torch.matmul(x, w).transpose(0, 1))
        return s.y
    if s.op == "latent":
        if own:
            s.be.attn_latent(s.cache, s.rowsd, s.d[0], c["H"], s.scale, s.d[1], c["S"])
        else:
            _plain_latent(s)
        return s.out
    if own:
        s.be.attn_latent_prompt(s.cache, s.d[0], s.pages.shape[0], c["start"], s.d[1], s.d[2], c["nope"], c["v"], s.d[3], c["H"], s.scale,
                                s.d[4], c["f32"], c["S"])
    else:
        _plain_prompt(s)
    return s.out


def _softmax(score, seen):
    score = score.masked_fill(~seen, -math.inf)
    e = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-3e38))
    return e / e.sum(-1, keepdim=True).clamp(min=1e-38)


def _plain_tree(s):
    c = s.c
    n, top, Hq, Hkv, dh, P = c["trees"], c["nodes"], c["Hq"], c["Hkv"], c["dh"], c["page"]
    owner, index = s.owner.long(), s.index.long()
    q = torch.zeros(n, top, Hq, dh, device="cuda")
    q[owner, index] = s.q
    sees, pos = (torch.zeros(n, top, dtype=torch.int64, device="cuda") for _ in range(2))
    sees[owner, index] = s.sees
    pos[owner, index] = s.pos.long()
    t = torch.arange(min(s.table.shape[1] * P, c["ctx"] + top), device="cuda")
    page = s.table.long()[:, t // P]
    k, v = (p[page, :, t % P].float().permute(0, 2, 1, 3).contiguous() for p in s.kv)          # [n, Hkv, t, dh]
    j = (t - s.base.long()[:, None]).clamp(max=63)                                             # the node whose cell t is
    seen = (j[:, None] >= 0) & ((sees[:, :, None] >> j[:, None].clamp(min=0)) & 1).bool() & (t < s.base.long()[:, None] + top)[:, None]
    old = (j < 0)[:, None] & ((t > pos[:, :, None] - c["window"]) if c["window"] else torch.ones_like(t, dtype=torch.bool))
    seen = (seen | old)[:, None, :, None]                                                      # [n, 1, node, 1, t]
    q = q.view(n, top, Hkv, Hq // Hkv, dh).transpose(1, 2).reshape(n, Hkv, -1, dh).contiguous()
    score = torch.matmul(q, k.transpose(2, 3).contiguous()).view(n, Hkv, top, Hq // Hkv, -1) * s.scale
    p = _softmax(score, seen).view(n, Hkv, -1, t.numel())
    o = torch.matmul(p, v).view(n, Hkv, top, Hq // Hkv, dh).transpose(1, 2).reshape(n, top, Hq, dh)
    s.out.copy_(o[owner, index])


def _plain_commit(s):
    c = s.c
    n, top, P = c["trees"], c["nodes"], c["page"]
    owner, index = s.owner.long(), s.index.long()
    parent, draft, tok = (torch.full((n, top), -9, dtype=torch.int64, device="cuda") for _ in range(3))
    parent[owner, index], draft[owner, index], tok[owner, index] = s.parent.long(), s.draft.long(), s.tok.long()
    # a node is accepted if its parent's pick drafted it and its parent is; nodes come after their parents
    up = parent.clamp(min=0)
    good = (parent >= 0) & (draft == tok.gather(1, up))
    good[:, 0] = True
    at = torch.arange(top, device="cuda").expand(n, top)
    up = torch.where(parent >= 0, up, at)
    for _ in range(max(1, math.ceil(math.log2(top + 1)))):       # a node's ancestors by doubling
        good = good & good.gather(1, up)
        up = up.gather(1, up)
    count = good.sum(1)
    path = torch.where(good, at, 10 ** 6).sort(1).values
    live = at < count[:, None]
    s.path.copy_(torch.where(live, path, -1))
    s.count.copy_(count)
    s.next.copy_(tok.gather(1, path.gather(1, (count - 1)[:, None])).squeeze(1))
    b = s.base.long()[:, None]
    src, dst = (b + path)[live], (b + at)[live]
    row = torch.arange(n, device="cuda")[:, None].expand(n, top)[live]
    table = s.table.long()
    s.kv[:, :, table[row, dst // P], :, dst % P] = s.kv[:, :, table[row, src // P], :, src % P].clone()


def _plain_append(s):
    c = s.c
    rank, rd, live = c["rank"], c["rope"], c["S"] - c["pad"]
    lat = s.ckv[:, :rank]
    if c["norm"]:
        lat = lat * torch.rsqrt((lat * lat).mean(-1, keepdim=True) + EPS) * s.norm
    angle = s.pos.double()[:, None] * s.freq
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    x = torch.cat([s.ckv[:, None, rank:], s.qin[..., c["nope"]:]], 1)
    y = x.clone()
    if c["interleaved"]:
        a, b = x[..., 0::2], x[..., 1::2]
        y[..., 0::2], y[..., 1::2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :rd // 2], x[..., rd // 2:]
        y[..., :rd // 2], y[..., rd // 2:] = a * cos - b * sin, b * cos + a * sin
    pos, seq = s.pos[:live].long(), s.seq[:live].long()
    s.q_nope[:live] = s.qin[:live, :, :c["nope"]].to(s.q_nope.dtype)
    s.q_abs[:live, :, rank:] = y[:live, 1:].to(s.q_abs.dtype)
    s.pool[s.table[seq, pos // c["page"]].long(), pos % c["page"]] = torch.cat([lat, y[:, 0]], 1)[:live].to(s.pool.dtype)


def _plain_latent(s):
    c = s.c
    P, rank = c["page"], c["rank"]
    t = torch.arange(c["ctx"], device="cuda")
    cells = s.pool[s.table.long()[:, t // P], t % P].float()                                   # [S, t, width]
    score = torch.matmul(s.q.float(), cells.transpose(1, 2).contiguous()) * s.scale
    p = _softmax(score, (t <= s.pos.long()[:, None])[:, None])
    s.out.copy_(torch.matmul(p, cells[..., :rank].contiguous()))


def _plain_prompt(s):
    c = s.c
    T, P, rank, nope = c["S"] + c["start"], c["page"], c["rank"], c["nope"]
    t = torch.arange(T, device="cuda")
    cells = s.pool[s.pages.long()[t // P], t % P].float()
    lat, turned = cells[:, :rank].contiguous(), cells[:, rank:]
    k = torch.matmul(lat, s.wk.float().transpose(1, 2).contiguous())                          # [H, T, nope]
    v = torch.matmul(lat, s.wv.float().transpose(1, 2).contiguous())
    q = s.q.float().transpose(0, 1)
    score = torch.matmul(q[..., :nope].contiguous(), k.transpose(1, 2).contiguous())
    score += torch.matmul(q[..., nope:].contiguous(), turned.T.contiguous())
    score *= s.scale
    p = _softmax(score, t <= c["start"] + torch.arange(c["S"], device="cuda")[:, None])
    s.out.copy_(torch.matmul(p, v).transpose(0, 1))


# ------------------------------------------------------------------- work ----

def work(case):
    c = case
    if c["op"] == "heads":
        S, H, a, b = c["S"], c["H"], c["n_in"], c["n_out"]
        return {"bytes": H * (2 * a * b + S * (2 * a + (4 if c["f32"] else 2) * b)), "flops": 2 * S * H * a * b}
    if c["op"] in ("tree", "commit"):
        b, top = 4 if c["type"] == "f32" else 2, c["nodes"]
        n = top if not c.get("ragged", True) else (top + max(1, top // 3)) / 2
        if c["op"] == "commit":
            depth = max(0.0, min(3.0, n / 4))                  # cells that move, about
            return {"bytes": c["trees"] * (4 * 4 * n + depth * 4 * c["layers"] * c["Hkv"] * c["dh"] * b), "flops": c["trees"] * n}
        w = c["window"] or c["ctx"]
        mean = (min(c["short"], w) + min(c["ctx"], w)) / 2 * (c["trees"] - 1) + min(c["ctx"], w)
        cells = mean + c["trees"] * n
        return {"bytes": cells * 2 * c["Hkv"] * c["dh"] * b + 8 * c["trees"] * n * c["Hq"] * c["dh"], "flops": 4 * cells * n * c["Hq"] * c["dh"]}
    width = c["rank"] + c["rope"]
    if c["op"] == "append":
        S = c["S"] - c["pad"]
        return {"bytes": S * 6 * (width + c["H"] * (c["nope"] + c["rope"])), "flops": S * (6 * c["rank"] + 6 * c["rope"] * (c["H"] + 1))}
    if c["op"] == "latent":
        S = c["S"] - c["pad"]
        cells = c["ctx"] + (S - 1) * (c["ctx"] + c["short"]) / 2
        return {"bytes": 2 * cells * width + 2 * S * c["H"] * (width + c["rank"]), "flops": 2 * cells * c["H"] * (width + c["rank"])}
    S, T, H = c["S"], c["S"] + c["start"], c["H"]
    pairs = S * c["start"] + S * (S + 1) / 2
    return {"bytes": 2 * T * width + 2 * H * (c["nope"] + c["v"]) * c["rank"] + S * H * (2 * (c["nope"] + c["rope"]) + 2 * c["v"]),
            "flops": 2 * T * c["rank"] * H * (c["nope"] + c["v"]) + 2 * pairs * H * (c["nope"] + c["rope"] + c["v"])}


# ------------------------------------------------------------------ exact ----

def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    return {"tree": _exact_tree, "commit": _exact_commit, "append": _exact_append, "heads": _exact_heads, "latent": _exact_latent,
            "prompt": _exact_prompt}[case["op"]](s)


def _exact_tree(s):
    c = s.c
    P, G = c["page"], c["Hq"] // c["Hkv"]
    out = torch.zeros(s.rows, c["Hq"], c["dh"], dtype=torch.float64, device="cuda")
    first, base, sees, pos = (t.tolist() for t in (s.first, s.base, s.sees, s.pos))
    for i in range(c["trees"]):
        a, b = first[i], first[i + 1]
        n = base[i] + b - a
        t = torch.arange(n, device="cuda")
        cells = (s.table[i, t // P].long(), t % P)
        see = torch.zeros(b - a, n, dtype=torch.bool, device="cuda")
        for r in range(a, b):
            see[r - a, max(0, pos[r] - c["window"] + 1) if c["window"] else 0:base[i]] = True
            for j in range(b - a):
                see[r - a, base[i] + j] = bool(sees[r] >> j & 1)
        for h in range(c["Hkv"]):
            k, v = (p[cells[0], h, cells[1]].double() for p in s.kv)
            x = (s.q[a:b, h * G:(h + 1) * G].double() @ k.T.contiguous()) * s.scale             # [node, G, t]
            x = torch.where(see[:, None], x, torch.tensor(-math.inf, dtype=torch.float64, device="cuda"))
            out[a:b, h * G:(h + 1) * G] = torch.softmax(x, -1).nan_to_num(0.0) @ v
    return out


def _exact_commit(s):
    c, P = s.c, s.c["page"]
    first, base, parent, draft, tok = (t.tolist() for t in (s.first, s.base, s.parent, s.draft, s.tok))
    path, count, nxt = np.full((c["trees"], c["nodes"]), -1, np.int32), np.zeros(c["trees"], np.int32), np.zeros(c["trees"], np.int32)
    table = s.table.tolist()
    for i in range(c["trees"]):
        a, way = first[i], [0]
        while True:
            kid = [j for j in range(way[-1] + 1, first[i + 1] - a) if parent[a + j] == way[-1] and draft[a + j] == tok[a + way[-1]]]
            if not kid:
                break
            way.append(kid[0])
        path[i, :len(way)], count[i], nxt[i] = way, len(way), tok[a + way[-1]]
        for to, at in enumerate(way):
            x, y = base[i] + at, base[i] + to
            s.kv[:, :, table[i][y // P], :, y % P].copy_(s.kv[:, :, table[i][x // P], :, x % P].clone())
    return {"kv": s.kv, "path": path, "count": count, "next": nxt}


def _exact_append(s):
    """pair by pair, as a product of complex numbers"""
    c, rank, half = s.c, s.c["rank"], s.c["rope"] // 2
    lat, q = s.ckv.double(), s.qin.double()
    cell = lat[:, :rank]
    if c["norm"]:
        cell = cell / ((cell * cell).sum(-1, keepdim=True) / rank + EPS).sqrt() * s.norm.double()
    turn = torch.polar(torch.ones(c["S"], half, dtype=torch.float64, device="cuda"), s.pos.double()[:, None] * s.freq)
    i = torch.arange(half, device="cuda")
    a, b = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half)
    for h, z in ((lat[:, rank:], turn), (q[..., c["nope"]:], turn[:, None])):
        y = torch.complex(h[..., a], h[..., b]) * z
        h[..., a], h[..., b] = y.real, y.imag
    pool, nope, ab = s.pool.double(), s.q_nope.double(), s.q_abs.double()
    for row, (p, n) in enumerate(zip(s.pos.tolist(), s.seq.tolist())):
        if p >= 0:
            nope[row], ab[row, :, rank:] = q[row, :, :c["nope"]], q[row, :, c["nope"]:]
            at = pool[int(s.table[n, p // c["page"]]), p % c["page"]]
            at[:rank], at[rank:] = cell[row], lat[row, rank:]
    return {"cells": pool, "q_nope": nope, "q_abs": ab}


def _exact_heads(s):
    y = torch.zeros(s.y.shape, dtype=torch.float64, device="cuda")
    for h in range(s.c["H"]):
        y[:, h] = s.x[:, h].double() @ s.w[h].double().T.contiguous()
    return y


def _exact_latent(s):
    c, P = s.c, s.c["page"]
    out = torch.zeros(s.out.shape, dtype=torch.float64, device="cuda")
    for row, last in enumerate(s.pos.tolist()):
        if last >= 0:
            cells = s.pool[s.table[row, :last // P + 1].long()].reshape(-1, c["rank"] + c["rope"])[:last + 1].double()
            p = torch.softmax(cells @ s.q[row].double().T.contiguous() * s.scale, 0)
            out[row] = p.T.contiguous() @ cells[:, :c["rank"]].contiguous()
    return out


def _exact_prompt(s):
    c, rank, T = s.c, s.c["rank"], s.c["S"] + s.c["start"]
    cells = s.pool[s.pages.long()].reshape(-1, rank + c["rope"])[:T].double()
    out = torch.zeros(s.out.shape, dtype=torch.float64, device="cuda")
    late = torch.arange(T, device="cuda")[None] > c["start"] + torch.arange(c["S"], device="cuda")[:, None]
    for h in range(c["H"]):
        keys = torch.cat([cells[:, :rank] @ s.wk[h].double().T.contiguous(), cells[:, rank:]], 1)
        x = s.q[:, h].double() @ keys.T.contiguous() * s.scale
        x[late] = -math.inf
        out[:, h] = torch.softmax(x, 1) @ (cells[:, :rank] @ s.wv[h].double().T.contiguous())
    return out

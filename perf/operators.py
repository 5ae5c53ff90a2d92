"""The operators of the attention half of a decode step, and of its end, as timed cases.

A case is a dict of plain values.  `op` says which operator it is:

  rope    `Backend.qk_rope_append`: a projection's q and k heads normalised, turned by their
          positions, k and v written into a paged cache (a decode step or a chunk of a prompt)
  attn    `Backend.attn_paged`: one new token of each stream against its pages
  pages   `Backend.kv_copy_pages`: pages of every layer's cache copied, for a fork or to compact
  sample  `Backend.sample`: a token of each row of logits by temperature, top-k, top-p and min-p,
          from given random numbers

`run` computes the operator in plain torch where `own` is false, and calls the framework where it
is true.  Both leave their results in the state's own buffers: a cache that is written in place, the
rows of an output.
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
        # one stream's decode step: one row of 32 + 2 x 8 heads, far into its context
        dict(name="rope_decode_1", op="rope", S=1, seqs=1, Hq=32, Hkv=8, dh=128, rd=128, interleaved=False, norm=True,
             scaled=False, type="bf16", page=16, ctx=32768, pad=0),
        # a server's batch with free places at its end: half of each head turned, pairs side by side, no norm
        dict(name="rope_decode_48", op="rope", S=48, seqs=48, Hq=40, Hkv=8, dh=128, rd=64, interleaved=True, norm=False,
             scaled=False, type="f16", page=32, ctx=8192, pad=3),
        # a chunk of prompts, 2048 tokens of three streams, frequencies stretched for long contexts
        dict(name="rope_prompt_2048", op="rope", S=2048, seqs=3, Hq=32, Hkv=8, dh=128, rd=128, interleaved=False, norm=True,
             scaled=True, type="bf16", page=64, ctx=131072, pad=0),
        # one stream, a short context: the smallest call
        dict(name="attn_1x900", op="attn", S=1, Hq=32, Hkv=8, dh=128, type="bf16", page=16, ctx=900, short=900, window=0, pad=0),
        # one stream, a long document
        dict(name="attn_1x131072", op="attn", S=1, Hq=32, Hkv=8, dh=128, type="bf16", page=64, ctx=131072, short=131072,
             window=0, pad=0),
        # a server's batch, every stream at another length, two places free
        dict(name="attn_32x8192", op="attn", S=32, Hq=32, Hkv=8, dh=128, type="bf16", page=32, ctx=8192, short=1, window=0, pad=2),
        # a sliding-window layer of many streams with small heads
        dict(name="attn_64x16384_w512", op="attn", S=64, Hq=64, Hkv=8, dh=64, type="f16", page=16, ctx=16384, short=100,
             window=512, pad=0),
        # no shared heads, a cache in full precision
        dict(name="attn_7x3000_f32", op="attn", S=7, Hq=16, Hkv=16, dh=128, type="f32", page=64, ctx=3000, short=600, window=0,
             pad=0),
        # a fork's last, partly filled pages: 8 branches of one page, 48 layers
        dict(name="pages_fork_8", op="pages", layers=48, Hkv=8, dh=128, type="bf16", page=16, pool=32, n=8, fork=True),
        # a cache made dense again: 64 pages of 64 tokens moved, 48 layers
        dict(name="pages_compact_64", op="pages", layers=48, Hkv=8, dh=128, type="bf16", page=64, pool=160, n=64, fork=False),
        # one stream's pick from the stack's vocabulary
        dict(name="sample_1x32000", op="sample", S=1, V=32000, top_k=50, top_p=0.95, min_p=0.0, temp=0.8, mixed=False, sigma=3.0),
        # a batch of requests, each with settings of its own, from a large vocabulary
        dict(name="sample_200x131072", op="sample", S=200, V=131072, top_k=40, top_p=0.9, min_p=0.05, temp=1.0, mixed=True,
             sigma=2.5),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope"] * 3 + ["attn"] * 5 + ["pages"] * 2 + ["sample"] * 3)
    Hkv = rng.choice([1, 2, 3, 4, 5, 8, 8, 8, 12, 16])
    G = rng.choice([1, 2, 3, 4, 4, 5, 6, 7, 8, 8, 12, 16, 20])
    if Hkv * G > 128:
        G = 128 // Hkv
    dh = rng.choice([32, 64, 64, 96, 128, 128, 128, 160, 192, 256])
    kind, page = rng.choice(["bf16", "bf16", "bf16", "f16", "f16", "f32"]), 1 << rng.randint(3, 8)
    if op == "rope":
        S = _log_int(rng, 1, 2048)
        if Hkv * (G + 2) * dh > 48 * 128:
            S = max(1, S * 48 * 128 // (Hkv * (G + 2) * dh))
        prompt = S > 4 and rng.random() < 0.5
        pad = rng.randint(0, min(3, S - 1))
        return dict(op="rope", S=S, seqs=rng.randint(1, 4) if prompt else S, Hq=Hkv * G, Hkv=Hkv, dh=dh,
                    rd=dh if rng.random() < 0.5 else 2 * rng.randint(1, dh // 2), interleaved=rng.random() < 0.5,
                    norm=rng.random() < 0.6, scaled=rng.random() < 0.4, type=kind, page=page,
                    ctx=max(_log_int(rng, 64, 131072), 2 * S), pad=pad)
    if op == "attn":
        S = _log_int(rng, 1, 128)
        # at most the long document's cells of the cache
        most = 131072 * 1024 // (S * Hkv * dh * (2 if kind == "f32" else 1))
        ctx = _log_int(rng, 1, max(2, min(131072, most)))
        return dict(op="attn", S=S, Hq=Hkv * G, Hkv=Hkv, dh=dh, type=kind, page=page, ctx=ctx, short=rng.randint(1, ctx),
                    window=0 if rng.random() < 0.7 else rng.randint(1, 2 * ctx), pad=rng.randint(0, min(2, S - 1)))
    if op == "pages":
        layers, n = _log_int(rng, 1, 60), _log_int(rng, 1, 300)
        one = layers * Hkv * dh * page * (4 if kind == "f32" else 2)
        n = max(1, min(n, (48 * 64 * 64 * 2048) // one))
        return dict(op="pages", layers=layers, Hkv=Hkv, dh=dh, type=kind, page=page, pool=2 * n + rng.randint(1, 20), n=n,
                    fork=rng.random() < 0.4)
    V = _log_int(rng, 200, 200000)
    S = min(_log_int(rng, 1, 256), max(1, 200 * 131072 // V))
    return dict(op="sample", S=S, V=V, top_k=rng.choice([0, 1, 5, 40, 50, 1000, V + 1]), top_p=rng.choice([1.0, 0.95, 0.9, 0.5, 0.1]),
                min_p=rng.choice([0.0, 0.0, 0.02, 0.1, 0.5]), temp=rng.choice([0.0, 0.3, 0.7, 1.0, 1.0, 1.5]),
                mixed=rng.random() < 0.5, sigma=rng.choice([1.0, 2.5, 4.0]))


# ----------------------------------------------------------------- inputs ----

class _Dev:
    """A torch tensor handed to the framework as device memory."""

    def __init__(self, t):
        self.t = t

    def __int__(self):
        return self.t.data_ptr()


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


def _frequencies(rd, theta, scaled):
    """the angle per position of each pair; scaled: the slow pairs 8 times slower, the fast ones as they are, between them a ramp"""
    i = np.arange(rd // 2, dtype=np.float64)
    f = theta ** (-2.0 * i / rd)
    if scaled:
        turns = 16384 * f / (2 * math.pi)
        keep = np.clip((turns - 1.0) / 31.0, 0.0, 1.0)
        f = f * keep + f / 8.0 * (1.0 - keep)
    return f


def prepare(case, seed):
    c, g, r = case, _gen(seed), np.random.default_rng([int(seed), 23])
    s = _State(op=c["op"], c=c)
    if c["op"] == "rope":
        S, dh = c["S"], c["dh"]
        live = S - c["pad"]
        if c["seqs"] == S:                        # a decode step: one row of each stream
            pos, seq = r.integers(0, c["ctx"], S), np.arange(S)
        else:                                     # chunks: consecutive positions of a few streams
            seq = np.sort(r.integers(0, c["seqs"], S))
            begin = r.integers(0, c["ctx"] - S + 1, c["seqs"])
            pos = begin[seq] + np.arange(S) - np.searchsorted(seq, seq)
        need = np.zeros(c["seqs"], np.int64)
        np.maximum.at(need, seq, pos + 1)
        # the positions before the rows share one page, so that the cache holds about what is written
        first = np.full(c["seqs"], 1 << 40)
        np.minimum.at(first, seq, pos)
        first = np.where(need > 0, first // c["page"], 0)
        own_pages = [int(-(-n // c["page"]) - f) if n else 0 for n, f in zip(need, first)]
        table = np.zeros((c["seqs"], max(1, int(-(-need.max() // c["page"])))), np.int32)
        ids, at = r.permutation(sum(own_pages)) + 1, 0
        for i, n in enumerate(own_pages):
            table[i, int(first[i]):int(first[i]) + n] = ids[at:at + n]
            at += n
        pos[live:] = -1                           # places that hold no stream
        s.n_pages = S // c["page"] + 2 * c["seqs"] + 1      # no fewer, wherever the chunks begin
        width = c["Hq"] + 2 * c["Hkv"]
        s.qkv = _randn(g, S, width * dh)
        s.kv = [_pool(g, s.n_pages, c["Hkv"], c["page"], dh, dtype=TYPES[c["type"]]) for _ in range(2)]
        s.q = torch.zeros(S, c["Hq"], dh, device="cuda")
        s.wq, s.wk = (1.0 + 0.1 * _randn(g, dh) for _ in range(2))
        s.freq = torch.from_numpy(_frequencies(c["rd"], 1e6 if c["scaled"] else 1e4, c["scaled"])).cuda()
        s.factor = 1.0 + 0.1 * math.log(8.0) if c["scaled"] else 1.0
        s.pos, s.seq, s.table = _i32(pos), _i32(seq), _i32(table)
    elif c["op"] == "attn":
        S = c["S"]
        length = r.integers(c["short"], c["ctx"] + 1, S)
        length[r.integers(0, S - c["pad"])] = c["ctx"]
        length[S - c["pad"]:] = 0
        table, s.n_pages = _tables(r, length, c["page"])
        s.kv = [_pool(g, s.n_pages, c["Hkv"], c["page"], c["dh"], dtype=TYPES[c["type"]]) for _ in range(2)]
        s.q = 1.5 * _randn(g, S, c["Hq"], c["dh"])
        s.out = torch.zeros_like(s.q)
        s.pos, s.table = _i32(length - 1), _i32(table)
        s.scale = 1.0 / math.sqrt(c["dh"])
    elif c["op"] == "pages":
        s.kv = _pool(g, 2, c["layers"], c["pool"], c["Hkv"], c["page"], c["dh"], dtype=TYPES[c["type"]])
        ids = r.permutation(c["pool"])
        s.dst = np.ascontiguousarray(ids[:c["n"]], np.int32)
        if c["fork"]:                             # several branches of a few pages
            s.src = np.ascontiguousarray(ids[c["n"] + r.integers(0, max(1, c["n"] // 8), c["n"])], np.int32)
        else:
            s.src = np.ascontiguousarray(ids[c["n"]:2 * c["n"]], np.int32)
    else:
        S, V = c["S"], c["V"]
        # a few likely tokens over a wide floor, as a head gives
        s.logits = c["sigma"] * _randn(g, S, V)
        s.logits[:, r.integers(0, V, 8)] += torch.from_numpy(r.uniform(2, 10, 8).astype(np.float32)).cuda()
        s.u = torch.rand(S, generator=g, device="cuda")
        s.tok = torch.zeros(S, dtype=torch.int32, device="cuda")
        n, f32 = np.ones(S), np.float32
        temp, top_k, top_p, min_p = c["temp"] * n, c["top_k"] * n, c["top_p"] * n, c["min_p"] * n
        if c["mixed"]:                            # each request's own, some of them without a filter, some greedy
            temp = r.choice([0.0, 0.5, 0.7, 1.0, 1.3], S) if S > 1 else temp
            top_k = np.where(r.random(S) < 0.4, 0, top_k)
            top_p = np.where(r.random(S) < 0.4, 1.0, r.uniform(0.3, 1.0, S))
            min_p = np.where(r.random(S) < 0.5, 0.0, min_p)
        s.temp, s.top_p, s.min_p = (torch.from_numpy(a.astype(f32)).cuda() for a in (temp, top_p, min_p))
        s.top_k = _i32(top_k)
    if own:
        _handles(s)
    torch.cuda.synchronize()
    return s


def _cache(be, s, k, v, n_pages):
    c = s.c
    return be.kv_cache(k.data_ptr(), v.data_ptr(), c["type"], n_pages, c["page"], c["Hkv"], c["dh"])


def _handles(s):
    """what a program keeps: the caches' and settings' descriptors"""
    be, c = _be(), s.c
    s.be = be
    if s.op in ("rope", "attn"):
        s.cache = _cache(be, s, s.kv[0], s.kv[1], s.n_pages)
        seq = _Dev(s.seq) if s.op == "rope" else None
        s.rows = be.kv_rows(_Dev(s.pos), _Dev(s.table), s.table.shape[0], s.table.shape[1], seq)
    if s.op == "rope":
        s.rope = be.rope(_Dev(s.freq), c["rd"], c["interleaved"], s.factor)
        s.norms = (_Dev(s.wq), _Dev(s.wk)) if c["norm"] else (None, None)
        s.d = _Dev(s.qkv), _Dev(s.q)
    elif s.op == "attn":
        s.d = _Dev(s.q), _Dev(s.out)
    elif s.op == "pages":
        s.caches = be.kv_caches([_cache(be, s, s.kv[0, i], s.kv[1, i], c["pool"]) for i in range(c["layers"])])
    else:
        s.params = be.sample_params(_Dev(s.temp), _Dev(s.top_k), _Dev(s.top_p), _Dev(s.min_p))
        s.d = _Dev(s.logits), _Dev(s.u), _Dev(s.tok)


# -------------------------------------------------------------------- run ----

def run(s):
    c = s.c
    if s.op == "rope":
        if own:
            s.be.qk_rope_append(s.cache, s.rows, s.rope, s.d[0], s.qkv.shape[1], s.norms[0], s.norms[1], EPS, c["Hq"], s.d[1], c["S"])
        else:
            _plain_rope(s)
        return {"q": s.q, "k": s.kv[0], "v": s.kv[1]}
    if s.op == "attn":
        if own:
            s.be.attn_paged(s.cache, s.rows, s.d[0], c["Hq"], s.scale, c["window"], s.d[1], c["S"])
        else:
            _plain_attn(s)
        return s.out
    if s.op == "pages":
        if own:
            s.be.kv_copy_pages(s.caches, s.src, s.dst)
        else:
            s.kv[:, :, torch.from_numpy(s.dst).long().cuda()] = s.kv[:, :, torch.from_numpy(s.src).long().cuda()]
        return s.kv
    if own:
        s.be.sample(s.d[0], c["S"], c["V"], s.params, s.d[1], s.d[2])
    else:
        _plain_sample(s)
    return s.tok


def _plain_rope(s):
    c = s.c
    S, Hq, Hkv, dh, rd = c["S"], c["Hq"], c["Hkv"], c["dh"], c["rd"]
    x = s.qkv.view(S, Hq + 2 * Hkv, dh)
    qk, v = x[:, :Hq + Hkv], x[:, Hq + Hkv:]
    if c["norm"]:
        w = torch.cat([s.wq.expand(Hq, dh), s.wk.expand(Hkv, dh)])
        qk = qk * torch.rsqrt((qk * qk).mean(-1, keepdim=True) + EPS) * w
    angle = s.pos.double()[:, None] * s.freq
    cos, sin = ((f(angle) * s.factor).float()[:, None] for f in (torch.cos, torch.sin))
    turned = qk.clone()
    if c["interleaved"]:
        a, b = qk[..., 0:rd:2], qk[..., 1:rd:2]
        turned[..., 0:rd:2], turned[..., 1:rd:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = qk[..., :rd // 2], qk[..., rd // 2:rd]
        turned[..., :rd // 2], turned[..., rd // 2:rd] = a * cos - b * sin, b * cos + a * sin
    live = S - c["pad"]
    pos, seq = s.pos[:live].long(), s.seq[:live].long()
    page, slot = s.table[seq, pos // c["page"]].long(), pos % c["page"]
    s.q[:live] = turned[:live, :Hq]
    s.kv[0][page, :, slot] = turned[:live, Hq:].to(s.kv[0].dtype)
    s.kv[1][page, :, slot] = v[:live].to(s.kv[1].dtype)


def _plain_attn(s):
    c = s.c
    S, Hq, Hkv, dh, P = c["S"], c["Hq"], c["Hkv"], c["dh"], c["page"]
    n = min(c["ctx"], c["window"] or c["ctx"])
    t = s.pos.long()[:, None] - n + 1 + torch.arange(n, device="cuda")          # [S, n], the newest last
    seen = t >= 0
    t = t.clamp(min=0)
    page = s.table.long().gather(1, t // P)
    k, v = (p[page, :, t % P].float().transpose(1, 2).contiguous() for p in s.kv)     # [S, Hkv, n, dh]
    q = s.q.view(S, Hkv, Hq // Hkv, dh)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * s.scale
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    e = torch.exp(score - score.amax(-1, keepdim=True).clamp(min=-3e38))
    o = torch.matmul(e, v) / e.sum(-1, keepdim=True).clamp(min=1e-38)           # a free place: zero
    s.out.copy_(o.view(S, Hq, dh))


def _plain_sample(s):
    l = s.logits.double()
    V, temp = l.shape[1], s.temp.double()[:, None]
    v, i = torch.sort(l, dim=1, descending=True, stable=True)
    w = torch.exp((v - v[:, :1]) / torch.where(temp > 0, temp, 1.0))
    at = torch.arange(V, device="cuda")
    k = torch.where(s.top_k > 0, s.top_k.clamp(max=V), V)[:, None]
    w = torch.where(at < k, w, 0.0)
    run_ = w.cumsum(1)
    keep = (run_ - w < s.top_p.double()[:, None] * run_[:, -1:]) & (w >= s.min_p.double()[:, None])
    keep |= s.top_p[:, None] >= 1
    keep &= (w >= s.min_p.double()[:, None]) & (at < torch.where(temp > 0, k, 1))
    keep[:, 0] = True
    w = torch.zeros_like(l).scatter_(1, i, torch.where(keep, w, 0.0)).cumsum(1)
    s.tok.copy_((w <= s.u.double()[:, None] * w[:, -1:]).sum(1))


# ------------------------------------------------------------------- work ----

def work(case):
    c = case
    if c["op"] == "sample":
        return {"bytes": 4 * c["S"] * (c["V"] + 6), "flops": 4 * c["S"] * c["V"]}
    b = 4 if c["type"] == "f32" else 2
    if c["op"] == "pages":
        one = 2 * c["layers"] * c["Hkv"] * c["page"] * c["dh"] * b
        n = c["n"]
        distinct = max(1, n // 8) if c["fork"] else n
        return {"bytes": one * (n + distinct), "flops": 0}
    S, Hq, Hkv, dh = c["S"] - c["pad"], c["Hq"], c["Hkv"], c["dh"]
    if c["op"] == "rope":
        return {"bytes": S * dh * (4 * (Hq + 2 * Hkv) + 4 * Hq + 2 * b * Hkv), "flops": 8 * S * dh * (Hq + Hkv)}
    w = c["window"] or c["ctx"]
    lo, hi = min(c["short"], w), min(c["ctx"], w)
    # the mean of min(length, window) over lengths from short to ctx, one row at ctx
    mean = hi if c["short"] >= w else ((lo + hi) / 2 * (hi - lo) + hi * (c["ctx"] - hi)) / max(1, c["ctx"] - c["short"]) \
        if c["ctx"] > c["short"] else hi
    tokens = hi + (S - 1) * mean
    return {"bytes": tokens * 2 * Hkv * dh * b + 8 * S * Hq * dh, "flops": 4 * tokens * Hq * dh}


# ------------------------------------------------------------------ exact ----

def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    c = case
    if c["op"] == "rope":
        return _exact_rope(s)
    if c["op"] == "attn":
        out = torch.zeros(c["S"], c["Hq"], c["dh"], dtype=torch.float64, device="cuda")
        G, P = c["Hq"] // c["Hkv"], c["page"]
        for row, last in enumerate(s.pos.tolist()):
            if last < 0:
                continue
            first = max(0, last + 1 - c["window"]) if c["window"] else 0
            pages = s.table[row, first // P:last // P + 1].long()
            a, n = first % P, last + 1 - first
            for h in range(c["Hkv"]):
                k, v = (p[pages, h].reshape(-1, c["dh"])[a:a + n].double() for p in s.kv)
                p = torch.softmax(k @ s.q[row, h * G:(h + 1) * G].double().T.contiguous() * s.scale, 0)
                out[row, h * G:(h + 1) * G] = p.T.contiguous() @ v
        return out
    if c["op"] == "pages":
        for a, b in zip(s.src.tolist(), s.dst.tolist()):
            s.kv[:, :, b].copy_(s.kv[:, :, a])
        return s.kv
    logits, u = s.logits.cpu().numpy(), s.u.cpu().numpy()
    rows = zip(s.temp.tolist(), s.top_k.tolist(), s.top_p.tolist(), s.min_p.tolist())
    return np.array([_exact_pick(logits[i].astype(np.float64), float(u[i]), *p) for i, p in enumerate(rows)], np.int32)


def _exact_rope(s):
    """pair by pair, as a product of complex numbers"""
    c = s.c
    S, Hq, Hkv, dh, half = c["S"], c["Hq"], c["Hkv"], c["dh"], c["rd"] // 2
    x = s.qkv.double().view(S, -1, dh)
    heads = [x[:, :Hq], x[:, Hq:Hq + Hkv]]
    if c["norm"]:
        heads = [h / ((h * h).sum(-1, keepdim=True) / dh + EPS).sqrt() * w.double() for h, w in zip(heads, (s.wq, s.wk))]
    turn = torch.polar(torch.full((S, half), float(s.factor), dtype=torch.float64, device="cuda"), s.pos.double()[:, None] * s.freq)
    i = torch.arange(half, device="cuda")
    first, second = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half)
    for h in heads:
        z = torch.complex(h[..., first], h[..., second]) * turn[:, None]
        h[..., first], h[..., second] = z.real, z.imag
    q, k, v = torch.zeros_like(s.q, dtype=torch.float64), s.kv[0].double(), s.kv[1].double()
    for row, (p, b) in enumerate(zip(s.pos.tolist(), s.seq.tolist())):
        if p >= 0:
            page = int(s.table[b, p // c["page"]])
            q[row] = heads[0][row]
            k[page, :, p % c["page"]] = heads[1][row]
            v[page, :, p % c["page"]] = x[row, Hq + Hkv:]
    return {"q": q, "k": k, "v": v}


def _exact_pick(l, u, temp, top_k, top_p, min_p):
    order = np.lexsort((np.arange(len(l)), -l))
    if temp <= 0:
        return int(order[0])
    if 0 < top_k < len(l):
        order = order[:top_k]
    w = np.exp((l[order] - l[order[0]]) / temp)
    if top_p < 1:
        n = int(np.searchsorted(np.cumsum(w), top_p * math.fsum(w), side="left")) + 1
        order, w = order[:n], w[:n]
    n = max(1, int((w >= min_p).sum()))
    order, w = order[:n], w[:n]
    by = np.argsort(order)
    run_ = np.cumsum(w[by])
    return int(order[by][min(n - 1, int(np.searchsorted(run_, u * run_[-1], side="right")))])

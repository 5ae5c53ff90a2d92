"""Trees of drafted tokens for the tests, and their operators in 64 bits from the definitions."""
import numpy as np


def tree(rng, n):
    """parents of n nodes, each after its own"""
    return np.array([-1] + [int(rng.integers(0, j)) for j in range(1, n)], np.int32)


def sees_of(parent):
    """(bits of each node's ancestors and itself, depths)"""
    sees, depth = np.zeros(len(parent), np.uint64), np.zeros(len(parent), np.int64)
    for j, p in enumerate(parent):
        sees[j] = np.uint64(1 << j) | (sees[p] if p >= 0 else np.uint64(0))
        depth[j] = depth[p] + 1 if p >= 0 else 0
    return sees, depth


def exact_tree(k, v, table, P, first, base, seq, sees, pos, q, scale, window, out):
    """k, v [pages, Hkv, P, dh], q and out [S, Hq, dh] in 64 bits -> (out with the trees' rows filled in, bound).  The bound is
    paged.exact_attention's."""
    S, Hq, dh = q.shape
    n_pages, Hkv = k.shape[:2]
    G, eps = Hq // Hkv, 2.0 ** -24
    out, bound = out.copy(), np.zeros(out.shape)
    for i in range(len(base)):
        for s in range(first[i], first[i + 1]):
            out[s] = 0.0
            if base[i] < 0 or not 0 <= seq[i] < table.shape[0]:
                continue
            lo = max(0, max(pos[s], base[i]) - window + 1) if window else 0
            t = np.concatenate([np.arange(lo, base[i]), [base[i] + j for j in range(first[i + 1] - first[i]) if int(sees[s]) >> j & 1]]).astype(np.int64)
            t = t[t // P < table.shape[1]]
            page = table[seq[i]][t // P]
            ok = (page >= 0) & (page < n_pages)
            t, page = t[ok], page[ok]
            if not len(t):
                continue
            for h in range(Hq):
                kk, vv = k[page, h // G, t % P], v[page, h // G, t % P]
                x = kk @ q[s, h] * scale
                p = np.exp(x - x.max())
                l = p.sum()
                out[s, h] = (p @ vv) / l
                score = (dh + 2) * eps * np.max(np.abs(kk) @ np.abs(q[s, h])) * abs(scale) + 4 * eps * (np.max(np.abs(x - x.max())) + 4)
                bound[s, h] = (2 * score + (2 * len(t) + 16) * eps) * (p @ np.abs(vv)) / l
    return out, bound


def exact_path(parent, draft, tok):
    """(path, next token) of one tree"""
    way = [0]
    while True:
        kid = [j for j in range(way[-1] + 1, len(parent)) if parent[j] == way[-1] and draft[j] == tok[way[-1]]]
        if not kid:
            return way, int(tok[way[-1]])
        way.append(kid[0])

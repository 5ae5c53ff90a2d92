"""Drafted tokens verified in one step: a tree of them for each sequence, its nodes the rows of a step over a
PagedCache (attention.py).

    rows, S = trees.place([(seq, parents, tokens), ...])
    stack.step(h, xn, logits, tok, S, cache=cache, rows=rows, trees=trees)
    accepted = trees.commit(tok)

Node 0 is the sequence's next token (the pick that the last step ended in), every other node a drafted token
behind its parent.  A step gives each node the pick that follows it; commit() keeps the longest path from node 0 on whose
drafted tokens are those picks, and the sequence goes on behind it.  The reference's tables have no slot for it.
"""
from operator import index

import numpy as np

from .latent import LatentCache


def tree_of(parents, max_nodes=64):
    """(depths [n], sees [n] u64) of a tree given by its nodes' parents: -1 for node 0, of every other an
    earlier node.  Bit j of sees[i]: node i attends to node j (itself and its ancestors)."""
    parents = [index(p) for p in parents]
    if not 1 <= len(parents) <= max_nodes or parents[0] != -1 or any(not 0 <= p < i for i, p in enumerate(parents[1:], 1)):
        raise ValueError(f"a tree: 1 to {max_nodes} nodes, -1 and then an earlier node of each as its parent")
    depth, sees = [0], [1]
    for i, p in enumerate(parents[1:], 1):
        depth.append(depth[p] + 1)
        sees.append(sees[p] | 1 << i)
    return np.array(depth, np.int32), np.array(sees, np.uint64)


class DraftTrees:
    """Trees of at most max_nodes nodes, up to max_trees of them in a step, over `cache`.  Its arrays stay where they are, so
    that a recorded step replays over what the next place() puts there."""

    def __init__(self, cache, max_trees=None, max_nodes=32):
        if isinstance(cache, LatentCache):
            raise ValueError("DraftTrees: over a PagedCache, not over latents")
        self.cache, self.be = cache, cache.be
        self.max_trees, self.max_nodes = max_trees or cache.max_seqs, max_nodes
        if not 1 <= self.max_trees <= 65535 or not 1 <= max_nodes <= 64:
            raise ValueError("DraftTrees: 1 to 65535 trees of 1 to 64 nodes")
        T, R = self.max_trees, cache.max_rows
        self._host = np.zeros(2 * R + (T + 1) + 2 * T + 3 * R, np.int32)   # sees, first, base, seq, at, parent, draft
        self.dev = self.be.upload(self._host)
        at, self._parts, self._addr = 0, [], []
        for n in (2 * R, T + 1, T, T, R, R, R):
            self._parts.append(self._host[at:at + n])
            self._addr.append(int(self.dev) + 4 * at)
            at += n
        sees, first, base, seq, self.at, self._parent, self._draft = self._addr
        self.dev_out = self.be.alloc(4 * T * (max_nodes + 2))              # count, next, path
        self.desc = self.be.trees(first, base, sees, int(cache.dev_table), T, cache.max_seqs, cache.max_pages, max_nodes, seq, self.at)
        self.window = 0                                                    # the narrowest of the layers that were run over the trees
        self._depth = 0                                                    # of the placed trees' deepest node
        self.rows_made = 0                                                 # the cache's when they were placed
        self._placed, self._marks, self.rows = None, (), 0                 # (rows: of the placed trees' step)

    def within(self, window):
        """A layer with such a window (0: none) is to run over the trees.  A node attends to all of its ancestors, so that a tree as deep as
        the window is refused: here, and by every later place(), whose trees a recorded step takes without asking."""
        if window and self._placed is not None and self._depth >= window:
            raise ValueError(f"DraftTrees: a tree {self._depth} deep, and a layer whose window is {window}")
        self.window = min(self.window or window, window or self.window)

    def place(self, batch, rows=None):
        """The nodes of a batch's trees get the next cells of their sequences: entries are (sequence, parents, tokens), tokens[0]
        the sequence's next token.  Returns (rows descriptor, number of rows), the trees' nodes in order; with `rows`
        the step has so many, free places behind the last tree's (as many as trees without a sequence have room for).
        Trees as deep as a layer's window are refused (see within).  CacheFull, or an upload that fails, leaves the sequences as
        they were."""
        cache, T = self.cache, self.max_trees
        if self._placed is not None:
            raise ValueError("DraftTrees.place: the trees before are neither committed nor dropped")
        batch = [(index(s), tree_of(parents, self.max_nodes), [index(p) for p in parents], np.array([index(t) for t in tokens], np.int32)) for s, parents, tokens in batch]
        used = sum(len(p) for _, _, p, _ in batch)
        rest = (used if rows is None else index(rows)) - used
        if not 1 <= len(batch) <= T or any(len(p) != len(t) for _, _, p, t in batch):
            raise ValueError(f"DraftTrees.place: 1 to {T} trees, a token of each node")
        if not 0 <= rest <= (T - len(batch)) * self.max_nodes:
            raise ValueError("DraftTrees.place: rows for fewer than the nodes, or more free places than trees without a sequence have room for")
        deepest = max(int(depth.max()) for _, (depth, _), _, _ in batch)
        if self.window and deepest >= self.window:
            raise ValueError(f"DraftTrees.place: a tree {deepest} deep, and a layer whose window is {self.window}")
        placed = [(s, cache.length(s), len(p)) for s, _, p, _ in batch]
        desc, total = cache.rows([(s, n) for s, _, n in placed] + ([(None, rest)] if rest else []))
        marks = [cache.mark(s) for s, _, _ in placed]
        sees, first, base, seq, at, parent, draft = self._parts
        sees = sees.view(np.uint64)
        base[:], seq[:], at[:], parent[:], draft[:] = -1, -1, -1, -1, -1
        sees[:] = 0
        row = 0
        for i, ((s, start, n), (_, (depth, see), p, tokens)) in enumerate(zip(placed, batch)):
            first[i], base[i], seq[i] = row, start, s
            sees[row:row + n], at[row:row + n], parent[row:row + n], draft[row:row + n] = see, start + depth, p, tokens
            row += n
        for i in range(len(batch), T + 1):                                 # free places share the rest
            first[i] = row
            row = min(row + self.max_nodes, total)
        try:
            self.be.h2d(self.dev, self._host)
        except BaseException:
            for s, start, _ in placed:
                cache.truncate(s, start)
            raise
        self._placed, self._marks, self._depth, self.rows, self.rows_made = placed, marks, deepest, total, cache.rows_made
        return desc, total

    def commit(self, tok):
        """Keep each tree's accepted path: its cells move to the sequence's next places in every layer, and the sequence
        ends behind them.  tok: the picks of the step's rows (device).  Returns for each tree (the path's nodes, the token
        that follows): the next tree's node 0.  Refused, with the trees as they were, where a sequence was closed (its place may be another's
        by now), went on, was truncated or forked since; drop() is the way out."""
        if self._placed is None:
            raise ValueError("DraftTrees.commit: no trees are placed")
        for (s, start, n), mark in zip(self._placed, self._marks):
            if self.cache.mark(s) != mark or any(self.cache._users[p] > 1 for p in self.cache._pages[s][start // self.cache.page_size:]):
                raise ValueError(f"DraftTrees.commit: sequence {s} is another, went on, was truncated or forked, with its tree in it")
        T, N = self.max_trees, self.max_nodes
        count, nxt, path = (int(self.dev_out) + 4 * n for n in (0, T, 2 * T))
        self.be.tree_commit(self.cache.layers, self.desc, self._parent, self._draft, tok, path, count, nxt, self.rows)
        out = self.be.d2h(self.dev_out, (T * (N + 2),), np.int32)
        count, nxt, path = out[:T], out[T:2 * T], out[2 * T:].reshape(T, N)
        kept = []
        for i, (s, start, _) in enumerate(self._placed):
            self.cache.truncate(s, start + int(count[i]))
            kept.append((path[i, :count[i]].tolist(), int(nxt[i])))
        self._placed, self.rows = None, 0
        return kept

    def drop(self):
        """forget the placed trees: their sequences are as before place(), but those that were closed, truncated or went on since"""
        for (s, start, _), mark in zip(self._placed or (), self._marks):
            if self.cache._pages[s] is not None and self.cache.mark(s) == mark:
                self.cache.truncate(s, start)
        self._placed, self.rows = None, 0

    def free(self):
        for b in (self.dev, self.dev_out):
            b.free()

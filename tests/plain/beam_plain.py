"""Beam search written down plainly, in 64 bits with numpy: the selection, the page tables and moves, a cache that follows, and a
whole search over a function that gives logits."""
from __future__ import annotations

import math

import numpy as np

PAGE = 64
BIG = float(np.finfo(np.float32).max)


def log_probs(row):
    """log softmax in 64 bits; NaN counts as -inf, +inf as the largest finite number of 32 bits; None for a row of nothing."""
    row = np.asarray(row, dtype=np.float64)
    row = np.minimum(np.where(np.isnan(row), -np.inf, row), BIG)
    top = row.max()
    if top == -np.inf:
        return None
    with np.errstate(under="ignore"):
        return (row - top) - math.log(np.exp(row - top).sum())


def select(logits, scores, beams, stops=(), ending=True):
    """(scores, parents, tokens, ended scores, ended parents, ended tokens), [groups, beams] each."""
    G, held = scores.shape
    V = logits.shape[1]
    f = lambda fill, t=np.float64: np.full((G, beams), fill, dtype=t)      # noqa: E731
    out = [f(-np.inf), np.tile(np.arange(beams), (G, 1)), f(0, np.int64), f(-np.inf), f(-1, np.int64), f(-1, np.int64)]
    stops = set(int(t) for t in stops)
    for g in range(G):
        cand = []
        for b in range(held):
            if not scores[g, b] > -np.inf:
                continue
            lp = log_probs(logits[g * held + b])
            if lp is None:
                continue
            total = float(scores[g, b]) + lp
            keep = min(V, beams + len(stops))
            order = np.argsort(-total, kind="stable")[:keep]
            cand += [(-total[t], b, int(t)) for t in order if total[t] > -np.inf]
        cand.sort()
        going = [c for c in cand if c[2] not in stops][:beams]
        first = {}
        for c in going:
            first.setdefault(c[1], c)
        places = dict(first)
        empty = [p for p in range(beams) if p not in first]
        rest = [c for c in going if first[c[1]] is not c]
        places.update(zip(empty, rest))
        for p, c in places.items():
            out[0][g, p], out[1][g, p], out[2][g, p] = -c[0], c[1], c[2]
        if ending:
            for rank, c in enumerate(cand[:beams]):
                if c[2] in stops:
                    out[3][g, rank], out[4][g, rank], out[5][g, rank] = -c[0], c[1], c[2]
    return out


def tables(tables_, homes, rings, slots, parents, lengths):
    """Changes the tables (lists of int arrays [slots + 1, columns]) and returns the moves [1 + tables][groups * beams] of (source,
    destination, rows)."""
    G, B = slots.shape
    moves = np.zeros((1 + len(tables_), G, B, 3), dtype=np.int64)
    for g in range(G):
        for b in range(B):
            if parents[g][b] != b:
                moves[0, g, b] = (slots[g][parents[g][b]], slots[g][b], 1)
        for k, (table, home, ring) in enumerate(zip(tables_, homes, rings)):
            L, W = lengths[g], table.shape[1]
            w = (L % ring if ring else L) // PAGE
            used = min(-(-L // PAGE), W, ring // PAGE if ring else W)
            old = {b: table[slots[g][parents[g][b]]].copy() for b in range(B)}
            for b in range(B):
                for c in range(used):
                    if c != w:
                        table[slots[g][b], c] = old[b][c]
            if w >= used:
                continue
            keeper = {}
            for b in range(B):
                if parents[g][b] == b:
                    keeper.setdefault(int(old[b][w]), b)
            spare = [int(home[slots[g][b], w]) for b in range(B) if int(home[slots[g][b], w]) not in keeper]
            rows = PAGE if ring and L >= ring else L % PAGE
            for b in range(B):
                page = int(old[b][w])
                if keeper.get(page) == b:
                    continue
                table[slots[g][b], w] = new = spare.pop(0)
                if rows:
                    moves[1 + k, g, b] = (page, new, rows)
    return moves.reshape(1 + len(tables_), G * B, 3)


def move(states, pages, moves):
    """Applies moves to torch or numpy tensors."""
    for src, dst, n in moves[0]:
        if n:
            for s in states:
                s[int(dst)] = s[int(src)]
    for k, of_table in enumerate(pages):
        for src, dst, n in moves[1 + k]:
            if n:
                for t in of_table:
                    t[:, int(dst), :, :int(n)] = t[:, int(src), :, :int(n)]


def search(logits_of, prompt, beams, max_new, stops=(), length_penalty=1.0, early_stopping=False, max_len=None):
    """The whole search without a cache: ``logits_of(tokens)`` gives the logits after them.  Returns [(value, score, tokens, reason)],
    best first, at most ``beams``: value = score / number of drawn tokens (a stop token counts) ** length_penalty."""
    limit = max_new if max_len is None else min(max_new, max_len - len(prompt))
    live, done = [(0.0, [])], []
    for step in range(1, limit + 1):
        cand = []
        for b, (score, toks) in enumerate(live):
            total = score + log_probs(logits_of(list(prompt) + toks))
            cand += [(-total[t], b, int(t)) for t in np.argsort(-total, kind="stable")[:beams + len(stops)] if total[t] > -np.inf]
        cand.sort()
        done += [(-c[0] / step ** length_penalty, -c[0], live[c[1]][1], "stop") for c in cand[:beams] if c[2] in stops]
        done = sorted(done, key=lambda d: -d[0])[:beams]
        live = [(-c[0], live[c[1]][1] + [c[2]]) for c in [c for c in cand if c[2] not in stops][:beams]]
        if not live:
            return done
        # a score only falls, and its value is best at the greatest length that it can reach
        if len(done) == beams and step < limit and (early_stopping or max(s for s, _ in live) / limit ** length_penalty <= done[-1][0]):
            return done
    done += [(s / limit ** length_penalty, s, t, "length" if limit == max_new else "context") for s, t in live]
    return sorted(done, key=lambda d: -d[0])[:beams]

"""NumPy restatement of beam search over the int4 KV cache: the choice of beams, and
the reordering of pages and of contiguous caches, step by step on the host.

TEST INFRASTRUCTURE ONLY.  The reference samples one continuation; it has no beams.
"""
from __future__ import annotations

import numpy as np

NEG = -np.inf


def totals(x, score, finished, pad):
    """scores + log-probabilities of one group, float64 [W, V]; -inf: no candidate."""
    W, V = x.shape
    out = np.full((W, V), NEG)
    for w in range(W):
        if not score[w] > NEG:
            continue
        if finished is not None and finished[w]:
            out[w, pad] = score[w]
            continue
        row = np.where(np.isnan(x[w]), NEG, x[w].astype(np.float64))
        top = row.max()
        if top == NEG:
            continue
        d = np.full(V, NEG)
        same = row == top
        d[same] = 0.0
        if top < np.inf:
            d[~same] = row[~same] - top
        with np.errstate(invalid="ignore"):
            t = float(score[w]) + (d - np.log(np.exp(d).sum()))
        out[w] = np.where(np.isnan(t), NEG, t)
    return out


def beam_select(x, scores, num_out, finished=None, pad=0):
    """x [B, W, V] -> (totals float64, parents, tokens), each [B, num_out]."""
    B, W, V = x.shape
    val = np.full((B, num_out), NEG)
    parents, tokens = np.full((B, num_out), -1, np.int32), np.full((B, num_out), -1, np.int32)
    for b in range(B):
        t = totals(x[b], scores[b], None if finished is None else finished[b], pad).ravel()
        order = np.argsort(-t, kind="stable")[:num_out]
        order = order[t[order] > NEG]
        k = len(order)
        val[b, :k], parents[b, :k], tokens[b, :k] = t[order], b * W + order // V, order % V
    return val, parents, tokens


def reorder(pool, parents):
    """The page reordering of an oracle.paged.Pool; returns what was granted."""
    S, P = pool.tables.shape
    old, lens = pool.tables.copy(), pool.lengths.copy()
    par = [int(p) if 0 <= p < S else -1 for p in parents]
    kids = [[c for c in range(S) if par[c] == p] for p in range(S)]
    for p in range(S):
        if not kids[p]:
            for e in old[p]:
                if pool._is_page(e):
                    pool.refs[e] -= 1
    free = [p for p, r in enumerate(pool.refs) if r <= 0]
    granted, copies, short = np.zeros(S, np.int32), [], False
    for s in range(S):
        p = par[s]
        if p == s:
            granted[s] = 1
            continue
        row, n, ok = np.full(P, -1, np.int32), 0, p >= 0
        if ok:
            n = min(max(int(lens[p]), 0), P * pool.page)
            full, rest = divmod(n, pool.page)
            if (p if p in kids[p] else kids[p][0]) == s:
                row = old[p].copy()
            else:
                if rest and pool._is_page(old[p][full]):
                    if short or not free:
                        short, ok = True, False
                    else:
                        row[full] = free.pop(0)
                        pool.refs[row[full]] = 1
                        copies.append((old[p][full], row[full]))
                if ok:
                    row[:full] = old[p][:full]
                    for e in row[:full]:
                        if pool._is_page(e):
                            pool.refs[e] += 1
        pool.tables[s], pool.lengths[s], granted[s] = row if ok else -1, n if ok else 0, ok
    for t in pool.pages:
        was = t.copy()
        for a, b in copies:
            t[:, b] = was[:, a]
    return granted


def reorder_rows(tensors, lengths, parents):
    """The contiguous caches [B, Hkv, cap, .] and lengths after the reordering."""
    B, cap = tensors[0].shape[0], tensors[0].shape[2]
    out, lens = [t.copy() for t in tensors], np.zeros_like(lengths)
    for s, p in enumerate(parents):
        if not 0 <= p < B:
            continue
        n = min(max(int(lengths[p]), 0), cap)
        lens[s] = lengths[p]
        for new, old in zip(out, tensors):
            new[s, :, :n] = old[p, :, :n]
    return out, lens

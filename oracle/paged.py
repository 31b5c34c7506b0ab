"""NumPy restatement of the paged int4 cache: appending, attention with a
sliding window and visible first tokens, and the page operations.

TEST INFRASTRUCTURE ONLY.  The reference has no paged cache; attention is the
rule of ``oracle.sdpa_int4`` over the rows that a block table names.
"""
from __future__ import annotations

import numpy as np

from oracle import oracle as O


def visible(n: int, limit: int, window: int, sinks: int) -> np.ndarray:
    """Which of keys 0 .. limit - 1 the query at position n - 1 attends."""
    t = np.arange(limit)
    ok = t < n
    return ok & ((t >= n - window) | (t < sinks)) if window > 0 else ok


def rows(pages, table, page_size: int, n: int):
    """K and V rows [Hkv, n, D] in float64, and whether each has a page."""
    num = pages[0].shape[0]
    t = np.arange(n)
    entry = np.asarray(table)[t // page_size] if n else np.zeros(0, np.int64)
    has = (entry >= 0) & (entry < num)
    at = np.where(has, entry, 0)
    out = []
    for i in (0, 3):
        w, s, b = (np.moveaxis(x[at, :, t % page_size], 0, 1) for x in pages[i:i + 3])
        with np.errstate(invalid="ignore"):
            out.append(O.dequantize(w, s, b))
    return out[0], out[1], has


def attend(q, k, v, keep, scale: float):
    """One query row over the kept keys, float64; none: 0."""
    if not keep.any():
        return np.zeros(v.shape[1])
    s = float(np.float32(scale)) * (k[keep] @ q.astype(np.float64))
    p = np.exp(s - s.max())
    return (p / p.sum()) @ v[keep]


def sdpa_int4_paged(q, pages, tables, seq_lens, page_size, gqa, scale=1.0, window=0, sinks=0, windows=None,
                    shared_prefix=0, max_kv_len=None):
    """q [B, Hq, D] -> [B, Hq, D] float64."""
    B, Hq, D = q.shape
    out = np.zeros((B, Hq, D))
    for b in range(B):
        table = np.array(tables[b])
        table[:shared_prefix // page_size] = tables[0][:shared_prefix // page_size]
        n = max(int(seq_lens[b]), 0)
        n = min(n, len(table) * page_size if max_kv_len is None else max_kv_len)
        k, v, has = rows(pages, table, page_size, n)
        keep = visible(n, n, int(windows[b]) if windows is not None else window, sinks) & has
        for h in range(Hq):
            out[b, h] = attend(q[b, h], k[h // gqa], v[h // gqa], keep, scale)
    return out


def sdpa_int4_paged_prefill(q, pages, table, n_prior, page_size, gqa, scale=1.0, window=0, sinks=0):
    """q [n_new, Hq, D] at positions n_prior + i -> [n_new, Hq, D] float64."""
    S, Hq, D = q.shape
    out = np.zeros((S, Hq, D))
    k, v, has = rows(pages, table, page_size, n_prior + S)
    for i in range(S):
        keep = visible(n_prior + i + 1, n_prior + S, window, sinks) & has
        for h in range(Hq):
            out[i, h] = attend(q[i, h], k[h // gqa], v[h // gqa], keep, scale)
    return out


def sdpa_int4_paged_chunks(q, pages, tables, starts, seq_lens, page_size, gqa, scale=1.0, window=0, sinks=0,
                           max_kv_len=None):
    """q [N, Hq, D], sequence b's in rows starts[b] .. starts[b + 1] - 1 -> [N, Hq, D] float64."""
    out = np.zeros(q.shape)
    for b in range(len(seq_lens)):
        n = max(int(seq_lens[b]), 0)
        n = min(n, tables.shape[1] * page_size if max_kv_len is None else max_kv_len)
        k, v, has = rows(pages, tables[b], page_size, n)
        new = int(starts[b + 1] - starts[b])
        for i in range(new):
            keep = visible(n - new + i + 1, n, window, sinks) & has
            for h in range(q.shape[1]):
                out[starts[b] + i, h] = attend(q[starts[b] + i, h], k[h // gqa], v[h // gqa], keep, scale)
    return out


def append(pages, k_new, v_new, tables, positions, page_size, sb, mode="mlx"):
    """Quantized rows into the page arrays, in place."""
    for i, x in ((0, k_new), (3, v_new)):
        parts = O.quantize_int4(x, sb, mode)
        for b in range(x.shape[0]):
            for t in range(x.shape[2]):
                r = int(positions[b]) + t
                if not 0 <= r < tables.shape[1] * page_size:
                    continue
                e = tables[b, r // page_size]
                if 0 <= e < pages[0].shape[0]:
                    for dst, src in zip(pages[i:i + 3], parts):
                        dst[e, :, r % page_size] = src[b, :, t]


class Pool:
    """The page operations, step by step on the host."""

    def __init__(self, tables, refs, lengths, page_size, pages=()):
        self.tables, self.refs, self.lengths = (np.array(x) for x in (tables, refs, lengths))
        self.page, self.pages = page_size, [np.array(p) for p in pages]  # [layers, num_pages, ..]

    def _is_page(self, e):
        return 0 <= e < len(self.refs)

    def reserve(self, n_new):
        granted = np.zeros(len(n_new), np.int32)
        free = [p for p, r in enumerate(self.refs) if r <= 0]
        short = False
        for s, new in enumerate(n_new):
            n = max(int(self.lengths[s]), 0)
            e1 = -(-(n + int(new)) // self.page)
            if new <= 0 or e1 > self.tables.shape[1]:
                continue
            lack = [e for e in range(n // self.page, e1) if not self._is_page(self.tables[s, e])]
            if lack and (short or len(lack) > len(free)):
                short = True
                continue
            for e in lack:
                self.tables[s, e] = free.pop(0)
                self.refs[self.tables[s, e]] = 1
            granted[s] = 1
        return granted

    def advance(self, n_new):
        advanced = np.zeros(len(n_new), np.int32)
        for s, new in enumerate(n_new):
            n, new = max(int(self.lengths[s]), 0), int(new)
            e1 = -(-(n + new) // self.page)
            if new < 0:
                self.lengths[s] = max(int(self.lengths[s]) + new, 0)
            elif new and e1 <= self.tables.shape[1] and all(
                    self._is_page(e) for e in self.tables[s, n // self.page:e1]):
                self.lengths[s], advanced[s] = n + new, 1
        return advanced

    def fork(self, parents):
        granted = np.zeros(len(parents), np.int32)
        free = [p for p, r in enumerate(self.refs) if r <= 0]
        short = False
        before = self.tables.copy(), self.lengths.copy()
        for s, par in enumerate(parents):
            if not 0 <= par < len(parents) or par == s or parents[par] >= 0 or before[1][s] != 0 or any(
                    self._is_page(e) for e in before[0][s]):
                continue
            n = min(max(int(before[1][par]), 0), self.tables.shape[1] * self.page)
            full, rest = divmod(n, self.page)
            row = np.full(self.tables.shape[1], -1, np.int32)
            row[:full] = before[0][par][:full]
            if rest and self._is_page(before[0][par][full]):
                if short or not free:
                    short = True
                    continue
                row[full] = free.pop(0)
                self.refs[row[full]] = 1
                for t in self.pages:
                    t[:, row[full]] = t[:, before[0][par][full]]
            for e in row[:full]:
                if self._is_page(e):
                    self.refs[e] += 1
            self.tables[s], self.lengths[s], granted[s] = row, n, 1
        return granted

    def free(self, which):
        for s in np.flatnonzero(which):
            for e in self.tables[s]:
                if self._is_page(e):
                    self.refs[e] -= 1
            self.tables[s], self.lengths[s] = -1, 0

    def evict(self, window, sinks, which=None):
        for s in range(len(self.lengths)):
            if which is not None and not which[s]:
                continue
            for e in range(self.tables.shape[1]):
                if e * self.page >= sinks and (e + 1) * self.page <= self.lengths[s] - window:
                    if self._is_page(self.tables[s, e]):
                        self.refs[self.tables[s, e]] -= 1
                    self.tables[s, e] = -1

    def compact(self):
        live = [p for p, r in enumerate(self.refs) if r > 0]
        n = len(live)
        to = {p: p for p in live}
        to.update(zip([p for p in live if p >= n], sorted(set(range(n)) - set(live))))
        for t in self.pages:
            old = t.copy()
            for a, b in to.items():
                t[:, b] = old[:, a]
        refs = np.zeros_like(self.refs)
        for a, b in to.items():
            refs[b] = self.refs[a]
        self.refs = refs
        num = len(refs)
        self.tables = np.array([[to.get(int(e), -1) if 0 <= e < num else e for e in row] for row in self.tables],
                               dtype=np.int32).reshape(self.tables.shape)
        return n

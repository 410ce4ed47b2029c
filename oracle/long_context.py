"""Oracles of long conversations over the paged cache, in 64 bits and plain Python (test oracle only): heads normed and
rotated by position, what a row sees of a window with sinks, and a pool of pages that sequences share."""
from __future__ import annotations

import numpy as np


def head_form(x, pos, weight=None, eps=1e-6, freq=None, rotary_dim=0, interleaved=False, amplitude=1.0):
    """x [rows, heads, hd] at positions pos [rows]: (result, bound on its error by its terms): the bound counts, for fp32
    arithmetic, 16 roundings of 2^-24 of a normed value (half of the sum of squares' 16 + 6, 3 of the root, 2 products)
    and, of a rotated pair, 4 of cos and sin (polynomial, remainder, amplitude) and 2 of the products and their sum, each
    relative to |a| + |b|; and 2^-51 of the angle (a position times a frequency in 64 bits, here and there)."""
    x = np.asarray(x, np.float64)
    hd = x.shape[2]
    err = np.zeros_like(x)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(2, keepdims=True) + eps) * np.asarray(weight, np.float64)
        err = 16 * 2.0 ** -24 * np.abs(x)
    if freq is None:
        return x, err
    out, tol = x.copy(), err.copy()
    n = (rotary_dim or hd) // 2
    i = np.arange(n)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    angle = np.asarray(pos, np.float64)[:, None] * np.asarray(freq, np.float64)
    c, s = (amplitude * f(angle)[:, None] for f in (np.cos, np.sin))
    out[:, :, a] = x[:, :, a] * c - x[:, :, b] * s
    out[:, :, b] = x[:, :, a] * s + x[:, :, b] * c
    size = abs(amplitude) * (np.abs(x[:, :, a]) + np.abs(x[:, :, b]))
    both = abs(amplitude) * (err[:, :, a] + err[:, :, b]) + size * (6 * 2.0 ** -24 + 2.0 ** -51 * np.abs(angle)[:, None])
    tol[:, :, a] = tol[:, :, b] = both
    return out, tol


def sees(pos: int, n: int, window: int, sinks: int) -> np.ndarray:
    """Which of n tokens a row at position pos sees."""
    t = np.arange(n)
    return (t <= pos) & ((t > pos - window) | (t < sinks))


class Pool:
    """Tables and users of pages; each page's content is any value, one per page, that copies carry along."""

    def __init__(self, table, refs, page, content):
        self.table, self.refs, self.page = np.array(table), np.array(refs), page
        self.content = list(content)

    def is_page(self, p):
        return 0 <= p < len(self.refs)

    def release(self, p):
        if self.is_page(p) and self.refs[p] > 0:
            self.refs[p] -= 1

    def new_page(self):
        free = np.nonzero(self.refs <= 0)[0]
        if not len(free):
            return -1
        self.refs[free[0]] = 1
        return int(free[0])

    def free(self, seqs, keep=0, end=None, behind=0):
        for i, b in enumerate(seqs):
            if not 0 <= b < len(self.table):
                continue
            for j in range(self.table.shape[1]):
                last = (j + 1) * self.page
                if j * self.page >= keep and (end is None or (end[i] >= 0 and last <= end[i] - behind)):
                    self.release(self.table[b, j])
                    self.table[b, j] = -1

    def reserve(self, seqs, start, count, stop=None, follow=False):
        """Entries are served in order; users change at the end only (a page given back is none of this call's).  ``follow``:
        an entry that begins before its start gets no page."""
        missing, begun = 0, []
        for i, b in enumerate(seqs):
            if not 0 <= b < len(self.table) or start[i] < 0:
                continue
            end = min(start[i] + count, self.table.shape[1] * self.page)
            end = end if stop is None else min(end, stop[i])
            for j in range(start[i] // self.page, -(-end // self.page) if end > start[i] else 0):
                if follow and j * self.page < start[i]:
                    begun.append((b, j))
                elif not self.is_page(self.table[b, j]):
                    p = self.new_page()
                    missing += p < 0
                    if p >= 0:
                        self.table[b, j] = p
        return missing + sum(not self.is_page(self.table[e]) for e in begun)

    def fork(self, parents, children, lengths):
        todo = [(p, c, n) for p, c, n in zip(parents, children, lengths)
                if 0 <= p < len(self.table) and 0 <= c < len(self.table) and p != c and n >= 0]
        for p, c, n in todo:
            row = [int(x) if j < n // self.page and self.is_page(x) else -1 for j, x in enumerate(self.table[p])]
            for x in row:
                if x >= 0:
                    self.refs[x] += 1
            for x in self.table[c]:
                self.release(x)
            self.table[c] = row
        missing = 0
        for p, c, n in todo:
            j = n // self.page
            if n % self.page == 0 or j >= self.table.shape[1] or not self.is_page(self.table[p, j]):
                continue
            new = self.new_page()
            missing += new < 0
            if new >= 0:
                self.content[new] = self.content[self.table[p, j]]
                self.table[c, j] = new
        return missing

    def compact(self):
        used = np.nonzero(self.refs > 0)[0]
        U = len(used)
        where = np.where(self.refs > 0, np.arange(len(self.refs)), -1)
        for a, b in zip(used[used >= U], np.nonzero(self.refs[:U] <= 0)[0]):
            where[a] = b
            self.content[b] = self.content[a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        for e in np.ndindex(self.table.shape):
            if self.is_page(self.table[e]):
                self.table[e] = where[self.table[e]]
        return where, U

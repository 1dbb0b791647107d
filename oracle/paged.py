"""numpy restatement in 64 bits of serving over a paged cache: the oracle of
firepit_b200's page tables, paged attention and sampling.

TEST INFRASTRUCTURE ONLY: the product never imports it.
"""
from __future__ import annotations

import math

import numpy as np


class Pool:
    """Page tables and the stack of free pages, one request after another."""

    def __init__(self, batch, pages, page_size, max_pages):
        self.p, self.max_pages = page_size, max_pages
        self.table = np.full((batch, max_pages), -1, np.int32)
        self.lengths = np.zeros(batch, np.int32)
        self.free = list(range(pages - 1, -1, -1))

    def _pages(self, tokens):
        return -(-int(tokens) // self.p)

    def extend(self, counts, rows, padded=False):
        """(slots, positions, requests, starts), as page_extend gives them."""
        batch = len(counts)
        out = np.full((3, rows), -1, np.int64)
        starts = []
        at, short = 0, False
        for b, n in enumerate(counts):
            n = int(n)
            first = b * (rows // batch) if padded else at
            starts.append(min(first, rows))
            at += max(n, 0)
            held = int(self.lengths[b])
            fits = n >= 0 and held + n <= self.max_pages * self.p and (
                n <= rows // batch if padded else first + n <= rows)
            need = self._pages(held + n) - self._pages(held) if fits else 0
            if need and (short or need > len(self.free)):
                short, fits = True, False
            if not fits:
                continue
            for j in range(need):
                self.table[b, self._pages(held) + j] = self.free.pop()
            for i in range(n):
                t = held + i
                out[:, first + i] = (self.table[b, t // self.p] * self.p + t % self.p, t, b)
            self.lengths[b] = held + n
        starts.append(rows if padded else min(at, rows))
        return out[0], out[1], out[2], np.array(starts)

    def truncate(self, lengths):
        given = []
        for b, n in enumerate(lengths):
            if 0 <= n < self.lengths[b]:
                lo, hi = self._pages(n), self._pages(self.lengths[b])
                given += list(self.table[b, lo:hi])
                self.table[b, lo:hi] = -1
                self.lengths[b] = n
        self.free += given[::-1]


def attend(q, k, v, scale):
    """One query q [d] over the tokens k, v [t, d]: (output, sum of p |v|, largest
    sum of |q_i k_i| * scale), the latter two for error bounds."""
    if len(k) == 0:
        return np.zeros_like(q), np.zeros_like(q), 0.0
    s = (k @ q) * scale
    p = np.exp(s - s.max())
    p /= p.sum()
    return p @ v, p @ np.abs(v), float((np.abs(k) @ np.abs(q)).max() * abs(scale))


def kept(logits, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(tokens kept, in order, and the log of each one's weight over the largest);
    temperature 0 or below keeps the first one."""
    x = np.where(np.isfinite(logits), logits, -math.inf).astype(np.float64)
    order = np.lexsort((np.arange(len(x)), -x))
    order = order[np.isfinite(x[order])]
    if len(order) == 0:
        return order, x[order]
    if not temperature > 0:
        return order[:1], np.zeros(1)
    d = (x[order] - x[order[0]]) / min(max(temperature, 1e-6), 1e6)
    n = len(order)
    if top_k > 0:
        n = min(n, top_k)
    if top_p < 1:
        w = np.exp(d[:n])
        n = max(1, int((np.cumsum(w) - w < top_p * w.sum()).sum()))
    if min_p > 0:
        n = min(n, int((d >= math.log(min(min_p, 1.0))).sum()))
    return order[:n], d[:n]


def sample(logits, noise, **filters):
    """(token, its log probability among what is kept, {token: log(w / noise)})."""
    order, d = kept(logits, **filters)
    if len(order) == 0:
        return -1, -math.inf, {}
    race = d - np.log(noise[order].astype(np.float64))
    best = int(order[race == race.max()].min())
    return best, float(d[list(order).index(best)] - np.log(np.exp(d).sum())), dict(zip(order.tolist(), race.tolist()))

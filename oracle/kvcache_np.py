"""The paged key-value cache and its attention in plain numpy: the bookkeeping
as a list-by-list restatement of what include/accel_hip.h says of each call,
attention in 64 bits from its definition."""
from __future__ import annotations

import numpy as np

NONE = 0xffffffff


class Pages:
    """refs, tables and lens, and the page data [layers, pages, kv_heads,
    page_size, head_dim] as raw bits or numbers.  `left_out` collects the
    entries a call did not serve."""

    def __init__(self, keys, values, sequences: int, slots: int):
        self.keys, self.values = np.array(keys), np.array(values)
        self.pages, self.page_size = self.keys.shape[1], self.keys.shape[3]
        self.refs = np.zeros(self.pages, np.uint32)
        self.tables = np.full((sequences, slots), NONE, np.uint32)
        self.lens = np.zeros(sequences, np.uint32)
        self.left_out = []

    def _free(self):
        return [p for p in range(self.pages) if self.refs[p] == 0]

    def reserve(self, grow, seqs=None):
        seqs = range(len(self.lens)) if seqs is None else seqs
        free, seen, slots = self._free(), set(), self.tables.shape[1]
        take = []
        for i, (s, g) in enumerate(zip(seqs, grow)):
            if s == NONE:
                continue
            if s >= len(self.lens) or s in seen:
                self.left_out.append(i)
                continue
            seen.add(s)
            n = int(self.lens[s])
            if n + int(g) > slots * self.page_size:
                self.left_out.append(i)
                continue
            have = -(-n // self.page_size)
            need = -(-(n + int(g)) // self.page_size) - have
            take.append((i, s, g, have, need))
        at = 0
        for i, s, g, have, need in take:
            if need and at + need > len(free):
                self.left_out.append(i)
            else:
                for j in range(need):
                    self.tables[s, have + j] = free[at + j]
                    self.refs[free[at + j]] = 1
                self.lens[s] += g
                at += need

    def append(self, layer, k, v, seqs=None, offsets=None):
        offsets = range(len(k) + 1) if offsets is None else offsets
        n = len(offsets) - 1
        seqs = range(n) if seqs is None else seqs
        for i in range(n):
            s = seqs[i]
            if s == NONE:
                continue
            if s >= len(self.lens):
                self.left_out.append(i)
                continue
            for t in range(offsets[i], min(offsets[i + 1], len(k))):
                pos = int(self.lens[s]) - int(offsets[i + 1]) + t
                page = self.tables[s, pos // self.page_size] if pos >= 0 else NONE
                if page >= self.pages or self.refs[page] > 1:
                    self.left_out.append(t)
                    continue
                self.keys[layer, page, :, pos % self.page_size] = k[t]
                self.values[layer, page, :, pos % self.page_size] = v[t]

    def fork(self, parents, children):
        free, seen, at = self._free(), set(), 0
        lens = self.lens.copy()
        tables = self.tables.copy()
        for i, (p, c) in enumerate(zip(parents, children)):
            again = c in seen
            seen.add(c)
            if p == NONE or c == NONE:
                # an index beside it outside the cache is still reported
                if NONE != p >= len(lens) or NONE != c >= len(lens):
                    self.left_out.append(i)
                continue
            if p >= len(lens) or c >= len(lens) or again or lens[c]:
                self.left_out.append(i)
                continue
            whole, part = divmod(int(lens[p]), self.page_size)
            if part:
                if at >= len(free):
                    self.left_out.append(i)
                    at += 1
                    continue
                src, dst = int(tables[p, whole]), free[at]
                at += 1
                self.keys[:, dst] = self.keys[:, src]
                self.values[:, dst] = self.values[:, src]
                self.refs[dst] = 1
                self.tables[c, whole] = dst
            for j in range(whole):
                page = tables[p, j]
                self.tables[c, j] = page
                if page < self.pages:
                    self.refs[page] += 1
            self.lens[c] = lens[p]

    def _drop(self, s, slots):
        for j in slots:
            page = self.tables[s, j]
            if page < self.pages:
                self.refs[page] -= 1
            self.tables[s, j] = NONE

    def free(self, seqs=None):
        for s in range(len(self.lens)) if seqs is None else seqs:
            if s < len(self.lens):
                self._drop(s, range(self.tables.shape[1]))
                self.lens[s] = 0

    def trim(self, window, sinks=0, seqs=None):
        P = self.page_size
        for s in range(len(self.lens)) if seqs is None else seqs:
            if s < len(self.lens):
                n = int(self.lens[s])
                self._drop(s, [j for j in range(self.tables.shape[1])
                               if j * P >= sinks and (j + 1) * P <= n - window])

    def compact(self):
        used = [p for p in range(self.pages) if self.refs[p]]
        L = len(used)
        src = [p for p in used if p >= L]
        dst = [p for p in range(L) if self.refs[p] == 0]
        for a, b in zip(src, dst):
            self.keys[:, b] = self.keys[:, a]
            self.values[:, b] = self.values[:, a]
            self.refs[b], self.refs[a] = self.refs[a], 0
            self.tables[self.tables == a] = b
        return L

    def copy(self, src, dst):
        keys, values = self.keys.copy(), self.values.copy()
        for a, b in zip(src, dst):
            if a < self.pages and b < self.pages:
                self.keys[:, b], self.values[:, b] = keys[:, a], values[:, a]


def visible(p: int, window: int, sinks: int) -> np.ndarray:
    """Positions the query at position p sees."""
    j = np.arange(p + 1)
    return j[(p - j < window) | (j < sinks)] if window else j


def attention(q, keys, values, tables, lens, seqs, offsets, scale, window=0, sinks=0):
    """q [T, heads, dim] over one layer's keys and values [pages, kv_heads,
    page_size, dim] (all 64-bit): out [T, heads, dim] and, per row and head,
    the sum of weight * |value| and the largest sum of |query * key| * scale
    and |score| spread (what error bounds are made of)."""
    T, H, D = q.shape
    KV, P = keys.shape[1], keys.shape[2]
    G = H // KV
    out = np.zeros((T, H, D))
    mass = np.zeros((T, H, D))
    size = np.zeros((T, H))
    for i in range(len(offsets) - 1):
        s = int(seqs[i])
        if s == NONE or s >= len(lens):
            continue
        n, end = int(lens[s]), int(offsets[i + 1])
        for t in range(int(offsets[i]), end):
            p = n - (end - t)
            if p < 0:
                continue
            pos = visible(p, window, sinks)
            page = tables[s, pos // P]
            pos, page = pos[page < len(keys)], page[page < len(keys)]
            if not len(pos):
                continue
            k = keys[page, :, pos % P]          # [n, KV, D]
            v = values[page, :, pos % P]
            for h in range(H):
                kh, vh = k[:, h // G], v[:, h // G]
                x = (kh @ q[t, h]) * scale
                e = np.exp(x - x.max())
                w = e / e.sum()
                out[t, h] = w @ vh
                mass[t, h] = w @ np.abs(vh)
                size[t, h] = (np.abs(kh) @ np.abs(q[t, h])).max() * scale + np.ptp(x)
    return out, mass, size

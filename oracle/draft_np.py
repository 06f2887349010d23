"""Drafts in plain numpy: attention of a tree's nodes in 64 bits from its
definition, the choice of a token from a row of logits, the walk down a tree and
what a cache keeps of it, each as include/accel_hip.h says of the call."""
from __future__ import annotations

import math

import numpy as np

NONE = 0xffffffff
NODES = 256
REFUSED = 0xfffffffe


def line_of(parents, t):
    """A node's path, from itself up to its root, or None where a parent is not
    below its child."""
    line = [t]
    while parents[t] != NONE:
        if parents[t] >= t:
            return None
        t = int(parents[t])
        line.append(t)
    return line


def attention(q, keys, values, tables, lens, seqs, offsets, parents, scale, window=0, sinks=0):
    """As kvcache_np.attention, of drafts' nodes; and the entries and rows left out."""
    T, H, D = q.shape
    P, G = keys.shape[2], H // keys.shape[1]
    out, mass, size = np.zeros((T, H, D)), np.zeros((T, H, D)), np.zeros((T, H))
    left_out = []
    for i in range(len(offsets) - 1):
        s, first = int(seqs[i]), int(offsets[i])
        m = int(offsets[i + 1]) - first
        if s == NONE or m <= 0:
            continue
        if s >= len(lens) or m > NODES or m > lens[s]:
            left_out.append(("entry", i))
            continue
        L = int(lens[s]) - m
        for t in range(m):
            line = line_of(parents[first:first + m], t)
            if line is None:
                left_out.append(("row", first + t))
                continue
            p = L + len(line) - 1
            # where each visible key lies, and the position that it stands for
            lies = list(range(L)) + [L + a for a in line]
            stands = list(range(L)) + [p - k for k in range(len(line))]
            pos = np.array(sorted(x for x, j in zip(lies, stands)
                                  if not window or p - j < window or j < sinks))
            page = tables[s, pos // P]
            if (page >= len(keys)).any():
                left_out.append(("page", first + t))
            pos, page = pos[page < len(keys)], page[page < len(keys)]
            if not len(pos):
                continue
            k, v = keys[page, :, pos % P], values[page, :, pos % P]
            for h in range(H):
                kh, vh = k[:, h // G], v[:, h // G]
                x = (kh @ q[first + t, h]) * scale
                e = np.exp(x - x.max())
                w = e / e.sum()
                out[first + t, h] = w @ vh
                mass[first + t, h] = w @ np.abs(vh)
                size[first + t, h] = ((np.abs(kh) @ np.abs(q[first + t, h])).max() * scale +
                                      np.ptp(x))
    return out, mass, size, left_out


def sample(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, log of its share, how near the choice was to falling otherwise) of
    one row of logits: the margin is the least distance of a border from a sum
    that it was compared with, as a share of the whole."""
    x = np.asarray(x, np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.lexsort((np.arange(len(x)), -x))
    top = x[order[0]]
    if top == -np.inf:
        return NONE, -math.inf, 1.0
    if not temperature > 0:
        return int(order[0]), 0.0, 1.0
    xs = x[order]
    with np.errstate(invalid="ignore", over="ignore"):
        if top == np.inf:
            w = (xs == np.inf).astype(np.float64)
        elif temperature == math.inf:
            w = (xs != -np.inf).astype(np.float64)
        else:
            w = np.exp((xs - top) / temperature)
    margin = 1.0
    keep = int((xs != -np.inf).sum())
    if top_k:
        keep = min(keep, int(top_k))
    if top_p < 1:
        run = np.cumsum(w[:keep])
        border = max(float(top_p), 0.0) * run[-1]
        margin = min(margin, np.abs(run - border).min() / run[-1])
        keep = min(keep, int((run < border).sum()) + 1)
    if min_p > 0:
        least = min(float(min_p), 1.0)
        margin = min(margin, np.abs(w[:keep] - least)[w[:keep] != 1].min(initial=1.0))
        keep = max(1, int((w[:keep] >= least).sum()))
    run = np.cumsum(w[:keep])
    u = min(max(float(u), 0.0), 1 - 2.0 ** -24) if u == u else 0.0
    border = u * run[-1]
    margin = min(margin, np.abs(run - border).min() / run[-1])
    j = min(int((run <= border).sum()), keep - 1)
    return int(order[j]), math.log(w[j] / run[-1]) if w[j] else -math.inf, margin


def accept(tokens, parents, offsets, sampled, width):
    n = len(offsets) - 1
    path = np.full((n, width), NONE, np.uint32)
    counts, nxt = np.zeros(n, np.uint32), np.full(n, NONE, np.uint32)
    left_out = []
    for i in range(n):
        first, m = int(offsets[i]), int(offsets[i + 1]) - int(offsets[i])
        if m > NODES:
            left_out.append(i)
            path[i, 0] = REFUSED
        if m <= 0 or m > NODES:
            continue
        at = 0
        while True:
            path[i, counts[i]] = at
            counts[i] += 1
            nxt[i] = sampled[first + at]
            if counts[i] == width or nxt[i] == NONE:
                break
            fits = [t for t in range(at + 1, m)
                    if parents[first + t] == at and tokens[first + t] == nxt[i]]
            if not fits:
                break
            at = fits[0]
    return path, counts, nxt, left_out


def keep(pages, path, counts, offsets, seqs=None):
    """On a kvcache_np.Pages."""
    P, cap = pages.page_size, pages.tables.shape[1] * pages.page_size
    n = len(offsets) - 1
    seqs = range(n) if seqs is None else seqs
    for i in range(n):
        s, m, k = int(seqs[i]), max(0, int(offsets[i + 1]) - int(offsets[i])), int(counts[i])
        if s == NONE:
            continue
        if s >= len(pages.lens) or m > pages.lens[s] or pages.lens[s] > cap:
            pages.left_out.append(i)
            continue
        L = int(pages.lens[s]) - m
        p = [int(x) for x in path[i][:k]]
        ok = k <= min(m, len(path[i])) and all(t < m for t in p)
        ok = ok and (k > 0 or int(path[i][0]) != REFUSED)
        ok = ok and all(a < b for a, b in zip(p, p[1:]))
        if ok:
            for c, t in enumerate(p):
                a, b = (int(pages.tables[s, (L + x) // P]) for x in (t, c))
                ok = ok and (t == c or (a < pages.pages and b < pages.pages and
                                        pages.refs[b] == 1))
        if not ok:
            pages.left_out.append(i)
            continue
        for c, t in enumerate(p):
            if t == c:
                continue
            a, b = (int(pages.tables[s, (L + x) // P]) for x in (t, c))
            for x in (pages.keys, pages.values):
                x[:, b, :, (L + c) % P] = x[:, a, :, (L + t) % P]
        pages._drop(s, range(-(-(L + k) // P), -(-(L + m) // P)))
        pages.lens[s] = L + k

"""Plain forms of the drafted trees' operators, on the CPU (numpy, 64 bits)."""
from __future__ import annotations

import numpy as np


def grow(rng, nodes, chain=0.4):
    """Parents (inside the request) of trees of `nodes` tokens each; roots beside node 0 too."""
    out = []
    for n in nodes:
        p = [-1] * min(n, 1)
        for j in range(1, n):
            u = rng.random()
            p.append(j - 1 if u < chain else -1 if u > 0.95 else int(rng.integers(0, j)))
        out += p
    return np.array(out, np.int32)


def line(parents, t0, j):
    """Node j and its ancestors."""
    out = []
    while j >= 0:
        out.append(j)
        j = int(parents[t0 + j])
    return out


def tree(parents, cu, lens, tokens, words):
    masks, pos = np.zeros((tokens, words), np.uint64), np.full(tokens, -1, np.int32)
    for r in range(len(lens)):
        n = cu[r + 1] - cu[r]
        for j in range(n):
            ln = line(parents, cu[r], j)
            for i in ln:
                masks[cu[r] + j, i // 64] |= np.uint64(1) << np.uint64(i % 64)
            pos[cu[r] + j] = lens[r] - n + len(ln) - 1
    return masks.view(np.int64), pos


def attend(q, k, v, cu, lens, table, page, scale, window, first, sink, masks, positions):
    """As kv_reference.attend, with the visibility of a tree."""
    q = np.asarray(q, np.float64)
    t, heads, d = q.shape
    g = heads // k.shape[1]
    out, smax, vmax = np.zeros_like(q), np.zeros((t, heads)), np.zeros((t, heads))
    bits = masks.view(np.uint64)
    for r, n in enumerate(lens):
        base = n - (cu[r + 1] - cu[r])
        for x in range(cu[r], cu[r + 1]):
            p = min(max(positions[x], base), n - 1)
            i = np.arange(n)
            own = np.zeros(n, bool)
            for j in range(max(0, -base), n - base):
                if j < 64 * bits.shape[1]:
                    own[base + j] = int(bits[x, j // 64]) >> (j % 64) & 1
            see = np.where(i >= base, own, (window == 0) | (i > p - window) | (i < first))
            i = i[see]
            if not i.size:
                continue
            kk, vv = k[table[r, i // page], :, i % page], v[table[r, i // page], :, i % page]
            for h in range(heads):
                with np.errstate(invalid="ignore", over="ignore"):
                    s = kk[:, h // g] @ q[x, h] * scale
                    m = np.nanmax(s) if np.isfinite(s).any() else 0.0
                    m = m if sink is None else max(m, sink[h])
                    w = np.exp(s - m)
                    z = w.sum() + (0.0 if sink is None else np.exp(sink[h] - m))
                    out[x, h] = (w[:, None] * vv[:, h // g]).sum(0) / z
                smax[x, h], vmax[x, h] = np.abs(s).max(), np.abs(vv[:, h // g]).max()
    return out, smax, vmax


def accept(page, parents, drafts, targets, cu, lens, table, free, top):
    """(counts, path, next, lens, free, top); inputs unchanged."""
    free, path = free.copy(), np.full(len(parents), -1, np.int32)
    counts, nxt, after = [], [], []
    for r in range(len(lens)):
        t0, n = cu[r], cu[r + 1] - cu[r]
        kept = [0] if n else []
        while kept:
            fit = [c for c in range(1, n)
                   if parents[t0 + c] == kept[-1] and drafts[t0 + c] == targets[t0 + kept[-1]]]
            if not fit:
                break
            kept.append(fit[0])
        path[t0:t0 + len(kept)] = kept
        counts.append(len(kept))
        nxt.append(targets[t0 + kept[-1]] if kept else -1)
        after.append(lens[r] - n + len(kept))
        for p in range(-(-after[-1] // page), -(-lens[r] // page)):
            free[top] = table[r, p]
            top += 1
    return counts, path, nxt, after, free, top


def commit(arrays, counts, path, cu, lens, table, page):
    """The arrays [blocks, heads, page, bytes] after the rows have moved."""
    out = [a.copy() for a in arrays]
    for r, k in enumerate(counts):
        base = lens[r] - (cu[r + 1] - cu[r])
        for i in range(k):
            a, b = base + path[cu[r] + i], base + i
            for x, y in zip(arrays, out):
                y[table[r, b // page], :, b % page] = x[table[r, a // page], :, a % page]
    return out

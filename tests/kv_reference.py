"""Plain 64-bit forms of the paged 4-bit cache's operators, on the CPU (numpy)."""
from __future__ import annotations

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantise(x):
    """x [..., d] -> (codes [..., d/2] uint8, scales [..., d/32] uint8)."""
    x = np.asarray(x, np.float64)
    b = x.reshape(*x.shape[:-1], -1, 32)
    fin = np.isfinite(b).all(-1)
    with np.errstate(invalid="ignore"):
        top = np.where(fin, np.abs(b).max(-1), 0.0)
    m, e = np.frexp(top)  # top = m 2^e, m in [0.5, 1): top <= 6 2^k = 0.75 2^(k+3)
    k = np.clip(np.where(m <= 0.75, e - 3, e - 2), -126, 125)
    y = np.abs(np.where(fin[..., None], b, 0.0)) / (2.0 ** k)[..., None]
    hi = np.clip(np.searchsorted(GRID, y), 1, 7)
    mid = (GRID[hi - 1] + GRID[hi]) / 2
    code = np.where((y > mid) | ((y == mid) & (hi % 2 == 0)), hi, hi - 1)
    code = np.where(y == 0, 0, code).astype(np.uint8)
    sign = np.signbit(b) & fin[..., None]
    code = (code | (sign.astype(np.uint8) << 3)).reshape(*x.shape)
    scale = np.where(~fin, 255, np.where(top == 0, 0, k + 127)).astype(np.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def values(codes, scales):
    """codes [..., d/2], scales [..., d/32] -> [..., d] float64."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    v = GRID[c & 7] * np.where(c & 8, -1.0, 1.0)
    s = scales.astype(np.float64)
    s = np.where(s >= 253, np.nan, np.where(s == 0, 0.0, 2.0 ** (s - 127)))
    return (v.reshape(*v.shape[:-1], -1, 32) * s[..., None]).reshape(v.shape)


def attend(q, k, v, cu_q, kv_lens, table, page, scale, window, first, sink):
    """q [t, heads, d]; k, v [blocks, kvh, page, d] values; float64 [t, heads, d],
    and the largest |score| and |value| that each query row sees."""
    q = np.asarray(q, np.float64)
    t, heads, d = q.shape
    kvh = k.shape[1]
    g = heads // kvh
    out = np.zeros_like(q)
    smax, vmax = np.zeros((t, heads)), np.zeros((t, heads))
    for r, n in enumerate(kv_lens):
        t0, t1 = cu_q[r], cu_q[r + 1]
        for j in range(t0, t1):
            p = n - (t1 - t0) + (j - t0)
            i = np.arange(0, max(0, p + 1))
            if window:
                i = i[(i > p - window) | (i < first)]
            if not i.size:
                continue
            kk = k[table[r, i // page], :, i % page]  # [n, kvh, d]
            vv = v[table[r, i // page], :, i % page]
            for h in range(heads):
                with np.errstate(invalid="ignore", over="ignore"):
                    s = kk[:, h // g] @ q[j, h] * scale
                    m = np.nanmax(s) if np.isfinite(s).any() else 0.0
                    m = m if sink is None else max(m, sink[h])
                    w = np.exp(s - m)
                    z = w.sum() + (0.0 if sink is None else np.exp(sink[h] - m))
                    out[j, h] = (w[:, None] * vv[:, h // g]).sum(0) / z
                smax[j, h] = np.abs(s).max()
                vmax[j, h] = np.abs(vv[:, h // g]).max()
    return out, smax, vmax


def plan(page, old, q, finished, table, free, top):
    """(table, free, top, lens, cu_q, slots, positions, requests); inputs unchanged."""
    table, free = table.copy(), free.copy()
    n = len(old)
    up = lambda x: -(-x // page)  # noqa: E731
    for r in range(n):
        if finished[r]:
            for p in range(up(old[r])):
                free[top] = table[r, p]
                top += 1
    slots, pos, who, lens, cu = [], [], [], [], [0]
    for r in range(n):
        lens.append(0 if finished[r] else old[r] + q[r])
        for p in range(up(old[r]), up(lens[-1])) if not finished[r] else ():
            top -= 1
            table[r, p] = free[top]
        for i in range(old[r], old[r] + q[r]):
            slots.append(int(table[r, i // page]) * page + i % page)
            pos.append(i)
            who.append(r)
        cu.append(cu[-1] + q[r])
    return table, free, top, lens, cu, slots, pos, who

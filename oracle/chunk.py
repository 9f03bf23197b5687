"""The operators around a chunk of new tokens, restated in plain Python and float64 (numpy): block
tables and slots, rotary positions, chunk attention."""
from __future__ import annotations

import numpy as np


def extend(table, seq_lens, query_start, free, top, n_tokens, page, num_blocks):
    """(table, slots, positions, blocks left, blocks short) of a step; inputs stay."""
    table = np.array(table)
    slots = np.full(n_tokens, -1, np.int64)
    positions = np.full(n_tokens, -1, np.int32)
    left, short = int(top), 0
    for r, length in enumerate(seq_lens):
        q0, q1 = int(query_start[r]), int(query_start[r + 1])
        start = int(length) - (q1 - q0)
        have, need = -(-max(start, 0) // page), min(-(-int(length) // page), table.shape[1])
        if q1 > q0:
            for p in range(have, need):
                ok = left > 0
                left -= ok
                short += not ok
                block = int(free[left]) if ok else -1
                table[r, p] = block if 0 <= block < num_blocks else -1
        for i in range(q1 - q0):
            pos = start + i
            if pos < 0:
                continue
            positions[q0 + i] = pos
            if pos // page < table.shape[1] and 0 <= table[r, pos // page] < num_blocks:
                slots[q0 + i] = int(table[r, pos // page]) * page + pos % page
    return table, slots, positions, left, short


def release(table, seq_lens, done, free, top, page, num_blocks):
    """(table, free, blocks left, dropped)."""
    table, free = np.array(table), np.array(free)
    top, dropped = int(top), 0
    for r, length in enumerate(seq_lens):
        if not done[r]:
            continue
        for p in range(min(-(-int(length) // page), table.shape[1])):
            if 0 <= table[r, p] < num_blocks:
                if top < len(free):
                    free[top] = table[r, p]
                    top += 1
                else:
                    dropped += 1
            table[r, p] = -1
    return table, free, top, dropped


def rotate(x, positions, w, amplitude, interleaved):
    """x (T, H, d) turned by angles positions * w (rot / 2,), float64."""
    x = np.array(x, np.float64)
    angle = np.asarray(positions, np.float64)[:, None, None] * np.asarray(w, np.float64)
    z = amplitude * np.exp(1j * angle)
    half = len(w)
    i = np.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    turned = (x[..., a] + 1j * x[..., b]) * z
    x[..., a], x[..., b] = turned.real, turned.imag
    return x


def attend(q, k, v, table, seq_lens, query_start, *, scale, causal, window, page):
    """Chunk attention row by row: q (T, H, d), k / v (NB, page, n_kv, d), float64.  Returns
    (out, lse, seen, size, reach): rows of no request are NaN in out; `size` is the weighted mean of
    |v| per channel and `reach` the row's largest scale sum_d |q_d k_d| (what rounding errors
    scale with)."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    T, H, d = q.shape
    n_kv = k.shape[2]
    G = H // n_kv
    out, size = np.full((T, H, d), np.nan), np.zeros((T, H, d))
    lse, reach = np.full((T, H), np.nan), np.zeros((T, H))
    seen = np.zeros(T, np.int64)
    for r, length in enumerate(seq_lens):
        q0, q1 = int(query_start[r]), int(query_start[r + 1])
        length = int(length)
        limit = min(length, table.shape[1] * page)
        js = np.arange(max(limit, 0))
        block = np.asarray(table[r])[js // page]
        good = (block >= 0) & (block < k.shape[0])
        js, block = js[good], block[good]
        kr, vr = k[block, js % page], v[block, js % page]
        for t in range(q0, q1):
            p = length - (q1 - q0) + (t - q0)
            see = np.zeros(len(js), bool)
            if p >= 0:
                see = np.ones(len(js), bool)
                if causal:
                    see &= js <= p
                if window:
                    see &= js > p - window
            out[t], lse[t] = 0.0, -np.inf
            seen[t] = see.sum()
            if not seen[t]:
                continue
            for h in range(H):
                kk, vv = kr[see, h // G], vr[see, h // G]
                s = scale * (kk @ q[t, h])
                m = s.max()
                if m == -np.inf:
                    continue
                e = np.exp(s - m)
                out[t, h] = (e @ vv) / e.sum()
                size[t, h] = (e @ np.abs(vv)) / e.sum()
                lse[t, h] = m + np.log(e.sum())
                reach[t, h] = scale * (np.abs(kk) @ np.abs(q[t, h])).max()
    return out, lse, seen, size, reach

"""The 8-bit paged cache, restated in plain Python and float64 (numpy): steps, the quantising write and
the numbers that codes stand for."""
from __future__ import annotations

import math

import numpy as np

MOST = {"int8": 127.0, "e4m3": 448.0}
LEAST_SCALE = 2.0 ** -64
MOST_SCALE = {"int8": 2.0 ** 121, "e4m3": 2.0 ** 119}


def step(m, code):
    """The scale that numbers of at most m take."""
    if m == 0.0:
        return LEAST_SCALE
    if code == "int8":
        _, e = math.frexp(m / 127.0)
        grid = 2.0 ** (e - 8)                               # 8 significant bits
        n = math.floor(m / 127.0 / grid)
        while n * grid * 127.0 < m:                         # (exact: 8 bits times 7)
            n += 1
        s = n * grid
    else:
        s = 2.0 ** (math.frexp(m)[1] - 12)
        while 448.0 * s < m:
            s *= 2.0
    return min(max(s, LEAST_SCALE), MOST_SCALE[code])


def to_code(y, code):
    """float64 quotients to codes, half to even, at most the largest."""
    y = np.clip(np.asarray(y, np.float64), -MOST[code], MOST[code])
    if code == "int8":
        return np.rint(y)
    _, e = np.frexp(np.maximum(np.abs(y), 2.0 ** -6))
    grid = 2.0 ** (e - 4.0)                                 # 4 significant bits, from 2^-6 on
    return np.rint(y / grid) * grid


def write(codes, scales, x, slots, page, code):
    """codes (NB, page, n_kv, d) and scales (NB, n_kv) of one half, as numbers, after x (T, n_kv, d) has
    entered at `slots`; inputs stay."""
    codes, scales = np.array(codes, np.float64), np.array(scales, np.float64)
    x = np.asarray(x, np.float64)
    nb, t, T = codes.shape[0], 0, len(slots)
    while t < T:
        b, a = divmod(int(slots[t]), page)
        n = 1
        while a + n < page and t + n < T and slots[t + n] == slots[t] + n:
            n += 1
        if 0 <= b < nb:
            for h in range(codes.shape[2]):
                part, old = x[t:t + n, h], scales[b, h] if a else 0.0
                if not np.isfinite(part).all() or np.isnan(old):
                    codes[b, a:a + n, h], scales[b, h] = 0.0, np.nan
                    continue
                s = max(step(np.abs(part).max(), code), old)
                if a and s > old:
                    codes[b, :a, h] = to_code(codes[b, :a, h] * old / s, code)
                codes[b, a:a + n, h] = to_code(part / s, code)
                scales[b, h] = s
        t += n
    return codes, scales

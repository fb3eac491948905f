"""The paged 8-bit cache's operators in plain Python and 64 bits: page planning, quantised append, attention.

Independent of the library: lists for the pages, float64 for the numbers, the definitions written out one token and one
row at a time.
"""
from __future__ import annotations

import math

import numpy as np

CODE_MAX = {"int8": 127.0, "e4m3": 448.0}
MIN_SCALE = 2.0 ** -100

#: the value of every e4m3 code: sign, 4 exponent bits (bias 7), 3 mantissa bits; 0x7f and 0xff are NaN
E4M3 = np.array([(-1.0 if c & 0x80 else 1.0) * (math.nan if c & 0x7F == 0x7F else
                 (c & 7) * 2.0 ** -9 if not c & 0x78 else (1 + (c & 7) / 8) * 2.0 ** (((c >> 3) & 15) - 7))
                 for c in range(256)])


def code_values(codes: np.ndarray, code: str) -> np.ndarray:
    """Values (float64) of uint8 code words."""
    return codes.view(np.int8).astype(np.float64) if code == "int8" else E4M3[codes]


def plan_step(lens, new_lens, table, free, page_len, max_tokens, capacity):
    """One step of page planning on Python lists (``table`` rows and the stack ``free`` are changed in place, unless
    the step is refused).  Returns (ok, lens, first, slots, positions, taken, given)."""
    width = len(table[0])
    ceil = lambda n: -(-n // page_len)  # noqa: E731
    ends = [0 if a < 0 else n + a for n, a in zip(lens, new_lens)]
    given = [p for r, (n, a) in enumerate(zip(lens, new_lens)) if a < 0 for p in table[r][:max(0, ceil(n))]]
    taken = sum(ceil(e) - ceil(n) for n, a, e in zip(lens, new_lens, ends) if a >= 0)
    total = sum(max(0, a) for a in new_lens)
    if (min(lens) < 0 or max(ceil(n) for n in lens + ends) > width or total > max_tokens
            or len(free) + len(given) > capacity or taken > len(free) + len(given)):
        return False, list(lens), [0] * (len(lens) + 1), [-1] * max_tokens, [-1] * max_tokens, 0, 0
    free.extend(given)
    first, slots, positions = [0], [], []
    for r, (n, a) in enumerate(zip(lens, new_lens)):
        for pos in range(n, n + max(0, a)):
            if pos // page_len >= ceil(n) and pos % page_len == 0 or pos == n and n % page_len == 0:
                table[r][pos // page_len] = free.pop()
            slots.append(table[r][pos // page_len] * page_len + pos % page_len)
            positions.append(pos)
        first.append(first[-1] + max(0, a))
    pad = [-1] * (max_tokens - total)
    return True, ends, first, slots + pad, positions + pad, taken, len(given)


def rope(x: np.ndarray, positions: np.ndarray, theta: float) -> np.ndarray:
    """rotate_half RoPE of rows [n, heads, 128] in float64 (gen_gqa_wrapper_vectors.py:25-35)."""
    half = x.shape[-1] // 2
    angle = positions[:, None].astype(np.float64) * theta ** (-np.arange(half) / half)
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a, b = x[..., :half].astype(np.float64), x[..., half:].astype(np.float64)
    return np.concatenate([a * c - b * s, a * s + b * c], -1)


def attend(q, k, v, m, seen, *, scale, cap=0.0, slopes=None):
    """Attention of one query row: q [heads, 128], k/v values [keys, kv_heads, 128], position m, visible keys ``seen``
    (a bool array).  Returns the output [heads, 128], the sum of weights times |v| and the largest sum of |q k| terms
    of a visible score (what error bounds are made of)."""
    heads, kv_heads = q.shape[0], k.shape[1]
    out, size = np.zeros((heads, 128)), np.zeros((heads, 128))
    most = 0.0
    p = np.flatnonzero(seen)
    if not len(p):
        return out, size, most
    for h in range(heads):
        kh, vh = k[p, h * kv_heads // heads], v[p, h * kv_heads // heads]
        z = scale * (kh @ q[h])
        if cap:
            z = cap * np.tanh(z / cap)
        if slopes is not None:
            z = z - slopes[h] * np.abs(m - p)
        w = np.exp(z - z.max())
        w /= w.sum()
        out[h], size[h] = w @ vh, w @ np.abs(vh)
        most = max(most, abs(scale) * (np.abs(kh) @ np.abs(q[h])).max())
    return out, size, most

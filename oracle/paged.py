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


def attend_diff(q, k, v, m, seen, lambdas, *, norm_weight=None, eps=1e-5, out_scale=1.0, **scores):
    """Differential attention of one query row: Q heads 2 j and 2 j + 1 are the maps of head j.  Returns the output
    [heads / 2, 128], the bound of what errors of the two maps' products would be a unit of, and :func:`attend`'s terms."""
    maps, size, most = attend(q, k, v, m, seen, **scores)
    lam = np.asarray(lambdas, np.float64)[:, None]
    out, size = maps[0::2] - lam * maps[1::2], size[0::2] + np.abs(lam) * size[1::2]
    if norm_weight is not None:
        rms = np.sqrt((out * out).mean(-1, keepdims=True) + eps)
        w = np.abs(norm_weight)
        # A change d of the row moves the result by d / rms, and by out / rms times that of the root mean square.
        size = w * (size / rms + np.abs(out) / rms ** 2 * np.sqrt((size * size).mean(-1, keepdims=True)))
        out = out / rms * norm_weight
    return out_scale * out, abs(out_scale) * size, most


def plan_eviction(weight, position, lens, evicted, keep, table, free, page_len, capacity, *, max_keep, sinks, recent):
    """The choice of what stays, on arrays and Python lists (``free``, the stack, grows unless the step is refused).
    Returns (ok, take, lens, evicted, requests cut, rows evicted, pages given back)."""
    requests, heads, room = weight.shape
    take = np.full((requests, heads, max_keep), -1, np.int64)
    ceil = lambda n: -(-n // page_len)  # noqa: E731
    after = [min(k, max_keep) if 0 < min(k, max_keep) < n else n for n, k in zip(lens, keep)]
    given = [p for r in range(requests) for p in table[r][ceil(after[r]):ceil(max(0, lens[r]))]]
    if any(n < 0 or ceil(n) > len(table[0]) or n > room for n in lens) or len(free) + len(given) > capacity:
        return False, take, list(lens), list(evicted), 0, 0, 0
    free.extend(given)
    for r in range(requests):
        n, k = lens[r], after[r]
        if k == n:
            continue
        for h in range(heads):
            def mark(i):
                w = float(weight[r, h, i])
                p = int(position[r, h, i])
                spared = p < sinks or p >= n + max(evicted[r], 0) - recent
                return (not spared, math.isfinite(w) or not math.isnan(w), -max(w, 0.0) if not math.isnan(w) else 0.0, i)
            stays = set(sorted(range(n), key=mark)[:k])
            holes = [i for i in range(k) if i not in stays]
            fills = [i for i in range(k, n) if i in stays]
            take[r, h, holes] = fills
    gone = [n - k for n, k in zip(lens, after)]
    return (True, take, after, [e + g for e, g in zip(evicted, gone)], sum(g > 0 for g in gone), sum(gone), len(given))


def evict(codes, scale, take, lens, table, page_len, code):
    """The move in one of K and V: ``codes`` [pages, heads, page_len, 128] (values in 64 bits) and ``scale`` [pages,
    heads], changed in place."""
    before, held = codes.copy(), scale.copy()
    top = CODE_MAX[code]
    requests, heads, max_keep = take.shape
    for r in range(requests):
        for column in range(-(-min(max_keep, lens[r]) // page_len)):
            to = table[r][column]
            for h in range(heads):
                rows = [(i, take[r, h, column * page_len + i]) for i in range(page_len)
                        if column * page_len + i < max_keep and take[r, h, column * page_len + i] >= 0]
                if not rows:
                    continue
                moves = {i: (table[r][s // page_len], s % page_len) for i, s in rows}
                values = {i: before[p, h, s] * np.float64(held[p, h]) for i, (p, s) in moves.items()}
                most = max(np.abs(x).max() for x in values.values())
                now = np.float64(np.float32(max(held[to, h], most / top, MIN_SCALE)))
                if now > held[to, h]:
                    codes[to, h] = round_code(before[to, h] * np.float64(held[to, h]) / now, code)
                for i, x in values.items():
                    codes[to, h, i] = round_code(x / now, code)
                scale[to, h] = now


def round_code(y, code):
    """The nearest code's value; of two as near the even one."""
    if code == "int8":
        return np.clip(np.rint(y), -127, 127)
    grid = np.unique(E4M3[np.isfinite(E4M3)])
    at = np.clip(np.searchsorted(grid, y), 1, len(grid) - 1)
    lo, hi = grid[at - 1], grid[at]
    even = lambda x: (np.abs(x) / 2.0 ** np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -9))) - 3, -9)) % 2 == 0  # noqa: E731
    return np.where(y - lo < hi - y, lo, np.where(y - lo > hi - y, hi, np.where(even(lo), lo, hi)))

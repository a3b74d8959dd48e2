"""What a paged cache holds and its attention, in float64, for the tests: the
quantizer belongs to the definition and is applied to the f16 values.

How far a kernel may be off, in units of the largest value of V that a row
sees: the queries and probabilities carry 22 bits or more (a pair of f16
values; three int8 digits carry 24), so with e = 2^-22 a score
s = scale * sum(q k) is off by at most

    d = e * scale * max|q| * sum|k|   (the query's rounding, at worst on every element)
      + 4 e * |s|max                  (f32 steps on the score, its difference from the maximum, exp2's argument)

and a probability relative to its block's largest by 2^d - 1 <= d (d < 1) plus
its own rounding e; numerator and denominator each carry that, and their f32
sums n 2^-24 for n sums one after another (blocks a wave, waves, chunks)."""

import numpy as np

BLOCK = 64


def f16(rows):
    """As the cache holds a value: f16, NaN where that is not finite."""
    with np.errstate(over="ignore"):
        h = np.asarray(rows, np.float32).astype(np.float16).astype(np.float64)
    return np.where(np.isfinite(h), h, np.nan)


def held(rows):
    """rows (tokens, heads, hd) as held: full blocks through their codes."""
    h = f16(rows)
    out = h.copy()
    for at in range(0, h.shape[0] // BLOCK * BLOCK, BLOCK):
        for g in range(h.shape[1]):
            b = h[at:at + BLOCK, g]
            a = np.max(np.abs(b))
            if np.isnan(b).any():
                out[at:at + BLOCK, g] = np.nan
            elif a == 0:
                out[at:at + BLOCK, g] = 0
            else:
                scale = np.float32(a) / np.float32(127)
                out[at:at + BLOCK, g] = (np.rint(127.0 * b / a).astype(np.int8).astype(np.float32) * scale).astype(np.float64)
    return out


def attention(q, k, v, seen, scale):
    """q (rows, heads, hd); k, v (tokens, kv_heads, hd) as held; row r sees its
    first seen[r] tokens. The result, and the bound above for each (row, head)."""
    rows, heads, hd = q.shape
    group = heads // k.shape[1]
    out, off = np.zeros((rows, heads, hd)), np.zeros((rows, heads, 1))
    e = 2.0 ** -22
    for h in range(heads):
        kk, vv = k[:, h // group], v[:, h // group]
        if len(kk) == 0:
            continue
        size = np.abs(kk).sum(axis=1)
        scores = scale * (q[:, h].astype(np.float64) @ kk.T)
        for r in range(rows):
            n = int(seen[r])
            if n == 0:
                continue
            s = scores[r, :n]
            p = np.exp(s - np.max(s))
            # A NaN value counts however small its probability is.
            out[r, h] = (p / p.sum()) @ vv[:n]
            d = e * scale * np.max(np.abs(q[r, h])) * np.max(size[:n]) + 4 * e * np.max(np.abs(s))
            vmax = np.nanmax(np.abs(vv[:n])) if not np.isnan(vv[:n]).all() else 0.0
            off[r, h] = vmax * (2 * (d + e) + (n / BLOCK + 24) * 2.0 ** -23)
    # Where every key's score is NaN the result is, and the bound says nothing.
    return out, np.nan_to_num(off)

"""Attention over the 8-bit cache in 64 bits, with a bound on what each kernel's
own arithmetic may add to a row.

The bound follows the kernels' roundings, computed for the row at hand instead of at their worst.
  Query: held in 3 bytes (2 for 16-bit rows of the prompt kernel) under a power of two.  What that
    does to each score is computed exactly; three bytes also drop up to 2^8 steps times the K scale.
  Scores: six FP32 roundings of |s| and of the maximum, 2^-21 of their sum; exponential 2^-22.
  Weights: bytes of the few-column kernel, half a step 2^-24 of the page's largest; f16 of the
    prompt kernel, 2^-11 of the weight (bfloat16 rows) or 2^-22 (two f16), and what rounds to 0 among them, 2^-22
    (2^-26) of the page's largest.  The relative part is taken as independent (6 times the root of the sum of squares),
    the other at its worst, weight by weight.
  Sums in FP32 round once a page (and a few times at the end), by 2^-24 of sum p |v| at most: (8 + 4 sqrt(pages))
    times that where the roundings fall to either side, (8 + pages) times where what is added is alike in all pages.
  Output: half a step of its type, and FP32's or float16's smallest numbers.
"""
import numpy as np

import kv8_ref as R

TINY = {"float32": 2.0 ** -124, "float16": 2.0 ** -25, "bfloat16": 2.0 ** -124}


def query_bytes(kernel, dtype):
    return 2 if kernel == "prompt" and dtype != "float32" else 3


def held_query(q, n):
    """q [..., dim] as n signed bytes a value under a power of two, and that step."""
    bits = 8 * n - 1
    most = 2.0 ** bits - 1 - (0x8080 if n == 3 else 0x80 if n == 2 else 0)
    mx = np.abs(q).max(-1, keepdims=True)
    e = bits - np.frexp(mx)[1]
    e = np.where(np.ldexp(mx, e) > most, e - 1, e)
    step = np.ldexp(1.0, -e)
    return np.rint(q / step) * step, step


def attend(c, table, n, pos, q, scale, causal, window, g, dtype, kernel, alike=False):
    """out, lse of rows q [rows][heads][dim] at positions pos, and the bounds of both (alike: see above)."""
    rows, heads, d = q.shape
    n = min(n, len(table) * R.PAGE)
    out, lse = np.zeros((rows, heads, d)), np.full((rows, heads), -np.inf)
    tol, ltol = np.zeros((rows, heads, d)), np.zeros((rows, heads))
    qb = query_bytes(kernel, dtype)
    if kernel == "few":
        rel, floor = 0.0, 2.0 ** -24
    else:
        rel, floor = (2.0 ** -11, 2.0 ** -22) if dtype == "bfloat16" else (2.0 ** -22, 2.0 ** -26)
    page = np.arange(n) // R.PAGE
    for h in range(heads):
        k, v, _, there = c.gather(table, n, h // g)
        sk = c.scales[table[page], h // g, 0].astype(np.float64)
        qh, step = held_query(q[:, h], qb)
        for r in range(rows):
            p0 = pos[r]
            a = max(0, p0 - window + 1) if window else 0
            b = min(n, p0 + 1) if causal else n
            if p0 < 0 or a >= b:
                continue
            assert there[a:b].all()
            s = (k[a:b] @ q[r, h]) * scale
            eps = np.abs((k[a:b] @ (qh[r] - q[r, h])) * scale)
            if qb == 3:
                eps += abs(scale) * sk[a:b] * 256 * step[r]
            eps += 2.0 ** -21 * (np.abs(s) + np.abs(s).max()) + 2.0 ** -22
            top = s.max()
            p = np.exp(s - top)
            lse[r, h] = top + np.log(p.sum())
            p /= p.sum()
            largest = np.maximum.reduceat(p, np.unique(page[a:b], return_index=True)[1])[page[a:b] - page[a]]
            x = v[a:b]
            out[r, h] = p @ x
            ax = np.abs(x)
            pages = page[b - 1] - page[a] + 1
            sums = (8 + (pages if alike else 4 * np.sqrt(pages))) * 2.0 ** -24
            tol[r, h] = (p * eps) @ np.abs(x - out[r, h]) + np.minimum(p, floor * largest) @ ax
            tol[r, h] += 6 * rel * np.sqrt((p ** 2) @ (x / max(ax.max(), 1e-300)) ** 2) * max(ax.max(), 1e-300)
            tol[r, h] += sums * (p @ ax) + R.EPS[dtype] * np.abs(out[r, h]) + TINY[dtype]
            ltol[r, h] = p @ eps + sums + 2.0 ** -22 * abs(lse[r, h])
    return out, lse, 1.05 * tol, 1.05 * ltol


def within(got, out, tol):
    """Whether every element is inside its bound (the same ones infinite, none NaN)."""
    fine = np.isfinite(out)
    return bool(np.array_equal(got[~fine], out[~fine]) and (np.abs(got[fine] - out[fine]) <= tol[fine]).all())

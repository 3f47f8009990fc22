"""Plain restatements in 64 bits of attention with sinks, gathered attention
weights, eviction and the verification of drafts."""
import numpy as np

import kv8_ref as R
from kv8_bounds import held_query


def sees(n, pos, causal, window, sinks):
    """[rows][tokens]: whether a row at a position sees a token."""
    j, p = np.arange(n)[None], np.asarray(pos)[:, None]
    see = np.repeat(p >= 0, n, 1)
    if causal:
        see = see & (j <= p)
    if window:
        see = see & ((j > p - window) | (j < sinks))
    return see


def attention(c, table, n, pos, q, scale, causal, window, sinks, g):
    """kv8_ref.attention with sinks: out, lse, and the size of each row's scores."""
    rows, heads, d = q.shape
    n = min(n, len(table) * R.PAGE)
    out, lse, err = np.zeros((rows, heads, d)), np.full((rows, heads), -np.inf), np.zeros((rows, heads))
    see = sees(n, pos, causal, window, sinks)
    for h in range(heads):
        k, v, bad, there = c.gather(table, n, h // g)
        s = (q[:, h] @ k.T) * scale
        size = np.abs(q[:, h]).max(1)[:, None] * np.abs(k).sum(1)[None] * abs(scale)
        for r in range(rows):
            m = see[r] & there
            if not m.any():
                continue
            if (bad & m).any():
                out[r, h], lse[r, h] = np.nan, np.nan
                continue
            p = np.exp(s[r, m] - s[r, m].max())
            out[r, h] = p @ v[m] / p.sum()
            lse[r, h] = s[r, m].max() + np.log(p.sum())
            err[r, h] = size[r, m].max()
    return out, lse, err


def gained(c, table, n, pos, q, lse, scale, causal, window, sinks, g):
    """What the rows give each token [kv heads][tokens], and a bound on what the kernels' roundings change.

    A score is off by what holding the query in three bytes does to it (or, as two f16 a value, 2^-22 of each
    product), by 2^-17 of the sum of its products' sizes (128 dims, each sum rounded to 2^-24), and by 2^-21 of itself and of
    lse, which are scaled to units of log2; the exponential adds 2^-21, the sum 2^-24 a term."""
    rows, heads, d = q.shape
    n = min(n, len(table) * R.PAGE)
    see = sees(n, pos, causal, window, sinks)
    w, tol = np.zeros((heads // g, n)), np.zeros((heads // g, n))
    for h in range(heads):
        k, _, _, there = c.gather(table, n, h // g)
        sk = np.array([c.scales[t, h // g, 0] if 0 <= t < len(c.k) else 0.0 for t in table], np.float64)[np.arange(n) // R.PAGE]
        fine = np.isfinite(lse[:, h])
        m = see & fine[:, None] & there[None]
        qh = np.where(fine[:, None], q[:, h], 0.0)
        held, step = held_query(qh, 3)
        s = (qh @ k.T) * scale
        e = np.where(m, np.exp(np.where(m, s - np.where(fine, lse[:, h], 0.0)[:, None], 0.0)), 0.0)
        eps = np.abs((held - qh) @ k.T * scale) + abs(scale) * sk[None] * 256 * step
        eps = eps + (np.abs(qh) @ np.abs(k).T) * abs(scale) * (2.0 ** -17 + 2.0 ** -22)
        eps = eps + 2.0 ** -21 * (np.abs(s) + np.abs(np.where(fine, lse[:, h], 0.0))[:, None] + 1)
        w[h // g] += e.sum(0)
        tol[h // g] += (e * np.expm1(np.minimum(eps, 1.0))).sum(0)
    return w, tol + w * (rows * g + 8) * 2.0 ** -24


def kept_tokens(weights, n, budget, first, recent):
    """Ascending ids of the tokens that a head keeps of n."""
    if n <= budget:
        return np.arange(n)
    mid = np.arange(first, n - recent)
    w = np.asarray(weights, np.float64)[mid]
    w = np.where(np.isnan(w), -np.inf, w)
    below = np.isnan(np.asarray(weights, np.float64)[mid])  # NaN below -inf
    order = np.lexsort((mid, below, -w))
    best = mid[order][:budget - first - recent]
    return np.sort(np.concatenate([np.arange(first), best, np.arange(n - recent, n)])).astype(np.int64)


def evict(c, weights, table, lens, slots, budget, first, recent):
    """Changes a copy of the cache c (k, v, scales, bad) and weights as the operator does: those, kept, lens."""
    k, v, scales, bad, wout = c.k.copy(), c.v.copy(), c.scales.copy(), c.bad.copy(), weights.copy()
    hk = k.shape[1]
    kept = np.full((len(lens), hk, budget), -1, np.int32)
    out = np.array(lens, np.int32).copy()
    for i, n in enumerate(lens):
        n = min(max(n, 0), table.shape[1] * R.PAGE)
        if n == 0:
            continue
        slot = slots[i]
        if not 0 <= slot < len(table):
            continue
        pages = table[slot, :-(-n // R.PAGE)]
        if ((pages < 0) | (pages >= len(k))).any():
            continue
        for h in range(hk):
            w = weights[pages, h].reshape(-1)[:n]
            tok = kept_tokens(w, n, budget, first, recent)
            kept[i, h, :len(tok)] = tok
            if n <= budget:
                continue
            for p in range(-(-budget // R.PAGE)):
                here = tok[p * R.PAGE:(p + 1) * R.PAGE]
                src, at, to, m = pages[here // R.PAGE], here % R.PAGE, pages[p], len(here)
                old = c.scales[src, h]
                new = old.max(0)
                with np.errstate(invalid="ignore", divide="ignore"):
                    ratio = np.where(new > 0, old / new, np.float32(0)).astype(np.float32)
                again = lambda x, r: np.clip(np.rint(x.astype(np.float32) * r), -127, 127).astype(np.int8)  # noqa: E731
                k[to, h, :m] = again(c.k[src, h, at], ratio[:, :1])
                v[to, h, :, :m] = again(c.v[src, h, :, at], ratio[:, 1:]).T
                scales[to, h] = new
                bits = sum(((int(c.bad[s, h]) >> int(a)) & 1) << x for x, (s, a) in enumerate(zip(src, at)))
                bad[to, h] = bits
                wout[to, h, :m] = w[here]
        if n > budget:
            out[i] = budget
    return k, v, scales, bad, wout, kept, out


def verify(logits, draft_logits, cu, drafts, accept_at, sample_at, temperature):
    """accepted and tokens, as the operator's definition has them."""
    def dist(x):
        if np.isnan(x).any() or (x == np.inf).any() or (x == -np.inf).all():
            return None
        if temperature == 0:
            return x
        p = np.exp((x - x.max()) / temperature)
        return p / p.sum()

    n = len(cu) - 1
    accepted, tokens = np.zeros(n, np.int32), np.full(n, -1, np.int32)
    for i in range(n):
        a, b = cu[i], cu[i + 1]
        while True:
            t = accepted[i]
            p = dist(logits[a + i + t])
            if p is None:
                break
            if a + t == b:
                r = p
            else:
                x = drafts[a + t]
                known = 0 <= x < logits.shape[1]
                if temperature == 0:
                    if x == np.argmax(p):
                        accepted[i] += 1
                        continue
                    r = p
                else:
                    q = None if draft_logits is None else dist(draft_logits[a + t])
                    if draft_logits is not None and q is None:
                        break
                    qx = 1.0 if q is None else q[x] if known else 0.0
                    assert not known or accept_at[a + t] * qx == 0 or abs(accept_at[a + t] * qx - p[x]) > 1e-6 * p[x]
                    if known and accept_at[a + t] * qx < p[x]:
                        accepted[i] += 1
                        continue
                    r = p.copy()
                    if q is not None:
                        r = np.maximum(p - q, 0)
                    elif known:
                        r[x] = 0
                    if r.sum() == 0:
                        r = p
            if temperature == 0:
                tokens[i] = np.argmax(p)
            else:
                c = np.cumsum(r)
                assert sample_at[i] == 0 or np.abs(c - sample_at[i] * c[-1]).min() > 1e-12 * c[-1]
                past = np.flatnonzero((c > sample_at[i] * c[-1]) & (r > 0))
                tokens[i] = past[0] if len(past) else np.flatnonzero(r > 0)[-1]
            break
    return accepted, tokens

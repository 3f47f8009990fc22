"""Plain restatements in 64 bits of the 8-bit paged key/value cache, attention
over it and the log probabilities of given tokens, and the arrays the tests
hand to the operators."""
import numpy as np

import codon_hip as ch
from codon_hip.devmem import DeviceArray

PAGE = 64
EPS = {"float32": 2.0 ** -24, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}  # half a step, relative


def bf16_bits(x):
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(np.asarray(x, np.float32)), np.uint16(0x7FC0), r)


def rounded(x, dtype):
    """x in the element type, as float64."""
    if dtype == "bfloat16":
        return (bf16_bits(x).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return np.asarray(x, np.float32).astype(dtype).astype(np.float64)


class View:
    """A strided window on a device array."""

    def __init__(self, base, offset, shape, stride):
        item = 4 if base.dtype == "float32" else 2
        self.base, self.shape, self._stride, self.dtype = base, tuple(shape), tuple(stride), base.dtype
        self._at = base.data_ptr() + offset * item

    def data_ptr(self):
        return self._at

    def stride(self):
        return self._stride


def put(hip, x, dtype):
    """x rounded to dtype on the device."""
    if dtype == "bfloat16":
        return DeviceArray(hip, bf16_bits(x), "bfloat16")
    return DeviceArray(hip, np.asarray(x, np.float32).astype(dtype))


def get(a):
    x = a.numpy()
    if a.dtype == "bfloat16":
        return (x.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return x.astype(np.float64)


class Cache:
    """A cache on the device, its contents made here."""

    def __init__(self, hip, rng, n_pages, heads, head_dim, fill=True):
        d = ch.Kv8Cache.dims(head_dim)
        self.hip, self.h, self.d = hip, heads, head_dim
        lo, hi = (-127, 128) if fill else (0, 1)
        self.k = rng.integers(lo, hi, (n_pages, heads, PAGE, d)).astype(np.int8)
        self.v = rng.integers(lo, hi, (n_pages, heads, d, PAGE)).astype(np.int8)
        self.k[..., head_dim:], self.v[:, :, head_dim:] = 0, 0
        self.scales = rng.uniform(0.01, 0.04, (n_pages, heads, 2)).astype(np.float32)
        self.bad = np.zeros((n_pages, heads), np.uint64)

    def upload(self):
        self.dev = [DeviceArray(self.hip, x) for x in (self.k, self.v, self.scales, self.bad)]
        self.cache = ch.Kv8Cache(*self.dev, self.d)
        return self.cache

    def download(self):
        return [x.numpy() for x in self.dev]

    def values(self, page, head):
        """K and V of a page's tokens as [64][head_dim]."""
        k = self.k[page, head, :, :self.d].astype(np.float64) * np.float64(self.scales[page, head, 0])
        v = self.v[page, head, :self.d].T.astype(np.float64) * np.float64(self.scales[page, head, 1])
        return k, v

    def gather(self, table, n, head):
        """K, V, bad of n tokens; tokens of pages outside the cache: None there (mask)."""
        k, v = np.zeros((n, self.d)), np.zeros((n, self.d))
        bad, there = np.zeros(n, bool), np.zeros(n, bool)
        for t0 in range(0, n, PAGE):
            page = table[t0 // PAGE]
            m = min(PAGE, n - t0)
            if 0 <= page < len(self.k):
                a, b = self.values(page, head)
                k[t0:t0 + m], v[t0:t0 + m] = a[:m], b[:m]
                bad[t0:t0 + m] = (int(self.bad[page, head]) >> np.arange(m).astype(object)).astype(object) % 2 == 1
                there[t0:t0 + m] = True
        return k, v, bad, there


def free(*arrays):
    for a in arrays:
        a.free()


def tables(rng, lens, n_pages, max_pages=None, rows=None):
    """Page tables of sequences of these lengths, pages in no order."""
    need = [-(-n // PAGE) for n in lens]
    order = rng.permutation(n_pages)
    t = np.full((rows or len(lens), max_pages or max(need + [1])), -1, np.int32)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = order[at:at + n]
        at += n
    assert at <= n_pages
    return t


def rope(x, pos, r):
    """x [rows][heads][dims] turned by positions pos, in 64 bits."""
    f = np.asarray(r.freq)
    half = len(f)
    a = pos[:, None, None] * f
    c, s = np.cos(a) * float(np.float32(r.gain)), np.sin(a) * float(np.float32(r.gain))
    y = x.copy()
    i0, i1 = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if r.struct.interleaved else (slice(0, half), slice(half, 2 * half))
    y[..., i0], y[..., i1] = x[..., i0] * c - x[..., i1] * s, x[..., i1] * c + x[..., i0] * s
    return y


def attention(cache, table, n, pos, q, scale, causal, window, g):
    """Rows q [rows][heads][dim] at positions pos over n tokens: out, lse and a
    bound on |out|'s error of scores and weights rounded as the kernels may."""
    rows, heads, d = q.shape
    n = min(n, len(table) * PAGE)
    out, lse = np.zeros((rows, heads, d)), np.full((rows, heads), -np.inf)
    err = np.zeros((rows, heads))
    j = np.arange(n)
    for h in range(heads):
        k, v, bad, there = cache.gather(table, n, h // g)
        s = (q[:, h] @ k.T) * scale
        size = np.abs(q[:, h]).max(1)[:, None] * np.abs(k).sum(1)[None] * abs(scale)
        see = there[None] & (pos[:, None] >= 0) & np.ones((rows, 1), bool)
        if causal:
            see = see & (j[None] <= pos[:, None])
        if window:
            see = see & (j[None] > pos[:, None] - window)
        for r in range(rows):
            m = see[r]
            if not m.any():
                continue
            if (bad & m).any():
                out[r, h], lse[r, h] = np.nan, np.nan
                continue
            x = s[r, m]
            p = np.exp(x - x.max())
            out[r, h] = p @ v[m] / p.sum()
            lse[r, h] = x.max() + np.log(p.sum())
            err[r, h] = size[r, m].max()
    return out, lse, err


def logprobs(x, targets, k):
    """log p(target), entropy, ids and log p of the k largest (ties: lowest id), in 64 bits."""
    n, vocab = x.shape
    lp, en = np.zeros(n), np.zeros(n)
    ids, top = np.full((n, k), -1), np.full((n, k), -np.inf)
    for r in range(n):
        row, t = x[r], None if targets is None else targets[r]
        if np.isnan(row).any() or (row == np.inf).any():
            lp[r], en[r], top[r] = np.nan, np.nan, np.nan
            if t is not None and t < 0:
                lp[r] = 0
            continue
        fine = row > -np.inf
        lse = -np.inf
        if fine.any():
            m = row[fine].max()
            lse = m + np.log(np.exp(row[fine] - m).sum())
            p = np.exp(row[fine] - lse)
            en[r] = -(p * (row[fine] - lse)).sum()
        if t is not None:
            lp[r] = 0 if t < 0 else np.nan if t >= vocab else -np.inf if not fine.any() else row[t] - lse
        order = np.argsort(-row, kind="stable")[:k]
        order = order[row[order] > -np.inf]
        ids[r, :len(order)], top[r, :len(order)] = order, row[order] - lse
    return lp, en, ids, top

"""Attention with sinks, gathered attention weights, eviction and shifted positions
over the 8-bit cache on the GPU, against the restatements in 64 bits.

Attention's tolerance is that of attention without sinks (test_gpu_kv8), the
weights' is derived in kv8_more_ref.gained, eviction is exact: ids are whole numbers, a
code's new value is one FP32 product and one rounding, which numpy does alike.
"""
import numpy as np
import pytest

import codon_hip as ch
import kv8_more_ref as M
import kv8_ref as R
from codon_hip.devmem import DeviceArray, Hip
from test_gpu_kv8 import check_attention

pytestmark = pytest.mark.gpu
TYPES = ["float32", "float16", "bfloat16"]


@pytest.fixture(scope="module")
def hip():
    return Hip()


def offsets(rows):
    return np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)


class Case:
    """A filled cache, its sequences, and a batch of rows over them."""

    def __init__(self, hip, rng, lens, rows, hk, g, d, dtype, change=None, slots=False, max_pages=None, spare=3):
        self.hip, self.lens, self.rows, self.d, self.g, self.dtype = hip, lens, rows, d, g, dtype
        self.c = R.Cache(hip, rng, sum(-(-n // R.PAGE) for n in lens) + 2, hk, d)
        n = len(lens)
        self.table = R.tables(rng, lens, len(self.c.k), max_pages, rows=2 * n if slots else None)
        self.slot = np.arange(n, dtype=np.int32)
        if slots:
            self.slot = rng.permutation(2 * n).astype(np.int32)[:n]
            moved = np.full_like(self.table, -1)
            moved[self.slot] = self.table[:n]
            self.table = moved
        if change:
            change(self.c, self.table)
        self.cu = offsets(rows)
        self.n, self.h = int(self.cu[-1]) + spare, hk * g
        self.q = R.rounded(rng.standard_normal((self.n, self.h, d)) * 2, dtype)
        width = (self.h + 2 * hk) * d  # Q within rows of Q | K | V
        self.base = R.put(hip, np.concatenate([self.q.reshape(self.n, -1), np.full((self.n, 2 * hk * d), 9.0)], 1), dtype)
        self.qv = R.View(self.base, 0, (self.n, self.h, d), (width, d, 1))
        self.arr = [DeviceArray(hip, x) for x in (self.cu, np.asarray(lens, np.int32), self.table, self.slot)]
        self.cache = self.c.upload()
        self.batch = ch.Kv8Batch(*self.arr[:3], self.n, max(rows), self.arr[3] if slots else None)

    def parts(self):
        for i, (m, r) in enumerate(zip(self.lens, self.rows)):
            if r:
                yield i, m, slice(int(self.cu[i]), int(self.cu[i + 1])), np.arange(m - r, m), self.table[self.slot[i]]

    def free(self):
        R.free(self.base, *self.arr, *self.c.dev)


# ---- attention with sinks -----------------------------------------------------------------

def run_sinks(hip, rng, lens, rows, hk, g, d, dtype, window, sinks, causal=True, change=None, **kw):
    x = Case(hip, rng, lens, rows, hk, g, d, dtype, change, **kw)
    mark = 7.0
    out, lse = R.put(hip, np.full((x.n, x.h, d), mark), dtype), DeviceArray(hip, np.full((x.n, x.h), mark, np.float32))
    ws = DeviceArray(hip, np.full(x.cache.attend_workspace(x.batch, x.h) + 16, 255, np.uint8))
    x.cache.attend(x.batch, x.qv, out, lse=lse, causal=causal, window=window, sinks=sinks, workspace=ws)
    got, glse, used = R.get(out), R.get(lse), np.zeros(x.n, bool)
    for i, m, a, pos, table in x.parts():
        used[a] = True
        ref, rlse, err = M.attention(x.c, table, m, pos, x.q[a], d ** -0.5, causal, window, sinks, g)
        check_attention(got[a], glse[a], ref, rlse, err, dtype, 127 * float(np.nanmax(x.c.scales)))
    assert (got[~used] == mark).all() and (glse[~used] == mark).all()
    R.free(out, lse, ws)
    x.free()
    return got, glse


@pytest.fixture(params=["0", "1"], ids=["few", "prompt"])
def kernel(request, monkeypatch):
    monkeypatch.setenv("CIH_KV8_PROMPT", request.param)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hk,g,d", [(2, 1, 16), (1, 3, 24), (2, 2, 32), (1, 1, 64), (2, 4, 128)])
def test_sinks_types_and_heads(hip, kernel, hk, g, d, dtype):
    run_sinks(hip, np.random.default_rng(d + g), [1, 64, 333, 0, 200, 700], [1, 3, 1, 0, 90, 20], hk, g, d, dtype, 70, 5)


@pytest.mark.parametrize("window,sinks", [(1, 1), (1, 64), (64, 1), (63, 65), (64, 64), (65, 128), (200, 500), (130, 4),
                                          (1000, 4), (10, 1 << 30), (2147483647, 3), (64, 0)])
def test_sinks_edges(hip, kernel, window, sinks):
    """Sinks that end inside a page, meet the window, pass the sequence or the rows."""
    run_sinks(hip, np.random.default_rng(window % 97 + sinks % 89), [1, 64, 65, 450, 512, 300], [1, 1, 2, 17, 40, 300], 1, 2, 64,
              "float32", window, sinks)


@pytest.mark.parametrize("dtype,d", [("float32", 64), ("bfloat16", 128), ("float16", 32)])
def test_sinks_long_and_split(hip, kernel, dtype, d):
    """Keys split over workgroups, some splits without a page; the gap's pages not in the table."""
    def gap(c, table):
        table[0, 3:40] = -1

    run_sinks(hip, np.random.default_rng(d), [5000, 70, 4097], [2, 1, 5], 2, 2, d, dtype, 1500, 100, change=gap)
    run_sinks(hip, np.random.default_rng(d + 1), [3000, 100], [150, 100], 1, 2, d, dtype, 700, 130)


@pytest.mark.parametrize("causal", [True, False])
def test_sinks_not_causal_slots_and_table_ends(hip, kernel, causal):
    rng = np.random.default_rng(4)
    run_sinks(hip, rng, [300, 65, 200], [7, 65, 1], 2, 2, 64, "float32", 90, 3, causal=causal, slots=True)
    # more tokens than the table's pages, and rows at negative positions
    x = Case(hip, rng, [128, 3], [2, 1], 1, 1, 64, "float32")
    x.arr[1] = DeviceArray(hip, np.array([1000, 3], np.int32))
    out = DeviceArray(hip, np.zeros((x.n, 1, 64), np.float32))
    ws = DeviceArray(hip, np.zeros(x.cache.attend_workspace(x.batch, 1) + 16, np.uint8))
    b = ch.Kv8Batch(*x.arr[:3], x.n, 2)
    x.cache.attend(b, x.qv, out, causal=causal, window=10, sinks=4, workspace=ws)
    ref, _, _ = M.attention(x.c, x.table[0], 1000, np.array([998, 999]), x.q[:2], 64 ** -0.5, causal, 10, 4, 1)
    assert np.allclose(R.get(out)[:2], ref, rtol=1e-4, atol=1e-4)


def test_sinks_bad_tokens(hip, kernel):
    """A bad token between the sinks and the window changes nothing; one among the sinks makes the rows NaN."""
    for token, lost in ((100, False), (2, True)):
        def mark(c, table):
            c.bad[table[0, token // 64], 0] = 1 << (token % 64)
            if not lost:
                c.scales[table[0, 2], 0] = np.nan  # a page that no row sees
        got, lse = run_sinks(hip, np.random.default_rng(1), [400], [20], 1, 1, 64, "float32", 90, 4, change=mark)
        assert np.isnan(got[:20]).all() == lost and np.isnan(lse[:20]).all() == lost


@pytest.mark.parametrize("dtype", TYPES)
def test_sinks_where_they_change_nothing(hip, kernel, dtype):
    """Without a window, and with all of a window's tokens among the sinks, every token is seen, in the same bits."""
    rng = lambda: np.random.default_rng(11)  # noqa: E731
    a = run_sinks(hip, rng(), [500, 77], [30, 1], 2, 2, 64, dtype, 0, 9)
    b = run_sinks(hip, rng(), [500, 77], [30, 1], 2, 2, 64, dtype, 0, 0)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


# ---- gathered weights ---------------------------------------------------------------------

def run_weigh(hip, rng, lens, rows, hk, g, d, dtype, window=0, sinks=0, causal=True, keep=1.0, change=None, lost=(), **kw):
    x = Case(hip, rng, lens, rows, hk, g, d, dtype, change, **kw)
    lse = np.full((x.n, x.h), 3.0, np.float32)
    for i, m, a, pos, table in x.parts():
        lse[a] = M.attention(x.c, table, m, pos, x.q[a], d ** -0.5, causal, window, sinks, g)[1]
    for r, h, value in lost:
        lse[r, h] = value
    was = rng.uniform(0.0, 4.0, x.c.k.shape[:3]).astype(np.float32)
    want, tol = was.astype(np.float64), np.zeros(was.shape)
    if keep == 0:
        was[:] = np.nan  # not read
    for i, m, a, pos, table in x.parts():
        w, t = M.gained(x.c, table, m, pos, x.q[a], lse[a].astype(np.float64), d ** -0.5, causal, window, sinks, g)
        for j in range(w.shape[1]):
            page = table[j // R.PAGE]
            if 0 <= page < len(want):
                old = 0.0 if keep == 0 or j >= pos[0] else keep * was[page, :, j % R.PAGE].astype(np.float64)
                want[page, :, j % R.PAGE] = old + w[:, j]
                tol[page, :, j % R.PAGE] = t[:, j] + 2.0 ** -23 * np.abs(old + w[:, j])
        if keep == 0:  # untouched ones are NaN, as they were
            pass
    if keep == 0:
        touched = np.zeros(was.shape, bool)
        for i, m, a, pos, table in x.parts():
            for j in range(min(m, table.shape[0] * R.PAGE)):
                if 0 <= table[j // R.PAGE] < len(want):
                    touched[table[j // R.PAGE], :, j % R.PAGE] = True
        want = np.where(touched, want, np.nan)
    wt, lv = DeviceArray(hip, was), DeviceArray(hip, lse)
    x.cache.weigh(x.batch, x.qv, lv, wt, causal=causal, window=window, sinks=sinks, keep=keep)
    got = wt.numpy().astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    off = np.abs(np.where(np.isnan(want), 0, got - want))
    assert (off <= tol + 1e-37).all(), (np.argwhere(off > tol)[:5], off.max(), tol[off > tol][:5])
    R.free(wt, lv)
    x.free()
    return got


@pytest.fixture(params=["0", "1"], ids=["few", "prompt"])
def weigh_kernel(request, monkeypatch):
    """The kernel that the sizes choose, and that of many columns for all."""
    monkeypatch.setenv("CIH_KV8_WEIGH", request.param)
    return request.param


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hk,g,d", [(2, 1, 16), (1, 3, 24), (2, 2, 32), (1, 1, 64), (2, 4, 128)])
@pytest.mark.parametrize("keep", [1.0, 0.9, 0.0])
def test_weigh_types_and_heads(hip, weigh_kernel, hk, g, d, dtype, keep):
    run_weigh(hip, np.random.default_rng(d + g), [1, 64, 333, 0, 65, 128], [1, 64, 2, 0, 3, 40], hk, g, d, dtype, keep=keep)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [24, 64, 128])
def test_weigh_prompts_and_long(hip, weigh_kernel, d, dtype):
    run_weigh(hip, np.random.default_rng(d), [700, 131, 1], [700, 131, 1], 2, 2, d, dtype, keep=0.0)
    run_weigh(hip, np.random.default_rng(d + 1), [2300, 900], [3, 1], 1, 8, d, dtype, keep=0.5)
    run_weigh(hip, np.random.default_rng(d + 2), [1500], [200], 1, 1, d, dtype, spare=0)


@pytest.mark.parametrize("window,sinks,causal", [(1, 0, True), (64, 4, True), (65, 100, True), (130, 0, False), (3, 70, False),
                                                 (0, 0, False), (1 << 30, 2, True), (2147483647, 0, False)])
def test_weigh_masks(hip, weigh_kernel, window, sinks, causal):
    run_weigh(hip, np.random.default_rng(window % 91), [300, 64, 450, 10], [150, 1, 9, 10], 1, 2, 32, "float32", window, sinks, causal)
    run_weigh(hip, np.random.default_rng(window % 91), [300, 450], [150, 9], 2, 1, 128, "bfloat16", window, sinks, causal, keep=0.25,
              slots=True)


def test_weigh_lost_rows_missing_pages_bad_tokens(hip, weigh_kernel):
    def edit(c, table):
        c.bad[table[0, 1], 0] = 1 << 5
        c.k[table[0, 1], 0, 5] = 0
        table[0, 2] = -1
        table[1, 0] = 99999

    for dtype in TYPES:
        run_weigh(hip, np.random.default_rng(3), [400, 200], [30, 2], 2, 2, 64, dtype, change=edit,
                  lost=[(3, 0, np.nan), (4, 1, np.inf), (5, 2, -np.inf), (30, 0, np.nan)])


def test_weigh_queries_that_are_not_finite(hip, weigh_kernel):
    """A row whose query is not finite has no lse: it adds nothing."""
    for dtype in TYPES:
        x = Case(hip, np.random.default_rng(8), [200], [40], 1, 1, 64, dtype)
        lse = M.attention(x.c, x.table[0], 200, np.arange(160, 200), x.q[:40], 0.125, True, 0, 0, 1)[1]
        lse = np.concatenate([lse, np.zeros((x.n - 40, 1))]).astype(np.float32)
        x.q[7, 0, 3], x.q[9, 0, 4] = np.nan, np.inf
        lse[7], lse[9] = np.nan, np.nan
        x.base.free()
        q = R.put(hip, x.q, dtype)
        wt, lv = DeviceArray(hip, np.zeros(x.c.k.shape[:3], np.float32)), DeviceArray(hip, lse)
        x.cache.weigh(x.batch, q, lv, wt)
        x.q[7], x.q[9] = 0, 0
        w, tol = M.gained(x.c, x.table[0], 200, np.arange(160, 200), x.q[:40], lse[:40].astype(np.float64), 0.125, True, 0, 0, 1)
        got = wt.numpy()[x.table[0], 0].reshape(-1)[:200]
        assert (np.abs(got - w[0]) <= tol[0] + 1e-37).all()
        x.base = q
        R.free(wt, lv)
        x.free()


def test_weigh_query_sizes(hip, weigh_kernel):
    """Tiny, large and sparse queries: every size of FP32 and float16 that attention takes."""
    for dtype, sizes in (("float32", (1e-30, 1e-3, 300.0, 1e5)), ("float16", (1e-6, 1e-3, 200.0)), ("bfloat16", (1e-30, 300.0))):
        for size in sizes:
            x = Case(hip, np.random.default_rng(8), [130], [33], 1, 1, 64, dtype)
            x.q = R.rounded(np.random.default_rng(9).standard_normal(x.q.shape) * size, dtype)
            x.q[5, 0, 1:] = 0
            scale = 2.0 / size / 8
            lse = M.attention(x.c, x.table[0], 130, np.arange(97, 130), x.q[:33], scale, True, 0, 0, 1)[1]
            lse = np.concatenate([lse, np.zeros((x.n - 33, 1))]).astype(np.float32)
            q = R.put(hip, x.q, dtype)
            wt, lv = DeviceArray(hip, np.zeros(x.c.k.shape[:3], np.float32)), DeviceArray(hip, lse)
            x.cache.weigh(x.batch, q, lv, wt, scale=scale)
            w, tol = M.gained(x.c, x.table[0], 130, np.arange(97, 130), x.q[:33], lse[:33].astype(np.float64), scale, True, 0, 0, 1)
            got = wt.numpy()[x.table[0], 0].reshape(-1)[:130]
            assert (np.abs(got - w[0]) <= tol[0] + 1e-37).all(), (dtype, size)
            R.free(q, wt, lv)
            x.free()


@pytest.mark.parametrize("dtype,small,large", [("float16", 3e-7, 1.0), ("float16", 2e-5, 60000.0), ("bfloat16", 1e-3, 1e37),
                                               ("bfloat16", 1e-37, 1.0), ("float32", 1e-3, 1e3)])
def test_weigh_small_values_beside_large_ones(hip, weigh_kernel, dtype, small, large):
    """A column's large value meets codes of 0, so that its small ones decide (FP32 rows: as far as 2^-22 of the large one holds them)."""
    x = Case(hip, np.random.default_rng(8), [130], [33], 1, 1, 64, dtype)
    R.free(*x.c.dev)
    x.c.k[:, :, :, 0] = 0
    x.cache = x.c.upload()
    q = np.random.default_rng(9).standard_normal(x.q.shape) * small
    q[..., 0] = large
    q = R.rounded(q, dtype)
    if weigh_kernel == "0" or dtype == "float32":
        q[..., 0] = R.rounded(np.array([small * 4]), dtype)  # three bytes hold a row to 2^-22 of its largest value
    scale = 0.25 / small
    lse = M.attention(x.c, x.table[0], 130, np.arange(97, 130), q[:33], scale, True, 0, 0, 1)[1]
    lse = np.concatenate([lse, np.zeros((x.n - 33, 1))]).astype(np.float32)
    dev, wt, lv = R.put(hip, q, dtype), DeviceArray(hip, np.zeros(x.c.k.shape[:3], np.float32)), DeviceArray(hip, lse)
    x.cache.weigh(x.batch, dev, lv, wt, scale=scale)
    # the restatement's bound without the large value, which adds nothing to a score
    q[..., 0] = 0
    w, tol = M.gained(x.c, x.table[0], 130, np.arange(97, 130), q[:33], lse[:33].astype(np.float64), scale, True, 0, 0, 1)
    got = wt.numpy()[x.table[0], 0].reshape(-1)[:130]
    off = (np.abs(got - w[0]) / (4 * tol[0] + 1e-37)).max()
    assert off <= 1, off
    R.free(dev, wt, lv)
    x.free()


# ---- eviction -----------------------------------------------------------------------------

def run_evict(hip, rng, lens, budget, first, recent, hk=2, d=64, slots=False, edit=None, weights=None, inplace=False,
              max_pages=None):
    x = Case(hip, rng, lens, [1] * len(lens), hk, 1, d, "float32", slots=slots, max_pages=max_pages)
    w = np.exp(2 * rng.standard_normal(x.c.k.shape[:3])).astype(np.float32) if weights is None else weights(x.c.k.shape[:3])
    x.c.bad[:] = rng.integers(0, 1 << 62, x.c.bad.shape).astype(np.uint64) & rng.integers(0, 1 << 62, x.c.bad.shape).astype(np.uint64)
    if edit:
        edit(x.c, x.table, w)
    R.free(*x.c.dev, x.arr[2])
    cache = x.c.upload()
    x.arr[2] = DeviceArray(hip, x.table)
    n = len(lens)
    batch = ch.Kv8Batch(*x.arr[:3], x.n, 1, x.arr[3] if slots else None)
    k, v, scales, bad, wout, kept, out = M.evict(x.c, w, x.table, lens, x.slot, budget, first, recent)
    wt = DeviceArray(hip, w)
    wo = wt if inplace else DeviceArray(hip, np.full_like(w, -5.0))
    lo = x.arr[1] if inplace else DeviceArray(hip, np.full(n, -9, np.int32))
    shifts = DeviceArray(hip, np.arange(n).astype(np.int32))
    kp = DeviceArray(hip, np.full((n, hk, budget), -7, np.int32))
    ws = DeviceArray(hip, np.full(cache.evict_workspace(batch, budget), 255, np.uint8))
    cache.evict(batch, wt, budget, first=first, recent=recent, weights_out=None if inplace else wo,
                lens_out=None if inplace else lo, shifts=shifts, kept=kp, workspace=ws)
    gk, gv, gs, gb = x.c.download()
    assert np.array_equal(kp.numpy(), kept), np.argwhere(kp.numpy() != kept)[:4]
    assert np.array_equal(lo.numpy(), out)
    real = np.minimum(np.maximum(lens, 0), x.table.shape[1] * R.PAGE)
    assert np.array_equal(shifts.numpy(), np.arange(n) + np.where(out < real, real - out, 0))
    got = wo.numpy()
    moved = np.zeros(w.shape, bool)
    for i in range(n):
        table = x.table[x.slot[i]]
        for h in range(hk):
            m = (kept[i, h] >= 0).sum()
            for t in range(m):
                page, at = table[t // R.PAGE], t % R.PAGE
                moved[page, h, at] = True
            if out[i] == lens[i]:
                continue
            for t in range(m):  # what is kept
                page, at = table[t // R.PAGE], t % R.PAGE
                assert np.array_equal(gk[page, h, at], k[page, h, at]) and np.array_equal(gv[page, h, :, at], v[page, h, :, at]), (i, h, t)
                assert int(gb[page, h]) >> at & 1 == int(bad[page, h]) >> at & 1
            for p in range(-(-m // R.PAGE)):
                assert np.array_equal(gs[table[p], h], scales[table[p], h])
    assert np.array_equal(got[moved].view(np.uint32), wout[moved].view(np.uint32))
    assert np.array_equal(got[~moved].view(np.uint32), (w if inplace else np.full_like(w, -5.0))[~moved].view(np.uint32))
    # pages of sequences that stay, and of none, are as they were
    left = np.ones(len(gk), bool)
    for i in range(n):
        if out[i] != lens[i]:
            left[x.table[x.slot[i], :-(-budget // R.PAGE)]] = False
    for a, b in ((gk, x.c.k), (gv, x.c.v), (gs, x.c.scales), (gb, x.c.bad)):
        assert np.array_equal(a[left], b[left])
    R.free(wt, shifts, kp, ws)
    if not inplace:
        R.free(wo, lo)
    x.free()


@pytest.mark.parametrize("d", [16, 24, 32, 64, 128])
@pytest.mark.parametrize("budget", [1, 63, 64, 65, 200])
def test_evict_budgets_and_heads(hip, budget, d):
    run_evict(hip, np.random.default_rng(budget + d), [0, 1, 64, 65, 201, 450, 128, 1100], budget, min(4, budget // 2), budget // 3, d=d)


@pytest.mark.parametrize("first,recent", [(0, 0), (100, 0), (0, 100), (40, 60), (99, 0), (0, 99), (1, 1)])
def test_evict_first_and_recent(hip, first, recent):
    run_evict(hip, np.random.default_rng(first), [101, 300, 164, 100, 99], 100, first, recent, inplace=True)


def test_evict_weights_at_the_edges(hip):
    """Ties, zeros of both signs, infinities, NaN, negative and tiny weights."""
    rng = np.random.default_rng(2)
    run_evict(hip, rng, [500, 70], 130, 3, 7, weights=lambda s: np.ones(s, np.float32))
    run_evict(hip, rng, [500, 70], 130, 0, 0, weights=lambda s: rng.integers(0, 3, s).astype(np.float32))
    values = np.array([0.0, -0.0, np.inf, -np.inf, np.nan, -1.0, 1e-40, -1e-40, 3e38], np.float32)
    run_evict(hip, rng, [500, 300, 1200], 140, 2, 5, weights=lambda s: rng.choice(values, s))
    run_evict(hip, rng, [500], 140, 0, 0, weights=lambda s: np.full(s, np.nan, np.float32))
    run_evict(hip, rng, [500], 140, 0, 0, weights=lambda s: np.zeros(s, np.float32) * rng.choice([1, -1], s).astype(np.float32))


def test_evict_scales_at_the_edges(hip):
    """Pages of zeros, scales of FP32's whole range, one that is not finite."""
    def edit(c, table, w):
        c.scales[:] = np.float32(10.0) ** np.random.default_rng(1).integers(-38, 38, c.scales.shape).astype(np.float32)
        c.scales[::3] = 0.0

    run_evict(hip, np.random.default_rng(3), [400, 1000, 64], 150, 4, 30, edit=edit)


def test_evict_slots_missing_pages_and_table_ends(hip):
    def missing(c, table, w):
        table[0, 2] = -1
        table[2, 0] = len(c.k)

    run_evict(hip, np.random.default_rng(5), [300, 300, 300, 500], 128, 4, 30, edit=missing)
    run_evict(hip, np.random.default_rng(6), [300, 20, 300, 500], 128, 4, 30, slots=True, inplace=True)


@pytest.mark.parametrize("n,budget", [(20000, 4000), (9000, 8999), (5000, 64), (8192, 8191), (70000, 3001), (131, 7)])
def test_evict_long(hip, n, budget):
    run_evict(hip, np.random.default_rng(n), [n, 77, n // 2], budget, 4, budget // 3, hk=1, d=32)


@pytest.mark.parametrize("max_pages", [32, 33, 128, 129, 1500])
def test_evict_short_sequences_in_wide_tables(hip, max_pages):
    rng = np.random.default_rng(max_pages)
    run_evict(hip, rng, [300, 0, 1, 1999, 64], 64, 4, 16, max_pages=max_pages)
    run_evict(hip, rng, [1999, 700], 650, 0, 0, max_pages=max_pages, weights=lambda s: rng.integers(0, 2, s).astype(np.float32), inplace=True)


@pytest.mark.parametrize("extra", [0, 63])
@pytest.mark.parametrize("budget,first,recent", [(700, 3, 40), (130, 64, 66), (4000, 0, 3000), (8900, 1, 0)])
def test_evict_long_tables_of_few_and_many_heads(hip, extra, budget, first, recent):
    """Several workgroups choose for a head of few, one for each of many: ties, edges and pages that are not there."""
    def missing(c, table, w):
        table[2, 70] = -1

    rng = np.random.default_rng(budget + extra)
    values = np.array([0.0, -0.0, np.inf, -np.inf, np.nan, -1.0, 1e-40, -1e-40, 3e38, 1.0, 1.0000001], np.float32)
    lens = [9001, 300, 5000, 8900] + [140] * extra
    run_evict(hip, rng, lens, budget, first, recent, d=16, weights=lambda s: rng.choice(values, s), edit=missing)
    run_evict(hip, rng, lens, budget, first, recent, d=16, weights=lambda s: rng.integers(0, 2, s).astype(np.float32), slots=True)


@pytest.mark.parametrize("pattern", ["last", "first", "even", "runs"])
def test_evict_where_the_kept_tokens_lie(hip, pattern):
    """Pages that all wait for one, that wait for none, and that take tokens from many."""
    def weights(shape):
        return np.zeros(shape, np.float32)

    def edit(c, table, w):
        for i, n in enumerate((2000, 4096)):
            j = np.arange(n)
            like = {"last": j, "first": -j, "even": j % 2, "runs": (j // 100) % 3}[pattern]
            w[table[i, j // 64], :, j % 64] = like[:, None]

    run_evict(hip, np.random.default_rng(1), [2000, 4096], 999, 1, 1, d=128, weights=weights, edit=edit)


def test_evict_again_and_again(hip):
    """A sequence at its budget takes 20 tokens and is cut again: its codes follow the restatement, step by step."""
    rng, hk, d, budget = np.random.default_rng(7), 2, 64, 100
    x = Case(hip, rng, [budget], [1], hk, 1, d, "float32", max_pages=2)
    w = rng.uniform(0, 1, x.c.k.shape[:3]).astype(np.float32)
    grown = DeviceArray(hip, np.array([budget + 20], np.int32))
    cu = DeviceArray(hip, np.array([0, 20], np.int32))
    wt, shifts = DeviceArray(hip, w), DeviceArray(hip, np.zeros(1, np.int32))
    batch = ch.Kv8Batch(cu, grown, x.arr[2], 20, 20)
    ws = DeviceArray(hip, np.zeros(x.cache.evict_workspace(batch, budget), np.uint8))
    held = DeviceArray(hip, np.zeros(1, np.int32))
    rope = ch.Rope(d)
    for step in range(4):
        k, v = (R.put(hip, rng.standard_normal((20, hk, d)) * (step + 1), "float32") for _ in range(2))
        x.cache.append(batch, k, v, rope=rope, shifts=shifts)
        x.c.k, x.c.v, x.c.scales, x.c.bad = x.c.download()
        w = wt.numpy()
        w[x.table[0, 1], :, budget - 64:] = rng.uniform(0, 1, (hk, 128 - budget))  # the new tokens'
        hip.h2d(wt.data_ptr(), w)
        want = M.evict(x.c, w, x.table, [budget + 20], [0], budget, 2, 10)
        x.cache.evict(batch, wt, budget, first=2, recent=10, lens_out=held, shifts=shifts, workspace=ws)
        assert held.numpy()[0] == budget and shifts.numpy()[0] == 20 * (step + 1)
        gk, gv, gs, gb = x.c.download()
        for p, m in ((0, 64), (1, budget - 64)):
            page = x.table[0, p]
            assert np.array_equal(gk[page, :, :m], want[0][page, :, :m])
            assert np.array_equal(gv[page, :, :, :m], want[1][page, :, :, :m])
            assert np.array_equal(gs[page], want[2][page])
            assert np.array_equal(wt.numpy()[page, :, :m], want[4][page, :, :m])
        R.free(k, v)
    R.free(grown, cu, wt, shifts, ws, held)
    x.free()


# ---- shifted positions --------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rot,inter", [(64, False), (24, True)])
def test_append_shifted(hip, dtype, rot, inter):
    """K's codes and q at positions of 20 to 10^6 more than their places; without shifts the bits of the call without them."""
    rng, d, hk, lens, rows = np.random.default_rng(rot), 64, 2, [70, 5, 130], [6, 5, 1]
    rope, shift = ch.Rope(rot, interleaved=inter), np.array([20, 1000000, -3], np.int32)
    n = sum(rows)
    got = []
    for call in ("shifted", "zero", "none"):
        rng = np.random.default_rng(rot)
        x = Case(hip, rng, lens, rows, hk, 1, d, dtype, spare=0)
        k, v, q = (R.rounded(rng.standard_normal((n, hk, d)), dtype) for _ in range(3))
        dev = [R.put(hip, a, dtype) for a in (k, v, q)]
        sh = DeviceArray(hip, shift if call == "shifted" else np.zeros(3, np.int32))
        x.cache.append(x.batch, dev[0], dev[1], q=dev[2], rope=rope, shifts=None if call == "none" else sh)
        got.append((R.get(dev[2]), [a.copy() for a in x.c.download()]))
        if call == "shifted":
            gk, gv, gs, _ = x.c.download()
            for i, m, a, pos, table in x.parts():
                want = R.rope(q[a], pos + shift[i], rope)
                assert (np.abs(got[0][0][a] - want) <= R.EPS[dtype] * np.abs(want) + 2.0 ** -20 * np.abs(want).max()).all()
                want = R.rope(k[a], pos + shift[i], rope)
                for r, p in enumerate(pos):
                    page, at = table[p // R.PAGE], p % R.PAGE
                    for h in range(hk):
                        off = np.abs(gk[page, h, at] - want[r, h] / np.float64(gs[page, h, 0]))
                        assert (off <= 0.5 + 1e-3).all()
        R.free(*dev, sh)
        x.free()
    for a, b in zip([got[1][0]] + got[1][1], [got[2][0]] + got[2][1]):
        assert np.array_equal(a, b)

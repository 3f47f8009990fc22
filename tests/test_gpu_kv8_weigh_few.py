"""The attention weight that cached tokens gather from few columns (at most 16 rows
times query heads of a kv head, as in single-token decoding), against the
restatement in 64 bits: both kernels, where a wave takes one page and where it takes many.

The tolerance is kv8_more_ref.gained's, and 2^-23 of a weight for the product with
keep and the sum.
"""
import numpy as np
import pytest

import kv8_more_ref as M
import kv8_ref as R
from codon_hip.devmem import DeviceArray, Hip
from test_gpu_kv8_more import Case

pytestmark = pytest.mark.gpu
TYPES = ["float32", "float16", "bfloat16"]


@pytest.fixture(scope="module")
def hip():
    return Hip()


@pytest.fixture(params=["0", "1"], ids=["few", "many"], autouse=True)
def weigh_kernel(request, monkeypatch):
    """The kernel of few columns, which these sizes choose, and that of many."""
    monkeypatch.setenv("CIH_KV8_WEIGH", request.param)


def weigh(hip, x, window=0, sinks=0, causal=True, keep=1.0, scale=None, lost=(), scales=None):
    """Weighs the rows of x.  lost: (row, head, lse) that add nothing; scales: (page, head, K scale) that only the
    device has, of pages whose tokens gather nothing."""
    assert max(x.rows) * x.g <= 16
    scale = x.d ** -0.5 if scale is None else scale
    lse = np.full((x.n, x.h), 3.0, np.float32)
    for i, m, a, pos, table in x.parts():
        lse[a] = M.attention(x.c, table, m, pos, x.q[a], scale, causal, window, sinks, x.g)[1]
    for r, h, value in lost:
        lse[r, h] = value
    was = np.random.default_rng(1).uniform(0.0, 4.0, x.c.k.shape[:3]).astype(np.float32)
    want, tol = was.astype(np.float64), np.zeros(was.shape)
    if keep == 0:
        was[:], want[:] = np.nan, np.nan  # not read
    odd = {(p, h) for p, h, _ in scales or ()}
    for i, m, a, pos, table in x.parts():
        w, t = M.gained(x.c, table, m, pos, x.q[a], lse[a].astype(np.float64), scale, causal, window, sinks, x.g)
        j = np.arange(w.shape[1])
        page = table[j // R.PAGE]
        there = (page >= 0) & (page < len(want))
        j, page, w, t = j[there], page[there], w[:, there], t[:, there]
        for h in range(len(w)):
            for p, hh in odd:
                if hh == h:
                    w[h, page == p], t[h, page == p] = 0, 0
            old = np.where(j >= pos[0], 0.0, keep * was[page, h, j % R.PAGE].astype(np.float64)) if keep else 0.0
            want[page, h, j % R.PAGE] = old + w[h]
            tol[page, h, j % R.PAGE] = t[h] + 2.0 ** -23 * np.abs(old + w[h])
    if scales:
        s = x.c.scales.copy()
        for p, h, value in scales:
            s[p, h, 0] = value
        hip.h2d(x.c.dev[2].data_ptr(), s)
    wt, lv = DeviceArray(hip, was), DeviceArray(hip, lse)
    x.cache.weigh(x.batch, x.qv, lv, wt, scale=scale, causal=causal, window=window, sinks=sinks, keep=keep)
    got = wt.numpy().astype(np.float64)
    R.free(wt, lv)
    x.free()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    off = np.abs(np.where(np.isnan(want), 0.0, got - want))
    assert (off <= tol + 1e-37).all(), (np.argwhere(off > tol)[:5], off.max(), tol[off > tol][:5])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hk,g,d", [(2, 1, 16), (1, 3, 24), (2, 2, 32), (1, 1, 64), (3, 5, 64), (2, 4, 128), (1, 8, 128), (2, 16, 64)])
@pytest.mark.parametrize("keep", [1.0, 0.9, 0.0])
def test_types_and_heads(hip, hk, g, d, dtype, keep):
    most = 16 // g
    rows = [min(r, most) for r in (1, 16, 2, 0, 3, 1, 16, 5)]
    x = Case(hip, np.random.default_rng(d + g), [1, 64, 333, 0, 65, 128, 700, 5], rows, hk, g, d, dtype)
    weigh(hip, x, keep=keep)


# pages of a workgroup: max_pages * sequences * kv heads / 2048, between 4 and 64; its four waves take them in turn
@pytest.mark.parametrize("dtype,d", [("float32", 16), ("bfloat16", 64), ("float16", 128), ("bfloat16", 24)])
@pytest.mark.parametrize("max_pages", [100, 200, 500, 1500])
def test_several_pages_a_wave(hip, max_pages, dtype, d):
    hk, lens = 8, [6000, 4097, 64, 0, 700, 1, 1500, 640, 2000, 3000, 65, 129]
    rows = [1, 2, 1, 0, 2, 1, 1, 2, 1, 1, 2, 1]

    def missing(c, table):
        table[0, 9], table[1, 0] = -1, len(c.k)

    x = Case(hip, np.random.default_rng(max_pages), lens, rows, hk, 2, d, dtype, change=missing, max_pages=max_pages)
    weigh(hip, x, keep=0.9)


@pytest.mark.parametrize("window,sinks,causal", [(1, 0, True), (64, 4, True), (65, 100, True), (130, 0, False), (3, 70, False), (0, 0, False),
                                                 (1 << 30, 2, True), (2147483647, 0, False), (200, 1 << 30, True)])
def test_masks(hip, window, sinks, causal):
    x = Case(hip, np.random.default_rng(window % 91), [300, 64, 450, 10, 5000], [8, 1, 7, 8, 3], 1, 2, 32, "float32")
    weigh(hip, x, window, sinks, causal)
    x = Case(hip, np.random.default_rng(window % 91), [300, 450, 3], [15, 9, 3], 2, 1, 128, "bfloat16", slots=True)
    weigh(hip, x, window, sinks, causal, keep=0.25)
    x = Case(hip, np.random.default_rng(window % 91), [4100] + [70] * 39, [1] * 40, 4, 1, 16, "float16", max_pages=130)
    weigh(hip, x, window, sinks, causal, keep=0.0)  # 10 pages a workgroup


@pytest.mark.parametrize("dtype", TYPES)
def test_lost_rows_missing_pages_bad_tokens(hip, dtype):
    def edit(c, table):
        c.bad[table[0, 1], 0] = 1 << 5
        c.k[table[0, 1], 0, 5] = 0
        table[0, 2] = -1
        table[1, 0] = 99999

    x = Case(hip, np.random.default_rng(3), [400, 200, 300], [8, 2, 1], 2, 2, 64, dtype, change=edit)
    weigh(hip, x, lost=[(3, 0, np.nan), (4, 1, np.inf), (5, 2, -np.inf), (8, 0, np.nan), (10, 3, np.inf)])


@pytest.mark.parametrize("dtype", TYPES)
def test_queries_that_are_not_finite(hip, dtype):
    """Such a row has no lse, and adds nothing; nor does it where an lse is given."""
    for given in (np.nan, 2.0):
        x = Case(hip, np.random.default_rng(8), [200], [8], 1, 2, 64, dtype)
        x.q[1, 0] = 0
        q = x.q.copy()
        q[3, 0, 3], q[5, 1, 4], q[6, 0, 63] = np.nan, np.inf, -np.inf
        wide = np.concatenate([q.reshape(x.n, -1), np.full((x.n, 2 * x.d), 9.0)], 1)
        x.base.free()
        x.base = R.put(hip, wide, dtype)
        x.qv = R.View(x.base, 0, (x.n, x.h, x.d), (wide.shape[1], x.d, 1))
        # (the restatement takes a row with this lse for lost)
        lost = [(3, 0, np.nan), (5, 1, np.nan), (6, 0, np.nan)]
        if given == given:
            weigh_given(hip, x, lost, given)
        else:
            weigh(hip, x, lost=lost)


def weigh_given(hip, x, lost, given):
    lse = M.attention(x.c, x.table[0], 200, np.arange(192, 200), x.q[:8], 0.125, True, 0, 0, 2)[1]
    none = lse.astype(np.float32).astype(np.float64)
    lse = np.concatenate([lse, np.zeros((x.n - 8, 2))]).astype(np.float32)
    for r, h, value in lost:
        none[r, h], lse[r, h] = value, given
    wt, lv = DeviceArray(hip, np.zeros(x.c.k.shape[:3], np.float32)), DeviceArray(hip, lse)
    x.cache.weigh(x.batch, x.qv, lv, wt)
    w, tol = M.gained(x.c, x.table[0], 200, np.arange(192, 200), x.q[:8], none, 0.125, True, 0, 0, 2)
    got = wt.numpy()[x.table[0], 0].reshape(-1)[:200]
    assert (np.abs(got - w[0]) <= tol[0] + 2.0 ** -23 * w[0] + 1e-37).all()
    R.free(wt, lv)
    x.free()


@pytest.mark.parametrize("dtype,sizes", [("float32", (1e-30, 1e-3, 300.0, 1e5)), ("float16", (1e-6, 1e-3, 200.0)), ("bfloat16", (1e-30, 300.0))])
def test_query_sizes(hip, dtype, sizes):
    """Tiny, large and sparse queries, scales of both signs."""
    for size in sizes:
        for sign in (1, -1):
            x = Case(hip, np.random.default_rng(8), [130, 700], [8, 4], 1, 2, 64, dtype, spare=0)
            x.q = R.rounded(np.random.default_rng(9).standard_normal(x.q.shape) * size, dtype)
            x.q[5, 0, 1:] = 0
            x.base.free()
            x.base = R.put(hip, x.q, dtype)
            x.qv = x.base
            weigh(hip, x, scale=sign * 2.0 / size / 8)


@pytest.mark.parametrize("dtype,small,large", [("float16", 1e-3, 1.0), ("bfloat16", 1e-37, 1e-35), ("float32", 1.0, 1e3)])
def test_small_values_beside_large_ones(hip, dtype, small, large):
    """A column's large value meets codes of 0: its small ones decide, as far as three bytes (two f16) hold them."""
    x = Case(hip, np.random.default_rng(8), [130], [8], 1, 2, 64, dtype, spare=0)
    R.free(*x.c.dev)
    x.c.k[:, :, :, 0] = 0
    x.cache = x.c.upload()
    x.q = np.random.default_rng(9).standard_normal(x.q.shape) * small
    x.q[..., 0] = large
    x.q = R.rounded(x.q, dtype)
    x.base.free()
    x.base = R.put(hip, x.q, dtype)
    x.qv = x.base
    weigh(hip, x, scale=0.25 / small)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, -0.02])
@pytest.mark.parametrize("dtype", TYPES)
def test_pages_whose_scale_is_none(hip, dtype, bad):
    """A page whose K scale is not finite or negative adds nothing to its tokens: hidden by a window, or seen."""
    for window in (0, 100):
        x = Case(hip, np.random.default_rng(6), [700, 90, 1], [2, 1, 1], 2, 2, 64, dtype)
        t = x.table
        weigh(hip, x, window, 3 if window else 0, keep=0.9,
              scales=[(t[0, 3], 0, bad), (t[0, 4], 1, bad), (t[0, 10], 1, bad), (t[1, 0], 0, bad)])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_offsets_past_32_bits(hip, dtype):
    """Codes, weights and rows at byte offsets beyond 2^31 and 2^32: as in a pool of five pages."""
    import codon_hip as ch
    from test_gpu_ops_streams import Raw, same

    d, hk, g, n, held = 128, 4, 2, 2, 300
    rng = np.random.default_rng(8)
    k, v = (R.put(hip, rng.standard_normal((held, hk, d)), dtype) for _ in range(2))
    q = R.put(hip, rng.standard_normal((n, hk * g, d)), dtype)
    full = [DeviceArray(hip, np.array(a, np.int32)) for a in ([0, held], [held])]
    cu = DeviceArray(hip, np.array([0, n], np.int32))
    got = []
    for pages, ids in ((5, [2, 0, 4, 3, 1]), (140000, [139999, 0, 70001, 131071, 139998])):
        arrays = [Raw(hip, (pages, hk, 64, d), "int8"), Raw(hip, (pages, hk, d, 64), "int8"),
                  Raw(hip, (pages, hk, 2), "float32"), Raw(hip, (pages, hk), "uint64"), Raw(hip, (pages, hk, 64), "float32")]
        cache, table = ch.Kv8Cache(*arrays[:4], d), DeviceArray(hip, np.array([ids], np.int32))
        cache.append(ch.Kv8Batch(full[0], full[1], table, held, held), k, v)
        b = ch.Kv8Batch(cu, full[1], table, n, n)
        out, lse = R.put(hip, np.zeros((n, hk * g, d)), dtype), DeviceArray(hip, np.zeros((n, hk * g), np.float32))
        ws = DeviceArray(hip, np.zeros(cache.attend_workspace(b, hk * g) + 16, np.uint8))
        cache.attend(b, q, out, lse=lse, workspace=ws)
        cache.weigh(b, q, lse, arrays[4], keep=0.0)
        cache.weigh(b, q, lse, arrays[4], window=90, sinks=5, keep=0.5)
        hip.sync()
        w = np.empty((5, hk, 64), np.float32)
        for i, page in enumerate(ids):
            one = np.empty((hk, 64), np.float32)
            hip.d2h(one, arrays[4].data_ptr() + page * hk * 64 * 4)
            w[i] = one
        w[4, :, held - 256:] = 0  # (places behind the last token are left as they were)
        got.append([lse.numpy(), w])
        R.free(table, out, lse, ws, *arrays)
    same(*got)
    assert got[0][1].sum() > 0 and (got[0][1] >= 0).all()
    R.free(k, v, q, cu, *full)

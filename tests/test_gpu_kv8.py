"""The 8-bit paged key/value cache on the GPU (cih_kv8_append, cih_kv8_read,
cih_kv8_attention) against the restatement in 64 bits.

Tolerances.  Codes: a rotated value carries at most four roundings of 2^-24 of
|x0| + |x1| <= 2 amax and its scale's and reciprocal's two, below 1e-4 of a code at 127
codes, so |code - x / s| <= 0.5 + 1e-4.  Attention: every product of codes is
exact; a query is held to 2^-21 of its row's largest value (FP32 rows; 2^-13
for 16-bit rows, whose own rounding is 2^-9 or 2^-12), so a score is off by
at most scale max|q| sum|k| times that and 2^-21 of itself, and moves the output by at most twice
that (and the exponential's own 2^-22) of the largest value; a weight is held to 2^-21 (2^-14) of the
largest of its page, whose 64 together move the output by at most 2^-16 (2^-9, 2^-8 with
bfloat16 weights), and sums add 2^-18.
"""
import numpy as np
import pytest

import codon_hip as ch
import kv8_ref as R
from codon_hip.devmem import DeviceArray, Hip

pytestmark = pytest.mark.gpu
LIMB = {"float32": 2.0 ** -21, "float16": 2.0 ** -12, "bfloat16": 2.0 ** -9}
WEIGHT = {"float32": 2.0 ** -16, "float16": 2.0 ** -9, "bfloat16": 2.0 ** -8}


@pytest.fixture(scope="module")
def hip():
    return Hip()


@pytest.fixture(params=["0", "1"], ids=["few", "prompt"])
def kernel(request, monkeypatch):
    """Both kernels, whichever the sizes would choose."""
    monkeypatch.setenv("CIH_KV8_PROMPT", request.param)


def offsets(rows):
    return np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)


def check_attention(got, lse, ref, rlse, err, dtype, vmax):
    nan = np.isnan(ref)
    assert np.array_equal(np.isnan(got), nan) and np.array_equal(np.isnan(lse), np.isnan(rlse))
    assert np.array_equal(np.isneginf(lse), np.isneginf(rlse))
    size = np.where(np.isfinite(rlse), err, 0)
    score = size * (LIMB[dtype] + 2.0 ** -21) + 2.0 ** -22
    tol = (2 * score + WEIGHT[dtype] + 2.0 ** -18)[..., None] * vmax + R.EPS[dtype] * np.abs(np.where(nan, 0, ref))
    bad = ~nan & (np.abs(got - ref) > tol)
    assert not bad.any(), (np.argwhere(bad)[:5], np.abs(got - ref)[bad][:5], tol[bad][:5])
    fine = np.isfinite(rlse)
    d = np.abs(np.where(fine, lse, 0) - np.where(fine, rlse, 0))
    assert (d <= 2 * score + WEIGHT[dtype] + 2.0 ** -22 * np.abs(np.where(fine, rlse, 0)))[fine].all(), d.max()


def run_attention(hip, rng, lens, rows, hk, g, d, dtype, causal=True, window=0, change=None, scale=None, n_pages=None,
                  max_pages=None, spare_rows=3, layout="packed", want_lse=True, slots=False):
    """One call against the restatement; change(cache, table) edits the cache first."""
    need = sum(-(-n // R.PAGE) for n in lens)
    c = R.Cache(hip, rng, n_pages or need + 2, hk, d)
    table = R.tables(rng, lens, len(c.k), max_pages, rows=2 * len(lens) if slots else None)
    slot = np.arange(len(lens), dtype=np.int32)
    if slots:  # sequences in other rows of the table
        slot = rng.permutation(2 * len(lens)).astype(np.int32)[:len(lens)]
        moved = np.full_like(table, -1)
        moved[slot] = table[:len(lens)]
        table = moved
    if change:
        change(c, table)
    cu, h = offsets(rows), hk * g
    n = int(cu[-1]) + spare_rows
    q = R.rounded(rng.standard_normal((n, h, d)) * 2, dtype)
    mark = 7.0
    if layout == "packed":  # Q within rows of Q | K | V
        width = (h + 2 * hk) * d
        qbase = R.put(hip, np.concatenate([q.reshape(n, -1), np.full((n, 2 * hk * d), 9.0)], 1), dtype)
        obase = R.put(hip, np.full((n, h * d + 5), mark), dtype)
        qv, ov = R.View(qbase, 0, (n, h, d), (width, d, 1)), R.View(obase, 5, (n, h, d), (h * d + 5, d, 1))
    else:  # heads first
        qbase, obase = R.put(hip, q.transpose(1, 0, 2), dtype), R.put(hip, np.full((h, n, d), mark), dtype)
        qv, ov = R.View(qbase, 0, (n, h, d), (d, n * d, 1)), R.View(obase, 0, (n, h, d), (d, n * d, 1))
    lse = DeviceArray(hip, np.full((n, h), mark, np.float32))
    arr = [DeviceArray(hip, x) for x in (cu, np.asarray(lens, np.int32), table, slot)]
    cache = c.upload()
    batch = ch.Kv8Batch(arr[0], arr[1], arr[2], n, max(rows), arr[3] if slots else None)
    ws = DeviceArray(hip, np.full(cache.attend_workspace(batch, h) + 16, 255, np.uint8))
    kw = {} if scale is None else {"scale": scale}
    cache.attend(batch, qv, ov, lse=lse if want_lse else None, causal=causal, window=window, workspace=ws, **kw)
    raw = R.get(obase)
    if layout == "packed":
        assert (raw[:, :5] == mark).all(), "elements between the rows were touched"
        got = raw[:, 5:].reshape(n, h, d)
    else:
        got = raw.transpose(1, 0, 2)
    glse = R.get(lse)
    sc = d ** -0.5 if scale is None else scale
    vmax = 127 * float(np.nanmax(c.scales))
    used = np.zeros(n, bool)
    for i, (m, r) in enumerate(zip(lens, rows)):
        if r == 0:
            continue
        a = slice(int(cu[i]), int(cu[i + 1]))
        used[a] = True
        pos = np.arange(m - r, m)
        ref, rlse, err = R.attention(c, table[slot[i]], m, pos, q[a], sc, causal, window, g)
        check_attention(got[a], glse[a] if want_lse else rlse, ref, rlse, err, dtype, vmax)
    assert (got[~used] == mark).all(), "rows behind the last sequence were touched"
    assert (glse[~used] == mark).all() and (want_lse or (glse == mark).all())
    R.free(qbase, obase, lse, ws, *arr, *c.dev)
    return got


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("d,hk,g", [(16, 3, 1), (24, 2, 2), (32, 1, 5), (64, 4, 1), (64, 1, 8), (128, 2, 3), (128, 1, 16)])
def test_steps(hip, kernel, dtype, d, hk, g):
    """One row a sequence, lengths around the pages' ends, an idle stream among them."""
    rng = np.random.default_rng(d + g)
    lens = [1, 2, 63, 64, 65, 0, 127, 128, 129, 300, 1000]
    run_attention(hip, rng, lens, [0 if n == 0 else 1 for n in lens], hk, g, d, dtype, layout="heads")


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("d,hk,g", [(16, 2, 1), (24, 2, 3), (32, 2, 1), (64, 2, 1), (64, 1, 4), (128, 1, 4)])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 50), (False, 33)])
def test_prompts_and_chunks(hip, kernel, dtype, d, hk, g, causal, window):
    """Ragged prompts, chunks behind a context, drafted rows: all masks."""
    rng = np.random.default_rng(d + g + window)
    run_attention(hip, rng, [1, 17, 64, 130, 200, 333, 90], [1, 17, 64, 130, 65, 3, 0], hk, g, d, dtype, causal, window,
                  layout="packed" if g == 1 else "heads")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("window", [0, 700, 1])
def test_long_sequences(hip, kernel, dtype, window):
    """Few rows over many pages: the keys are split and joined again."""
    rng = np.random.default_rng(3)
    run_attention(hip, rng, [9001, 5], [1, 1], 1, 1, 64, dtype, window=window, layout="heads")
    run_attention(hip, rng, [4097, 4500], [2, 7], 1, 4, 128, dtype, window=window, layout="heads")


@pytest.mark.parametrize("rows", [1, 40])
def test_bad_tokens(hip, kernel, rows):
    """A token that is not finite makes the rows that see it NaN, and no other."""
    rng = np.random.default_rng(5)

    def change(c, table):
        c.bad[table[0, 1], 0] = np.uint64(1 << 20)              # token 84 of sequence 0, head 0
        c.bad[table[1, 0], 1] = np.uint64((1 << 63) | 1)        # tokens 0 and 63 of sequence 1, head 1
        c.bad[table[2, 2], 0] = np.uint64(2 ** 64 - 2 ** 22)    # sequence 2: only tokens past its end (150)

    run_attention(hip, rng, [100, 100, 150], [rows] * 3, 2, 1, 32, "float32", change=change, layout="heads")
    run_attention(hip, rng, [100, 100, 150], [rows] * 3, 2, 2, 64, "bfloat16", change=change, window=16, layout="heads")


@pytest.mark.parametrize("rows", [1, 30])
def test_garbage_past_the_end_and_missing_pages(hip, kernel, rows):
    """Codes past a sequence's length, scales of pages it does not own, page ids outside the cache."""
    rng = np.random.default_rng(6)

    def change(c, table):
        table[1, 1] = 10 ** 6
        table[2, 0] = -5
        owned = set(table[0].tolist()) | set(table[1].tolist()) | set(table[2].tolist())
        for p in range(len(c.k)):
            if p not in owned:
                c.scales[p] = np.nan

    run_attention(hip, rng, [70, 190, 64], [rows] * 3, 1, 2, 64, "float32", change=change, n_pages=12, max_pages=5,
                  layout="heads")
    run_attention(hip, rng, [70, 190, 64], [rows] * 3, 2, 1, 16, "float16", causal=False, change=change, n_pages=12,
                  max_pages=5, layout="heads")


def test_rows_before_the_first_position(hip, kernel):
    """A padded batch: more rows than tokens; the rows at negative positions give 0 and -inf."""
    rng = np.random.default_rng(7)
    got = run_attention(hip, rng, [3, 0, 70], [5, 4, 1], 2, 1, 64, "float32", layout="heads")
    assert (got[:2] == 0).all() and (got[5:9] == 0).all()
    run_attention(hip, rng, [3, 0, 70], [5, 4, 1], 2, 1, 64, "float32", causal=False, layout="heads")


def test_lengths_past_the_table(hip, kernel):
    """A length beyond the table's pages reads what the table has."""
    rng = np.random.default_rng(8)
    c = R.Cache(hip, rng, 4, 1, 32)
    table = np.array([[2, 0]], np.int32)
    q = rng.standard_normal((2, 1, 32))
    arr = [DeviceArray(hip, x) for x in (np.array([0, 2], np.int32), np.array([200], np.int32), table)]
    qd, od = R.put(hip, q, "float32"), R.put(hip, q * 0, "float32")
    cache = c.upload()
    b = ch.Kv8Batch(arr[0], arr[1], arr[2], 2, 2)
    ws = DeviceArray(hip, np.zeros(cache.attend_workspace(b, 1) + 16, np.uint8))
    cache.attend(b, qd, od, workspace=ws)
    ref, rlse, err = R.attention(c, table[0], 200, np.array([198, 199]), R.rounded(q, "float32"), 32 ** -0.5, True, 0, 1)
    check_attention(R.get(od), rlse, ref, rlse, err, "float32", 127 * float(c.scales.max()))
    R.free(*arr, qd, od, ws, *c.dev)


def test_slots_shared_pages_and_no_lse(hip, kernel):
    rng = np.random.default_rng(9)
    run_attention(hip, rng, [100, 1, 64], [1, 1, 2], 2, 2, 64, "float16", slots=True, layout="heads", want_lse=False)

    def share(c, table):  # two sequences with the same first page
        table[1, 0] = table[0, 0]

    run_attention(hip, rng, [100, 140], [1, 30], 2, 1, 64, "float32", change=share, layout="heads")


@pytest.mark.parametrize("scale", [0.0, -0.3, 3.0])
def test_scales(hip, kernel, scale):
    """Uniform weights, turned order, nearly one-hot rows."""
    rng = np.random.default_rng(10)
    run_attention(hip, rng, [150, 77], [1, 77], 2, 1, 64, "float32", scale=scale, layout="heads")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_query_extremes(hip, kernel, dtype):
    """Rows of zeros and of very small and large values (scores stay finite)."""
    rng = np.random.default_rng(11)
    c = R.Cache(hip, rng, 5, 1, 64)
    table = R.tables(rng, [300], 5)
    q = rng.standard_normal((4, 1, 64)) * np.array([0.0, 1e-30, 1e4, 1e-3])[:, None, None]
    q = R.rounded(q, dtype)
    arr = [DeviceArray(hip, x) for x in (np.array([0, 4], np.int32), np.array([300], np.int32), table)]
    qd, od = R.put(hip, q, dtype), R.put(hip, q * 0, dtype)
    lse = DeviceArray(hip, np.zeros((4, 1), np.float32))
    cache = c.upload()
    b = ch.Kv8Batch(arr[0], arr[1], arr[2], 4, 4)
    ws = DeviceArray(hip, np.zeros(cache.attend_workspace(b, 1) + 16, np.uint8))
    cache.attend(b, qd, od, lse=lse, workspace=ws)
    ref, rlse, err = R.attention(c, table[0], 300, np.arange(296, 300), q, 64 ** -0.5, True, 0, 1)
    check_attention(R.get(od), R.get(lse), ref, rlse, err, dtype, 127 * float(c.scales.max()))
    R.free(*arr, qd, od, lse, ws, *c.dev)


def test_query_not_finite(hip, kernel):
    """A query row with NaN or infinity gives NaN for its own head only."""
    rng = np.random.default_rng(12)
    for rows in (1, 33):
        c = R.Cache(hip, rng, 3, 2, 64)
        table = R.tables(rng, [100], 3)
        q = rng.standard_normal((rows, 2, 64))
        q[0, 0, 3], q[-1, 1, 5] = np.nan, np.inf
        arr = [DeviceArray(hip, x) for x in (np.array([0, rows], np.int32), np.array([100], np.int32), table)]
        qd, od = R.put(hip, q, "float32"), R.put(hip, q * 0, "float32")
        cache = c.upload()
        b = ch.Kv8Batch(arr[0], arr[1], arr[2], rows, rows)
        ws = DeviceArray(hip, np.zeros(cache.attend_workspace(b, 2) + 16, np.uint8))
        cache.attend(b, qd, od, workspace=ws)
        got = R.get(od)
        bad = np.isnan(got).any(-1)
        want = np.zeros((rows, 2), bool)
        want[0, 0] = want[-1, 1] = True
        assert np.array_equal(bad, want), (rows, np.argwhere(bad != want))
        R.free(*arr, qd, od, ws, *c.dev)


def test_v_scales_far_apart(hip, kernel):
    """Pages whose V is huge or zero beside ordinary ones: rows that do not see the huge page keep their precision."""
    rng = np.random.default_rng(14)

    def change(c, table):
        c.scales[table[0, 1], :, 1] = 1e30   # tokens 64 .. 127: seen by the later rows only
        c.scales[table[1, 0], :, 1] = 0      # a page of zeros first
        c.v[table[1, 0]] = 0
        c.scales[table[2, 1], :, 1] = 1e-20

    for rows, n in ((64, 64), (100, 130)):
        c = R.Cache(hip, rng, 12, 2, 64)
        table = R.tables(rng, [n] * 3, 12, 3)
        if n > 64:
            change(c, table)
        q = R.rounded(rng.standard_normal((3 * rows, 2, 64)), "float32")
        arr = [DeviceArray(hip, x) for x in (offsets([rows] * 3), np.array([n] * 3, np.int32), table)]
        qd, od = R.put(hip, q, "float32"), R.put(hip, q * 0, "float32")
        cache = c.upload()
        b = ch.Kv8Batch(*arr, 3 * rows, rows)
        ws = DeviceArray(hip, np.zeros(cache.attend_workspace(b, 2) + 16, np.uint8))
        cache.attend(b, qd, od, workspace=ws)
        got = R.get(od)
        for i in range(3):
            for r in range(rows):
                pos = n - rows + r
                a = slice(i * rows + r, i * rows + r + 1)
                ref, rlse, err = R.attention(c, table[i], n, np.array([pos]), q[a], 1 / 8, True, 0, 1)
                vmax = 127 * max(float(c.scales[table[i, p], :, 1].max()) for p in range(pos // 64 + 1))
                check_attention(got[a], rlse, ref, rlse, err, "float32", vmax)
        R.free(*arr, qd, od, ws, *c.dev)


def test_the_sizes_choose_the_prompt_kernel(hip):
    """Enough columns for it without being told so."""
    rng = np.random.default_rng(15)
    lens = [int(x) for x in rng.integers(60, 100, 24)]
    run_attention(hip, rng, lens, [max(n - 5 * i, 1) for i, n in enumerate(lens)], 8, 1, 32, "bfloat16", layout="heads")


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("d,hk,g", [(16, 2, 1), (24, 2, 2), (64, 1, 4), (128, 1, 3)])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 900), (False, 1500)])
def test_prompts_over_split_keys(hip, kernel, dtype, d, hk, g, causal, window):
    """Chunks of rows over long keys, which are split and joined: splits that a sequence is too short for, that the
    window hides, with bad tokens and missing pages in them."""
    rng = np.random.default_rng(16 + d)

    def change(c, table):
        c.bad[table[0, 30], 0] = np.uint64(1 << 9)    # token 1929 of sequence 0, head 0
        table[2, 17:19] = -1                          # 1088 .. 1215 of sequence 2
        c.scales[table[2, 30:34], :, 1] *= 2.0 ** -12  # a split whose values are far below the others'

    run_attention(hip, rng, [2111, 70, 3000, 1], [85, 70, 40, 1], hk, g, d, dtype, causal, window, change=change, layout="heads")


def test_the_sizes_choose_split_prompts(hip):
    rng = np.random.default_rng(17)
    for dtype in ("float32", "bfloat16"):
        run_attention(hip, rng, [2500], [100], 2, 1, 64, dtype)
        run_attention(hip, rng, [2100, 2500], [30, 33], 1, 4, 128, dtype, layout="heads")


# ---- append and read ---------------------------------------------------------

def append_ref(c, table, start, k, v):
    """The restatement of one sequence's append on the host copy; k, v [rows][heads][dim], rotated.  Returns
    what the codes should be before they are rounded, by (page, head): arrays [tokens][dim] and kept tokens."""
    want = {}
    n = len(k)
    for pg in range(start // R.PAGE, (start + n + R.PAGE - 1) // R.PAGE):
        page = table[pg]
        lo, hi = max(start - pg * R.PAGE, 0), min(start + n - pg * R.PAGE, R.PAGE)
        r0 = pg * R.PAGE + lo - start
        for h in range(c.h):
            kn, vn = k[r0:r0 + hi - lo, h], v[r0:r0 + hi - lo, h]
            fine = np.isfinite(kn).all(1) & np.isfinite(vn).all(1)
            old = c.scales[page, h].astype(np.float64)
            new = []
            for x, o in ((kn, old[0]), (vn, old[1])):
                s = np.abs(x[fine]).max() / 127 if fine.any() else 0.0
                s = 0.0 if s < 2.0 ** -126 else s  # too small to be inverted
                new.append(max(s, o) if lo else s)
            bad = int(c.bad[page, h]) & ((1 << lo) - 1)
            for t in np.flatnonzero(~fine):
                bad |= 1 << int(lo + t)
            parts = []
            for x, kept, o, s in ((kn, c.k[page, h, :lo, :c.d], old[0], new[0]), (vn, c.v[page, h, :c.d, :lo].T, old[1], new[1])):
                y = np.where(fine[:, None], x, 0.0) / s if s else np.zeros_like(x)
                parts.append(np.concatenate([kept * (o / s) if s else kept * 0.0, y]))
            want[page, h] = (parts, np.array(new), bad, lo, hi)
    return want


def run_append(hip, rng, lens, rows, hk, g, d, dtype, rope=None, edit=None, q=True, inplace=False, n_pages=None, gap=0):
    need = sum(-(-n // R.PAGE) for n in lens)
    c = R.Cache(hip, rng, n_pages or need + 2, hk, d)
    table = R.tables(rng, lens, len(c.k))
    cu = offsets(rows)
    n, h = int(cu[-1]) + 2, hk * g
    k = R.rounded(rng.standard_normal((n, hk, d)), dtype)
    v = R.rounded(rng.standard_normal((n, hk, d)) * 3, dtype)
    qx = R.rounded(rng.standard_normal((n, h, d)), dtype)
    if edit:
        edit(k, v, c, table)
    width = (h + 2 * hk) * d + gap
    base = R.put(hip, np.concatenate([x.reshape(n, -1) for x in (qx, k, v)] + [np.zeros((n, gap))], 1), dtype)
    qo = base if inplace else R.put(hip, np.full((n, h, d), 5.0), dtype)
    arr = [DeviceArray(hip, x) for x in (cu, np.asarray(lens, np.int32), table)]
    cache = c.upload()
    b = ch.Kv8Batch(*arr, n, max(rows))
    views = [R.View(base, o, (n, x, d), (width, d, 1)) for o, x in ((0, h), (h * d, hk), ((h + hk) * d, hk))]
    qv = views[0] if q else None
    cache.append(b, views[1], views[2], q=qv, q_out=None if inplace or not q else qo, rope=rope)
    kg, vg, sg, bg = c.download()
    turn = lambda x, p: R.rope(x, p, rope) if rope else x  # noqa: E731
    touched = set()
    for i, (m, r) in enumerate(zip(lens, rows)):
        a = slice(int(cu[i]), int(cu[i + 1]))
        pos = np.arange(m - r, m)
        # rotated values that leave FP32 are infinite there
        with np.errstate(over="ignore", invalid="ignore"):
            kr = turn(k[a], pos)
            kr = np.where(np.abs(kr) > np.finfo(np.float32).max, np.inf, kr)
        skip = max(0, r - m)
        for (page, hh), (parts, s, bad, lo, hi) in append_ref(c, table[i], m - r + skip, kr[skip:], v[a][skip:]).items():
            touched.add((page, hh))
            assert int(bg[page, hh]) == bad, (i, page, hh, hex(int(bg[page, hh])), hex(bad))
            assert np.allclose(sg[page, hh], s, rtol=2.0 ** -21, atol=1.2e-38), (sg[page, hh], s)
            for got, want in ((kg[page, hh, :hi, :d], parts[0]), (vg[page, hh, :d, :hi].T, parts[1])):
                off = np.abs(got - want)
                assert (off <= 0.5 + 1e-4).all(), (i, page, hh, off.max(), np.argwhere(off > 0.5 + 1e-4)[:4])
        if q:
            want = turn(qx[a], pos)[skip:]
            got = R.get(qo).reshape(n, -1)[:, :h * d].reshape(n, h, d)[a][skip:]
            assert (np.abs(got - want) <= R.EPS[dtype] * np.abs(want) + 2.0 ** -21 * (np.abs(want).max(initial=0))).all()
    for page in range(len(kg)):
        for hh in range(hk):
            if (page, hh) not in touched:
                assert np.array_equal(kg[page, hh], c.k[page, hh]) and np.array_equal(vg[page, hh], c.v[page, hh])
                assert np.array_equal(sg[page, hh], c.scales[page, hh]) and bg[page, hh] == c.bad[page, hh]
    if q and not inplace:
        assert (R.get(qo)[int(cu[-1]):] == 5.0).all()
    # read back: codes times scales
    ko, vo = R.put(hip, np.full((n, hk, d), 5.0), dtype), R.put(hip, np.full((n, hk, d), 5.0), dtype)
    cache.read(b, ko, vo)
    kb, vb = R.get(ko), R.get(vo)
    for i, (m, r) in enumerate(zip(lens, rows)):
        for x, p in zip(range(int(cu[i]), int(cu[i + 1])), range(m - r, m)):
            if p < 0:
                assert (kb[x] == 5.0).all()
                continue
            page, t = table[i, p // R.PAGE], p % R.PAGE
            for hh in range(hk):
                if int(bg[page, hh]) >> t & 1:
                    assert np.isnan(kb[x, hh]).all() and np.isnan(vb[x, hh]).all()
                else:
                    # one rounding of code * scale to the type, or one to FP32 (2^-24) before it; subnormals: half a step
                    for got, want in ((kb[x, hh], kg[page, hh, t, :d] * np.float64(sg[page, hh, 0])),
                                      (vb[x, hh], vg[page, hh, :d, t] * np.float64(sg[page, hh, 1]))):
                        tiny = 2.0 ** -25 if dtype == "float16" else 2.0 ** -134
                        assert (np.abs(got - want) <= (R.EPS[dtype] + 2.0 ** -23) * np.abs(want) + tiny).all()
    assert (kb[int(cu[-1]):] == 5.0).all() and (vb[int(cu[-1]):] == 5.0).all()
    R.free(base, ko, vo, *arr, *c.dev)
    if not inplace:
        qo.free()


ROPES = [None, dict(interleaved=False), dict(interleaved=True), dict(interleaved=False, scaling="linear", factor=4.0),
         dict(interleaved=True, scaling="ntk", factor=8.0), dict(interleaved=False, scaling="yarn", factor=8.0, trained_len=64)]


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("d,hk,g", [(16, 3, 1), (24, 2, 2), (32, 1, 4), (64, 2, 1), (128, 2, 3)])
@pytest.mark.parametrize("kind", range(len(ROPES)))
def test_append(hip, dtype, d, hk, g, kind):
    rng = np.random.default_rng(d + kind)
    part = d if kind % 2 else d // 2 + d // 2 % 2
    rope = None if ROPES[kind] is None else ch.Rope(part, **ROPES[kind])
    run_append(hip, rng, [1, 64, 65, 130, 200, 77, 128], [1, 64, 1, 130, 70, 1, 64], hk, g, d, dtype, rope,
               inplace=kind == 2, q=kind != 3)


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("d,hk,g", [(16, 3, 1), (24, 2, 2), (32, 1, 4), (64, 2, 1), (128, 2, 3)])
@pytest.mark.parametrize("kind", [0, 1, 2])
def test_append_few_rows(hip, dtype, d, hk, g, kind):
    """One to four rows a sequence, over a page's end, an idle stream among them; kept codes of all word offsets."""
    rng = np.random.default_rng(d + kind)
    rope = None if ROPES[kind] is None else ch.Rope(d, **ROPES[kind])
    run_append(hip, rng, [1, 2, 7, 64, 66, 65, 130, 0, 99], [1, 2, 3, 4, 4, 1, 2, 0, 1], hk, g, d, dtype, rope)
    run_append(hip, rng, [6, 64, 130], [1, 1, 1], hk, g, d, dtype, rope)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows", [1, 70])
def test_append_rows_of_any_alignment(hip, dtype, rows):
    rng = np.random.default_rng(rows)
    run_append(hip, rng, [100, 71], [rows, rows], 2, 2, 64, dtype, ch.Rope(64), gap=1)
    run_append(hip, rng, [100, 71], [rows, rows], 2, 1, 32, dtype, ch.Rope(10, interleaved=True))


def test_append_far_positions(hip):
    """Angles of positions that FP32 products of position and frequency lose."""
    rng = np.random.default_rng(1)
    c = R.Cache(hip, rng, 3, 1, 64)
    n = 1_000_003
    table = np.full((1, n // R.PAGE + 1), -1, np.int32)
    table[0, -1] = 1
    k = rng.standard_normal((2, 1, 64))
    kd, qd = R.put(hip, k, "float32"), R.put(hip, k * 0, "float32")
    arr = [DeviceArray(hip, x) for x in (np.array([0, 2], np.int32), np.array([n], np.int32), table)]
    cache = c.upload()
    rope = ch.Rope(64)
    cache.append(ch.Kv8Batch(*arr, 2, 2), kd, kd, q=kd, q_out=qd, rope=rope)
    want = R.rope(R.rounded(k, "float32"), np.array([n - 2, n - 1]), rope)
    # position * frequency in turns, about 1.6e5, is off by at most 2^-35 in 64 bits; 32-bit sine, cosine and products
    assert np.abs(R.get(qd) - want).max() <= 2.0 ** -20 * np.abs(want).max()
    R.free(*arr, kd, qd, *c.dev)


def test_append_not_finite_and_extremes(hip):
    """NaN, infinities and a rotation that overflows mark their token in their head; zeros, tiny and huge pages."""
    rng = np.random.default_rng(2)

    def edit(k, v, c, table):
        k[0, 0, 3], v[5, 1, 7] = np.nan, np.inf
        k[9, 1] = -np.inf
        k[12, 0], k[12, 0, 0], k[12, 0, 32] = 0, 3e38, 3e38      # turned: beyond FP32
        k[70:, 0], v[70:, 1] = 0, 0                              # a page of zeros (sequence 1)
        k[70:, 1] *= 1e-44                                       # values that have no scale
        v[70:, 0] *= 1e30
    run_append(hip, rng, [70, 40], [70, 40], 2, 1, 64, "float32", ch.Rope(64), edit=edit)
    run_append(hip, rng, [70, 40], [70, 40], 2, 1, 64, "float32", ch.Rope(64), edit=edit, gap=3)

    def keep(k, v, c, table):  # a page whose kept tokens are small, bad, or without a scale
        c.scales[table[0, 0], 0] = 1e-6
        c.scales[table[0, 0], 1] = 0
        c.k[table[0, 0], 1], c.v[table[0, 0], 1] = 0, 0
        c.bad[table[0, 0], 0] = np.uint64(0xF0F0F0F0F0F0F0F0)
        k[0, 1], v[0, 1] = 0, 0
    run_append(hip, rng, [30], [1], 2, 2, 64, "float32", edit=keep)

    def lost(k, v, c, table):
        keep(k, v, c, table)
        k[0, 0, 5], v[2, 0, 63] = np.inf, np.nan
    run_append(hip, rng, [31], [3], 2, 2, 64, "float32", edit=lost)
    run_append(hip, rng, [50], [20], 2, 2, 64, "float32", edit=lost)
    run_append(hip, rng, [30], [9], 2, 2, 128, "bfloat16", edit=keep)


def test_append_padded_batch(hip):
    """More rows than tokens: the rows at negative positions are not stored."""
    run_append(hip, np.random.default_rng(3), [3, 70], [5, 2], 1, 2, 32, "float32", ch.Rope(32))


def test_append_many_times_equals_the_reference_step_by_step(hip):
    """Tokens one by one: the page's scale only grows, codes follow it."""
    rng = np.random.default_rng(4)
    c = R.Cache(hip, rng, 3, 1, 32, fill=False)
    table = np.array([[1, 2]], np.int32)
    cache = c.upload()
    td = DeviceArray(hip, table)
    cu = DeviceArray(hip, np.array([0, 1], np.int32))
    last = 0.0
    for p in range(70):
        x = (rng.standard_normal((1, 1, 32)) * (1 + p / 10)).astype(np.float32)
        kd = R.put(hip, x, "float32")
        ln = DeviceArray(hip, np.array([p + 1], np.int32))
        before = c.download()
        cache.append(ch.Kv8Batch(cu, ln, td, 1, 1), kd, kd)
        kg, vg, sg, bg = c.download()
        page, t = table[0, p // 64], p % 64
        s = max(float(sg[page, 0, 0]), 1e-30)
        assert s >= last * (t > 0) and np.isclose(s, max(np.abs(x).max() / 127, last if t else 0), rtol=1e-6)
        assert (np.abs(kg[page, 0, t] - x[0, 0] / s) <= 0.5 + 1e-4).all() and np.array_equal(kg[page, 0, t], vg[page, 0, :, t])
        old = before[0][page, 0, :t] * (float(before[2][page, 0, 0]) / s)
        assert (np.abs(kg[page, 0, :t] - old) <= 0.5 + 1e-4).all()
        last = s
        R.free(kd, ln)
    R.free(td, cu, *c.dev)


def test_append_read_attend_together(hip):
    """A prompt, then steps, as a program runs them: the attention of the rows equals the restatement over what
    was appended, to the cache's own rounding (half a code of K and V)."""
    rng = np.random.default_rng(13)
    d, hk, g, n0, steps = 64, 2, 2, 75, 60
    rope = ch.Rope(d)
    c = R.Cache(hip, rng, 4, hk, d)
    cache = c.upload()
    table = np.array([[3, 0, 2]], np.int32)
    td = DeviceArray(hip, table)
    ks, vs, lens = np.zeros((0, hk, d)), np.zeros((0, hk, d)), 0
    for n in [n0] + [1] * steps:
        x = [rng.standard_normal((n, w, d)).astype(np.float32) for w in (hk * g, hk, hk)]
        lens += n
        arr = [DeviceArray(hip, np.array([0, n], np.int32)), DeviceArray(hip, np.array([lens], np.int32))]
        q, k, v = [R.put(hip, y, "float32") for y in x]
        out = R.put(hip, x[0] * 0, "float32")
        b = ch.Kv8Batch(arr[0], arr[1], td, n, n)
        ws = DeviceArray(hip, np.zeros(cache.attend_workspace(b, hk * g) + 16, np.uint8))
        cache.append(b, k, v, q=q, rope=rope)
        cache.attend(b, q, out, workspace=ws)
        pos = np.arange(lens - n, lens)
        ks, vs = np.concatenate([ks, R.rope(x[1].astype(np.float64), pos, rope)]), np.concatenate([vs, x[2]])
        qr, got = R.rope(x[0].astype(np.float64), pos, rope), R.get(out)
        # codes: half a step of amax / 127 and as much again for every time the scale grew (the first appends only)
        sk, sv = np.abs(ks).max() / 127, np.abs(vs).max() / 127
        for h in range(hk * g):
            s = qr[:, h] @ ks[:, h // g].T / 8
            s[pos[:, None] < np.arange(lens)] = -np.inf
            p = np.exp(s - s.max(1, keepdims=True))
            p /= p.sum(1, keepdims=True)
            ref = p @ vs[:, h // g]
            ds = 2 * sk * np.abs(qr[:, h]).sum(1) / 8
            tol = 2 * sv + 2 * ds[:, None] * np.abs(vs).max()
            assert (np.abs(got[:, h] - ref) <= tol).all(), (lens, h, np.abs(got[:, h] - ref).max(), tol.max())
        R.free(*arr, q, k, v, out, ws)
    R.free(td, *c.dev)

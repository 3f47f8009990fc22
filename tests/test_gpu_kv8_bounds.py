"""Attention over the 8-bit cache on the GPU, both kernels, within the bounds of
tests/kv8_bounds.py: what the kernels' own roundings add to a row, and no more."""
import numpy as np
import pytest

import codon_hip as ch
import kv8_bounds as B
import kv8_ref as R
from codon_hip.devmem import DeviceArray, Hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    return Hip()


def offsets(rows):
    return np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)


def attend(hip, c, table, lens, rows, q, dtype, causal=True, window=0, scale=None):
    """The call's out and lse as float64."""
    n, h, d = q.shape
    arr = [DeviceArray(hip, x) for x in (offsets(rows), np.asarray(lens, np.int32), table)]
    qd, od = R.put(hip, q, dtype), R.put(hip, q * 0 + 7, dtype)
    lse = DeviceArray(hip, np.full((n, h), 7, np.float32))
    cache = c.upload()
    b = ch.Kv8Batch(*arr, n, max(rows))
    ws = DeviceArray(hip, np.full(cache.attend_workspace(b, h) + 16, 255, np.uint8))
    kw = {} if scale is None else {"scale": scale}
    cache.attend(b, qd, od, lse=lse, causal=causal, window=window, workspace=ws, **kw)
    got = R.get(od), R.get(lse)
    R.free(*arr, qd, od, lse, ws, *c.dev)
    return got


def check(hip, monkeypatch, kernel, c, table, lens, rows, q, dtype, causal=True, window=0, only=None, scale=None,
          seqs=None, alike=False):
    """One call against the bounds (only: rows of a sequence that are looked at; seqs: sequences)."""
    monkeypatch.setenv("CIH_KV8_PROMPT", "1" if kernel == "prompt" else "0")
    got, glse = attend(hip, c, table, lens, rows, q, dtype, causal, window, scale)
    g = q.shape[1] // c.h
    cu = offsets(rows)
    for i, (n, r) in enumerate(zip(lens, rows)):
        if seqs is not None and i not in seqs:
            continue
        at = np.arange(r) if only is None else np.unique(np.clip(only, 0, r - 1)) if r else np.arange(0)
        ref, rlse, tol, ltol = B.attend(c, table[i], n, n - r + at, q[cu[i] + at], c.d ** -0.5 if scale is None else scale,
                                        causal, window, g, dtype, kernel, alike)
        mine, mlse = got[cu[i] + at], glse[cu[i] + at]
        bad = ~(np.abs(mine - ref) <= tol)
        assert not bad.any(), (i, np.argwhere(bad)[:4], mine[bad][:4], ref[bad][:4], tol[bad][:4], bad.mean())
        fine = np.isfinite(rlse)
        assert np.array_equal(mlse[~fine], rlse[~fine])
        off = np.abs(mlse[fine] - rlse[fine])
        assert (off <= ltol[fine]).all(), (i, (off - ltol[fine]).max())


# ---- V scales of any size ----------------------------------------------------

# three pages each: a fall, a rise, both, over most of what FP32 holds
SCALES = [(1.0, 1e-36, 0.02), (1e34, 0.02, 1e-30), (1e-36, 1.0, 1e34), (0.02, 1e36, 1e-4), (1e-37, 1e-37, 1e36),
          (2.6e36, 1e-37, 2.6e36)]


def far_apart(hip, monkeypatch, kernel, g=1):
    """Rows of which some see a page of other size and some do not: each keeps the precision of what it sees."""
    rng = np.random.default_rng(31)
    lens = [180] * len(SCALES)
    c = R.Cache(hip, rng, 3 * len(SCALES), 1, 64)
    table = R.tables(rng, lens, len(c.k))
    for i, sv in enumerate(SCALES):
        c.scales[table[i, :3], 0, 1] = sv
    q = R.rounded(rng.standard_normal((180 * len(SCALES), g, 64)) * 0.5, "float32")
    check(hip, monkeypatch, kernel, c, table, lens, lens, q, "float32",
          only=[0, 1, 30, 62, 63, 64, 65, 66, 70, 90, 126, 127, 128, 129, 131, 150, 179])


def test_prompts_over_v_scales_far_apart(hip, monkeypatch):
    far_apart(hip, monkeypatch, "prompt")
    far_apart(hip, monkeypatch, "prompt", g=3)


def test_rows_over_v_scales_far_apart(hip, monkeypatch):
    far_apart(hip, monkeypatch, "few")
    far_apart(hip, monkeypatch, "few", g=3)


@pytest.mark.parametrize("kernel", ["few", "prompt"])
@pytest.mark.parametrize("rows", [1, 100])
def test_split_keys_over_v_scales_far_apart(hip, monkeypatch, kernel, rows):
    """Splits joined: pages of 10^-37 to 10^36, and values near the largest that FP32 has, of one sign and of both."""
    rng = np.random.default_rng(34)
    for lo, hi, one_sign in ((-37, 36.4, False), (36.4, 36.42, True), (-37, -36, False)):
        n = 4500
        c = R.Cache(hip, rng, 71, 1, 64)
        table = R.tables(rng, [n], 71)
        c.scales[:, 0, 1] = 10.0 ** rng.uniform(lo, hi, 71)
        if one_sign:
            c.v = np.abs(c.v)
        q = R.rounded(rng.standard_normal((rows, 1, 64)) * 0.3, "float32")
        check(hip, monkeypatch, kernel, c, table, [n], [rows], q, "float32", only=[0, 1, 33, 64, 99])


# ---- long sums ---------------------------------------------------------------

@pytest.mark.parametrize("kernel", ["few", "prompt"])
@pytest.mark.parametrize("scale", [0.0, 0.05])
def test_long_sums_of_one_sign(hip, monkeypatch, kernel, scale):
    """Values of one sign under flat weights, the keys not split: roundings that all fall to one side add up."""
    rng = np.random.default_rng(38)
    n, d, hk, seqs = 30000, 16, 32, 32
    c = R.Cache(hip, rng, 469, hk, d)
    table = np.repeat(R.tables(rng, [n], 469), seqs, 0)
    c.scales[:] = 0.02, 0.01
    c.v[:] = rng.integers(60, 120, c.v.shape)
    q = R.rounded(rng.standard_normal((17 * seqs, hk, d)), "float32")
    check(hip, monkeypatch, kernel, c, table, [n] * seqs, [17] * seqs, q, "float32", scale=scale, only=[3], seqs=[0, 31])


# ---- many small weights behind a large one -----------------------------------

@pytest.mark.parametrize("behind", ["first", "middle"])
def test_prompts_with_a_key_above_all_others(hip, monkeypatch, behind):
    """A key of weight 1 and 16,000 of e^-19.5 to e^-21, whose values differ from its: together they move the output
    by 4e-5, each by less than float16 can say beside 1.  So many sequences and heads that the keys are not split; they
    share their pages."""
    rng = np.random.default_rng(32)
    n, d, hk, seqs = 16000, 16, 32, 32
    c = R.Cache(hip, rng, 250, hk, d)
    table = np.repeat(R.tables(rng, [n], 250), seqs, 0)
    c.scales[:] = 25 / 127, 0.01
    c.k[:] = 0
    c.k[..., 0] = rng.integers(20, 28, (250, hk, 64))
    c.v[:] = rng.integers(60, 120, c.v.shape)
    one = 0 if behind == "first" else 7777
    c.k[table[0, one // 64], :, one % 64, 0] = 127
    c.v[table[0, one // 64], :, :, one % 64] = -100
    q = np.zeros((17 * seqs, hk, d))
    q[..., 0] = 1
    for kernel in ("prompt", "few"):
        check(hip, monkeypatch, kernel, c, table, [n] * seqs, [17] * seqs, q, "float32", scale=1.0, only=[0, 16], seqs=[0, 31],
              alike=True)


def test_prompts_of_uneven_scores(hip, monkeypatch):
    """Scores that differ by some 30 from page to page, in both directions."""
    rng = np.random.default_rng(33)
    for dtype in ("float32", "bfloat16"):
        for spread in (2.0, 8.0):
            n = 700
            c = R.Cache(hip, rng, 11, 1, 64)
            table = R.tables(rng, [n], 11)
            q = R.rounded(rng.standard_normal((n, 2, 64)) * spread, dtype)
            check(hip, monkeypatch, "prompt", c, table, [n], [n], q, dtype, only=np.arange(0, n, 23))


# ---- ordinary rows -----------------------------------------------------------

@pytest.mark.parametrize("kernel", ["few", "prompt"])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("d,hk,g", [(16, 2, 1), (24, 2, 2), (32, 1, 3), (64, 1, 4), (64, 2, 1), (128, 1, 4)])
def test_rows(hip, monkeypatch, kernel, dtype, d, hk, g):
    """Flat and peaked softmaxes: single tokens, drafted rows, prompts, chunks, windows."""
    rng = np.random.default_rng(35 + d)
    lens, rows = [1, 65, 130, 333, 700, 700], [1, 65, 130, 40, 1, 5]
    for causal, window, spread in ((True, 0, 0.5), (True, 100, 2.0), (False, 0, 0.5)):
        c = R.Cache(hip, rng, 40, hk, d)
        table = R.tables(rng, lens, 40)
        q = R.rounded(rng.standard_normal((sum(rows), hk * g, d)) * spread, dtype)
        check(hip, monkeypatch, kernel, c, table, lens, rows, q, dtype, causal, window, only=[0, 1, 17, 39, 63, 64, 100, 129])


@pytest.mark.parametrize("kernel", ["few", "prompt"])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_rows_over_split_keys(hip, monkeypatch, kernel, dtype):
    rng = np.random.default_rng(36)
    lens, rows = [9001, 4100], [1, 80]
    c = R.Cache(hip, rng, 210, 1, 64)
    table = R.tables(rng, lens, 210)
    for window in (0, 1500):
        q = R.rounded(rng.standard_normal((81, 2, 64)) * 0.5, dtype)
        check(hip, monkeypatch, kernel, c, table, lens, rows, q, dtype, window=window, only=[0, 1, 40, 79])


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n_seq,rows,hk,g,d,kernel", [(64, 17, 20, 1, 64, "prompt"), (8, 1, 20, 1, 64, "few"),
                                                      (1, 100, 4, 1, 64, "few"), (1, 100, 4, 4, 128, "prompt")])
def test_the_kernel_that_the_sizes_choose(hip, monkeypatch, dtype, n_seq, rows, hk, g, d, kernel):
    """... is the one that is meant: bit by bit what it gives when it is asked for."""
    rng = np.random.default_rng(37)
    n = 2100 if kernel == "prompt" and n_seq == 1 else 150
    lens, counts = [n] * n_seq, [rows] * n_seq
    need = sum(-(-x // 64) for x in lens)
    c = R.Cache(hip, rng, need, hk, d)
    table = R.tables(rng, lens, need)
    q = R.rounded(rng.standard_normal((sum(counts), hk * g, d)), dtype)
    monkeypatch.delenv("CIH_KV8_PROMPT", raising=False)
    chosen = attend(hip, c, table, lens, counts, q, dtype)
    got = {}
    for name, e in (("few", "0"), ("prompt", "1")):
        monkeypatch.setenv("CIH_KV8_PROMPT", e)
        got[name] = attend(hip, c, table, lens, counts, q, dtype)
    assert all(np.array_equal(a, b) for a, b in zip(chosen, got[kernel]))
    assert not all(np.array_equal(a, b) for a, b in zip(*got.values()))

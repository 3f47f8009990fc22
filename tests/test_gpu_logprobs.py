"""Log probabilities of given tokens, entropy and top alternatives on the GPU
(cih_token_logprobs) against the restatement in 64 bits.

Tolerances: a sum of at most V exponentials in FP32 by lanes and trees of at
most 2^-24 (V / 64 + 32) relative, log and exp 2^-22 each, the difference
x - lse one rounding of |x| + |lse|: below 2^-18 (1 + |x| + |lse|) for V up to
140000.  The entropy adds the products p x, with |x - max| up to the logits' range.
"""
import numpy as np
import pytest

import codon_hip as ch
import kv8_ref as R
from codon_hip.devmem import DeviceArray, Hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    return Hip()


def run(hip, x, targets, k, dtype, stride=None, want=("logprob", "entropy", "top")):
    n, vocab = x.shape
    stride = stride or vocab
    wide = np.full((n, stride), 1e4)
    wide[:, :vocab] = x
    base = R.put(hip, wide, dtype)
    x = R.rounded(x, dtype)
    logits = R.View(base, 0, (n, vocab), (stride, 1))
    t = None if targets is None else DeviceArray(hip, np.asarray(targets, np.int32))
    lp, en = [DeviceArray(hip, np.full(n, 7, np.float32)) for _ in range(2)]
    ids, top = DeviceArray(hip, np.full((n, k), 7, np.int32)), DeviceArray(hip, np.full((n, k), 7, np.float32))
    ws = DeviceArray(hip, np.full(ch.token_logprobs_workspace(n, vocab, k) + 16, 255, np.uint8))
    pair = (ids, top) if "top" in want else (None, None)
    ch.token_logprobs(logits, t, lp if "logprob" in want else None, en if "entropy" in want else None, *pair, workspace=ws)
    g = [a.numpy() for a in (lp, en, ids, top)]
    ref = R.logprobs(x, targets, k)
    fin = np.where(np.isfinite(x), np.abs(x), 0).max(initial=0)
    tol = 2.0 ** -18 * (1 + 2 * fin + np.log(vocab))
    for name, got, want_ in (("logprob", g[0], ref[0]), ("entropy", g[1], ref[1]), ("top", g[3], ref[3])):
        if name not in want:
            assert (got == 7).all()
            continue
        assert np.array_equal(np.isnan(got), np.isnan(want_)), name
        assert np.array_equal(np.isneginf(got), np.isneginf(want_)), name
        f = np.isfinite(want_)
        assert np.abs(got[f] - want_[f]).max(initial=0) <= tol, (name, np.abs(got[f] - want_[f]).max(), tol)
    if "top" in want:
        assert np.array_equal(g[2], ref[2]), np.argwhere(g[2] != ref[2])[:5]
    R.free(base, lp, en, ids, top, ws, *([] if t is None else [t]))


@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n,vocab,k", [(1, 1, 1), (5, 2, 2), (8, 33, 5), (70, 33, 33), (3, 64, 20), (3, 65, 64), (9, 257, 8),
                                       (4, 1000, 32), (2, 1023, 1), (2, 1025, 40), (3, 4097, 20), (2, 16385, 20), (2, 33000, 7),
                                       (2, 70001, 64), (1, 140000, 20), (600, 1500, 3), (1100, 40, 4)])
def test_random(hip, dtype, n, vocab, k):
    rng = np.random.default_rng(vocab)
    run(hip, 3 * rng.standard_normal((n, vocab)), rng.integers(0, vocab, n), k, dtype)


@pytest.mark.parametrize("n,vocab,k", [(3, 4096, 64), (70, 4095, 9), (2, 49153, 64), (90, 49999, 5), (2, 65536, 33),
                                       (2, 65537, 64), (1, 98305, 64), (257, 98304, 2), (128, 131072, 20)])
def test_around_the_sizes_that_choose(hip, n, vocab, k):
    """Threads a row and chunks a row change between these."""
    rng = np.random.default_rng(vocab + k)
    run(hip, 3 * rng.standard_normal((n, vocab)), rng.integers(0, vocab, n), k, "bfloat16" if n % 2 else "float32")


@pytest.mark.parametrize("vocab", [33, 60, 300, 5000, 20000, 70000])
def test_ties(hip, vocab):
    """Equal logits: the lowest ids, also where every logit is the same."""
    rng = np.random.default_rng(1)
    x = rng.integers(0, 4, (4, vocab)).astype(float)
    x[1] = 2.5
    x[2] = -np.arange(vocab) // 7
    x[3] = np.arange(vocab) // 7 * 0.25
    run(hip, x, rng.integers(0, vocab, 4), min(vocab, 30), "float32")


@pytest.mark.parametrize("n,vocab", [(4, 1500), (4, 16000), (520, 16000), (2, 140001), (513, 70000)])
@pytest.mark.parametrize("period", [64, 512, 2048, 4096, 8192])
def test_large_logits_in_a_pattern(hip, n, vocab, period):
    """The largest logits lie a period apart or ascend, so that a few threads see most of them."""
    rng = np.random.default_rng(period)
    x = rng.standard_normal((n, vocab))
    i = np.arange(vocab)
    x[0] += 50 * (i % period < 8)
    x[1] = i * 1e-3 if n > 2 else -i * 1e-3
    if n > 2:
        x[2] += 50 * (i % period < 300)
        x[3] = np.where(i % period < 100, 8.0, x[3])
    run(hip, x, rng.integers(0, vocab, n), 64, "float32" if n > 500 else "bfloat16" if period % 3 else "float16")


@pytest.mark.parametrize("vocab", [33, 200, 5000, 70000])
def test_masked_lost_and_odd_rows(hip, vocab):
    """Rows of -inf but one, few or none; the type's lowest values; NaN and infinities; targets outside; wide ranges."""
    rng = np.random.default_rng(2)
    x = 3 * rng.standard_normal((12, vocab))
    x[0] = -np.inf
    x[1, :-1] = -np.inf
    x[2, 3:] = -np.inf
    x[3, ::2] = -np.inf
    x[4, 7] = np.nan
    x[5, vocab - 1] = np.inf
    x[6, :5] = np.finfo(np.float32).min
    x[7] = np.finfo(np.float32).min
    x[8] *= 30
    x[9] += 1000
    x[10, vocab // 2:] = np.nan
    t = rng.integers(0, vocab, 12)
    t[1], t[2], t[3] = vocab - 1, 5, 0
    run(hip, x, t, 20, "float32")
    t[:] = -1
    t[9], t[10], t[11] = vocab, vocab + 5, -2 ** 31
    run(hip, x, t, 1, "float32")


def test_outputs_left_out_and_strides(hip):
    rng = np.random.default_rng(3)
    for vocab in (33, 1000, 40001):
        x = rng.standard_normal((6, vocab))
        for want in (("logprob",), ("entropy",), ("top",), ("logprob", "top")):
            run(hip, x, rng.integers(0, vocab, 6) if "logprob" in want else None, 4, "bfloat16", stride=vocab + 7, want=want)
        run(hip, x, rng.integers(0, vocab, 6), 0, "float16", stride=vocab + 1, want=("logprob", "entropy"))


@pytest.mark.parametrize("n,vocab,k", [((1 << 26) + 77, 2, 0), ((1 << 23) + 5, 3, 2), ((1 << 22) + 9, 70, 3)])
def test_more_rows_than_a_launch_has_threads(hip, n, vocab, k):
    """Rows past 2^22, which several launches share, and past 2^26, whose waves have more than 2^32 lanes: every row is
    the one of its place in a block of rows that repeats."""
    rng = np.random.default_rng(vocab)
    period = 1009
    x = R.rounded(rng.standard_normal((period, vocab)) * 3, "float16")
    t = rng.integers(0, vocab, period).astype(np.int32)
    want = R.logprobs(x, t, k)
    reps = -(-n // period)
    base = DeviceArray(hip, np.tile(x.astype(np.float16), (reps, 1))[:n])
    targets = DeviceArray(hip, np.tile(t, reps)[:n])
    lp, en = [DeviceArray(hip, np.full(n, 7, np.float32)) for _ in range(2)]
    ids, top = DeviceArray(hip, np.full((n, k), 7, np.int32)), DeviceArray(hip, np.full((n, k), 7, np.float32))
    assert ch.token_logprobs_workspace(n, vocab, k) == 0
    ch.token_logprobs(base, targets, lp, en, *((ids, top) if k else (None, None)))
    tol = 2.0 ** -18 * (1 + 2 * np.abs(x).max() + np.log(vocab))
    for a, w in ((lp, want[0]), (en, want[1])) + (((top, want[3]),) if k else ()):
        got = a.numpy()
        first = got[:period]
        assert np.abs(first - w).max() <= tol
        whole = got[:n // period * period].reshape(-1, *first.shape)
        assert (whole == first).all() and (got[whole.shape[0] * period:] == first[:n % period]).all()
    if k:
        got = ids.numpy()
        assert np.array_equal(got[:period], want[2]) and np.array_equal(got[-(n % period):], want[2][:n % period])
        assert (got[:n // period * period].reshape(-1, period, k) == want[2]).all()
    R.free(base, targets, lp, en, ids, top)


@pytest.mark.parametrize("vocab,k", [(900, 1), (5000, 3), (70000, 20)])
def test_alternatives_among_both_signs(hip, vocab, k):
    """The threads' largest logits differ in their sign: few or many of them positive, all but one, none but one."""
    rng = np.random.default_rng(k)
    x = -np.abs(rng.standard_normal((6, vocab))) * 3 - 1
    x[1] *= -1
    for r, n in ((2, 1), (3, k), (4, 2 * k + 9), (5, vocab // 2)):
        x[r, rng.permutation(vocab)[:n]] *= -1
    run(hip, x, rng.integers(0, vocab, 6), k, "float32")

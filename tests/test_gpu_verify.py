"""Verification of drafted tokens on the GPU against its definition in 64 bits: whole numbers, equal.

The seeds are fixed, and none of their random numbers lies where roundings decide: accept_at within 10^-6
(relative) of p(x) / q(x), or sample_at within 10^-12 of a running sum.  The restatement checks it.
"""
import numpy as np
import pytest

import codon_hip as ch
import kv8_more_ref as M
import kv8_ref as R
from codon_hip.devmem import DeviceArray, Hip

pytestmark = pytest.mark.gpu
TYPES = ["float32", "float16", "bfloat16"]


@pytest.fixture(scope="module")
def hip():
    return Hip()


def call(hip, logits, about, cu, drafts, u, v, temperature, dtype, gap=0, want=None):
    n, d, vocab = len(cu) - 1, len(drafts), logits.shape[1]

    def rows(x):
        base = R.put(hip, np.concatenate([x, np.full((len(x), gap), 99.0)], 1), dtype)
        return base, R.View(base, 0, x.shape, (vocab + gap, 1))

    lb, lv = rows(logits)
    db, dv = (None, None) if about is None else rows(about)
    arr = [DeviceArray(hip, x) for x in (np.asarray(drafts, np.int32), np.asarray(cu, np.int32), np.asarray(u, np.float32), np.asarray(v, np.float32))]
    acc, tok = (DeviceArray(hip, np.full(n + 1, -77, np.int32)) for _ in range(2))
    av, tv = R.View(acc, 0, (n,), (1,)), R.View(tok, 0, (n,), (1,))
    av.dtype = tv.dtype = "int32"
    ws = DeviceArray(hip, np.full(ch.verify_drafts_workspace(n, d, vocab) + 16, 255, np.uint8))
    draws = temperature > 0
    for _ in range(2):  # the workspace as the first call left it
        ch.verify_drafts(lv, arr[0], arr[1], av, tv, draft_logits=dv, accept_at=arr[2] if draws else None,
                         sample_at=arr[3] if draws else None, temperature=temperature, workspace=ws)
    got = acc.numpy(), tok.numpy()
    assert got[0][-1] == -77 and got[1][-1] == -77
    if want is None:
        want = M.verify(logits, about, cu, drafts, np.asarray(u, np.float32), np.asarray(v, np.float32), float(np.float32(temperature)))
    assert np.array_equal(got[0][:-1], want[0]), (got[0][:-1], want[0])
    assert np.array_equal(got[1][:-1], want[1]), (got[1][:-1], want[1])
    R.free(lb, acc, tok, ws, *arr)
    if db is not None:
        db.free()
    return want


def make(rng, counts, vocab, dtype, temperature, spread=3.0, off=1.0):
    cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    n, d = len(counts), int(cu[-1])
    logits = R.rounded(rng.standard_normal((n + d, vocab)) * spread, dtype)
    row = np.arange(d) + np.repeat(np.arange(n), counts)
    about = R.rounded(logits[row] + off * rng.standard_normal((d, vocab)), dtype)
    heat = max(temperature, 1e-3)
    drafts = np.argmax(about / heat + rng.gumbel(size=about.shape), 1).astype(np.int32) if d else np.zeros(0, np.int32)
    u = rng.random(d).astype(np.float32)
    v = np.minimum(rng.random(n), 0.9999999).astype(np.float32)
    return logits, about, cu, drafts, u, v


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 33, 64, 65, 257, 1000, 4099, 32003])
@pytest.mark.parametrize("temperature", [0.0, 0.7, 1.0])
def test_verify_vocabularies(hip, vocab, dtype, temperature):
    rng = np.random.default_rng(vocab)
    counts = [4, 0, 1, 7, 3, 2]
    logits, about, cu, drafts, u, v = make(rng, counts, vocab, dtype, temperature)
    call(hip, logits, about, cu, drafts, u, v, temperature, dtype)
    call(hip, logits, None, cu, drafts, u, v, temperature, dtype, gap=3)


@pytest.mark.parametrize("counts", [[0], [1], [0, 0, 0], [40], [3] * 70, [200]])
def test_verify_counts(hip, counts):
    for vocab in (33, 2000):
        rng = np.random.default_rng(len(counts))
        a = make(rng, counts, vocab, "float32", 1.0, off=0.2)
        want = call(hip, *a, 1.0, "float32", gap=1)
        if counts == [200]:
            assert want[0][0] > 3  # many are accepted


def test_verify_many_rows_and_wide(hip):
    rng = np.random.default_rng(5)
    call(hip, *make(rng, [5] * 300, 33, "float32", 1.0), 1.0, "float32")
    call(hip, *make(rng, [5, 3, 6], 131072, "bfloat16", 0.8), 0.8, "bfloat16")
    call(hip, *make(rng, [2], 262147, "float32", 1.3), 1.3, "float32")


@pytest.mark.parametrize("vocab", [33, 3000])
def test_verify_all_accepted_and_none(hip, vocab):
    rng = np.random.default_rng(6)
    logits, about, cu, drafts, u, v = make(rng, [5, 5], vocab, "float32", 1.0)
    row = np.arange(10) + np.repeat([0, 1], 5)
    same = logits[row]
    assert (call(hip, logits, same, cu, drafts, u, v, 1.0, "float32")[0] == 5).all()  # q = p: never refused
    far = np.where(np.arange(vocab)[None] == drafts[:, None], -200.0, logits[row])
    flat = logits.copy()
    flat[row] = far  # the target all but excludes the drafts
    assert (call(hip, flat, about, cu, drafts, np.full(10, 0.5), v, 1.0, "float32")[0] == 0).all()


@pytest.mark.parametrize("vocab", [40, 5000])
def test_verify_infinities_and_nan(hip, vocab):
    """-inf logits are never drawn; rows without a distribution end their sequence at -1."""
    rng = np.random.default_rng(7)
    logits, about, cu, drafts, u, v = make(rng, [3] * 8, vocab, "float32", 1.0, off=0.01)
    row = lambda i, t: 3 * i + i + t  # noqa: E731
    hide = rng.random(logits.shape) < 0.5
    keep = np.zeros_like(hide)
    for r in range(24):
        keep[r + r // 3, drafts[r]] = True
    logits = np.where(hide & ~keep, -np.inf, logits)
    about[rng.random(about.shape) < 0.3] = -np.inf
    for r in range(24):
        about[r, drafts[r]] = logits[r + r // 3, drafts[r]]
    u[:] = 0.0  # everything that has a probability is accepted
    logits[row(0, 0), 3] = np.nan
    logits[row(1, 1), 0] = np.inf
    logits[row(2, 2)] = -np.inf
    logits[row(3, 3), vocab - 1] = np.nan
    about[3 * 4 + 1, 5] = np.nan
    about[3 * 5 + 2] = -np.inf
    drafts[3 * 6 + 1] = -1
    drafts[3 * 7] = vocab
    for temperature in (1.0, 0.0):
        want = call(hip, logits, about, cu, drafts, u, v, temperature, "float32")
        if temperature:
            assert list(want[0][:6]) == [0, 1, 2, 3, 1, 2] and (want[1][:6] == -1).all() and want[0][6] == 1 and want[0][7] == 0
    call(hip, logits, None, cu, drafts, u, v, 1.0, "float32")


@pytest.mark.parametrize("vocab", [48, 4096])
def test_verify_ties_and_borders(hip, vocab):
    """The lowest id among equal logits; sample_at of 0 and just below 1 end at the first and last token."""
    logits, drafts = np.zeros((4, vocab)), np.array([0, 5], np.int32)
    cu = np.array([0, 1, 2], np.int32)
    assert list(call(hip, logits, None, cu, drafts, [0, 0], [0, 0], 0.0, "float32")[0]) == [1, 0]
    for at in (0.0, 1.0 - 2.0 ** -24, 0.503):
        call(hip, logits, None, cu, drafts, [0.999, 0.999], [at, at], 1.0, "float32")
    # a refused draft of a certain distribution is never the next token
    one = np.full((2, vocab), -np.inf)
    one[:, 7] = 0.0
    a, t = call(hip, one, None, np.array([0, 1], np.int32), [8], [0.0], [0.5], 1.0, "float32")
    assert (a[0], t[0]) == (0, 7)
    # q = p and a refusal by hand (accept_at beyond 1): nothing is left of p - q, so p itself
    two = np.random.default_rng(1).standard_normal((2, vocab)).astype(np.float32).astype(np.float64)
    call(hip, two, two[:1], np.array([0, 1], np.int32), [3], [1.5], [0.4], 1.0, "float32")


@pytest.mark.parametrize("vocab", [33, 200, 3000, 40000])
@pytest.mark.parametrize("change", [0.5, -0.5, 0.01])
def test_verify_drafts_that_differ_in_few_tokens(hip, vocab, change):
    """What is left of p hangs on the last bits of the sums' ratio: all other tokens have the same p / q."""
    rng = np.random.default_rng(vocab)
    n = 24
    logits = R.rounded(rng.standard_normal((2 * n, vocab)) * 2, "float32")
    about = logits[::2].copy()
    at = rng.integers(0, vocab, (n, 3))
    for i in range(n):
        about[i, at[i]] += change
    about = R.rounded(about, "float32")
    # accept_at beyond 1 refuses whatever was drafted
    v = rng.random(n).astype(np.float32)
    acc, tok = call(hip, logits, about, np.arange(n + 1), rng.integers(0, vocab, n), np.full(n, 3e38), v, 1.0, "float32")
    assert (acc == 0).all()
    if change < 0:  # the draft is below the target at three tokens only
        assert all(t in a for t, a in zip(tok, at))


def test_verify_temperatures(hip):
    rng = np.random.default_rng(9)
    for temperature in (1e-3, 0.05, 10.0, 1e30):
        for vocab in (33, 700):
            call(hip, *make(rng, [3, 2], vocab, "float32", min(temperature, 10.0)), temperature, "float32")


def test_verify_follows_the_target(hip):
    """4,000 sequences of one draft: what is emitted first has the target's frequencies (5 standard deviations)."""
    rng = np.random.default_rng(10)
    vocab, n = 9, 4000
    p, q = rng.standard_normal(vocab), rng.standard_normal(vocab)
    logits, about = np.tile(p, (2 * n, 1)), np.tile(q, (n, 1))
    about, logits = about.astype(np.float32).astype(np.float64), logits.astype(np.float32).astype(np.float64)
    drafts = np.argmax(about + rng.gumbel(size=about.shape), 1).astype(np.int32)
    u, v = rng.random(n).astype(np.float32), np.minimum(rng.random(n), 0.999999).astype(np.float32)
    acc, tok = call(hip, logits, about, np.arange(n + 1), drafts, u, v, 1.0, "float32")
    first = np.where(acc == 1, drafts, tok)
    want = np.exp(p) / np.exp(p).sum()
    got = np.bincount(first, minlength=vocab) / n
    assert (np.abs(got - want) <= 5 * np.sqrt(want * (1 - want) / n)).all()

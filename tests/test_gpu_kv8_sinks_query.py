"""What attention with sinks holds of a query: three bytes a value, whatever the rows' type and the
kernel, so that small values beside a large one count (tests/kv8_bounds.py with three bytes).

With more sinks than tokens a row sees all tokens up to its own, as without a window.
"""
import numpy as np
import pytest

import kv8_bounds as B
import kv8_ref as R
from codon_hip.devmem import DeviceArray, Hip
from test_gpu_kv8_more import Case

TYPES = ["float32", "float16", "bfloat16"]


@pytest.fixture(scope="module")
def hip():
    return Hip()


@pytest.fixture(autouse=True)
def three_bytes(monkeypatch):
    monkeypatch.setattr(B, "query_bytes", lambda kernel, dtype: 3)


def with_outlier(q, size, dtype):
    """Queries whose first value is `size` times as large as the others."""
    q = q.copy()
    q[..., 0] = size
    return R.rounded(q, dtype)


@pytest.mark.parametrize("dtype,size", [("float32", 3000.0), ("float16", 3.0), ("float16", 200.0), ("bfloat16", 3.0), ("bfloat16", 3000.0)])
@pytest.mark.parametrize("d", [16, 24, 64, 128])
@pytest.mark.parametrize("kernel", ["few", "prompt"])
@pytest.mark.gpu
def test_small_values_beside_a_large_one(hip, monkeypatch, kernel, d, dtype, size):
    """Scores that the small values decide: the large one meets codes of 0 (3: no value is large)."""
    monkeypatch.setenv("CIH_KV8_PROMPT", "0" if kernel == "few" else "1")
    x = Case(hip, np.random.default_rng(d), [400, 70, 5], [40, 70, 1], 1, 2, d, dtype, spare=0)
    R.free(*x.c.dev)
    if size > 3:
        x.c.k[:, :, :, 0] = 0
    x.cache = x.c.upload()
    x.q = with_outlier(x.q, size, dtype)
    x.base.free()
    x.base = R.put(hip, x.q, dtype)
    out, lse = R.put(hip, np.zeros(x.q.shape), dtype), DeviceArray(hip, np.zeros((x.n, x.h), np.float32))
    ws = DeviceArray(hip, np.zeros(x.cache.attend_workspace(x.batch, x.h) + 16, np.uint8))
    x.cache.attend(x.batch, x.base, out, lse=lse, window=50, sinks=1 << 30, workspace=ws)
    got, glse = R.get(out), R.get(lse)
    for _, m, a, pos, table in x.parts():
        ref, rlse, tol, ltol = B.attend(x.c, table, m, pos, x.q[a], d ** -0.5, True, 0, 2, dtype, kernel)
        assert B.within(glse[a], rlse, ltol), np.abs(glse[a] - rlse).max()
        assert B.within(got[a], ref, tol), np.abs(got[a] - ref).max()
    R.free(out, lse, ws)
    x.free()


@pytest.mark.parametrize("dtype,size", [("float16", 200.0), ("bfloat16", 3000.0)])
def test_two_bytes_would_not_do(dtype, size):
    """On the CPU: the same attention of queries held in two bytes is outside the bound, of those in three within."""
    rng, d, n = np.random.default_rng(1), 64, 200
    c = R.Cache(None, rng, 4, 1, d)
    c.k[:, :, :, 0] = 0
    table = np.arange(4)
    q = with_outlier(rng.standard_normal((20, 2, d)) * 2, size, dtype)
    pos = np.arange(n - 20, n)
    ref, rlse, tol, ltol = B.attend(c, table, n, pos, q, d ** -0.5, True, 0, 2, dtype, "prompt")
    for held, inside in ((2, False), (3, True)):
        out, lse, _ = R.attention(c, table, n, pos, B.held_query(q, held)[0], d ** -0.5, True, 0, 2)
        assert B.within(R.rounded(out, dtype), ref, tol) == inside and B.within(lse, rlse, ltol) == inside

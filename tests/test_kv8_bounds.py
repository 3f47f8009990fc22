"""The bounds of tests/kv8_bounds.py hold the right result and none of some wrong
ones: mistakes planted in the restatement, on the CPU."""
import numpy as np
import pytest

import kv8_bounds as B
import kv8_ref as R


def mistaken(c, table, n, pos, q, d, dtype, drop=0, v=1.0, query=None, zero=False, weight=None):
    q = q if query is None else B.held_query(q, query)[0]
    out = np.zeros_like(q)
    k, x, _, _ = c.gather(table, n, 0)
    for r, p0 in enumerate(pos):
        b = p0 + 1 - drop
        for h in range(q.shape[1]):
            s = (k[:b] @ q[r, h]) * d ** -0.5
            p = np.exp(s - s.max())
            w = p if weight is None else np.rint(p * weight) / weight
            out[r, h] = v * (w @ x[:b]) / p.sum()
    return R.rounded(out * (not zero), dtype)


@pytest.mark.parametrize("kernel", ["few", "prompt"])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("d,n", [(16, 131), (64, 300), (128, 1100)])
def test_bounds_hold_and_catch(kernel, dtype, d, n):
    rng = np.random.default_rng(d)
    c = R.Cache(None, rng, -(-n // 64) + 1, 1, d)
    table = R.tables(rng, [n], len(c.k))[0]
    pos = np.arange(n - 6, n)
    q = R.rounded(rng.standard_normal((6, 2, d)) * 0.5, dtype)
    out, lse, tol, ltol = B.attend(c, table, n, pos, q, d ** -0.5, True, 0, 2, dtype, kernel)
    ref, rlse, _ = R.attention(c, table, n, pos, q, d ** -0.5, True, 0, 2)
    assert np.abs(out - ref).max() < 1e-12 and np.abs(lse - rlse).max() < 1e-12
    call = lambda **kw: mistaken(c, table, n, pos, q, d, dtype, **kw)  # noqa: E731
    assert B.within(call(), out, tol)
    assert (ltol < 1e-3).all()
    for name, kw in (("last key left out", dict(drop=1)), ("values 1% large", dict(v=1.01)),
                     ("query in one byte", dict(query=1)), ("zeros", dict(zero=True)), ("weights in 7 bits", dict(weight=127.0))):
        got = call(**kw)
        caught = sum(not B.within(got[r], out[r], tol[r]) for r in range(len(pos)))
        # (a last key of hardly any weight may be left out of a row)
        assert caught >= (len(pos) / 2 if name == "last key left out" else len(pos)), (name, caught)

"""Eviction where the smaller tests do not reach: tables whose keys fill registers, LDS
and more.
"""
import numpy as np
import pytest

from codon_hip.devmem import Hip
from test_gpu_kv8_more import run_evict

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    return Hip()


@pytest.mark.parametrize("budget,first,recent", [(3001, 4, 1000), (20000, 0, 0), (50, 50, 0), (40001, 16, 39000)])
def test_long_tables_of_many_heads(hip, budget, first, recent):
    """Of more than 128 heads in all each has one workgroup: a wave keeps the keys of its first 32 pages in
    registers, of the next 32 in LDS (40,000 tokens: 40 pages a wave) and reads those behind again (70,000: 69)."""
    rng = np.random.default_rng(budget)
    values = np.array([0.0, -0.0, np.inf, -np.inf, np.nan, -1.0, 1e-40, -1e-40, 3e38, 1.0, 1.0000001], np.float32)
    lens = [40000, 140, 70000] + [140] * 62
    run_evict(hip, rng, lens, budget, first, recent, d=16)
    run_evict(hip, rng, lens, budget, first, recent, d=16, weights=lambda s: rng.choice(values, s))
    run_evict(hip, rng, lens, budget, first, recent, d=16, weights=lambda s: rng.integers(0, 2, s).astype(np.float32), inplace=True)


def test_many_heads_pages_behind_that_are_not_there(hip):
    """A page that is missing among those in LDS, or behind them, leaves its sequence alone."""
    def missing(c, table, w):
        table[0, 35] = -1    # in LDS
        table[1, 1090] = 1 << 30  # behind it

    run_evict(hip, np.random.default_rng(2), [40000, 70000, 45000] + [140] * 62, 3001, 4, 100, d=16, edit=missing)

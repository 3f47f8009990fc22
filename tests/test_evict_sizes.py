"""Sizes of an eviction that one launch may have: the workspace's query and the call refuse the same ones
(CPU: no call gets as far as a device)."""
import pytest

from test_ops_args import Fake, batch, cache, code


class Heads:
    """A cache and a batch of given sizes."""

    def __init__(self, n_seq, heads, d, max_pages):
        self.cache = cache(1, heads, d)
        self.batch = batch(n_seq, 1, n_seq, table=Fake((n_seq, max_pages), "int32"))
        self.weights = Fake((1, heads, 64))


# sequences, heads, head size, pages of the table, budget; what is launched is next to 2^32 threads
FITS = [(4095, 1024, 64, 40, 64), (1023, 4095, 16, 33, 100), (2047, 4098, 64, 32, 64),  # that choose
        (1023, 128, 128, 200, 64 * 128), (1023, 128, 64, 400, 64 * 256), (1023, 128, 24, 800, 64 * 512),  # that move
        (128, 32, 128, 1025, 65536), (1023, 128, 128, 128, 1 << 30), (65600, 1, 16, 65, 4096)]
MORE = [(4096, 1024, 64, 40, 64), (2048, 4096, 64, 32, 64), (4095, 4096, 64, 32, 64), (4096, 4096, 64, 32, 64),
        (1024, 128, 128, 200, 64 * 128), (1024, 128, 64, 400, 64 * 256), (1024, 128, 24, 800, 64 * 512), (1023, 128, 128, 200, 64 * 131), (1 << 20, 32, 128, 1024, 65536), (1023, 129, 128, 128, 1 << 30)]


@pytest.mark.parametrize("sizes", FITS)
def test_sizes_that_a_launch_may_have(sizes):
    x, budget = Heads(*sizes[:4]), sizes[4]
    assert x.cache.evict_workspace(x.batch, budget) > 0
    # the next check refuses it
    assert code(x.cache.evict, x.batch, x.weights, budget) == -3


@pytest.mark.parametrize("sizes", MORE)
def test_sizes_that_it_may_not_have(sizes):
    x, budget = Heads(*sizes[:4]), sizes[4]
    assert code(x.cache.evict_workspace, x.batch, budget) == -2
    assert code(x.cache.evict, x.batch, x.weights, budget) == -2

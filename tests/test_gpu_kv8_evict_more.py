"""Eviction where the smaller tests do not reach: tables whose keys fill registers, LDS
and more, grids of many pages, sequences longer than their tables, waits that end,
and the error that a cache gathers over many steps.
"""
import numpy as np
import pytest

import codon_hip as ch
import kv8_more_ref as M
import kv8_ref as R
from codon_hip.devmem import DeviceArray, Hip
from test_gpu_kv8_more import Case, run_evict
from test_gpu_ops_streams import Raw

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


def test_grids_of_many_pages(hip):
    """65,600 heads with room for 64 pages each (they launch 2^28 threads), most of them of sequences without tokens."""
    rng = np.random.default_rng(5)
    n, budget, at, held = 65600, 4096, [0, 37, 40000, 65599], [4130, 4097, 4096, 4160]
    x = Case(hip, rng, held, [1] * 4, 1, 1, 16, "float32", max_pages=65)
    w = np.exp(rng.standard_normal(x.c.k.shape[:3])).astype(np.float32)
    want = M.evict(x.c, w, x.table, held, range(4), budget, 4, 100)
    lens, table = np.zeros(n, np.int32), np.full((n, 65), -1, np.int32)
    lens[at], table[at] = held, x.table
    dev = [DeviceArray(hip, a) for a in (np.zeros(n + 1, np.int32), lens, table, w, np.zeros(n, np.int32))]
    batch = ch.Kv8Batch(*dev[:3], 1, 1)
    ws = Raw(hip, (x.cache.evict_workspace(batch, budget),), "uint8")
    x.cache.evict(batch, dev[3], budget, first=4, recent=100, shifts=dev[4], workspace=ws)
    lens[at], shifts = want[6], np.zeros(n, np.int32)
    shifts[at] = np.array(held) - want[6]
    assert np.array_equal(dev[1].numpy(), lens) and np.array_equal(dev[4].numpy(), shifts)
    gk, gv, gs, _ = x.c.download()
    gw = dev[3].numpy()
    for i, m in enumerate(want[6]):
        j = np.arange(m)
        page = x.table[i, j // 64]
        assert np.array_equal(gk[page, 0, j % 64], want[0][page, 0, j % 64])
        assert np.array_equal(gv[page, 0, :, j % 64], want[1][page, 0, :, j % 64])
        assert np.array_equal(gs[page], want[2][page]) and np.array_equal(gw[page, 0, j % 64], want[4][page, 0, j % 64])
    R.free(ws, *dev)
    x.free()


def test_lengths_past_the_table(hip):
    """A sequence that is longer than its table holds the table's tokens: those are cut, and positions go on behind its length."""
    rng, d, budget, lens = np.random.default_rng(3), 64, 100, [1000, 300, 321, 90, 1 << 30]
    x = Case(hip, rng, [320, 300, 320, 90, 320], [1] * 5, 2, 1, d, "float32")
    w = rng.uniform(0, 1, x.c.k.shape[:3]).astype(np.float32)
    want = M.evict(x.c, w, x.table, lens, range(5), budget, 4, 30)
    dev = [DeviceArray(hip, a) for a in (np.array(lens, np.int32), w, np.arange(5).astype(np.int32), np.zeros((5, 2, budget), np.int32))]
    batch = ch.Kv8Batch(x.arr[0], dev[0], x.arr[2], 5, 1)
    ws = DeviceArray(hip, np.zeros(x.cache.evict_workspace(batch, budget), np.uint8))
    x.cache.evict(batch, dev[1], budget, first=4, recent=30, shifts=dev[2], kept=dev[3], workspace=ws)
    assert np.array_equal(dev[3].numpy(), want[5])
    held = dev[0].numpy()
    assert list(held) == [100, 100, 100, 90, 100]
    shifts = dev[2].numpy()
    assert np.array_equal(shifts, np.arange(5) + lens - held)
    # the next row of each: its place follows what is held, its angle the length there was
    k, v = rng.standard_normal((5, 2, d)), rng.standard_normal((5, 2, d))
    rows = [R.put(hip, a, "float32") for a in (k, v)]
    grown, cu = DeviceArray(hip, held + 1), DeviceArray(hip, np.arange(6, dtype=np.int32))
    rope = ch.Rope(d)
    x.cache.append(ch.Kv8Batch(cu, grown, x.arr[2], 5, 1), *rows, rope=rope, shifts=dev[2])
    gk, _, gs, _ = x.c.download()
    for i in range(5):
        page, at = x.table[i, held[i] // 64], held[i] % 64
        turned = R.rope(R.rounded(k[i:i + 1], "float32"), np.array([lens[i] + i]), rope)[0]
        assert (np.abs(gk[page, :, at] - turned / gs[page, :, :1].astype(np.float64)) <= 0.5 + 1e-3).all()
    # a budget that is more than the table holds: the sequence stays as it is, its length too
    hip.h2d(dev[0].data_ptr(), np.array(lens, np.int32))
    ws2 = DeviceArray(hip, np.zeros(x.cache.evict_workspace(batch, 350), np.uint8))
    x.cache.evict(batch, dev[1], 350, first=4, recent=30, shifts=dev[2], workspace=ws2)
    assert list(dev[0].numpy()) == lens and np.array_equal(dev[2].numpy(), shifts)
    R.free(ws, ws2, grown, cu, *rows, *dev)
    x.free()


@pytest.mark.parametrize("d", [16, 24, 64, 128])
def test_a_wait_that_ends_shows(hip, monkeypatch, d):
    """Pages that do not hear in time (here: that do not listen) that their tokens were read are left as they
    are, with all tokens bad; the others move."""
    monkeypatch.setenv("CIH_KV8_EVICT_POLLS", "0")
    rng, hk, budget, lens = np.random.default_rng(d), 2, 1500, [4000, 1400, 1700]
    x = Case(hip, rng, lens, [1] * 3, hk, 1, d, "float32")
    w = rng.uniform(0, 1, x.c.k.shape[:3]).astype(np.float32)
    k, v, scales, bad, wout, kept, out = M.evict(x.c, w, x.table, lens, range(3), budget, 70, 200)
    dev = [DeviceArray(hip, a) for a in (w, np.zeros((3, hk, budget), np.int32))]
    ws = DeviceArray(hip, np.zeros(x.cache.evict_workspace(x.batch, budget), np.uint8))
    x.cache.evict(x.batch, dev[0], budget, first=70, recent=200, kept=dev[1], workspace=ws)
    assert np.array_equal(dev[1].numpy(), kept) and np.array_equal(x.arr[1].numpy(), out)
    got, gw = x.c.download(), dev[0].numpy()
    run = {16: 8, 24: 8, 64: 4, 128: 2}[d]
    left = 0
    for i, h in np.ndindex(3, hk):
        tok = kept[i, h, :out[i]]
        for p in range(-(-out[i] // 64)):
            m, page = min(64, out[i] - p * 64), x.table[i, p]
            r0, r1 = np.searchsorted(tok, [p * 64, p * 64 + 64])  # its tokens' new places
            stays = m == 64 and tok[p * 64 + 63] == p * 64 + 63
            waits = lens[i] > budget and not stays and r0 < r1 and r0 // 64 < p // run * run
            assert np.array_equal(gw[page, h, :m], wout[page, h, :m])
            want = (x.c.k, x.c.v, x.c.scales) if waits else (k, v, scales)
            n = 64 if waits else m
            assert np.array_equal(got[0][page, h, :n], want[0][page, h, :n])
            assert np.array_equal(got[1][page, h, :, :n], want[1][page, h, :, :n])
            assert np.array_equal(got[2][page, h], want[2][page, h])
            if waits:
                assert int(got[3][page, h]) == 2 ** 64 - 1
            left += waits
    assert 20 < left < hk * 2 * -(-budget // 64)
    # such pages read as NaN
    cu, back = DeviceArray(hip, np.array([0, budget], np.int32)), [R.put(hip, np.zeros((budget, hk, d)), "float32") for _ in range(2)]
    one = DeviceArray(hip, np.array([budget], np.int32))
    x.cache.read(ch.Kv8Batch(cu, one, x.arr[2], budget, budget), *back)
    lost = np.isnan(R.get(back[0])).all(2).sum()
    assert lost >= 64 and lost == np.isnan(R.get(back[1])).any(2).sum()
    R.free(cu, one, ws, *back, *dev)
    x.free()


@pytest.mark.parametrize("d", [16, 64, 128])
def test_cut_again_and_again_keeps_the_values(hip, d):
    """A sequence at its budget takes rows and is cut, 60 times, with an outlier now and then: what the cache holds of a
    token is its own K (turned) and V, off by half a step of each scale that its code was rounded to."""
    rng, hk, budget, new = np.random.default_rng(d), 2, 150, 13
    x = Case(hip, rng, [budget + new], [1], hk, 1, d, "float32")
    x.c.k[:], x.c.v[:], x.c.scales[:], x.c.bad[:] = 0, 0, 0, 0
    for a, b in zip(x.c.dev, (x.c.k, x.c.v, x.c.scales, x.c.bad)):
        hip.h2d(a.data_ptr(), b)
    table, rope = x.table[0], ch.Rope(d)
    wt, shifts = DeviceArray(hip, np.zeros(x.c.k.shape[:3], np.float32)), DeviceArray(hip, np.zeros(1, np.int32))
    held, kept = DeviceArray(hip, np.zeros(1, np.int32)), DeviceArray(hip, np.zeros((1, hk, budget), np.int32))
    ws = DeviceArray(hip, np.zeros(x.cache.evict_workspace(x.batch, budget), np.uint8))
    own = np.zeros((hk, 0, 2, d))    # what each place's token was
    off = np.zeros((hk, 0, 2))       # how far the cache may be from it
    scale = np.zeros((hk, 0, 2))     # of the code that it has

    def follow(own, off, scale, fresh):
        """Half a step where a code was made or made again; what the cache holds is within that."""
        gk, gv, gs, _ = x.c.download()
        j = np.arange(own.shape[1])
        page = table[j // 64]
        now = gs[page].astype(np.float64).transpose(1, 0, 2)
        again = (now != scale) | (j >= fresh)[None, :, None]
        off = off + again * now * (0.5 + 1e-3)
        got = np.stack((gk[page, :, j % 64, :d], gv[page, :, :d, j % 64]), 2).transpose(1, 0, 2, 3) * now[..., None]
        assert (np.abs(got - own) <= off[..., None]).all()
        return off, now

    for step in range(60):
        n0 = own.shape[1]
        m = budget + new - n0
        k, v = (rng.standard_normal((m, hk, d)) * np.where(rng.random((m, hk, 1)) < 0.05, 6.0, 1.0) for _ in range(2))
        k, v = R.rounded(k, "float32"), R.rounded(v, "float32")
        rows, cu = [R.put(hip, a, "float32") for a in (k, v)], DeviceArray(hip, np.array([0, m], np.int32))
        lens = DeviceArray(hip, np.array([budget + new], np.int32))
        batch = ch.Kv8Batch(cu, lens, x.arr[2], m, m)
        x.cache.append(batch, *rows, rope=rope, shifts=shifts)
        pos = np.arange(n0, budget + new) + int(shifts.numpy()[0])
        both = np.stack((R.rope(k, pos, rope), v), 2).transpose(1, 0, 2, 3)
        own, off = np.concatenate([own, both], 1), np.concatenate([off, np.zeros((hk, m, 2))], 1)
        scale = np.concatenate([scale, np.zeros((hk, m, 2))], 1)
        off, scale = follow(own, off, scale, n0)
        hip.h2d(wt.data_ptr(), rng.random(x.c.k.shape[:3]).astype(np.float32))
        x.cache.evict(batch, wt, budget, first=2, recent=20, lens_out=held, shifts=shifts, kept=kept, workspace=ws)
        tok = kept.numpy()[0]
        own, off, scale = (np.stack([a[h, tok[h]] for h in range(hk)]) for a in (own, off, scale))
        off, scale = follow(own, off, scale, budget)
        R.free(cu, lens, *rows)
    assert shifts.numpy()[0] == 60 * new
    R.free(wt, shifts, held, kept, ws)
    x.free()

"""The device operators away from one null-stream call: on streams of their
own, two at once, captured and replayed, in place, over a cache of more than
2^32 bytes.  Every result equals the plain eager call's bit for bit: a
call's sums have a fixed order.
"""
import ctypes

import numpy as np
import pytest

import codon_hip as ch
import kv8_ref as R
from codon_hip.devmem import DeviceArray, Hip

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    return Hip()


@pytest.fixture
def streams(hip):
    made = []
    for _ in range(2):
        s = ctypes.c_void_p()
        assert hip.L.hipStreamCreate(ctypes.byref(s)) == 0
        made.append(s.value)
    yield made
    hip.sync()
    for s in made:
        hip.L.hipStreamDestroy(ctypes.c_void_p(s))


class Raw:
    """Device memory that nothing initialises."""

    def __init__(self, hip, shape, dtype):
        self._hip, self.shape, self.dtype = hip, shape, dtype
        self._ptr = hip.malloc(int(np.prod(shape, dtype=np.int64)) * np.dtype(dtype).itemsize)

    data_ptr = DeviceArray.data_ptr
    stride = DeviceArray.stride
    free = DeviceArray.free


class Program:
    """Steps of a serving loop on buffers of its own: append, attention, read
    back, log probabilities of the attention's output as logits."""

    D, HK, G, V = 64, 2, 3, 384

    def __init__(self, hip, seed, rows, lens, max_pages=40, dtype="bfloat16"):
        self.hip, self.dtype, rng = hip, dtype, np.random.default_rng(seed)
        self.rng, self.rows = rng, rows
        n, self.n = len(rows), int(sum(rows))
        self.pages = n * max_pages
        d, hk, h = self.D, self.HK, self.HK * self.G
        self.cache_arrays = [Raw(hip, (self.pages, hk, 64, d), "int8"), Raw(hip, (self.pages, hk, d, 64), "int8"),
                             Raw(hip, (self.pages, hk, 2), "float32"), Raw(hip, (self.pages, hk), "uint64")]
        self.cache = ch.Kv8Cache(*self.cache_arrays, d)
        table = rng.permutation(self.pages).astype(np.int32).reshape(n, max_pages)
        cu = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        self.cu, self.table = DeviceArray(hip, cu), DeviceArray(hip, table)
        self.lens = DeviceArray(hip, np.array(lens, np.int32))
        self.batch = ch.Kv8Batch(self.cu, self.lens, self.table, self.n, max(rows))
        one = lambda w: R.put(hip, np.zeros((self.n, w, d)), dtype)  # noqa: E731
        self.q, self.k, self.v, self.out, self.kr, self.vr = one(h), one(hk), one(hk), one(h), one(hk), one(hk)
        self.lse = R.put(hip, np.zeros((self.n, h)), "float32")
        self.targets = DeviceArray(hip, rng.integers(0, self.V, self.n).astype(np.int32))
        self.lp, self.en = R.put(hip, np.zeros(self.n), "float32"), R.put(hip, np.zeros(self.n), "float32")
        self.ids, self.tl = DeviceArray(hip, np.zeros((self.n, 7), np.int32)), R.put(hip, np.zeros((self.n, 7)), "float32")
        self.ws = DeviceArray(hip, np.zeros(self.cache.attend_workspace(self.batch, h) + 16, np.uint8))
        self.lws = DeviceArray(hip, np.zeros(ch.token_logprobs_workspace(self.n, self.V, 7) + 16, np.uint8))
        self.rope = ch.Rope(d)
        # every sequence's history
        hist = [max(l - r, 0) for l, r in zip(lens, rows)]
        hcu = DeviceArray(hip, np.concatenate([[0], np.cumsum(hist)]).astype(np.int32))
        hl, m = DeviceArray(hip, np.array(hist, np.int32)), sum(hist)
        hk_, hv = (R.put(hip, rng.standard_normal((m, hk, d)), dtype) for _ in range(2))
        self.cache.append(ch.Kv8Batch(hcu, hl, self.table, m, max(hist)), hk_, hv, rope=self.rope)
        hip.sync()
        R.free(hcu, hl, hk_, hv)

    def feed(self, lens, seed):
        """New rows and lengths, between calls."""
        rng = np.random.default_rng(seed)
        for a in (self.q, self.k, self.v):
            x = rng.standard_normal(a.shape)
            host = R.bf16_bits(x) if self.dtype == "bfloat16" else x.astype(np.float32)
            self.hip.h2d(a.data_ptr(), np.ascontiguousarray(host))
        self.hip.h2d(self.lens.data_ptr(), np.array(lens, np.int32))

    def run(self, stream=None):
        self.cache.append(self.batch, self.k, self.v, q=self.q, rope=self.rope, stream=stream)
        self.cache.attend(self.batch, self.q, self.out, lse=self.lse, workspace=self.ws, stream=stream)
        self.cache.read(self.batch, self.kr, self.vr, stream=stream)
        logits = R.View(self.out, 0, (self.n, self.V), (self.V, 1))
        ch.token_logprobs(logits, self.targets, self.lp, self.en, self.ids, self.tl, workspace=self.lws, stream=stream)

    def results(self):
        return [a.numpy() for a in (self.q, self.out, self.lse, self.kr, self.vr, self.lp, self.en, self.ids, self.tl)]

    def free(self):
        R.free(self.cu, self.table, self.lens, self.q, self.k, self.v, self.out, self.kr, self.vr, self.lse, self.targets,
               self.lp, self.en, self.ids, self.tl, self.ws, self.lws, *self.cache_arrays)


def same(a, b):
    for x, y in zip(a, b):
        assert np.array_equal(x.view(np.uint8), y.view(np.uint8))


ROWS, LENS = [1, 1, 1], [2100, 5, 700]
PROMPT_ROWS, PROMPT_LENS = [70, 3, 1], [900, 3, 65]


def grown(lens, i, rows):
    return [n + i * r for n, r in zip(lens, rows)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("rows,lens", [(ROWS, LENS), (PROMPT_ROWS, PROMPT_LENS)], ids=["steps", "prompts"])
def test_two_streams_at_once(hip, streams, rows, lens, dtype):
    pair = [Program(hip, s, rows, lens, dtype=dtype) for s in (1, 2)]
    plain = [Program(hip, s, rows, lens, dtype=dtype) for s in (1, 2)]
    for i in range(4):
        for s in (0, 1):
            for p in (pair[s], plain[s]):
                p.feed(grown(lens, i, rows), 10 * i + s)
        hip.sync()
        for s in (0, 1):
            pair[s].run(streams[s])
        hip.sync()
        for s in (0, 1):
            plain[s].run()
            same(pair[s].results(), plain[s].results())
    for p in pair + plain:
        p.free()


def test_the_threads_own_stream(hip):
    a, b = (Program(hip, 7, PROMPT_ROWS, PROMPT_LENS) for _ in range(2))
    for p in (a, b):
        p.feed(PROMPT_LENS, 8)
    hip.sync()
    a.run(2)  # hipStreamPerThread
    b.run()
    hip.sync()
    same(a.results(), b.results())
    for p in (a, b):
        p.free()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("rows,lens", [(ROWS, LENS), (PROMPT_ROWS, PROMPT_LENS)], ids=["steps", "prompts"])
def test_captured_and_replayed(hip, streams, rows, lens, dtype):
    """Two graphs over buffers of their own, captured once and replayed with new rows and lengths, the programs' eager
    work between."""
    L, graphs = hip.L, []
    pair = [Program(hip, s, rows, lens, dtype=dtype) for s in (3, 4)]
    plain = [Program(hip, s, rows, lens, dtype=dtype) for s in (3, 4)]
    for p, st in zip(pair, streams):
        st = ctypes.c_void_p(st)
        assert L.hipStreamBeginCapture(st, 0) == 0  # global capture mode
        try:
            p.run(st.value)
        finally:
            g = ctypes.c_void_p()
            e = L.hipStreamEndCapture(st, ctypes.byref(g))
        assert e == 0
        ex = ctypes.c_void_p()
        assert L.hipGraphInstantiate(ctypes.byref(ex), g, None, None, 0) == 0
        assert L.hipGraphDestroy(g) == 0
        graphs.append(ex)
    for i in range(5):
        for s in (0, 1):
            for p in (pair[s], plain[s]):
                p.feed(grown(lens, i, rows), 100 * i + s)
        hip.sync()
        for ex, st in zip(graphs, streams):
            assert L.hipGraphLaunch(ex, ctypes.c_void_p(st)) == 0
        hip.sync()
        for s in (0, 1):
            plain[s].run()
            same(pair[s].results(), plain[s].results())
    for ex in graphs:
        assert L.hipGraphExecDestroy(ex) == 0
    for p in pair + plain:
        p.free()


@pytest.mark.parametrize("choice", ["0", "1"], ids=["few", "prompt"])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
def test_output_in_the_queries_place(hip, monkeypatch, choice, dtype):
    monkeypatch.setenv("CIH_KV8_PROMPT", choice)
    rows, lens = [40, 1, 7], [300, 1200, 7]
    p = Program(hip, 5, rows, lens, dtype="bfloat16")
    x = np.random.default_rng(6).standard_normal((p.n, p.HK * p.G, p.D))
    q, out = R.put(hip, x, dtype), R.put(hip, x * 0, dtype)
    p.cache.attend(p.batch, q, out, workspace=p.ws)
    p.cache.attend(p.batch, q, q, workspace=p.ws)
    assert np.array_equal(q.numpy().view(np.uint8), out.numpy().view(np.uint8))
    R.free(q, out)
    p.free()


@pytest.mark.parametrize("choice", ["0", "1"], ids=["few", "prompt"])
def test_offsets_past_32_bits(hip, monkeypatch, choice):
    """Codes at byte offsets beyond 2^31 and 2^32 of a pool: as in a pool of four pages."""
    monkeypatch.setenv("CIH_KV8_PROMPT", choice)
    d, hk, g, n, dtype = 128, 4, 2, 200, "bfloat16"
    rng = np.random.default_rng(8)
    x = [R.put(hip, rng.standard_normal((n, w, d)), dtype) for w in (hk * g, hk, hk)]
    cu, lens = DeviceArray(hip, np.array([0, n], np.int32)), DeviceArray(hip, np.array([n], np.int32))
    got = []
    for pages, ids in ((4, [2, 0, 3, 1]), (140000, [139999, 0, 70001, 131071])):
        assert pages == 4 or max(ids) * hk * 64 * d > 2 ** 32
        arrays = [Raw(hip, (pages, hk, 64, d), "int8"), Raw(hip, (pages, hk, d, 64), "int8"),
                  Raw(hip, (pages, hk, 2), "float32"), Raw(hip, (pages, hk), "uint64")]
        cache, table = ch.Kv8Cache(*arrays, d), DeviceArray(hip, np.array([ids], np.int32))
        b = ch.Kv8Batch(cu, lens, table, n, n)
        out, kr, vr = (R.put(hip, np.zeros((n, w, d)), dtype) for w in (hk * g, hk, hk))
        ws = DeviceArray(hip, np.zeros(cache.attend_workspace(b, hk * g) + 16, np.uint8))
        cache.append(b, x[1], x[2], rope=ch.Rope(d))
        cache.read(b, kr, vr)
        cache.attend(b, x[0], out, workspace=ws)
        got.append([a.numpy() for a in (out, kr, vr)])
        hip.sync()
        R.free(table, out, kr, vr, ws, *arrays)
    same(*got)
    assert np.abs(got[0][1].astype(np.int64)).max() > 0
    R.free(cu, lens, *x)

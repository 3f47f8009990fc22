"""Decoding with a bounded cache, as a program does it: new rows appended at shifted
positions, attention over a window and sinks (or all that is left), their weights
gathered, the cache cut to its budget, the rows' drafts verified.  Every step against
the restatements in 64 bits; on two streams at once and replayed from graphs the bits of
the plain eager calls.
"""
import ctypes

import numpy as np
import pytest

import codon_hip as ch
import kv8_more_ref as M
import kv8_ref as R
from codon_hip.devmem import DeviceArray, Hip
from test_gpu_kv8 import check_attention
from test_gpu_ops_streams import Raw, same, streams  # noqa: F401 (streams is a fixture)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    return Hip()


class Loop:
    """Sequences at their budget that take rows at each step.  `lens` (budget and rows) stays, so that a step can be replayed."""

    D, HK, G = 64, 2, 2
    FIRST, RECENT = 4, 20

    def __init__(self, hip, seed, rows, budget, vocab, window=0, sinks=0, dtype="bfloat16", heat=1.0):
        self.hip, self.dtype, self.budget, self.vocab, self.heat = hip, dtype, budget, vocab, heat
        self.window, self.sinks, self.rows = window, sinks, rows
        rng = np.random.default_rng(seed)
        n, self.n, d, hk, h = len(rows), int(sum(rows)), self.D, self.HK, self.HK * self.G
        pages = -(-(budget + max(rows)) // 64)
        self.table_np = rng.permutation(n * pages + 3)[:n * pages].astype(np.int32).reshape(n, pages)
        self.cu_np = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        every = n * pages + 3  # (nothing reads what no call has written)
        self.cache_arrays = [DeviceArray(hip, x) for x in (
            np.full((every, hk, 64, d), 85, np.int8), np.full((every, hk, d, 64), 85, np.int8),
            np.full((every, hk, 2), np.nan, np.float32), np.full((every, hk), 2 ** 64 - 1, np.uint64))]
        self.cache = ch.Kv8Cache(*self.cache_arrays, d)
        up = lambda x: DeviceArray(hip, np.asarray(x))  # noqa: E731
        self.weights = up(np.zeros((n * pages + 3, hk, 64), np.float32))
        self.cu, self.table = up(self.cu_np), up(self.table_np)
        self.lens = up((budget + np.array(rows)).astype(np.int32))
        self.held, self.shifts = up(np.zeros(n, np.int32)), up(np.zeros(n, np.int32))
        self.kept = up(np.zeros((n, hk, budget), np.int32))
        self.batch = ch.Kv8Batch(self.cu, self.lens, self.table, self.n, max(rows))
        one = lambda w: R.put(hip, np.zeros((self.n, w, d)), dtype)  # noqa: E731
        self.q, self.k, self.v, self.out = one(h), one(hk), one(hk), one(h)
        self.lse = up(np.zeros((self.n, h), np.float32))
        # drafts: a row each but the last of a sequence
        self.drafts_n = self.n - n
        self.cu_drafts_np = (self.cu_np - np.arange(n + 1)).astype(np.int32)
        self.cu_drafts = up(self.cu_drafts_np)
        self.drafts = up(np.zeros(self.drafts_n, np.int32))
        self.u, self.w = up(np.zeros(self.drafts_n, np.float32)), up(np.zeros(n, np.float32))
        self.about = R.put(hip, np.zeros((self.drafts_n, vocab)), dtype)
        self.accepted, self.tokens = up(np.zeros(n, np.int32)), up(np.zeros(n, np.int32))
        byte = lambda size: up(np.full(size + 16, 255, np.uint8))  # noqa: E731
        self.ws = byte(self.cache.attend_workspace(self.batch, h))
        self.ews = byte(self.cache.evict_workspace(self.batch, budget))
        self.vws = byte(ch.verify_drafts_workspace(n, self.drafts_n, vocab))
        self.rope = ch.Rope(d)
        # the budget's tokens
        full = up(np.full(n, budget, np.int32))
        fcu = up((np.arange(n + 1) * budget).astype(np.int32))
        kv = [R.put(hip, rng.standard_normal((n * budget, hk, d)), dtype) for _ in range(2)]
        self.cache.append(ch.Kv8Batch(fcu, full, self.table, n * budget, budget), *kv, rope=self.rope)
        hip.sync()
        R.free(full, fcu, *kv)

    def feed(self, seed):
        rng = np.random.default_rng(seed)
        self.host = {}
        for name in ("q", "k", "v", "about"):
            a = getattr(self, name)
            x = rng.standard_normal(a.shape) * (2 if name in ("q", "about") else 1)
            self.host[name] = R.rounded(x, self.dtype)
            bits = R.bf16_bits(x) if self.dtype == "bfloat16" else self.host[name].astype(self.dtype)
            self.hip.h2d(a.data_ptr(), np.ascontiguousarray(bits))
        for name, x in (("drafts", rng.integers(0, self.vocab, self.drafts_n).astype(np.int32)),
                        ("u", (rng.random(self.drafts_n) * 1e-4).astype(np.float32)),
                        ("w", np.minimum(rng.random(len(self.rows)), 0.999999).astype(np.float32))):
            self.host[name] = x
            self.hip.h2d(getattr(self, name).data_ptr(), x)

    def run(self, stream=None, check=None):
        check = check or (lambda what: None)
        self.cache.append(self.batch, self.k, self.v, q=self.q, rope=self.rope, shifts=self.shifts, stream=stream)
        check("append")
        self.cache.attend(self.batch, self.q, self.out, lse=self.lse, window=self.window, sinks=self.sinks, workspace=self.ws,
                          stream=stream)
        check("attend")
        self.cache.weigh(self.batch, self.q, self.lse, self.weights, window=self.window, sinks=self.sinks, keep=0.9, stream=stream)
        check("weigh")
        self.cache.evict(self.batch, self.weights, self.budget, first=self.FIRST, recent=self.RECENT, lens_out=self.held,
                         shifts=self.shifts, kept=self.kept, workspace=self.ews, stream=stream)
        check("evict")
        logits = R.View(self.out, 0, (self.n, self.vocab), (self.HK * self.G * self.D, 1))
        ch.verify_drafts(logits, self.drafts, self.cu_drafts, self.accepted, self.tokens, draft_logits=self.about,
                         accept_at=self.u, sample_at=self.w, temperature=self.heat, workspace=self.vws, stream=stream)
        check("verify")

    def results(self):
        used = [a.numpy()[self.table_np[:, :self.budget // 64]] for a in (*self.cache_arrays, self.weights)]
        return [a.numpy() for a in (self.q, self.out, self.lse, self.held, self.shifts, self.kept, self.accepted, self.tokens)] + used

    def free(self):
        R.free(self.weights, self.cu, self.table, self.lens, self.held, self.shifts, self.kept, self.q, self.k, self.v, self.out,
               self.lse, self.cu_drafts, self.drafts, self.u, self.w, self.about, self.accepted, self.tokens, self.ws, self.ews,
               self.vws, *self.cache_arrays)


class Cut:
    """What kv8_ref.Cache offers, of arrays that were read back."""

    gather, values = R.Cache.gather, R.Cache.values

    def __init__(self, p):
        self.k, self.v, self.scales, self.bad = [a.numpy() for a in p.cache_arrays]
        self.d = p.D


STEPS, PROMPTS = [1, 4, 3], [40, 1, 9]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("rows,budget,vocab,window,sinks", [(STEPS, 300, 40, 0, 0), (PROMPTS, 128, 256, 90, 5), ([1], 1000, 33, 200, 70)],
                         ids=["steps", "chunks", "one"])
def test_steps_follow_the_restatements(hip, rows, budget, vocab, window, sinks, dtype):
    p = Loop(hip, 1, rows, budget, vocab, window, sinks, dtype)
    shift = np.zeros(len(rows), np.int64)
    state = {}

    def check(what):
        hip.sync()
        c, seqs = Cut(p), range(len(rows))
        lens = budget + np.array(rows)
        w = p.weights.numpy()
        if what == "append":
            got = R.get(p.q)
            for i in seqs:
                a = slice(p.cu_np[i], p.cu_np[i + 1])
                pos = np.arange(budget, lens[i])
                want = R.rope(p.host["q"][a], pos + shift[i], p.rope)
                assert (np.abs(got[a] - want) <= R.EPS[dtype] * np.abs(want) + 2.0 ** -20 * np.abs(want).max()).all()
                k = R.rope(p.host["k"][a], pos + shift[i], p.rope)
                for r, t in enumerate(pos):
                    page = p.table_np[i, t // 64]
                    off = np.abs(c.k[page, :, t % 64] - k[r] / c.scales[page, :, :1].astype(np.float64))
                    assert off.max() <= 0.5 + 1e-3
            state["w"] = w
        if what == "attend":
            out, lse, q = R.get(p.out), p.lse.numpy(), R.get(p.q)
            for i in seqs:
                a = slice(p.cu_np[i], p.cu_np[i + 1])
                ref = M.attention(c, p.table_np[i], lens[i], np.arange(budget, lens[i]), q[a], p.D ** -0.5, True, window, sinks, p.G)
                check_attention(out[a], lse[a], *ref, dtype, 127 * float(c.scales.max()))
        if what == "weigh":
            lse, q = p.lse.numpy().astype(np.float64), R.get(p.q)
            for i in seqs:
                a = slice(p.cu_np[i], p.cu_np[i + 1])
                g, tol = M.gained(c, p.table_np[i], lens[i], np.arange(budget, lens[i]), q[a], lse[a], p.D ** -0.5, True, window, sinks, p.G)
                j = np.arange(lens[i])
                page = p.table_np[i, j // 64]
                old = np.where(j < budget, np.float64(np.float32(0.9)) * state["w"][page, :, j % 64].T, 0)
                assert (np.abs(w[page, :, j % 64].T - old - g) <= tol + 2.0 ** -23 * (old + g)).all()
            state["w"], state["c"] = w, c
        if what == "evict":
            k, v, scales, bad, wout, kept, out = M.evict(state["c"], state["w"], p.table_np, list(lens), np.arange(len(rows)), budget, p.FIRST, p.RECENT)
            assert np.array_equal(p.kept.numpy(), kept) and np.array_equal(p.held.numpy(), out) and (out == budget).all()
            shift[:] += np.array(rows)
            assert np.array_equal(p.shifts.numpy(), shift)
            for i in seqs:
                j = np.arange(budget)
                page = p.table_np[i, j // 64]
                assert np.array_equal(c.k[page, :, j % 64], k[page, :, j % 64]) and np.array_equal(c.v[page, :, :, j % 64], v[page, :, :, j % 64])
                assert np.array_equal(c.scales[page], scales[page]) and np.array_equal(w[page, :, j % 64], wout[page, :, j % 64])
        if what == "verify":
            logits = R.get(p.out).reshape(p.n, -1)[:, :vocab]
            want = M.verify(logits, p.host["about"], p.cu_drafts_np, p.host["drafts"], p.host["u"], p.host["w"], p.heat)
            assert np.array_equal(p.accepted.numpy(), want[0]) and np.array_equal(p.tokens.numpy(), want[1])

    for i in range(5):
        p.feed(20 + i)
        p.run(check=check)
    p.free()


LOOPS = [(STEPS, 300, 40, 0, 0), (PROMPTS, 192, 256, 90, 5), ([2, 3], 2200, 250, 0, 0)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("args", LOOPS, ids=["steps", "chunks", "long"])
def test_two_streams_at_once(hip, streams, args, dtype):  # noqa: F811
    pair, plain = ([Loop(hip, s, *args, dtype=dtype) for s in (1, 2)] for _ in range(2))
    for i in range(4):
        for s in (0, 1):
            for p in (pair[s], plain[s]):
                p.feed(10 * i + s)
        hip.sync()
        for s in (0, 1):
            pair[s].run(streams[s])
        hip.sync()
        for s in (0, 1):
            plain[s].run()
            same(pair[s].results(), plain[s].results())
    for p in pair + plain:
        p.free()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("args", LOOPS, ids=["steps", "chunks", "long"])
def test_captured_and_replayed(hip, streams, args, dtype):  # noqa: F811
    """Two graphs over buffers of their own, captured once and replayed on new rows, the programs' eager work between."""
    L, graphs = hip.L, []
    pair, plain = ([Loop(hip, s, *args, dtype=dtype) for s in (3, 4)] for _ in range(2))
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
                p.feed(100 * i + s)
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


def test_long_tables_at_once_and_replayed(hip, streams):  # noqa: F811
    """Tables of more than 8,192 tokens, where several workgroups choose for a head."""
    args = ([130, 7, 1], 8800, 250, 0, 0)
    test_two_streams_at_once(hip, streams, args, "float16")
    test_captured_and_replayed(hip, streams, args, "float16")


def test_offsets_past_32_bits(hip):
    """Codes and weights at byte offsets beyond 2^31 and 2^32: as in a pool of five pages."""
    d, hk, g, n, budget, dtype = 128, 4, 2, 300, 130, "bfloat16"
    rng = np.random.default_rng(8)
    x = [R.put(hip, rng.standard_normal((n, w, d)), dtype) for w in (hk * g, hk, hk)]
    cu, lens = DeviceArray(hip, np.array([0, n], np.int32)), DeviceArray(hip, np.array([n], np.int32))
    got = []
    for pages, ids in ((5, [2, 0, 4, 3, 1]), (140000, [139999, 0, 70001, 131071, 139998])):
        arrays = [Raw(hip, (pages, hk, 64, d), "int8"), Raw(hip, (pages, hk, d, 64), "int8"),
                  Raw(hip, (pages, hk, 2), "float32"), Raw(hip, (pages, hk), "uint64"), Raw(hip, (pages, hk, 64), "float32")]
        cache, table = ch.Kv8Cache(*arrays[:4], d), DeviceArray(hip, np.array([ids], np.int32))
        b = ch.Kv8Batch(cu, lens, table, n, n)
        out, kr, vr = (R.put(hip, np.zeros((n, w, d)), dtype) for w in (hk * g, hk, hk))
        lse = DeviceArray(hip, np.zeros((n, hk * g), np.float32))
        ws = DeviceArray(hip, np.zeros(max(cache.attend_workspace(b, hk * g), cache.evict_workspace(b, budget)), np.uint8))
        held, kept = DeviceArray(hip, np.zeros(1, np.int32)), DeviceArray(hip, np.zeros((1, hk, budget), np.int32))
        cache.append(b, x[1], x[2], rope=ch.Rope(d))
        cache.attend(b, x[0], out, lse=lse, window=90, sinks=5, workspace=ws)
        cache.weigh(b, x[0], lse, arrays[4], window=90, sinks=5, keep=0.0)
        cache.evict(b, arrays[4], budget, first=5, recent=20, lens_out=held, kept=kept, workspace=ws)
        few = DeviceArray(hip, np.array([0, budget], np.int32))
        cache.read(ch.Kv8Batch(few, held, table, n, budget), kr, vr)
        got.append([a.numpy() for a in (out, lse, kept, held, kr, vr)])
        hip.sync()
        R.free(table, out, kr, vr, ws, lse, held, kept, few, *arrays)
    same(*got)
    assert np.abs(got[0][4].astype(np.int64)).max() > 0
    R.free(cu, lens, *x)


def test_torch_tensors_and_streams():
    """The calls on torch tensors: torch's current stream, outputs in place, what the plain null-stream calls give."""
    torch = pytest.importorskip("torch")
    dev, d, hk, n = "cuda", 64, 2, 200
    gen = torch.Generator(device=dev).manual_seed(3)
    results = []
    for stream in (None, torch.cuda.Stream()):
        gen.manual_seed(3)
        rand = lambda *s: torch.randn(*s, device=dev, generator=gen)  # noqa: E731
        cache = ch.Kv8Cache(torch.empty(4, hk, 64, d, dtype=torch.int8, device=dev), torch.empty(4, hk, d, 64, dtype=torch.int8, device=dev),
                            torch.empty(4, hk, 2, device=dev), torch.empty(4, hk, dtype=torch.int64, device=dev), d)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        lens, shifts = i32([n]), i32([0])
        b = ch.Kv8Batch(i32([0, n]), lens, i32([[3, 1, 0, 2]]), n, n)
        q, k, v = rand(n, 2 * hk, d), rand(n, hk, d), rand(n, hk, d)
        out, lse, w = torch.empty_like(q), torch.empty(n, 2 * hk, device=dev), torch.empty(4, hk, 64, device=dev)
        ws = torch.empty(max(cache.attend_workspace(b, 2 * hk), cache.evict_workspace(b, 100)), dtype=torch.uint8, device=dev)
        logits, about, drafts = rand(6, 500), rand(4, 500), i32([1, 2, 3, 4])
        acc, tok, u, s = i32([0, 0]), i32([0, 0]), torch.rand(4, device=dev, generator=gen), torch.rand(2, device=dev, generator=gen)
        vws = torch.empty(ch.verify_drafts_workspace(2, 4, 500), dtype=torch.uint8, device=dev)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            cache.append(b, k, v, q=q, rope=ch.Rope(d), shifts=shifts)
            cache.attend(b, q, out, lse=lse, window=64, sinks=4, workspace=ws)
            cache.weigh(b, q, lse, w, window=64, sinks=4, keep=0.0)
            cache.evict(b, w, 100, first=4, recent=10, shifts=shifts, workspace=ws)
            ch.verify_drafts(logits, drafts, i32([0, 3, 4]), acc, tok, draft_logits=about, accept_at=u, sample_at=s, workspace=vws)
        torch.cuda.synchronize()
        assert lens.item() == 100 and shifts.item() == n - 100
        results.append([x.clone() for x in (out, lse, w[torch.tensor([3])], acc, tok)])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    with pytest.raises(ValueError):
        cache.weigh(b, q, lse, w.cpu())
    with pytest.raises(ValueError):
        ch.verify_drafts(logits, drafts, i32([0, 3, 4]), acc.cpu(), tok, temperature=0.0)

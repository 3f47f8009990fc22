"""Decoders over the 8-bit paged cache (cih_decoder_create_kv8), scores of
given sequences (cih_decoder_score) and reading the cache back.

A step is checked against the model in 64 bits over the keys and values that
the decoder holds (read back from it), so that what is left is the GPU's FP32
arithmetic: logits within 1e-3 absolute, as the decoder over FP32 caches.  The
cache itself is checked in the first layer, whose inputs do not depend on it.
"""
import numpy as np
import pytest

import codon_hip as ch
from codon_hip import _lib as C
from ref64 import _gelu, _ln, dense_weights
from test_gpu_decode import overflow_model

pytestmark = pytest.mark.gpu
TOL = 1e-3


def turn(x, pos, rope, hd):
    """Rows [n][heads][hd] by the decoder's rotary positions (None: the reference's)."""
    half = hd // 2 if rope is None else len(rope.freq)
    f = 10000.0 ** (-2.0 * np.arange(half) / hd) if rope is None else np.asarray(rope.freq)
    gain = 1.0 if rope is None else float(rope.gain)
    a = pos[:, None, None] * f
    c, s = gain * np.cos(a), gain * np.sin(a)
    y = x.copy()
    i0, i1 = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if rope is not None and rope.struct.interleaved else \
        (slice(0, half), slice(half, 2 * half))
    y[..., i0], y[..., i1] = x[..., i0] * c - x[..., i1] * s, x[..., i1] * c + x[..., i0] * s
    return y


def rows64(cfg, W, tokens, pos, caches, rope=None):
    """Logits of rows (token, position) of one sequence over caches[layer] = (K, V) [positions][dim]."""
    d, F, L, H, V = cfg.dim, cfg.hidden_dim, cfg.n_layers, cfg.n_heads, cfg.vocab_size
    hd, n = d // H, len(tokens)
    pos = np.asarray(pos)
    emb = W["token_embedding_table"].reshape(V, d)
    x = np.stack([np.zeros(d) if t == 32 else emb[t] * np.float64(np.float32(0.88)) for t in tokens])

    def mat(name, l, o, i):
        return W[name].reshape(L, o, i)[l]

    def vec(name, l, o):
        return W[name].reshape(L, o)[l]

    for l in range(L):
        h = _ln(x, vec("ln_1_weight", l, d), vec("ln_1_bias", l, d))
        q = turn((h @ mat("wq", l, d, d).T + vec("bq", l, d)).reshape(n, H, hd), pos, rope, hd)
        K, Vv = (c.astype(np.float64).reshape(-1, H, hd) for c in caches[l])
        s = np.einsum("qhe,khe->hqk", q, K) / np.sqrt(hd)
        s = np.where(np.arange(len(K))[None, None] <= pos[None, :, None], s, -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        p /= p.sum(-1, keepdims=True)
        x = x + np.einsum("hqk,khe->qhe", p, Vv).reshape(n, d) @ mat("wo", l, d, d).T + vec("bo", l, d)
        h = _ln(x, vec("ln_2_weight", l, d), vec("ln_2_bias", l, d))
        x = x + _gelu(h @ mat("fc1_weight", l, F, d).T + vec("fc1_bias", l, F)) @ mat("fc2_weight", l, d, F).T + vec("fc2_bias", l, d)
    x = _ln(x, W["ln_f_weight"], W["ln_f_bias"])
    cw = W["classifier_weights"]
    if cw.size < 3 * d + d * d + V * d + V:
        return x @ emb.T
    dw, db = cw[2 * d:2 * d + d * d].reshape(d, d), cw[2 * d + d * d:3 * d + d * d]
    decw, decb = cw[3 * d + d * d:3 * d + d * d + V * d].reshape(V, d), cw[3 * d + d * d + V * d:3 * d + d * d + V * d + V]
    return _ln(_gelu(x @ dw.T + db), cw[:d], cw[d:2 * d]) @ decw.T + decb


def held(dec, cfg, slot, n):
    return [dec.read_cache(l, slot, 0, n) for l in range(cfg.n_layers)]


def make(hd, fmt="q8", heads=4, layers=2, seed=0, **kw):
    cfg = ch.EsmConfig(heads * hd, 4 * heads * hd, layers, heads)
    w = ch.EsmWeights.random(cfg, seed=seed + hd, std=0.06, bias_std=0.02)
    w = {"fp32": lambda: w, "q8": w.quantize_q8, "q4": w.quantize_q4}[fmt]()
    return cfg, w, ch.GpuModel(cfg, w, max_batch=1, max_len=16)


def tokens(n, seed):
    return np.concatenate([[0], 4 + np.random.default_rng(seed).integers(0, 20, n - 1)]).astype(np.int32)


ROPES = {None: None, "part": dict(interleaved=True), "yarn": dict(scaling="yarn", factor=4.0, trained_len=64)}


@pytest.mark.parametrize("hd,fmt,rope", [(16, "q8", None), (24, "q8", "yarn"), (32, "q4", "part"), (64, "q8", None),
                                         (64, "fp32", "yarn"), (64, "q4", "part"), (32, "fp32", None)])
def test_prompts_and_steps(hd, fmt, rope):
    """Prompts of two slots in one call (their rows mixed), then steps of both, across a page's end."""
    heads = 8 if hd == 24 else 4
    cfg, w, m = make(hd, fmt, heads)
    W = dense_weights(cfg, w)
    r = None if rope is None else ch.Rope(hd // 2 if rope == "part" else hd, **ROPES[rope])
    dec = ch.GpuDecoder(m, n_slots=3, max_len=200, max_rows=128, kv8=True, rope=r)
    ta, tb = tokens(70, 1), tokens(41, 2)
    na, nb = 60, 37
    order = sorted([(p * 37, 2, p) for p in range(na)] + [(p * 60, 0, p) for p in range(nb)])
    slots, pos = [o[1] for o in order], [o[2] for o in order]
    got = dec.decode(slots, [ta[p] if s == 2 else tb[p] for s, p in zip(slots, pos)], pos)
    for s, t, n in ((2, ta, na), (0, tb, nb)):
        ref = rows64(cfg, W, t[:n], np.arange(n), held(dec, cfg, s, n), r)
        mine = np.stack([got[i] for i in range(len(slots)) if slots[i] == s])
        assert np.abs(mine - ref).max() <= TOL, (s, np.abs(mine - ref).max())
    for i in range(8):
        got = dec.decode([0, 2], [tb[nb + i % 4], ta[na + i]], [nb + i, na + i])
        for j, (s, t, p) in enumerate(((0, tb[nb + i % 4], nb + i), (2, ta[na + i], na + i))):
            ref = rows64(cfg, W, [t], [p], held(dec, cfg, s, p + 1), r)
            assert np.abs(got[j] - ref[0]).max() <= TOL, (s, p)
    dec.close()
    m.close()


def test_first_layer_cache():
    """K and V of the first layer against the FP32 decoder's: half a code, and half a code more for every time a later
    call raised the page's scale."""
    cfg, w, m = make(64)
    a = ch.GpuDecoder(m, n_slots=1, max_len=150, max_rows=64)
    b = ch.GpuDecoder(m, n_slots=2, max_len=150, max_rows=64, kv8=True)
    t = tokens(140, 3)
    at = 0
    for n in (50, 1, 1, 60, 28):
        for dec, s in ((a, 0), (b, 1)):
            dec.decode([s] * n, t[at:at + n], np.arange(at, at + n))
        at += n
    for x, y in zip(a.read_cache(0, 0, 0, at), b.read_cache(0, 1, 0, at)):
        x, y = x.reshape(at, 4, 64), y.reshape(at, 4, 64)
        for p0 in range(0, at, 64):
            step = np.abs(x[p0:p0 + 64]).max((0, 2)) / 127
            # the FP32 decoder's angles are FP32 products: off by 2^-24 of the position, times the value
            off = np.abs(x[p0:p0 + 64] - y[p0:p0 + 64]).max((0, 2))
            assert (off <= 5 * 0.5 * step * 1.01 + 150 * 2.0 ** -23 * 127 * step).all(), (p0, off / step)
    u, v = b.read_cache(0, 1, 70, 20), b.read_cache(0, 1, 0, at)
    assert np.array_equal(u[0], v[0][70:90]) and np.array_equal(u[1], v[1][70:90])
    for dec in (a, b):
        dec.close()
    m.close()


def test_pool_of_pages():
    """Slots share a pool: a call that needs more pages than are free changes nothing; reset and rewriting give back."""
    cfg, w, m = make(32)
    W = dense_weights(cfg, w)
    dec = ch.GpuDecoder(m, n_slots=4, max_len=640, max_rows=256, kv8=True, n_pages=5)
    t = tokens(300, 4)
    dec.decode([0] * 200, t[:200], np.arange(200))          # 4 pages
    dec.decode([1] * 10, t[:10], np.arange(10))             # the fifth
    for bad in (([2], [0], [0]), ([0] * 57, t[200:257], np.arange(200, 257))):
        with pytest.raises(ch.CihError) as e:
            dec.decode(*bad)
        assert e.value.code == -3
    got = dec.decode([0, 1], [t[200], t[10]], [200, 10])    # still as they were
    for j, (s, p) in enumerate(((0, 200), (1, 10))):
        ref = rows64(cfg, W, [t[p]], [p], held(dec, cfg, s, p + 1))
        assert np.abs(got[j] - ref[0]).max() <= TOL
    dec.decode([0], [t[100]], [100])                        # rewrites: 101 tokens, two pages go back
    with pytest.raises(ch.CihError):
        dec.read_cache(0, 0, 101, 1)
    with pytest.raises(ch.CihError):
        dec.decode([0], [5], [103])                         # does not continue
    got = dec.decode([2] * 100 + [0], np.concatenate([t[:100], t[101:102]]), list(range(100)) + [101])
    ref = rows64(cfg, W, t[:100], np.arange(100), held(dec, cfg, 2, 100))
    assert np.abs(got[:100] - ref).max() <= TOL
    assert np.abs(got[100] - rows64(cfg, W, [t[101]], [101], held(dec, cfg, 0, 102))[0]).max() <= TOL
    dec.reset(2)
    dec.reset(0)
    dec.decode([3] * 250, t[:250], np.arange(250))          # four pages again
    dec.reset()
    dec.decode([3] * 256, np.resize(t, 256), np.arange(256))
    dec.close()
    m.close()


@pytest.mark.parametrize("fmt,streams", [("q8", 3), ("q4", 1), ("fp32", 2)])
def test_graph_replays_match_eager(fmt, streams, monkeypatch):
    """Captured steps against kernel by kernel, bit for bit, over a page's end, with other calls in between."""
    cfg, w, m = make(64, fmt)
    t = [tokens(90, 10 + s) for s in range(streams)]
    sl = list(range(streams))
    out = {}
    for env in ("1", "0"):
        monkeypatch.setenv("CIH_DECODE_GRAPH", env)
        dec = ch.GpuDecoder(m, n_slots=streams + 1, max_len=128, max_rows=64, kv8=True)
        got = []
        for s in sl:
            got.append(dec.decode([s] * 50, t[s][:50], np.arange(50)))
        for p in range(50, 80):
            got.append(dec.decode(sl, [t[s][p] for s in sl], [p] * streams))
            if p % 7 == 0:
                got.append(dec.decode([streams] * 3, [5, 6, 7], np.arange(3)))
                got.append(dec.decode([streams, streams], [8, 9], [3, 4]))
        out[env] = got
        dec.close()
    for i, (x, y) in enumerate(zip(out["1"], out["0"])):
        assert np.array_equal(x, y), i
    m.close()


@pytest.mark.parametrize("hd,fmt", [(64, "q8"), (24, "fp32")])
def test_many_streams(hd, fmt):
    """More streams than the GEMV takes, each at its own position; pages that start, fill and end."""
    cfg, w, m = make(hd, fmt, heads=8 if hd == 24 else 4)
    W = dense_weights(cfg, w)
    n = 20
    dec = ch.GpuDecoder(m, n_slots=n, max_len=2048, max_rows=64, kv8=True, n_pages=60)
    t = [tokens(140, 40 + s) for s in range(n)]
    at = [(7 * s) % 64 + 64 * (s % 2) for s in range(n)]
    for s in range(n):
        for p in range(0, at[s], 50):
            k = min(50, at[s] - p)
            dec.decode([s] * k, t[s][p:p + k], np.arange(p, p + k))
    for i in range(3):
        got = dec.decode(list(range(n)), [t[s][at[s] + i] for s in range(n)], [at[s] + i for s in range(n)])
        for s in range(n):
            ref = rows64(cfg, W, [t[s][at[s] + i]], [at[s] + i], held(dec, cfg, s, at[s] + i + 1))
            assert np.abs(got[s] - ref[0]).max() <= TOL, (i, s)
    dec.close()
    m.close()


@pytest.mark.parametrize("hd,fmt", [(16, "q8"), (24, "q4"), (32, "fp32"), (64, "q8")])
def test_steps_from_the_first_token(hd, fmt):
    """A sequence token by token, through every place of a page and into the next, then again from the middle of it."""
    cfg, w, m = make(hd, fmt, heads=8 if hd == 24 else 4)
    W = dense_weights(cfg, w)
    dec = ch.GpuDecoder(m, n_slots=2, max_len=130, max_rows=8, kv8=True)
    t = tokens(140, 50 + hd)
    for p in [*range(70), *range(45, 52)]:
        got = dec.decode([1], [t[p]], [p])
        ref = rows64(cfg, W, [t[p]], [p], held(dec, cfg, 1, p + 1))
        assert np.abs(got[0] - ref[0]).max() <= TOL, p
    dec.close()
    m.close()


@pytest.mark.parametrize("rows", [1, 12])
def test_limb_overflow_runs_full_range(rows):
    """Steps and prompts whose activations overflow the f16 limbs run again in full range and write the same positions:
    the kept tokens of their page survive the first run."""
    cfg, w = overflow_model("ln1", 99)
    W = dense_weights(cfg, w)
    m = ch.GpuModel(cfg, w, max_batch=1, max_len=16)
    dec = ch.GpuDecoder(m, n_slots=1, max_len=64, max_rows=16, kv8=True)
    t = tokens(40, 5)
    for p in range(0, 24, rows):
        got = dec.decode([0] * rows, t[p:p + rows], np.arange(p, p + rows))
        ref = rows64(cfg, W, t[p:p + rows], np.arange(p, p + rows), held(dec, cfg, 0, p + rows))
        assert np.abs(got - ref).max() <= TOL, p
    dec.close()
    m.close()


def test_generate():
    """Greedy generation equals stepping; a stream's tokens do not depend on the others'."""
    cfg, w, m = make(64, "q4")
    dec = ch.GpuDecoder(m, n_slots=3, max_len=128, max_rows=32, kv8=True, n_pages=6)
    prompts = [tokens(n, n) for n in (5, 61, 30)]
    got, _, _ = dec.generate(prompts, 0.0, 20, [1, 2, 3])
    solo = [dec.generate([p], 0.0, 20, [i + 1], slots=[2])[0][0] for i, p in enumerate(prompts)]
    for x, y in zip(got, solo):
        assert np.array_equal(x, y)
    dec.reset()
    logits = dec.decode([1] * 30, prompts[2], np.arange(30))[-1]
    for i, tok in enumerate(got[2]):
        ok = [2] + list(range(4, 24))
        assert tok == ok[int(np.argmax(logits[ok]))] or logits[ok].max() - logits[tok] < 1e-4
        logits = dec.decode([1], [tok], [30 + i])[0]
    dec.close()
    m.close()


def test_positions_past_the_fp32_decoder():
    """A prompt beyond 15000 positions with scaled rotary positions, in chunks, and a step after it."""
    cfg, w, m = make(32, "q8", heads=2, layers=1)
    W = dense_weights(cfg, w)
    n = 15500
    rope = ch.Rope(32, scaling="yarn", factor=16.0, trained_len=1024)
    dec = ch.GpuDecoder(m, n_slots=1, max_len=n + 10, max_rows=4096, kv8=True, rope=rope)
    t = tokens(n + 1, 6)
    for p in range(0, n, 4096):
        k = min(4096, n - p)
        got = dec.decode([0] * k, t[p:p + k], np.arange(p, p + k))
    c = held(dec, cfg, 0, n)
    ref = rows64(cfg, W, t[n - 3:n], np.arange(n - 3, n), c, rope)
    assert np.abs(got[-3:] - ref).max() <= TOL
    got = dec.decode([0], [t[n]], [n])
    assert np.abs(got[0] - rows64(cfg, W, [t[n]], [n], held(dec, cfg, 0, n + 1), rope)[0]).max() <= TOL
    dec.close()
    m.close()


@pytest.mark.parametrize("kv8", [False, True])
def test_score(kv8):
    """Scores of ragged sequences against log softmax in 64 bits of the logits that the same calls (48 rows each) give:
    the sums' and logarithms' FP32 roundings only, below 2^-18 of the logits' size."""
    cfg, w, m = make(64)
    seqs, slots = [tokens(n, 20 + n) for n in (1, 70, 33, 100)], [2, 0, 3, 1]
    rows = [(sl, int(t), p) for sl, s in zip(slots, seqs) for p, t in enumerate(s)]
    other = ch.GpuDecoder(m, n_slots=4, max_len=128, max_rows=48, kv8=kv8)
    lg = np.concatenate([other.decode(*zip(*rows[p:p + 48])) for p in range(0, len(rows), 48)]).astype(np.float64)
    lp = lg - (lg.max(1) + np.log(np.exp(lg - lg.max(1, keepdims=True)).sum(1)))[:, None]
    tol = 2.0 ** -18 * (1 + 2 * np.abs(lg).max() + np.log(33))
    dec = ch.GpuDecoder(m, n_slots=4, max_len=128, max_rows=48, kv8=kv8)
    for top in (0, 5, 33):
        res, at = dec.score(seqs, top, slots=slots), 0
        for s, r in zip(seqs, res):
            x = lp[at:at + len(s)]
            at += len(s)
            assert r["logprob"].shape == (len(s),) and r["top_ids"].shape == (len(s), top)
            assert np.abs(r["logprob"][:-1] - x[np.arange(len(s) - 1), s[1:]]).max(initial=0) <= tol
            assert r["logprob"][-1] == 0
            assert np.abs(r["entropy"] + (np.exp(x) * x).sum(1)).max() <= tol
            order = np.argsort(-lg[at - len(s):at], axis=1, kind="stable")[:, :top]
            assert np.array_equal(r["top_ids"], order)
            assert np.abs(np.take_along_axis(x, order, 1) - r["top_logprobs"]).max(initial=0) <= tol
    # the slots hold the sequences
    got = dec.decode([1], [5], [100])
    assert np.abs(got - other.decode([1], [5], [100])).max() == 0
    other.close()
    dec.close()
    m.close()


def test_score_large_vocabulary():
    """Rows of 500,000 logits, which are split over workgroups and joined, with as many alternatives as there may be."""
    cfg = ch.EsmConfig(64, 256, 1, 2, vocab_size=500_000)
    m = ch.GpuModel(cfg, ch.EsmWeights.random(cfg, seed=5, std=0.06, bias_std=0.02), max_batch=1, max_len=16)
    dec = ch.GpuDecoder(m, n_slots=1, max_len=64, max_rows=4, kv8=True)
    lg = dec.decode([0], [400_000], [0]).astype(np.float64)[0]
    lse = lg.max() + np.log(np.exp(lg - lg.max()).sum())
    tol = 2.0 ** -18 * (1 + 2 * np.abs(lg).max() + np.log(lg.size))
    for top in (0, 33, 64):
        r = dec.score([[400_000]], top)[0]
        best = np.argsort(-lg, kind="stable")[:top]
        assert np.array_equal(r["top_ids"][0], best)
        assert np.abs(r["top_logprobs"][0] - (lg[best] - lse)).max(initial=0) <= tol
        assert abs(r["entropy"][0] - (lse - np.exp(lg - lse) @ lg)) <= tol
    dec.close()
    m.close()


def test_refusals():
    cfg, w, m = make(16)
    for kw in (dict(max_len=1 << 21), dict(n_pages=-1), dict(n_slots=0), dict(rope=ch.Rope(32))):
        with pytest.raises(ch.CihError):
            ch.GpuDecoder(m, **{**dict(n_slots=1, max_len=64, max_rows=8, kv8=True), **kw})
    with pytest.raises(ValueError):
        ch.GpuDecoder(m, n_slots=1, max_len=64, max_rows=8, n_pages=3)
    dec = ch.GpuDecoder(m, n_slots=2, max_len=64, max_rows=8, kv8=True)
    for seqs, kw, code in (([[0, 99]], {}, -8), ([[0, -1]], {}, -8), ([[]], {}, -1), ([[0], [0]], dict(slots=[1, 1]), -1),
                           ([[0]], dict(slots=[2]), -1), ([[0] * 65], {}, -3), ([[0]], dict(top_k=34), -2)):
        with pytest.raises(ch.CihError) as e:
            dec.score(seqs, **kw)
        assert e.value.code == code, (seqs, kw)
    zero, offs = np.zeros(8, np.int32), np.array([-1, 1], np.int32)
    assert C.lib().cih_decoder_score(dec._h, 1, zero.ctypes.data, zero.ctypes.data + 4, offs.ctypes.data, 0, None, None, None,
                                     None) == -1
    dec.decode([0, 0], [0, 5], [0, 1])
    for a in ((2, 0, 0, 1), (-1, 0, 0, 1), (0, 2, 0, 1), (0, 0, 0, 3), (0, 0, -1, 1), (0, 1, 0, 1)):
        with pytest.raises(ch.CihError):
            dec.read_cache(*a)
    dec.close()
    m.close()


def test_generate_again_over_a_tight_pool():
    """The slots' pages of the call before go back before the first prompt takes any: 4 + 1 pages fit where 1 + 3 are held."""
    cfg, w, m = make(32, "q8", heads=2, layers=1)
    dec = ch.GpuDecoder(m, n_slots=3, max_len=300, max_rows=64, kv8=True, n_pages=6)
    dec.generate([tokens(60, 1), tokens(180, 2)], 0.0, 2, [1, 2])
    again = [tokens(250, 3), tokens(50, 4)]
    got, _, _ = dec.generate(again, 0.0, 4, [1, 2])
    fresh = ch.GpuDecoder(m, n_slots=2, max_len=300, max_rows=64, kv8=True)
    want, _, _ = fresh.generate(again, 0.0, 4, [1, 2])
    assert all(np.array_equal(a, b) for a, b in zip(got, want))
    # one that does not fit leaves no slot with what it held before
    dec.decode([2], [0], [0])
    dec.read_cache(0, 2, 0, 1)
    with pytest.raises(ch.CihError) as e:
        dec.generate([tokens(290, 5), tokens(128, 6), tokens(40, 7)], 0.0, 2, [1, 2, 3])
    assert e.value.code == -3
    with pytest.raises(ch.CihError):
        dec.read_cache(0, 2, 0, 1)
    for d in (dec, fresh):
        d.close()
    m.close()


def test_rope_not_finite():
    cfg, w, m = make(16)
    for field in ("gain", "freq"):
        r = ch.Rope(16)
        if field == "gain":
            r.struct.gain = np.inf
        else:
            r.struct.freq[7] = np.nan
        with pytest.raises(ch.CihError) as e:
            ch.GpuDecoder(m, n_slots=1, max_len=64, max_rows=8, kv8=True, rope=r)
        assert e.value.code == -1
    m.close()

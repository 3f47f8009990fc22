"""The decoder's operators on their own: the 8-bit paged key/value cache
(append with rotary positions, reading back), attention over it, and the log
probabilities of given tokens.

`own` false: plain torch in 32 bits.  `own` true: the calls a program makes of
codon_hip (Kv8Cache.append / .read / .attend, token_logprobs).

A case is a dict: "op" (append, attend, logprobs), "dtype" and its sizes.
"lens" are the tokens that each sequence holds after its new rows, "rows" the
new rows; a sequence's rows are its last ones.  Keys and values are N(0, 1),
queries N(0, 1.5) (softmaxes with a few large weights), logits N(0, 3), all
made on the GPU from the seed.
"""
import math
import os
import sys

import torch

own = False

PAGE = 64  # tokens that share a scale
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def spread(lo, hi, n):
    """n lengths from lo to hi in no order, as a text."""
    return ",".join(str(lo + (hi - lo) * (i * 37 % n) // max(1, n - 1)) for i in range(n))


def listed():
    return [
        # one decode step of eight streams of ESM-2 650M (20 heads of 64): a row each, rotated and appended
        dict(name="append_step_f32", op="append", dtype="f32", heads=20, kv_heads=20, head_dim=64,
             lens=spread(130, 700, 8), rows=spread(1, 1, 8), rot=64, interleaved=False, scaling="none", factor=1.0),
        # prompts of eight proteins on ESM-2 35M, whose 24-wide heads do not fill a tile
        dict(name="append_prompts_f32", op="append", dtype="f32", heads=20, kv_heads=20, head_dim=24,
             lens="512,131,387,254,449,173,318,505", rows="512,131,387,254,449,173,318,505", rot=24,
             interleaved=False, scaling="none", factor=1.0),
        # a chunk of long prompts with shared heads, part of each head rotated, positions scaled eight times
        dict(name="append_long_bf16", op="append", dtype="bf16", heads=32, kv_heads=8, head_dim=128,
             lens=spread(20001, 60000, 16), rows=spread(513, 1024, 16), rot=64, interleaved=True, scaling="yarn",
             factor=8.0),
        # one stream of ESM-2 8M: the smallest step
        dict(name="attend_step_8m_f32", op="attend", dtype="f32", heads=20, kv_heads=20, head_dim=16, lens="131",
             rows="1", window=0, causal=True),
        # eight streams of ESM-2 650M around position 700
        dict(name="attend_step_650m_f32", op="attend", dtype="f32", heads=20, kv_heads=20, head_dim=64,
             lens=spread(450, 701, 8), rows=spread(1, 1, 8), window=0, causal=True),
        # a full serving batch with shared heads and long contexts: the cache's bytes
        dict(name="attend_batch_bf16", op="attend", dtype="bf16", heads=32, kv_heads=8, head_dim=128,
             lens=spread(1025, 8190, 64), rows=spread(1, 1, 64), window=0, causal=True),
        # one very long sequence: the keys have to be split over the GPU
        dict(name="attend_one_long_f16", op="attend", dtype="f16", heads=40, kv_heads=40, head_dim=64, lens="65003",
             rows="1", window=0, causal=True),
        # the prompts of a small ragged batch on ESM-2 650M
        dict(name="attend_prompts_650m_f32", op="attend", dtype="f32", heads=20, kv_heads=20, head_dim=64,
             lens="512,131,387,254,449,173,318,505", rows="512,131,387,254,449,173,318,505", window=0, causal=True),
        # a chunk of a long prompt behind a cached context, shared heads
        dict(name="attend_chunk_bf16", op="attend", dtype="bf16", heads=32, kv_heads=8, head_dim=128, lens="16000",
             rows="2047", window=0, causal=True),
        # scores of one decode step of eight streams over ESM-2's 33 tokens
        dict(name="logprobs_step_f32", op="logprobs", dtype="f32", rows=8, vocab=33, top=5),
        # scores of a batch of proteins over the 33 tokens
        dict(name="logprobs_batch_f32", op="logprobs", dtype="f32", rows=8192, vocab=33, top=5),
        # a large vocabulary in 16 bits
        dict(name="logprobs_wide_bf16", op="logprobs", dtype="bf16", rows=512, vocab=131072, top=20),
    ]


def draw(rng):
    """One more case: steps, prompts and chunks over all head sizes, types and ragged lengths; narrow and wide vocabularies."""
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    dtype = rng.choice(["f32", "f16", "bf16"])
    op = rng.choice(["append", "attend", "attend", "logprobs"])
    if op == "logprobs":
        vocab = rng.choice([33, log_int(2, 1000), log_int(1000, 140000)])
        rows = log_int(1, max(2, min(8192, 60_000_000 // vocab)))
        return dict(op=op, dtype=dtype, rows=rows, vocab=vocab, top=min(vocab, rng.randint(1, 32)))
    head_dim = rng.choice([16, 24, 32, 64, 64, 128])
    kv_heads = rng.choice([1, 2, 5, 8, 20])
    heads = kv_heads * rng.choice([x for x in (1, 1, 2, 3, 4, 8) if x * kv_heads <= 40])
    kind = rng.choice(["step", "step", "prompt", "chunk", "few"])
    if kind == "prompt":  # whole prompts
        n, top = log_int(1, 16), log_int(1, 1024)
        rows = lens = [rng.randint(1, top) for _ in range(n)]
    elif kind == "chunk":  # more rows behind a cached context
        n = log_int(1, 4)
        rows = [log_int(2, 1024) for _ in range(n)]
        lens = [r + log_int(1, 6000) for r in rows]
    else:  # one row a sequence, or a few (drafted tokens to be checked)
        n = log_int(1, 64)
        top = log_int(64, min(20000, 250_000_000 // (n * kv_heads * padded(head_dim))))
        rows = [rng.randint(1, 1 if kind == "step" else 6) for _ in range(n)]
        lens = [r + rng.randint(0, top) for r in rows]
        if op == "attend" and n > 2:  # a stream that is not running
            lens[1] = rows[1] = 0
    case = dict(op=op, dtype=dtype, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                lens=",".join(map(str, lens)), rows=",".join(map(str, rows)))
    if op == "append":
        scaling = rng.choice(["none", "linear", "ntk", "yarn"])
        return dict(case, rot=rng.choice([head_dim, head_dim // 2 if head_dim > 16 else 8]),
                    interleaved=rng.random() < 0.5, scaling=scaling,
                    factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0]))
    return dict(case, window=rng.choice([0, 0, log_int(16, 4096)]), causal=rng.random() < 0.9)


def ints(text):
    return [int(x) for x in text.split(",")]


def padded(head_dim):
    return 16 if head_dim <= 16 else 32 if head_dim <= 32 else 64 if head_dim <= 64 else 128


def visible(case):
    """(sum over the sequences of (row, key) pairs a head sees, of keys that any row sees)."""
    pairs = keys = 0
    w = case["window"]
    for n, r in zip(ints(case["lens"]), ints(case["rows"])):
        last = [p + 1 if case["causal"] else n for p in range(n - r, n)]
        first = [max(0, p + 1 - w) if w else 0 for p in range(n - r, n)]
        pairs += sum(b - a for a, b in zip(first, last))
        keys += (max(last) - min(first)) if r else 0
    return pairs, keys


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "logprobs":
        n, v, k = case["rows"], case["vocab"], case["top"]
        return {"bytes": float(n * (v * size + 4 + 8 + 8 * k)), "flops": 5.0 * n * v}
    d, hk, h = case["head_dim"], case["kv_heads"], case["heads"]
    rows = sum(ints(case["rows"]))
    if case["op"] == "append":
        # kept codes are counted read and written once
        kept = sum((n - r) % PAGE for n, r in zip(ints(case["lens"]), ints(case["rows"])))
        moved = size * rows * d * (2 * hk + 2 * h) + 2 * rows * d * hk + 4 * kept * d * hk  # rows in, codes out
        back = 2 * (rows + kept) * d * hk * (1 + 2)  # codes in, values out
        return {"bytes": float(moved + back), "flops": 6.0 * rows * d * (h + 2 * hk)}
    pairs, keys = visible(case)
    return {"bytes": float(2 * keys * d * hk + 2 * size * rows * d * h + 4 * rows * h),
            "flops": 4.0 * pairs * d * h}


def frequencies(case):
    """Rotary angle per position of each pair, and the factor on cosine and sine (numbers of 64 bits)."""
    rot, s, base, trained = case["rot"], case["factor"], 10000.0, 1024
    if case["scaling"] == "ntk":
        base *= s ** (rot / (rot - 2))
    f = [base ** (-2.0 * j / rot) for j in range(rot // 2)]
    if case["scaling"] == "linear":
        f = [x / s for x in f]
    if case["scaling"] == "yarn":
        share = [min(1.0, max(0.0, (trained * x / (2 * math.pi) - 1) / 31)) for x in f]
        f = [x * ((1 - g) / s + g) for x, g in zip(f, share)]
        return f, 0.1 * math.log(s) + 1
    return f, 1.0


def cache(case, g, lens):
    """A filled cache: pages in no order, codes [pages][kv heads][64][dims] of K and [dims][64] of V, scales, and
    the sequences' tables."""
    dev, d, hk = "cuda", case["head_dim"], case["kv_heads"]
    need = [-(-n // PAGE) for n in lens]
    total = sum(need) + 3
    order = torch.randperm(total, device=dev, generator=g).int()
    table = torch.zeros(len(lens), max(1, max(need)), dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    k = torch.zeros(total, hk, PAGE, padded(d), dtype=torch.int8, device=dev)
    v = torch.zeros(total, hk, padded(d), PAGE, dtype=torch.int8, device=dev)
    x = torch.randn(total, hk, PAGE, d, device=dev, generator=g)
    sk = x.abs().amax((2, 3)) / 127
    k[..., :d] = torch.round(x / sk[..., None, None]).to(torch.int8)
    x = torch.randn(total, hk, d, PAGE, device=dev, generator=g)
    sv = x.abs().amax((2, 3)) / 127
    v[:, :, :d] = torch.round(x / sv[..., None, None]).to(torch.int8)
    return dict(codes_k=k, codes_v=v, scales=torch.stack((sk, sv), -1).contiguous(),
                bad=torch.zeros(total, hk, dtype=torch.int64, device=dev), table=table)


def offsets(rows):
    cu = [0]
    for r in rows:
        cu.append(cu[-1] + r)
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


def framework():
    path = os.path.join(os.getcwd(), "codon-infer_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import codon_hip
    return codon_hip


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, dev = DTYPES[case["dtype"]], "cuda"
    if case["op"] == "logprobs":
        n, v, k = case["rows"], case["vocab"], case["top"]
        st = dict(case, logits=(3 * torch.randn(n, v, device=dev, generator=g)).to(t),
                  targets=torch.randint(v, (n,), device=dev, generator=g, dtype=torch.int32),
                  logprob=torch.empty(n, device=dev), entropy=torch.empty(n, device=dev),
                  top_ids=torch.empty(n, k, device=dev, dtype=torch.int32),
                  top_logprobs=torch.empty(n, k, device=dev))
        if own:
            ch = framework()
            st["workspace"] = torch.empty(ch.token_logprobs_workspace(n, v, k), dtype=torch.uint8, device=dev)
            st["call"] = ch.token_logprobs
        return st
    lens, rows = ints(case["lens"]), ints(case["rows"])
    h, hk, d, n = case["heads"], case["kv_heads"], case["head_dim"], sum(rows)
    st = dict(case, **cache(case, g, lens), cu=offsets(rows),
              held=torch.tensor(lens, dtype=torch.int32, device=dev), most=max(rows), total=n,
              q=(1.5 * torch.randn(n, h, d, device=dev, generator=g)).to(t),
              out=torch.empty(n, h, d, device=dev, dtype=t))
    if case["op"] == "attend":
        st["lse"] = torch.empty(n, h, device=dev)
        if own:
            ch = framework()
            st["cache"] = ch.Kv8Cache(st["codes_k"], st["codes_v"], st["scales"], st["bad"], d)
            st["batch"] = ch.Kv8Batch(st["cu"], st["held"], st["table"], n, max(rows))
            st["workspace"] = torch.empty(st["cache"].attend_workspace(st["batch"], h), dtype=torch.uint8, device=dev)
        return st
    back = [r + (m - r) % PAGE for m, r in zip(lens, rows)]  # read back: the new rows and their first page's others
    rd = torch.bfloat16 if case["dtype"] == "bf16" else torch.float16
    f, m = frequencies(case)
    st.update(k=torch.randn(n, hk, d, device=dev, generator=g).to(t), v=torch.randn(n, hk, d, device=dev, generator=g).to(t),
              back=offsets(back), k_back=torch.empty(sum(back), hk, d, device=dev, dtype=rd),
              v_back=torch.empty(sum(back), hk, d, device=dev, dtype=rd), most_back=max(back),
              freq=torch.tensor(f, dtype=torch.float64, device=dev), gain=m)
    if own:
        ch = framework()
        st["cache"] = ch.Kv8Cache(st["codes_k"], st["codes_v"], st["scales"], st["bad"], d)
        st["batch"] = ch.Kv8Batch(st["cu"], st["held"], st["table"], n, max(rows))
        st["batch_back"] = ch.Kv8Batch(st["back"], st["held"], st["table"], sum(back), max(back))
        st["rope"] = ch.Rope(case["rot"], base=10000.0, interleaved=case["interleaved"], scaling=case["scaling"],
                             factor=case["factor"], trained_len=1024)
    return st


def run(st):
    if st["op"] == "logprobs":
        if own:
            st["call"](st["logits"], st["targets"], st["logprob"], st["entropy"], st["top_ids"], st["top_logprobs"],
                       workspace=st["workspace"])
            return [st[x] for x in ("logprob", "entropy", "top_ids", "top_logprobs")]
        return plain_logprobs(st)
    if st["op"] == "attend":
        if own:
            st["cache"].attend(st["batch"], st["q"], st["out"], lse=st["lse"], causal=st["causal"],
                               window=st["window"], workspace=st["workspace"])
            return [st["out"], st["lse"]]
        return plain_attend(st)
    if own:
        st["cache"].append(st["batch"], st["k"], st["v"], q=st["q"], q_out=st["out"], rope=st["rope"])
        st["cache"].read(st["batch_back"], st["k_back"], st["v_back"])
    else:
        st["out"] = plain_append(st)
        st["k_back"], st["v_back"] = plain_read(st, st["k_back"].dtype)
    return [st["out"], st["k_back"], st["v_back"], st["scales"], st["bad"]]


def plain_logprobs(st):
    x, t = st["logits"].float(), st["targets"].long()[:, None]
    lse = torch.log(torch.exp(x - x.amax(1, keepdim=True)).sum(1, keepdim=True)) + x.amax(1, keepdim=True)
    lp = x - lse
    entropy = -(torch.exp(lp) * lp).sum(1)
    ids = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :st["top"]]
    return [lp.gather(1, t)[:, 0], entropy, ids.int(), lp.gather(1, ids)]


def place(cu, held, most):
    """Of each sequence's rows, padded to the longest: row, position, whether there is one."""
    rows = (cu[1:] - cu[:-1])[:, None]
    i = torch.arange(most, device=cu.device)[None]
    return (cu[:-1, None] + i).long(), (held[:, None] - rows + i).long(), i < rows


def plain_attend(st):
    h, hk, d = st["heads"], st["kv_heads"], st["head_dim"]
    table = st["table"].long()
    n, pages = table.shape
    row, pos, there = place(st["cu"], st["held"], st["most"])
    scale = st["scales"][table]
    k = st["codes_k"][table][..., :d].float() * scale[..., 0, None, None]
    k = k.permute(0, 2, 1, 3, 4).reshape(n, hk, pages * PAGE, d)
    v = st["codes_v"][table][..., :d, :].float() * scale[..., 1, None, None]
    v = v.permute(0, 2, 1, 4, 3).reshape(n, hk, pages * PAGE, d)
    q = st["q"][row.clamp(max=st["total"] - 1)].float().view(n, st["most"], hk, h // hk, d).permute(0, 2, 3, 1, 4)
    s = torch.matmul(q.reshape(n, hk, -1, d), k.transpose(2, 3).contiguous()).mul_(1 / math.sqrt(d))
    s = s.view(n, hk, h // hk, st["most"], pages * PAGE)
    j = torch.arange(pages * PAGE, device=s.device)
    see = (j < st["held"][:, None])[:, None].expand(n, st["most"], -1)
    if st["causal"]:
        see = see & (j <= pos[..., None])
    if st["window"]:
        see = see & (j > pos[..., None] - st["window"])
    s.masked_fill_(~see[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s.sub_(torch.where(top == -math.inf, 0.0, top)))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(n, hk, -1, pages * PAGE), v).view(n, hk, h // hk, st["most"], d)
    out = torch.where(total > 0, out / total, 0.0)
    lse = (top + torch.log(total))[..., 0]
    out, lse = out.permute(0, 3, 1, 2, 4).reshape(n, st["most"], h, d), lse.permute(0, 3, 1, 2).reshape(n, st["most"], h)
    return [out[there].to(st["q"].dtype), lse[there]]


def rotate(st, x, pos):
    """x [rows][heads][dims] in 32 bits, turned by its positions' angles."""
    half = st["rot"] // 2
    a = pos.double()[:, None, None] * st["freq"]
    c, s = (torch.cos(a) * st["gain"]).float(), (torch.sin(a) * st["gain"]).float()
    y = x.clone()
    if st["interleaved"]:
        x0, x1 = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2], y[..., 1:2 * half:2] = x0 * c - x1 * s, x1 * c + x0 * s
    else:
        x0, x1 = x[..., :half], x[..., half:2 * half]
        y[..., :half], y[..., half:2 * half] = x0 * c - x1 * s, x1 * c + x0 * s
    return y


def plain_append(st):
    d = st["head_dim"]
    row, pos, there = place(st["cu"], st["held"], st["most"])
    row, at = row[there], pos[there]
    seq = torch.arange(there.shape[0], device=row.device)[:, None].expand_as(there)[there]
    page = st["table"][seq, at // PAGE].long()
    k, v = rotate(st, st["k"].float()[row], at), st["v"].float()[row]
    fine = torch.isfinite(k).all(-1) & torch.isfinite(v).all(-1)
    k, v = torch.where(fine[..., None], k, 0.0), torch.where(fine[..., None], v, 0.0)
    # the largest value of each (page, head): scales of pages that keep tokens do not shrink
    start = (st["held"] - (st["cu"][1:] - st["cu"][:-1])).long()
    first = start[seq] // PAGE == at // PAGE
    kept = torch.where(first, start[seq] % PAGE, 0)
    new = torch.stack((k.abs().amax(-1), v.abs().amax(-1)), -1) / 127
    old = st["scales"].clone()
    scales, touched = torch.zeros_like(old), torch.zeros(old.shape[0], dtype=torch.int64, device=row.device)
    touched[page] = 1
    keeps = torch.zeros_like(touched).scatter_reduce(0, page, kept, "amax")
    scales = scales.scatter_reduce(0, page[:, None, None].expand_as(new), new, "amax")
    scales = torch.where((keeps > 0)[:, None, None], torch.maximum(scales, old), scales)
    scales = torch.where((touched > 0)[:, None, None], scales, old)
    ratio = torch.where(scales > 0, old / scales, 0.0)
    again = (touched > 0) & (keeps > 0)
    pages = torch.nonzero(again)[:, 0]
    st["codes_k"][pages] = torch.round(st["codes_k"][pages].float() * ratio[pages, :, 0, None, None]).clamp(-127, 127).to(torch.int8)
    st["codes_v"][pages] = torch.round(st["codes_v"][pages].float() * ratio[pages, :, 1, None, None]).clamp(-127, 127).to(torch.int8)
    inv = torch.where(scales > 0, 1 / scales, 0.0)[page]
    st["codes_k"][page, :, at % PAGE, :d] = torch.round(k * inv[..., 0, None]).clamp(-127, 127).to(torch.int8)
    st["codes_v"][page, :, :d, at % PAGE] = torch.round(v * inv[..., 1, None]).clamp(-127, 127).to(torch.int8)
    st["scales"].copy_(scales)
    bit = torch.ones_like(at) << (at % PAGE)
    below = torch.where(keeps > 0, (torch.ones_like(keeps) << keeps) - 1, 0)
    bad = torch.where((touched > 0)[:, None], st["bad"] & below[:, None], st["bad"])
    st["bad"].copy_(bad.index_add(0, page, torch.where(fine, 0, bit[:, None])))
    return rotate(st, st["q"].float()[row], at).to(st["q"].dtype)


def plain_read(st, dtype):
    row, pos, there = place(st["back"], st["held"], st["most_back"])
    at = pos[there]
    seq = torch.arange(there.shape[0], device=row.device)[:, None].expand_as(there)[there]
    page = st["table"][seq, at // PAGE].long()
    d, lost = st["head_dim"], (st["bad"][page] >> (at % PAGE)[:, None] & 1)[..., None] > 0
    k = st["codes_k"][page, :, at % PAGE, :d].float() * st["scales"][page][..., 0, None]
    v = st["codes_v"][page, :, :d, at % PAGE].float() * st["scales"][page][..., 1, None]
    return torch.where(lost, math.nan, k).to(dtype), torch.where(lost, math.nan, v).to(dtype)


def exact(case, seed):
    """The outputs from the definitions in 64 bits, sequence by sequence."""
    st = prepare(case, seed)
    if case["op"] == "logprobs":
        x = st["logits"].double()
        p = torch.softmax(x, 1)
        lse = torch.logsumexp(x, 1)
        picked = x[torch.arange(len(x), device=x.device), st["targets"].long()] - lse
        highest = torch.topk(x, st["top"], dim=1).values - lse[:, None]
        return [picked, -(torch.xlogy(p, p)).sum(1), None, highest]
    lens, rows = ints(case["lens"]), ints(case["rows"])
    g, d = case["heads"] // case["kv_heads"], case["head_dim"]
    outs, first = [], 0
    for i, (n, r) in enumerate(zip(lens, rows)):
        if r == 0:
            continue
        q = st["q"][first:first + r].double()
        page = st["table"][i, :-(-n // PAGE)].long()
        pos = torch.arange(n - r, n, device=q.device)
        outs.append((exact_attend if case["op"] == "attend" else exact_append)(st, case, q, page, pos, first, n, r, g, d))
        first += r
    if case["op"] == "attend":
        return [torch.cat([o[0] for o in outs]), torch.cat([o[1] for o in outs])]
    return [torch.cat([o[0] for o in outs]), torch.cat([o[1] for o in outs]), torch.cat([o[2] for o in outs]),
            st["exact_scales"], None]


def exact_attend(st, case, q, page, pos, first, n, r, g, d):
    out = torch.empty_like(q)
    lse = torch.empty(q.shape[:2], dtype=torch.float64, device=q.device)
    j = torch.arange(n, device=q.device)
    hidden = torch.zeros(r, n, dtype=torch.bool, device=q.device)
    if case["causal"]:
        hidden |= j[None] > pos[:, None]
    if case["window"]:
        hidden |= j[None] <= pos[:, None] - case["window"]
    for kv in range(case["kv_heads"]):
        k = (st["codes_k"][page, kv, :, :d].double() * st["scales"][page, kv, 0].double()[:, None, None]).reshape(-1, d)[:n]
        v = st["codes_v"][page, kv, :d].double() * st["scales"][page, kv, 1].double()[:, None, None]
        v = v.transpose(1, 2).reshape(-1, d)[:n]
        for h in range(kv * g, kv * g + g):
            s = (q[:, h] @ k.T) / math.sqrt(d)
            s[hidden] = -math.inf
            lse[:, h] = torch.logsumexp(s, 1)
            out[:, h] = torch.softmax(s, 1) @ v
    return out, lse


def exact_append(st, case, q, page, pos, first, n, r, g, d):
    f, gain = frequencies(case)
    pairs = case["rot"] // 2
    ang = pos.double()[:, None] * torch.tensor(f, dtype=torch.float64, device=q.device)
    turn = torch.polar(torch.full_like(ang, gain), ang)[:, None]

    def turned(x):
        if case["interleaved"]:
            z = torch.view_as_complex(x[..., :2 * pairs].reshape(*x.shape[:-1], pairs, 2).contiguous()) * turn
            return torch.cat((torch.view_as_real(z).flatten(-2), x[..., 2 * pairs:]), -1)
        z = torch.complex(x[..., :pairs].contiguous(), x[..., pairs:2 * pairs].contiguous()) * turn
        return torch.cat((z.real, z.imag, x[..., 2 * pairs:]), -1)

    if "exact_scales" not in st:
        st["exact_scales"] = st["scales"].double()
    k, v = turned(st["k"][first:first + r].double()), st["v"][first:first + r].double()
    start, backs = n - r, []
    for which, x, codes in ((0, k, st["codes_k"]), (1, v, st["codes_v"].transpose(2, 3))):
        got = []
        for b in range(start // PAGE, len(page)):
            a0, a1 = max(start, b * PAGE), min(n, (b + 1) * PAGE)
            new = x[a0 - start:a1 - start]
            top = new.abs().amax((0, 2)) / 127
            if a0 > b * PAGE:
                was = st["scales"][page[b], :, which].double()
                s = torch.maximum(was, top)
                held = torch.round(codes[page[b], :, :a0 - b * PAGE, :d].double() * (was / s)[:, None, None])
                got.append(held.transpose(0, 1) * s[:, None])
            else:
                s = top
            st["exact_scales"][page[b], :, which] = s
            got.append(torch.round(new / s[:, None]) * s[:, None])
        backs.append(torch.cat(got))
    return turned(q), backs[0], backs[1]

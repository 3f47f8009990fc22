"""The operators of long and of drafted decoding on their own: attention over the
8-bit cache with a sliding window and first tokens that stay visible (sinks), the
attention weight that cached tokens gather, eviction by it, and the verification
of drafted tokens.

`own` false: plain torch.  `own` true: the calls a program makes of codon_hip
(Kv8Cache.attend / .weigh / .evict / .read, verify_drafts).

A case is a dict: "op" (attend, weigh, evict, verify), "dtype" and its sizes.
"lens" are the tokens that each sequence holds, "rows" the new rows among them (its
last ones).  Keys and values are N(0, 1), queries N(0, 1.5) (softmaxes with a few
large weights), gathered weights log-normal, logits N(0, 3) with a draft's N(0, 1)
off them, all made on the GPU from the seed.
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
        # one stream of ESM-2 650M (20 heads of 64) past its window: the smallest step
        dict(name="sinks_step_f32", op="attend", dtype="f32", heads=20, kv_heads=20, head_dim=64, lens="701", rows="1",
             window=256, sinks=4),
        # a full serving batch with shared heads, long past its window
        dict(name="sinks_batch_bf16", op="attend", dtype="bf16", heads=32, kv_heads=8, head_dim=128,
             lens=spread(4097, 16384, 64), rows=spread(1, 1, 64), window=4096, sinks=4),
        # a chunk of a long prompt: a few first tokens and the window before each row
        dict(name="sinks_chunk_f16", op="attend", dtype="f16", heads=32, kv_heads=8, head_dim=128, lens="16000",
             rows="2047", window=4096, sinks=4),
        # what eight streams' steps on ESM-2 650M add to the cached tokens' weights
        dict(name="weigh_step_f32", op="weigh", dtype="f32", heads=20, kv_heads=20, head_dim=64,
             lens=spread(450, 701, 8), rows=spread(1, 1, 8), window=0, sinks=0, keep=1.0),
        # a full serving batch with shared heads: the keys' bytes
        dict(name="weigh_batch_bf16", op="weigh", dtype="bf16", heads=32, kv_heads=8, head_dim=128,
             lens=spread(1025, 8190, 64), rows=spread(1, 1, 64), window=0, sinks=0, keep=0.98),
        # a chunk of a long prompt, weighed before the cache is cut to its budget
        dict(name="weigh_chunk_bf16", op="weigh", dtype="bf16", heads=32, kv_heads=8, head_dim=128, lens="16000",
             rows="2047", window=0, sinks=0, keep=1.0),
        # eight streams of ESM-2 650M, a page over their budget
        dict(name="evict_step_f16", op="evict", dtype="f16", kv_heads=20, head_dim=64, lens=spread(577, 577, 8),
             budget=512, first=4, recent=64),
        # ragged prompts cut to one budget after their prefill; some are within it
        dict(name="evict_batch_bf16", op="evict", dtype="bf16", kv_heads=8, head_dim=128, lens=spread(1900, 6000, 32),
             budget=2048, first=4, recent=256),
        # one very long sequence cut to a sixteenth
        dict(name="evict_one_long_f16", op="evict", dtype="f16", kv_heads=40, head_dim=64, lens="65003", budget=4001,
             first=16, recent=512),
        # four drafted residues of each of eight streams, over ESM-2's 33 tokens
        dict(name="verify_step_f32", op="verify", dtype="f32", vocab=33, drafts="4,4,4,4,4,4,4,4", draft_logits=True,
             temperature=1.0),
        # a full serving batch over a large vocabulary in 16 bits
        dict(name="verify_batch_bf16", op="verify", dtype="bf16", vocab=131072, drafts=spread(3, 7, 64),
             draft_logits=True, temperature=0.8),
        # one stream whose drafts were looked up in its own text, without a distribution
        dict(name="verify_lookup_f16", op="verify", dtype="f16", vocab=32003, drafts="7", draft_logits=False,
             temperature=0.7),
    ]


def draw(rng):
    """One more case: steps, drafts, prompts and chunks over all head sizes, types and ragged lengths; budgets of a page to most of a sequence; narrow and wide vocabularies."""
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    dtype = rng.choice(["f32", "f16", "bf16"])
    op = rng.choice(["attend", "weigh", "evict", "verify"])
    if op == "verify":
        vocab = rng.choice([33, log_int(2, 1000), log_int(1000, 140000), log_int(1000, 140000)])
        n = log_int(1, max(2, min(512, 8_000_000 // vocab)))
        return dict(op=op, dtype=dtype, vocab=vocab, drafts=",".join(str(rng.randint(0, 7)) for _ in range(n)),
                    draft_logits=rng.random() < 0.7, temperature=rng.choice([0.0, 0.5, 1.0, 1.3]))
    head_dim = rng.choice([16, 24, 32, 64, 64, 128])
    kv_heads = rng.choice([1, 2, 5, 8, 20])
    if op == "evict":
        n = log_int(1, 64)
        budget = log_int(64, min(8192, 60_000_000 // (n * kv_heads * padded(head_dim))))
        top = log_int(budget + 1, min(40000, 8 * budget))
        first, recent = rng.choice([0, 4, 16]), rng.choice([0, budget // 8, budget // 2])
        return dict(op=op, dtype=dtype, kv_heads=kv_heads, head_dim=head_dim, budget=budget, first=first, recent=recent,
                    lens=",".join(str(rng.randint(budget // 2, top)) for _ in range(n)))
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
        if n > 2:  # a stream that is not running
            lens[1] = rows[1] = 0
    case = dict(op=op, dtype=dtype, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                lens=",".join(map(str, lens)), rows=",".join(map(str, rows)))
    if op == "attend":
        return dict(case, window=log_int(16, 4096), sinks=rng.choice([1, 4, 4, 64, 100, 500]))
    window = rng.choice([0, 0, 0, log_int(16, 4096)])
    return dict(case, window=window, sinks=rng.choice([0, 4]) if window else 0, keep=rng.choice([0.0, 0.9, 1.0]))


def ints(text):
    return [int(x) for x in text.split(",")]


def padded(head_dim):
    return 16 if head_dim <= 16 else 32 if head_dim <= 32 else 64 if head_dim <= 64 else 128


def visible(case):
    """(sum over the sequences of (row, key) pairs a head sees, of keys that any row sees)."""
    pairs = keys = 0
    w, s = case["window"], case["sinks"]
    for n, r in zip(ints(case["lens"]), ints(case["rows"])):
        last = range(n - r + 1, n + 1)  # of each row, the first key that it does not see
        first = [max(0, p - w) if w else 0 for p in last]
        pairs += sum(b - a + min(a, s) for a, b in zip(first, last))
        keys += (n - first[0] + min(first[0], s)) if r else 0
    return pairs, keys


def work(case):
    size = SIZE[case["dtype"]]
    if case["op"] == "verify":
        drafts = ints(case["drafts"])
        n, d, v = len(drafts), sum(drafts), case["vocab"]
        logits = (n + d + (d if case["draft_logits"] else 0)) * v
        return {"bytes": float(logits * size + 8 * d + 12 * n), "flops": 5.0 * logits}
    d, hk = case["head_dim"], case["kv_heads"]
    if case["op"] == "evict":
        lens = ints(case["lens"])
        kept = sum(min(x, case["budget"]) for x in lens)
        moved = sum(case["budget"] for x in lens if x > case["budget"])
        # weights in and out, ids, codes in and out, and the kept codes read back as values
        return {"bytes": float(hk * (4 * sum(lens) + 8 * kept + 4 * d * moved + 2 * d * kept * 3)),
                "flops": float(hk * (2 * sum(lens) + 4 * d * kept))}
    h, rows = case["heads"], sum(ints(case["rows"]))
    pairs, keys = visible(case)
    if case["op"] == "weigh":
        return {"bytes": float(keys * hk * (d + 8) + size * rows * d * h + 4 * rows * h), "flops": 2.0 * pairs * d * h}
    return {"bytes": float(2 * keys * d * hk + 2 * size * rows * d * h + 4 * rows * h), "flops": 4.0 * pairs * d * h}


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
    if case["op"] == "verify":
        return prepare_verify(case, g, t, dev)
    lens = ints(case["lens"])
    hk, d = case["kv_heads"], case["head_dim"]
    st = dict(case, **cache(case, g, lens), held=torch.tensor(lens, dtype=torch.int32, device=dev))
    pages = st["table"].shape[1]
    weights = torch.exp(2 * torch.randn(st["scales"].shape[0], hk, PAGE, device=dev, generator=g))
    if case["op"] == "evict":
        n, keep = len(lens), [min(x, case["budget"]) for x in lens]
        total = sum(keep)
        st.update(weights=weights, weights_out=torch.zeros_like(weights), lens_out=torch.empty_like(st["held"]),
                  kept=torch.empty(n, hk, case["budget"], dtype=torch.int32, device=dev), cu=offsets([1] * n),
                  cu_back=offsets(keep), most_back=max(keep),
                  k_back=torch.empty(total, hk, d, device=dev, dtype=t), v_back=torch.empty(total, hk, d, device=dev, dtype=t))
        if own:
            ch = framework()
            st["cache"] = ch.Kv8Cache(st["codes_k"], st["codes_v"], st["scales"], st["bad"], d)
            st["batch"] = ch.Kv8Batch(st["cu"], st["held"], st["table"], n, 1)
            st["batch_back"] = ch.Kv8Batch(st["cu_back"], st["lens_out"], st["table"], total, max(keep))
            st["workspace"] = torch.empty(st["cache"].evict_workspace(st["batch"], case["budget"]), dtype=torch.uint8,
                                          device=dev)
        return st
    rows, h = ints(case["rows"]), case["heads"]
    n = sum(rows)
    st.update(cu=offsets(rows), most=max(rows), total=n, causal=True,
              q=(1.5 * torch.randn(n, h, d, device=dev, generator=g)).to(t))
    if own:
        ch = framework()
        st["cache"] = ch.Kv8Cache(st["codes_k"], st["codes_v"], st["scales"], st["bad"], d)
        st["batch"] = ch.Kv8Batch(st["cu"], st["held"], st["table"], n, max(rows))
    if case["op"] == "weigh":  # lse: as the attention before it gives it
        st.update(weights=weights, lse=plain_lse(st))
    else:
        st.update(out=torch.empty(n, h, d, device=dev, dtype=t), lse=torch.empty(n, h, device=dev))
        if own:
            st["workspace"] = torch.empty(st["cache"].attend_workspace(st["batch"], h), dtype=torch.uint8, device=dev)
    return st


def prepare_verify(case, g, t, dev):
    drafts = ints(case["drafts"])
    n, d, v, heat = len(drafts), sum(drafts), case["vocab"], case["temperature"]
    cu = offsets(drafts)
    row = torch.arange(d, device=dev) + torch.repeat_interleave(
        torch.arange(n, device=dev), torch.tensor(drafts, device=dev))  # the target's row of each draft
    logits = 3 * torch.randn(n + d, v, device=dev, generator=g)
    about = (logits[row] + torch.randn(d, v, device=dev, generator=g)).to(t)
    race = -torch.log(-torch.log(torch.rand(d, v, device=dev, generator=g).clamp(1e-20, 1 - 1e-7)))
    drafted = (about.float() + heat * race).argmax(1).int() if d else torch.zeros(0, dtype=torch.int32, device=dev)
    st = dict(case, logits=logits.to(t), cu=cu, row=row, drafted=drafted, most=max(drafts),
              about=about if case["draft_logits"] else None, u=torch.rand(d, device=dev, generator=g),
              v=torch.rand(n, device=dev, generator=g), accepted=torch.empty(n, dtype=torch.int32, device=dev),
              token=torch.empty(n, dtype=torch.int32, device=dev))
    if own:
        ch = framework()
        st["workspace"] = torch.empty(ch.verify_drafts_workspace(n, d, v), dtype=torch.uint8, device=dev)
        st["call"] = ch.verify_drafts
    return st


def run(st):
    if own:
        if st["op"] == "verify":
            st["call"](st["logits"], st["drafted"], st["cu"], st["accepted"], st["token"], draft_logits=st["about"],
                       accept_at=st["u"], sample_at=st["v"], temperature=st["temperature"], workspace=st["workspace"])
            return [st["accepted"], st["token"]]
        if st["op"] == "weigh":
            st["cache"].weigh(st["batch"], st["q"], st["lse"], st["weights"], window=st["window"], sinks=st["sinks"],
                              keep=st["keep"])
            return [st["weights"]]
        if st["op"] == "attend":
            st["cache"].attend(st["batch"], st["q"], st["out"], lse=st["lse"], window=st["window"], sinks=st["sinks"],
                               workspace=st["workspace"])
            return [st["out"], st["lse"]]
        st["cache"].evict(st["batch"], st["weights"], st["budget"], first=st["first"], recent=st["recent"],
                          weights_out=st["weights_out"], lens_out=st["lens_out"], kept=st["kept"],
                          workspace=st["workspace"])
        st["cache"].read(st["batch_back"], st["k_back"], st["v_back"])
        return [st[x] for x in ("kept", "lens_out", "weights_out", "scales", "bad", "k_back", "v_back")]
    return {"verify": plain_verify, "weigh": plain_weigh, "attend": plain_attend, "evict": plain_evict}[st["op"]](st)


def place(cu, held, most):
    """Of each sequence's rows, padded to the longest: row, position, whether there is one."""
    rows = (cu[1:] - cu[:-1])[:, None]
    i = torch.arange(most, device=cu.device)[None]
    return (cu[:-1, None] + i).long(), (held[:, None] - rows + i).long(), i < rows


def plain_scores(st):
    """Scores [sequences][kv heads][group][rows][keys], -inf where a row does not see a key; rows as place() has them."""
    h, hk, d = st["heads"], st["kv_heads"], st["head_dim"]
    table = st["table"].long()
    n, pages = table.shape
    row, pos, there = place(st["cu"], st["held"], st["most"])
    k = st["codes_k"][table][..., :d].float() * st["scales"][table][..., 0, None, None]
    k = k.permute(0, 2, 1, 3, 4).reshape(n, hk, pages * PAGE, d)
    q = st["q"][row.clamp(max=st["total"] - 1)].float().view(n, st["most"], hk, h // hk, d).permute(0, 2, 3, 1, 4)
    s = torch.matmul(q.reshape(n, hk, -1, d), k.transpose(2, 3).contiguous()).mul_(1 / math.sqrt(d))
    s = s.view(n, hk, h // hk, st["most"], pages * PAGE)
    j = torch.arange(pages * PAGE, device=s.device)
    see = (j < st["held"][:, None])[:, None] & (j <= pos[..., None]) & there[..., None]
    if st["window"]:
        see = see & ((j > pos[..., None] - st["window"]) | (j < st["sinks"]))
    return s.masked_fill_(~see[:, None, None], -math.inf), row, there


def by_rows(x, there):
    """[sequences][kv heads][group][rows] and what follows, as [rows][heads] and what follows."""
    order = [0, 3, 1, 2] + list(range(4, x.dim()))
    return x.permute(order).flatten(2, 3)[there]


def plain_softmax(st):
    s, row, there = plain_scores(st)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s.sub_(torch.where(top == -math.inf, 0.0, top)))
    total = p.sum(-1, keepdim=True)
    return p, total, by_rows((top + torch.log(total))[..., 0], there), there


def plain_lse(st):
    return plain_softmax(st)[2].contiguous()


def plain_attend(st):
    hk, d = st["kv_heads"], st["head_dim"]
    table = st["table"].long()
    n, pages = table.shape
    p, total, lse, there = plain_softmax(st)
    v = st["codes_v"][table][..., :d, :].float() * st["scales"][table][..., 1, None, None]
    v = v.permute(0, 2, 1, 4, 3).reshape(n, hk, pages * PAGE, d)
    out = torch.matmul(p.view(n, hk, -1, pages * PAGE), v).view(*p.shape[:4], d)
    out = torch.where(total > 0, out / total, 0.0)
    return [by_rows(out, there).to(st["q"].dtype), lse]


def plain_weigh(st):
    hk, pages = st["kv_heads"], st["table"].shape[1]
    s, row, there = plain_scores(st)
    lse = st["lse"][row.clamp(max=st["total"] - 1)].view(s.shape[0], st["most"], hk, -1).permute(0, 2, 3, 1)
    fine = torch.isfinite(lse)[..., None]
    p = torch.where(fine, torch.exp(s.sub_(torch.where(fine, lse[..., None], 0.0))), 0.0)
    gained = p.sum((2, 3)).view(-1, hk, pages, PAGE).transpose(1, 2)  # [sequences][pages][kv heads][tokens]
    j = torch.arange(pages * PAGE, device=s.device).view(1, pages, 1, PAGE)
    held, rows = st["held"].view(-1, 1, 1, 1), (st["cu"][1:] - st["cu"][:-1]).view(-1, 1, 1, 1)
    table = st["table"].long()
    old = torch.where(j < held - rows, st["keep"] * st["weights"][table], 0.0)
    seq, page, head, at = torch.nonzero((j < held).expand(gained.shape), as_tuple=True)
    st["weights"][table[seq, page], head, at] = (old + gained)[seq, page, head, at]
    return [st["weights"]]


def plain_kept(st):
    """Ids of the kept tokens [sequences][kv heads][budget], -1 behind them, and how many are kept."""
    hk, budget = st["kv_heads"], st["budget"]
    table = st["table"].long()
    w = st["weights"][table].transpose(1, 2).flatten(2, 3)  # [sequences][kv heads][tokens]
    j = torch.arange(w.shape[2], device=w.device)
    held = st["held"].view(-1, 1, 1)
    key = torch.where((j < st["first"]) | (j >= held - st["recent"]), math.inf, w)
    key = torch.where(j < held, key, -math.inf)
    best = torch.sort(key, dim=2, descending=True, stable=True).indices[..., :budget]
    if best.shape[2] < budget:
        best = torch.nn.functional.pad(best, (0, budget - best.shape[2]))
    there = torch.arange(budget, device=w.device) < held
    kept = torch.sort(torch.where(there, best, 1 << 40), dim=2).values
    return torch.where(there, kept, -1), held[:, 0, 0].clamp(max=budget)


def plain_evict(st):
    d, hk = st["head_dim"], st["kv_heads"]
    kept, lens = plain_kept(st)
    table = st["table"].long()
    there = kept >= 0
    at = torch.nonzero(there, as_tuple=True)
    seq, head, to = at
    tok = kept[at]
    page, slot = table[seq, tok // PAGE], tok % PAGE
    page_to, slot_to = table[seq, to // PAGE], to % PAGE
    # a page's new scales: the largest of the pages that its tokens come from
    old = st["scales"][page, head]
    new = torch.zeros_like(st["scales"]).view(-1, 2)
    new = new.scatter_reduce(0, (page_to * hk + head)[:, None].expand(-1, 2), old, "amax").view_as(st["scales"])
    here = new[page_to, head]
    ratio = torch.where(here > 0, old / here, 0.0)
    k = torch.round(st["codes_k"][page, head, slot].float() * ratio[:, :1]).clamp(-127, 127).to(torch.int8)
    v = torch.round(st["codes_v"][page, head, :, slot].float() * ratio[:, 1:]).clamp(-127, 127).to(torch.int8)
    lost = st["bad"][page, head] >> slot & 1
    st["weights_out"][page_to, head, slot_to] = st["weights"][page, head, slot]
    moved = (st["held"] > st["budget"])[seq]  # sequences within their budget stay as they are
    m = torch.nonzero(moved)[:, 0]
    st["codes_k"][page_to[m], head[m], slot_to[m]] = k[m]
    st["codes_v"][page_to[m], head[m], :, slot_to[m]] = v[m]
    st["scales"][page_to[m], head[m]] = here[m]
    bits = torch.zeros_like(st["bad"]).view(-1).index_add(0, page_to * hk + head, lost << slot_to).view_as(st["bad"])
    st["bad"][page_to[m], head[m]] = bits[page_to[m], head[m]]
    st["lens_out"] = lens.int()
    k, v = plain_read(st)
    return [kept.int(), st["lens_out"], st["weights_out"], st["scales"], st["bad"], k, v]


def plain_read(st):
    row, pos, there = place(st["cu_back"], st["lens_out"], st["most_back"])
    at = pos[there]
    seq = torch.arange(there.shape[0], device=row.device)[:, None].expand_as(there)[there]
    page = st["table"][seq, at // PAGE].long()
    d, lost = st["head_dim"], (st["bad"][page] >> (at % PAGE)[:, None] & 1)[..., None] > 0
    k = st["codes_k"][page, :, at % PAGE, :d].float() * st["scales"][page][..., 0, None]
    v = st["codes_v"][page, :, :d, at % PAGE].float() * st["scales"][page][..., 1, None]
    t = st["k_back"].dtype
    return torch.where(lost, math.nan, k).to(t), torch.where(lost, math.nan, v).to(t)


def plain_verify(st):
    """In 64 bits: a token is the first whose running sum passes a border, which sums of 32 bits move across tokens."""
    cu, n = st["cu"].long(), len(st["v"])
    number, k = torch.arange(n, device=cu.device), cu[1:] - cu[:-1]
    x, drafted = st["logits"].double(), st["drafted"].long()[:, None]
    if st["temperature"] > 0:
        p = torch.exp((x - x.amax(1, keepdim=True)) / st["temperature"])
        p = p / p.sum(1, keepdim=True)
        if st["about"] is not None:
            q = st["about"].double()
            q = torch.exp((q - q.amax(1, keepdim=True)) / st["temperature"]) if len(q) else q
            q = q / q.sum(1, keepdim=True)
        else:
            q = torch.zeros_like(p[st["row"]]).scatter_(1, drafted, 1.0)
        takes = st["u"] * q.gather(1, drafted)[:, 0] < p[st["row"]].gather(1, drafted)[:, 0]
    else:
        best = (x == x.amax(1, keepdim=True)).int().argmax(1)
        takes = best[st["row"]] == drafted[:, 0]
    # drafts that are taken up to the first that is not
    i = torch.arange(st["most"], device=cu.device)
    padded_takes = torch.zeros(n, st["most"] + 1, dtype=torch.int64, device=cu.device)
    there = i < k[:, None]
    if len(takes):
        padded_takes[:, :-1] = torch.where(there, takes[(cu[:-1, None] + i).clamp(max=len(takes) - 1)], 0)
    accepted = padded_takes.cumprod(1).sum(1)
    row = cu[:-1] + number + accepted
    if st["temperature"] > 0:
        r = p[row]
        refused = accepted < k
        if len(takes):
            left = (r - q[(cu[:-1] + accepted).clamp(max=len(takes) - 1)]).clamp(min=0)
            r = torch.where((refused & (left.sum(1) > 0))[:, None], left, r)
        c = r.cumsum(1)
        token = (c <= st["v"].double()[:, None] * c[:, -1:]).sum(1)
    else:
        token = best[row]
    return [accepted.int(), token.int()]


def exact(case, seed):
    """The outputs from the definitions in 64 bits, sequence by sequence."""
    st = prepare(case, seed)
    if case["op"] == "verify":
        return exact_verify(st, case)
    if case["op"] == "evict":
        return exact_evict(st, case)
    lens, rows = ints(case["lens"]), ints(case["rows"])
    g, d = case["heads"] // case["kv_heads"], case["head_dim"]
    outs, lses, first = [], [], 0
    weights = st["weights"].double() if case["op"] == "weigh" else None
    for i, (n, r) in enumerate(zip(lens, rows)):
        if n == 0:
            continue
        q = st["q"][first:first + r].double()
        page = st["table"][i, :-(-n // PAGE)].long()
        pos, j = torch.arange(n - r, n, device=q.device)[:, None], torch.arange(n, device=q.device)
        hidden = j > pos
        if case["window"]:
            hidden |= (j <= pos - case["window"]) & (j >= case["sinks"])
        out, lse = torch.empty_like(q), torch.empty(q.shape[:2], dtype=torch.float64, device=q.device)
        for kv in range(case["kv_heads"]):
            k = st["codes_k"][page, kv, :, :d].double() * st["scales"][page, kv, 0].double()[:, None, None]
            k = k.reshape(-1, d)[:n]
            v = st["codes_v"][page, kv, :d].double() * st["scales"][page, kv, 1].double()[:, None, None]
            v = v.transpose(1, 2).reshape(-1, d)[:n]
            gained = torch.zeros(n, dtype=torch.float64, device=q.device)
            for h in range(kv * g, kv * g + g):
                s = (q[:, h] @ k.T) / math.sqrt(d)
                s[hidden] = -math.inf
                if weights is not None:
                    gained += torch.exp(s - st["lse"][first:first + r, h].double()[:, None]).sum(0)
                else:
                    lse[:, h] = torch.logsumexp(s, 1)
                    out[:, h] = torch.softmax(s, 1) @ v
            if weights is not None:
                was = weights[page, kv].reshape(-1)[:n] * case["keep"]
                was[n - r:] = 0
                weights[page[j // PAGE], kv, j % PAGE] = was + gained
        outs.append(out)
        lses.append(lse)
        first += r
    return [weights] if weights is not None else [torch.cat(outs), torch.cat(lses)]


def exact_evict(st, case):
    hk, d, budget = case["kv_heads"], case["head_dim"], case["budget"]
    lens = ints(case["lens"])
    dev = st["table"].device
    kept = torch.full((len(lens), hk, budget), -1, dtype=torch.int32, device=dev)
    scales, weights = st["scales"].double(), torch.zeros_like(st["weights_out"]).double()
    backs = [], []
    for i, n in enumerate(lens):
        page = st["table"][i].long()
        m = min(n, budget)
        pages = -(-m // PAGE)
        both = [torch.empty(m, hk, d, dtype=torch.float64, device=dev) for _ in range(2)]
        to = torch.arange(m, device=dev)
        for h in range(hk):
            tok = torch.arange(n, device=dev)
            if n > budget:
                lo, hi = min(case["first"], n), max(min(case["first"], n), n - case["recent"])
                middle = st["weights"][page[tok // PAGE], h, tok % PAGE][lo:hi].double()
                more = max(0, budget - lo - (n - hi))
                chosen = torch.argsort(-middle, stable=True)[:more] + lo
                tok = torch.sort(torch.cat((tok[:lo], chosen, tok[hi:]))).values
            kept[i, h, :m] = tok.int()
            weights[page[to // PAGE], h, to % PAGE] = st["weights"][page[tok // PAGE], h, tok % PAGE].double()
            for which, codes in ((0, st["codes_k"]), (1, st["codes_v"].transpose(2, 3))):
                was = st["scales"][page[tok // PAGE], h, which].double()
                x = codes[page[tok // PAGE], h, tok % PAGE, :d].double()
                if n > budget:
                    s = torch.stack([was[b * PAGE:(b + 1) * PAGE].max() for b in range(pages)])
                    scales[page[:pages], h, which] = s
                    s = s[to // PAGE]
                    x = torch.round(x * (was / s)[:, None])
                    was = s
                both[which][:, h] = x * was[:, None]
        backs[0].append(both[0])
        backs[1].append(both[1])
    return [kept, torch.tensor([min(n, budget) for n in lens], dtype=torch.int32, device=dev), weights, scales, None,
            torch.cat(backs[0]), torch.cat(backs[1])]


def exact_verify(st, case):
    drafts, heat = ints(case["drafts"]), case["temperature"]
    got, first = [], 0
    for i, k in enumerate(drafts):
        x = st["logits"][first + i:first + i + k + 1].double()
        drafted = st["drafted"][first:first + k].long().tolist()
        taken, token = 0, None
        if heat == 0:
            best = [int(torch.nonzero(r == r.max())[0]) for r in x]
            while taken < k and best[taken] == drafted[taken]:
                taken += 1
            token = best[taken]
        else:
            p = torch.softmax(x / heat, 1)
            q = torch.softmax(st["about"][first:first + k].double() / heat, 1) if case["draft_logits"] else None
            while taken < k:
                t = drafted[taken]
                if not float(st["u"][first + taken]) * (1.0 if q is None else float(q[taken, t])) < float(p[taken, t]):
                    break
                taken += 1
            r = p[taken].clone()
            if taken < k:
                if q is None:
                    r[drafted[taken]] = 0
                else:
                    r = (r - q[taken]).clamp(min=0)
                r = r if float(r.sum()) > 0 else p[taken]
            c = torch.cumsum(r, 0)
            token = int(torch.searchsorted(c, st["v"][i].double() * c[-1], right=True))
        got.append((taken, token))
        first += k
    return [torch.tensor([a for a, _ in got], dtype=torch.int32), torch.tensor([b for _, b in got], dtype=torch.int32)]

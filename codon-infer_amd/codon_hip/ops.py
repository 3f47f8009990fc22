"""The device operators of the C ABI on arrays in GPU memory: the 8-bit paged
key/value cache with rotary positions (cih_kv8_append, cih_kv8_read), attention
over it (cih_kv8_attention), the attention weight that its tokens gather and
eviction by it (cih_kv8_weigh, cih_kv8_evict), the log probabilities of given
tokens (cih_token_logprobs) and the verification of drafted ones
(cih_verify_drafts).  None of them has a counterpart in the reference.

Arrays are anything with data_ptr(), shape, stride() in elements and dtype:
torch tensors on the GPU, or devmem.DeviceArray.  Outputs are written into
arrays the caller brings.  Calls are enqueued and return without waiting: on
`stream` (a hipStream_t as an integer) if given, else for torch tensors on
torch's current stream, else on the null stream.  The arrays must live on the
current device, and must not be freed before the work has run.
"""
import ctypes
import sys

from . import _lib as C

_FLOATS = {"float32": C.F32, "float16": C.F16, "bfloat16": C.BF16}
_names = {}  # dtype object -> its name


def _dtype(a):
    d = a.dtype
    try:
        return _names[d]
    except KeyError:
        n = _names[d] = str(d).rpartition(".")[2]
        return n


def _float(a, what):
    try:
        return _FLOATS[_dtype(a)]
    except KeyError:
        raise TypeError(f"{what} is {_dtype(a)}: float32, float16 or bfloat16 is needed") from None


def _where(arrays):
    """The GPU that the torch tensors among the arrays are on; None without one."""
    torch = sys.modules.get("torch")
    if torch is None:
        return None
    at, tensor = None, torch.Tensor
    for a in arrays:
        if isinstance(a, tensor):
            d = a.get_device()
            if d != at:
                if d < 0 or at is not None:
                    raise ValueError("tensors on the CPU or on different GPUs")
                at = d
    return at


def _stream(at, stream):
    """The stream to enqueue on for tensors on GPU `at`, which must be the current one."""
    if at is None:
        return stream or 0
    now, raw = _torch_now()
    if at != now():
        raise ValueError(f"a tensor is on cuda:{at}, the current device is cuda:{now()}")
    return raw(at) if stream is None else stream


_now = None


def _torch_now():
    """torch's current device, and its current stream on a device: the plain
    integers where this torch gives them (a Stream object costs 1 us)."""
    global _now
    if _now is None:
        torch = sys.modules["torch"]
        torch.cuda.current_device()  # torch is set up
        raw = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        _now = (getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device),
                raw or (lambda d: torch.cuda.current_stream(d).cuda_stream))
    return _now


def _same(at, kept):
    if at is None:
        return kept
    if kept is not None and kept != at:
        raise ValueError("tensors on different GPUs")
    return at


def _dense(a):
    n = 1
    for d, st in zip(reversed(a.shape), reversed(a.stride())):
        if d != 1 and st != n:
            return False
        n *= d
    return True


def _plain(a, what, dtype, shape=None):
    """The address of an array without gaps, of this type (and shape)."""
    try:
        name = _names[a.dtype]
    except KeyError:
        name = _dtype(a)
    if name not in dtype:
        raise TypeError(f"{what} is {name}: {' or '.join(dtype)} is needed")
    if shape is not None and a.shape != shape:
        raise ValueError(f"{what} has shape {tuple(a.shape)}: {tuple(shape)} is needed")
    try:
        dense = a.is_contiguous()
    except AttributeError:
        dense = _dense(a)
    if not dense:
        raise ValueError(f"{what} must be contiguous")
    return a.data_ptr()


def _rows(a, what, shape, new=C.RowsStruct):
    """A [rows][heads][dim] array as a cih_rows; the last axis without gaps."""
    if a.shape != shape:
        raise ValueError(f"{what} has shape {tuple(a.shape)}: {shape} is needed")
    rs, hs, one = a.stride()
    if one != 1:
        raise ValueError(f"{what}: the last axis must be contiguous")
    return new(a.data_ptr(), rs, hs)


_lib = C.lib()
_at = ctypes.addressof


class Rope:
    """Rotary positions (cih_rope_init): the first rot_dim dims of a head in
    pairs (j, j + rot_dim / 2), or neighbours with interleaved; scaling "none",
    "linear", "ntk" or "yarn" by factor for contexts beyond trained_len."""

    SCALINGS = {"none": C.ROPE_NONE, "linear": C.ROPE_LINEAR, "ntk": C.ROPE_NTK, "yarn": C.ROPE_YARN}

    def __init__(self, rot_dim, base=10000.0, interleaved=False, scaling="none", factor=1.0, trained_len=1024):
        if scaling not in self.SCALINGS:
            raise ValueError(f"scaling {scaling!r} is none of {', '.join(self.SCALINGS)}")
        self.struct = C.RopeStruct()
        C.check(_lib.cih_rope_init(_at(self.struct), rot_dim, int(interleaved), float(base),
                                      self.SCALINGS[scaling], float(factor), int(trained_len)))

    @property
    def freq(self):
        """Radians per position of each pair."""
        return list(self.struct.freq[:self.struct.rot_dim // 2])

    @property
    def gain(self):
        return self.struct.gain


class Kv8Batch:
    """Sequences and their new rows (cih_kv8_batch): int32 arrays cu_rows
    [n_seq + 1], lens [n_seq], table [table_rows][max_pages] and slots [n_seq]
    (None: row i of the table is sequence i's).  n_rows: rows of the row arrays;
    max_rows: the most of any sequence."""

    def __init__(self, cu_rows, lens, table, n_rows, max_rows, slots=None):
        n = lens.shape[0]
        i32 = ("int32",)
        if len(table.shape) != 2 or (table.shape[1] != 1 and table.stride()[1] != 1):
            raise ValueError("table must be a matrix with contiguous rows")
        if _dtype(table) != "int32":
            raise TypeError(f"table is {_dtype(table)}: int32 is needed")
        stride = table.stride()[0] if table.shape[0] > 1 else table.shape[1]
        self.lens = lens
        self._arrays = (cu_rows, lens, table) + (() if slots is None else (slots,))
        self.n_rows, self.n_seq = n_rows, n
        self.struct = C.Kv8BatchStruct(_plain(cu_rows, "cu_rows", i32, (n + 1,)), _plain(lens, "lens", i32, (n,)),
                                       table.data_ptr(), None if slots is None else _plain(slots, "slots", i32, (n,)),
                                       n, n_rows, max_rows, table.shape[0], stride, table.shape[1])
        self._at = _at(self.struct)
        self._gpu = _where(self._arrays)


class Kv8Cache:
    """The paged cache (cih_kv8_cache) over the caller's buffers: k int8
    [n_pages][kv_heads][64][dims], v int8 [n_pages][kv_heads][dims][64], scales
    float32 [n_pages][kv_heads][2], bad int64 or uint64 [n_pages][kv_heads];
    dims = Kv8Cache.dims(head_dim)."""

    def __init__(self, k, v, scales, bad, head_dim):
        n, h, page, d = k.shape
        if page != C.KV8_PAGE or d != self.dims(head_dim):
            raise ValueError(f"k has shape {tuple(k.shape)}: pages of [{C.KV8_PAGE}][{self.dims(head_dim)}] are needed")
        self._arrays = (k, v, scales, bad)
        self.kv_heads, self.head_dim = h, head_dim
        self.struct = C.Kv8CacheStruct(_plain(k, "k", ("int8",)), _plain(v, "v", ("int8",), (n, h, d, page)),
                                       _plain(scales, "scales", ("float32",), (n, h, 2)),
                                       _plain(bad, "bad", ("int64", "uint64"), (n, h)), n, h, head_dim)
        self._at = _at(self.struct)
        self._gpu = _where(self._arrays)
        self._scale = head_dim ** -0.5
        self._weights = (n, h, page)

    @staticmethod
    def dims(head_dim):
        """Dims of a head as stored."""
        return 32 if head_dim == 24 else head_dim

    def append(self, batch, k, v, q=None, q_out=None, rope=None, stream=None, shifts=None):
        """Writes the batch's rows k and v [n_rows][kv_heads][head_dim] into the
        cache at their positions, k rotated by rope; q [n_rows][q_heads][head_dim]
        rotated goes to q_out (default: q itself).  shifts: int32 [n_seq], added to
        a sequence's positions for their angles (what evict took)."""
        t, shape = _float(k, "k"), (batch.n_rows, self.kv_heads, self.head_dim)
        ks, vs = _rows(k, "k", shape), _rows(v, "v", shape)
        if _float(v, "v") != t:
            raise TypeError("k and v differ in type")
        qs = qo = None
        heads = 0
        if q is not None:
            q_out = q if q_out is None else q_out
            heads = q.shape[1]
            shape = (batch.n_rows, heads, self.head_dim)
            qs, qo = _rows(q, "q", shape), _rows(q_out, "q_out", shape)
            if _float(q, "q") != t or _float(q_out, "q_out") != t:
                raise TypeError("q, q_out and k differ in type")
        sh = None if shifts is None else _plain(shifts, "shifts", ("int32",), (batch.n_seq,))
        at = _same(_same(_where((k, v, shifts) if q is None else (k, v, q, q_out, shifts)), self._gpu), batch._gpu)
        a = _at
        C.check(_lib.cih_kv8_append_shifted(self._at, batch._at, t, a(ks), a(vs), heads, a(qs) if qs else None,
                                            a(qo) if qo else None, a(rope.struct) if rope else None, sh,
                                            _stream(at, stream)))

    def read(self, batch, k, v, stream=None):
        """The batch's rows read back into k and v [n_rows][kv_heads][head_dim]."""
        t, shape = _float(k, "k"), (batch.n_rows, self.kv_heads, self.head_dim)
        ks, vs = _rows(k, "k", shape), _rows(v, "v", shape)
        if _float(v, "v") != t:
            raise TypeError("k and v differ in type")
        at = _same(_same(_where((k, v)), self._gpu), batch._gpu)
        C.check(_lib.cih_kv8_read(self._at, batch._at, t, _at(ks), _at(vs),
                                     _stream(at, stream)))

    def attend_workspace(self, batch, q_heads):
        """Bytes of workspace that attend needs for a batch of these sizes."""
        n = ctypes.c_size_t()
        C.check(_lib.cih_kv8_attention_workspace(self._at, batch._at, q_heads, ctypes.byref(n)))
        return n.value

    def attend(self, batch, q, out, lse=None, scale=None, causal=True, window=0, workspace=None, stream=None, sinks=0):
        """Attention of the batch's rows q [n_rows][q_heads][head_dim] over the
        cache into out (q's shape and type) and lse float32 [n_rows][q_heads].
        scale: default 1 / sqrt(head_dim).  sinks: first tokens that a window
        leaves visible.  workspace: uint8, of attend_workspace bytes at least."""
        t, heads = _float(q, "q"), q.shape[1]
        shape = (batch.n_rows, heads, self.head_dim)
        qs, os = _rows(q, "q", shape), _rows(out, "out", shape)
        if _float(out, "out") != t:
            raise TypeError("q and out differ in type")
        ls = None if lse is None else _plain(lse, "lse", ("float32",), shape[:2])
        ws, size = _workspace(workspace)
        at = _same(_same(_where((q, out, lse, workspace)), self._gpu), batch._gpu)
        C.check(_lib.cih_kv8_attention_sinks(self._at, batch._at, t, heads, _at(qs), _at(os), ls,
                                             self._scale if scale is None else scale, 1 if causal else 0, window, sinks,
                                             ws, size, _stream(at, stream)))

    def weigh(self, batch, q, lse, weights, scale=None, causal=True, window=0, sinks=0, keep=1.0, stream=None):
        """Adds to weights (float32 [n_pages][kv_heads][64], beside the cache) what
        the batch's rows q give each token they see: the sum of exp(scale q.k - lse)
        over rows and the query heads of a kv head, with lse [n_rows][q_heads] from
        attend with the same arguments.  keep: the share that earlier weights keep
        (0: start anew)."""
        t, heads = _float(q, "q"), q.shape[1]
        shape = (batch.n_rows, heads, self.head_dim)
        qs = _rows(q, "q", shape)
        ls = _plain(lse, "lse", ("float32",), shape[:2])
        wt = _plain(weights, "weights", ("float32",), self._weights)
        at = _same(_same(_where((q, lse, weights)), self._gpu), batch._gpu)
        C.check(_lib.cih_kv8_weigh(self._at, batch._at, t, heads, _at(qs), ls, self._scale if scale is None else scale,
                                   1 if causal else 0, window, sinks, keep, wt, _stream(at, stream)))

    def evict_workspace(self, batch, budget):
        """Bytes of workspace that evict needs for a batch of these sizes."""
        n = ctypes.c_size_t()
        C.check(_lib.cih_kv8_evict_workspace(self._at, batch._at, budget, ctypes.byref(n)))
        return n.value

    def evict(self, batch, weights, budget, first=0, recent=0, weights_out=None, lens_out=None, shifts=None, kept=None,
              workspace=None, stream=None):
        """Cuts the batch's sequences to at most budget tokens: each kv head keeps its
        first `first`, its last `recent` and of the others those with the largest
        weights, in their order.  The kept tokens' weights go to weights_out
        (default: weights itself), the new lengths to lens_out (default: the
        batch's lens), how many tokens went (its length less the budget) is added to
        shifts (int32 [n_seq]), the places that the kept ones had go to kept (int32 [n_seq][kv_heads][budget],
        -1 behind them)."""
        n, i32 = batch.n_seq, ("int32",)
        weights_out = weights if weights_out is None else weights_out
        lens_out = batch.lens if lens_out is None else lens_out
        wt = _plain(weights, "weights", ("float32",), self._weights)
        wo = _plain(weights_out, "weights_out", ("float32",), self._weights)
        lo = _plain(lens_out, "lens_out", i32, (n,))
        sh = None if shifts is None else _plain(shifts, "shifts", i32, (n,))
        kp = None if kept is None else _plain(kept, "kept", i32, (n, self.kv_heads, budget))
        ws, size = _workspace(workspace)
        at = _same(_same(_where((weights, weights_out, lens_out, shifts, kept, workspace)), self._gpu), batch._gpu)
        C.check(_lib.cih_kv8_evict(self._at, batch._at, budget, first, recent, wt, wo, lo, sh, kp, ws, size,
                                   _stream(at, stream)))


def _workspace(w):
    return (None, 0) if w is None else (_plain(w, "workspace", ("uint8",)), w.shape[0])


def token_logprobs_workspace(n_rows, vocab, top_k):
    """Bytes of workspace that token_logprobs needs."""
    n = ctypes.c_size_t()
    C.check(_lib.cih_token_logprobs_workspace(n_rows, vocab, top_k, ctypes.byref(n)))
    return n.value


def token_logprobs(logits, targets=None, logprob=None, entropy=None, top_ids=None, top_logprobs=None, workspace=None,
                   stream=None):
    """Of each row of logits [n][vocab]: the log probability of targets [n]
    (int32) into logprob, the entropy (nats) into entropy, the largest logits'
    ids and log probabilities into top_ids (int32) and top_logprobs [n][k]
    (all outputs float32 but the ids; None: not wanted)."""
    n, vocab = logits.shape
    if vocab != 1 and logits.stride()[1] != 1:
        raise ValueError("logits: the last axis must be contiguous")
    if (top_ids is None) != (top_logprobs is None):
        raise ValueError("top_ids and top_logprobs go together")
    if logprob is not None and targets is None:
        raise ValueError("logprob needs targets")
    f32 = ("float32",)
    tg = None if targets is None else _plain(targets, "targets", ("int32",), (n,))
    lp = None if logprob is None else _plain(logprob, "logprob", f32, (n,))
    en = None if entropy is None else _plain(entropy, "entropy", f32, (n,))
    k, ids, tl = 0, None, None
    if top_ids is not None:
        k = top_ids.shape[1]
        ids = _plain(top_ids, "top_ids", ("int32",), (n, k))
        tl = _plain(top_logprobs, "top_logprobs", f32, (n, k))
    ws, size = _workspace(workspace)
    at = _where((logits, targets, logprob, entropy, top_ids, top_logprobs, workspace))
    C.check(_lib.cih_token_logprobs(_float(logits, "logits"), logits.data_ptr(), logits.stride()[0], n, vocab, tg, lp,
                                       en, k, ids, tl, ws, size, _stream(at, stream)))


def verify_drafts_workspace(n_seq, n_drafts, vocab):
    """Bytes of workspace that verify_drafts needs."""
    n = ctypes.c_size_t()
    C.check(_lib.cih_verify_drafts_workspace(n_seq, n_drafts, vocab, ctypes.byref(n)))
    return n.value


def verify_drafts(logits, drafts, cu_drafts, accepted, tokens, draft_logits=None, accept_at=None, sample_at=None,
                  temperature=1.0, workspace=None, stream=None):
    """Speculative sampling: of the drafts of sequence i (int32 [n_drafts], from
    cu_drafts[i] to cu_drafts[i + 1]), how many are accepted (int32 [n_seq]) and the
    token after them (int32 [n_seq]).  logits [n_drafts + n_seq][vocab]: the target's,
    a row for each draft of a sequence and one after them; draft_logits
    [n_drafts][vocab]: what the drafts were drawn from (None: they are certain).
    accept_at float32 [n_drafts] and sample_at float32 [n_seq]: random numbers in
    [0, 1), not needed at temperature 0."""
    (n,), (d,), (rows, vocab) = tokens.shape, drafts.shape, logits.shape
    f32, i32 = ("float32",), ("int32",)
    t, (stride, one) = _float(logits, "logits"), logits.stride()
    if rows != n + d:
        raise ValueError(f"logits has {rows} rows: {n + d} are needed")
    if vocab != 1 and one != 1:
        raise ValueError("logits: the last axis must be contiguous")
    dl, ds = None, 0
    if draft_logits is not None:
        if draft_logits.shape != (d, vocab):
            raise ValueError(f"draft_logits has shape {tuple(draft_logits.shape)}: {(d, vocab)} is needed")
        ds, one = draft_logits.stride()
        if vocab != 1 and one != 1:
            raise ValueError("draft_logits: the last axis must be contiguous")
        if _float(draft_logits, "draft_logits") != t:
            raise TypeError("logits and draft_logits differ in type")
        dl = draft_logits.data_ptr()
    dr = _plain(drafts, "drafts", i32, (d,))
    cu = _plain(cu_drafts, "cu_drafts", i32, (n + 1,))
    ac, tk = _plain(accepted, "accepted", i32, (n,)), _plain(tokens, "tokens", i32, (n,))
    ua = None if accept_at is None else _plain(accept_at, "accept_at", f32, (d,))
    us = None if sample_at is None else _plain(sample_at, "sample_at", f32, (n,))
    ws, size = _workspace(workspace)
    at = _where((logits, drafts, cu_drafts, accepted, tokens, draft_logits, accept_at, sample_at, workspace))
    C.check(_lib.cih_verify_drafts(t, logits.data_ptr(), stride, dl, ds, n, d, vocab, cu, dr, ua, us,
                                   temperature, ac, tk, ws, size, _stream(at, stream)))

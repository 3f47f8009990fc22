// C entries of the 8-bit paged key/value cache, of the token log probabilities and
// of the verification of drafts: argument checks on the host, then the launches.
#include <cmath>

#include "kv8.h"
#include "model.h"

using namespace cih;

namespace {

bool aligned(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

size_t float_size(int dtype) { return dtype == CIH_F32 ? 4 : 2; }

// A launch goes to the stream's device, the kernels to the current one.
int check_stream(hipStream_t st) {
    if (!st || st == hipStreamPerThread) return 0;  // the current device's
    int now = -1;
    hipDevice_t of = -1;
    HIPCHK(hipGetDevice(&now));
    HIPCHK(hipStreamGetDevice(st, &of));
    if (of != now) return set_error(CIH_ERR_ARG, "the stream belongs to device %d, the current device is %d", of, now);
    return 0;
}

// memory: the cache's buffers are looked at too (not for sizes of a workspace)
int check_cache(const cih_kv8_cache *c, Kv8View &v, bool memory) {
    if (!c) return set_error(CIH_ERR_ARG, "null cache");
    const int d = c->head_dim;
    if (d != 16 && d != 24 && d != 32 && d != 64 && d != 128)
        return set_error(CIH_ERR_SHAPE, "head_dim %d is not 16, 24, 32, 64 or 128", d);
    if (c->kv_heads < 1 || c->kv_heads > 65535 || c->n_pages < 1)
        return set_error(CIH_ERR_SHAPE, "%d pages of %d heads", c->n_pages, c->kv_heads);
    if (memory) {
        if (!c->k || !c->v || !c->scales || !c->bad) return set_error(CIH_ERR_ARG, "null cache buffer");
        if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->scales, 8) || !aligned(c->bad, 8))
            return set_error(CIH_ERR_ARG, "codes must be 16-byte, scales and bad 8-byte aligned");
    }
    v = {static_cast<signed char *>(c->k), static_cast<signed char *>(c->v), reinterpret_cast<float2 *>(c->scales),
         reinterpret_cast<unsigned long long *>(c->bad), c->n_pages, c->kv_heads, d, kv8_dims(d)};
    return 0;
}

int check_batch(const cih_kv8_batch *b, Kv8Seqs &s, bool memory) {
    if (!b) return set_error(CIH_ERR_ARG, "null batch");
    if (b->n_seq < 0 || b->n_rows < 0 || b->max_rows < 0 || b->table_rows < 0)
        return set_error(CIH_ERR_ARG, "negative size in the batch");
    if (b->max_pages < 1 || b->max_pages > (1 << 24) || b->table_stride < b->max_pages)
        return set_error(CIH_ERR_SHAPE, "a table of %d pages a row, %d apart", b->max_pages, b->table_stride);
    if (b->max_rows > (1 << 30) || b->n_rows > (1 << 30)) return set_error(CIH_ERR_SHAPE, "more than 2^30 rows");
    if (memory && b->n_seq > 0) {
        if (!b->cu_rows || !b->lens || !b->table) return set_error(CIH_ERR_ARG, "null batch array");
        if (!aligned(b->cu_rows, 4) || !aligned(b->lens, 4) || !aligned(b->table, 4) || !aligned(b->slots, 4))
            return set_error(CIH_ERR_ARG, "batch arrays must be 4-byte aligned");
        if (!b->slots && b->table_rows < b->n_seq)
            return set_error(CIH_ERR_SHAPE, "a table of %d rows for %d sequences", b->table_rows, b->n_seq);
    }
    s = {b->cu_rows, b->lens, b->table, b->slots, b->n_seq, b->n_rows, std::min(b->max_rows, b->n_rows), b->table_rows,
         b->table_stride, b->max_pages};
    return 0;
}

int check_rows(const cih_rows *r, const char *what, int dtype, RowsView &v) {
    if (!r || !r->data) return set_error(CIH_ERR_ARG, "null %s", what);
    if (!aligned(r->data, float_size(dtype))) return set_error(CIH_ERR_ARG, "%s is not aligned to its type", what);
    const int64_t most = (int64_t)1 << 31;
    if (r->row_stride < 0 || r->head_stride < 0 || r->row_stride > most || r->head_stride > most)
        return set_error(CIH_ERR_SHAPE, "%s: strides of %lld and %lld elements", what, (long long)r->row_stride,
                         (long long)r->head_stride);
    v = {r->data, r->row_stride, r->head_stride};
    return 0;
}

// Rows that are written must not share elements.
int check_out(const RowsView &v, const char *what, int64_t rows, int64_t heads, int64_t d) {
    const bool by_row = (heads <= 1 || v.hs >= d) && (rows <= 1 || v.rs >= (heads - 1) * v.hs + d);
    const bool by_head = (rows <= 1 || v.rs >= d) && (heads <= 1 || v.hs >= (rows - 1) * v.rs + d);
    if (!by_row && !by_head) return set_error(CIH_ERR_SHAPE, "%s: its strides make heads or rows overlap", what);
    return 0;
}

int check_float(int dtype) {
    if (dtype != CIH_F32 && dtype != CIH_F16 && dtype != CIH_BF16) return set_error(CIH_ERR_ARG, "bad element type %d", dtype);
    return 0;
}

int check_heads(int heads, int hk, const Kv8Seqs &s) {
    if (heads < 1 || heads > 65535 || heads % hk)
        return set_error(CIH_ERR_SHAPE, "%d query heads over %d key/value heads", heads, hk);
    if ((int64_t)s.max_rows * (heads / hk) > 1 << 30)
        return set_error(CIH_ERR_SHAPE, "%d rows of %d query heads a key/value head", s.max_rows, heads / hk);
    return 0;
}

// What attention and the weights that it leaves have in common.
int check_call(const cih_kv8_cache *cache, const cih_kv8_batch *batch, int dtype, int heads, float scale, int causal,
               int window, int sinks, Kv8Attention &a) {
    if (int rc = check_float(dtype)) return rc;
    if (int rc = check_cache(cache, a.c, true)) return rc;
    if (int rc = check_batch(batch, a.s, true)) return rc;
    if (int rc = check_heads(heads, a.c.hk, a.s)) return rc;
    if (window < 0) return set_error(CIH_ERR_ARG, "window %d", window);
    if (sinks < 0) return set_error(CIH_ERR_ARG, "%d sinks", sinks);
    if (!std::isfinite(scale)) return set_error(CIH_ERR_ARG, "the scale is not finite");
    a.dtype = dtype;
    a.heads = heads;
    a.scale = scale;
    a.causal = causal != 0;
    a.window = window;
    a.sinks = window > 0 ? sinks : 0;  // without a window all of them are visible anyway
    return 0;
}

int check_budget(int budget, int first, int recent) {
    if (budget < 1 || budget > 1 << 30) return set_error(CIH_ERR_SHAPE, "a budget of %d tokens", budget);
    if (first < 0 || recent < 0 || (int64_t)first + recent > budget)
        return set_error(CIH_ERR_ARG, "%d first and %d recent tokens in a budget of %d", first, recent, budget);
    return 0;
}

int check_evict_size(const Kv8View &c, const Kv8Seqs &s, int budget) {
    if (!kv8_evict_fits(c, s, budget))
        return set_error(CIH_ERR_SHAPE, "%d sequences of %d heads to %d tokens: more than one launch may have", s.n_seq, c.hk, budget);
    return 0;
}

}  // namespace

int cih::kv8_rope(const cih_rope *r, int head_dim, RopeArg &a) {
    if (!r) return 0;
    if (r->rot_dim < 2 || r->rot_dim > head_dim || r->rot_dim % 2)
        return set_error(CIH_ERR_SHAPE, "%d rotary dims in a head of %d", r->rot_dim, head_dim);
    a.rot = r->rot_dim;
    a.inter = r->interleaved != 0;
    a.gain = r->gain;
    if (!std::isfinite(a.gain)) return set_error(CIH_ERR_ARG, "the rotary gain is not finite");
    const double turn = 6.283185307179586476925;
    for (int j = 0; j < a.rot / 2; j++) {
        if (!std::isfinite(r->freq[j])) return set_error(CIH_ERR_ARG, "rotary frequency %d is not finite", j);
        a.turns[j] = r->freq[j] / turn;
    }
    return 0;
}

#define CIH_TRY(expr)                    \
    do {                                 \
        if (int rc_ = (expr)) return rc_; \
    } while (0)

extern "C" {

int cih_rope_init(cih_rope *r, int32_t rot_dim, int32_t interleaved, double base, int32_t scaling, double factor,
                  int32_t trained_len) {
    if (!r) return set_error(CIH_ERR_ARG, "null rope");
    if (rot_dim < 2 || rot_dim > 128 || rot_dim % 2) return set_error(CIH_ERR_SHAPE, "%d rotary dims", rot_dim);
    if (!(base > 0.0) || !std::isfinite(base)) return set_error(CIH_ERR_ARG, "the base must be positive");
    if (scaling < CIH_ROPE_NONE || scaling > CIH_ROPE_YARN) return set_error(CIH_ERR_ARG, "bad scaling %d", scaling);
    if (scaling != CIH_ROPE_NONE && (!(factor >= 1.0) || !std::isfinite(factor)))
        return set_error(CIH_ERR_ARG, "the scaling factor must be at least 1");
    if (scaling == CIH_ROPE_NTK && rot_dim < 4) return set_error(CIH_ERR_SHAPE, "NTK scaling needs 4 rotary dims");
    if (scaling == CIH_ROPE_YARN && trained_len < 1) return set_error(CIH_ERR_ARG, "trained_len must be at least 1");
    *r = cih_rope{};
    r->rot_dim = rot_dim;
    r->interleaved = interleaved != 0;
    r->gain = 1.0f;
    if (scaling == CIH_ROPE_NTK) base *= std::pow(factor, rot_dim / (rot_dim - 2.0));
    for (int j = 0; j < rot_dim / 2; j++) {
        double f = std::pow(base, -2.0 * j / rot_dim);
        if (scaling == CIH_ROPE_LINEAR) f /= factor;
        if (scaling == CIH_ROPE_YARN) {
            const double turns = trained_len * f / 6.283185307179586476925;
            const double g = std::min(1.0, std::max(0.0, (turns - 1.0) / 31.0));
            f *= (1.0 - g) / factor + g;
        }
        r->freq[j] = f;
    }
    if (scaling == CIH_ROPE_YARN) r->gain = (float)(0.1 * std::log(factor) + 1.0);
    return CIH_OK;
}

int cih_kv8_append_shifted(const cih_kv8_cache *cache, const cih_kv8_batch *batch, int32_t dtype, const cih_rows *k,
                           const cih_rows *v, int32_t q_heads, const cih_rows *q, const cih_rows *q_out,
                           const cih_rope *rope, const int32_t *shifts, void *stream) {
    Kv8View c;
    Kv8Seqs s;
    RowsView kv, vv, qv{}, qo{};
    RopeArg ra;
    CIH_TRY(check_float(dtype));
    CIH_TRY(check_cache(cache, c, true));
    CIH_TRY(check_batch(batch, s, true));
    CIH_TRY(kv8_rope(rope, c.d, ra));
    if (!aligned(shifts, 4)) return set_error(CIH_ERR_ARG, "shifts must be 4-byte aligned");
    ra.shift = shifts;
    if (s.n_rows == 0 || s.n_seq == 0 || s.max_rows == 0) return CIH_OK;
    CIH_TRY(check_rows(k, "k", dtype, kv));
    CIH_TRY(check_rows(v, "v", dtype, vv));
    if (q) {
        CIH_TRY(check_heads(q_heads, c.hk, s));
        CIH_TRY(check_rows(q, "q", dtype, qv));
        CIH_TRY(check_rows(q_out, "q_out", dtype, qo));
        CIH_TRY(check_out(qo, "q_out", s.n_rows, q_heads, c.d));
        if (qo.p == qv.p && (qo.rs != qv.rs || qo.hs != qv.hs))
            return set_error(CIH_ERR_ARG, "q_out in q's place must have q's strides");
    }
    hipStream_t st = static_cast<hipStream_t>(stream);
    CIH_TRY(check_stream(st));
    const hipError_t e = launch_kv8_append(c, s, dtype, kv, vv, q ? q_heads : c.hk, qv, qo, ra, st);
    if (e != hipSuccess) return set_error(CIH_ERR_HIP, "cache append failed: %s", hipGetErrorString(e));
    return CIH_OK;
}

int cih_kv8_append(const cih_kv8_cache *cache, const cih_kv8_batch *batch, int32_t dtype, const cih_rows *k,
                   const cih_rows *v, int32_t q_heads, const cih_rows *q, const cih_rows *q_out, const cih_rope *rope,
                   void *stream) {
    return cih_kv8_append_shifted(cache, batch, dtype, k, v, q_heads, q, q_out, rope, nullptr, stream);
}

int cih_kv8_read(const cih_kv8_cache *cache, const cih_kv8_batch *batch, int32_t dtype, const cih_rows *k,
                 const cih_rows *v, void *stream) {
    Kv8View c;
    Kv8Seqs s;
    RowsView kv, vv;
    CIH_TRY(check_float(dtype));
    CIH_TRY(check_cache(cache, c, true));
    CIH_TRY(check_batch(batch, s, true));
    if (s.n_rows == 0 || s.n_seq == 0 || s.max_rows == 0) return CIH_OK;
    CIH_TRY(check_rows(k, "k", dtype, kv));
    CIH_TRY(check_rows(v, "v", dtype, vv));
    CIH_TRY(check_out(kv, "k", s.n_rows, c.hk, c.d));
    CIH_TRY(check_out(vv, "v", s.n_rows, c.hk, c.d));
    hipStream_t st = static_cast<hipStream_t>(stream);
    CIH_TRY(check_stream(st));
    const hipError_t e = launch_kv8_read(c, s, dtype, kv, vv, st);
    if (e != hipSuccess) return set_error(CIH_ERR_HIP, "cache read failed: %s", hipGetErrorString(e));
    return CIH_OK;
}

int cih_kv8_attention_workspace(const cih_kv8_cache *cache, const cih_kv8_batch *batch, int32_t q_heads, size_t *bytes) {
    Kv8View c;
    Kv8Seqs s;
    if (!bytes) return set_error(CIH_ERR_ARG, "null bytes");
    CIH_TRY(check_cache(cache, c, false));
    CIH_TRY(check_batch(batch, s, false));
    CIH_TRY(check_heads(q_heads, c.hk, s));
    *bytes = kv8_attention_floats(c, s, q_heads) * sizeof(float);
    return CIH_OK;
}

int cih_kv8_attention_sinks(const cih_kv8_cache *cache, const cih_kv8_batch *batch, int32_t dtype, int32_t q_heads,
                            const cih_rows *q, const cih_rows *out, float *lse, float scale, int32_t causal,
                            int32_t window, int32_t sinks, void *workspace, size_t workspace_bytes, void *stream) {
    Kv8Attention a{};
    CIH_TRY(check_call(cache, batch, dtype, q_heads, scale, causal, window, sinks, a));
    if (a.s.n_rows == 0 || a.s.n_seq == 0 || a.s.max_rows == 0) return CIH_OK;
    CIH_TRY(check_rows(q, "q", dtype, a.q));
    CIH_TRY(check_rows(out, "out", dtype, a.out));
    CIH_TRY(check_out(a.out, "out", a.s.n_rows, q_heads, a.c.d));
    if (a.out.p == a.q.p && (a.out.rs != a.q.rs || a.out.hs != a.q.hs))
        return set_error(CIH_ERR_ARG, "out in q's place must have q's strides");
    if (lse && !aligned(lse, 4)) return set_error(CIH_ERR_ARG, "lse must be 4-byte aligned");
    const size_t need = kv8_attention_floats(a.c, a.s, q_heads) * sizeof(float);
    if (need > 0 && (!workspace || !aligned(workspace, 16) || workspace_bytes < need))
        return set_error(CIH_ERR_CAPACITY, "the call needs a 16-byte aligned workspace of %zu bytes", need);
    a.lse = lse;
    hipStream_t st = static_cast<hipStream_t>(stream);
    CIH_TRY(check_stream(st));
    const hipError_t e = launch_kv8_attention(a, static_cast<float *>(workspace), need > 0 ? workspace_bytes / sizeof(float) : 0, st);
    if (e != hipSuccess) return set_error(CIH_ERR_HIP, "attention over the cache failed: %s", hipGetErrorString(e));
    return CIH_OK;
}

int cih_kv8_attention(const cih_kv8_cache *cache, const cih_kv8_batch *batch, int32_t dtype, int32_t q_heads,
                      const cih_rows *q, const cih_rows *out, float *lse, float scale, int32_t causal, int32_t window,
                      void *workspace, size_t workspace_bytes, void *stream) {
    return cih_kv8_attention_sinks(cache, batch, dtype, q_heads, q, out, lse, scale, causal, window, 0, workspace,
                                   workspace_bytes, stream);
}

int cih_kv8_weigh(const cih_kv8_cache *cache, const cih_kv8_batch *batch, int32_t dtype, int32_t q_heads,
                  const cih_rows *q, const float *lse, float scale, int32_t causal, int32_t window, int32_t sinks,
                  float keep, float *weights, void *stream) {
    Kv8Weigh w{};
    CIH_TRY(check_call(cache, batch, dtype, q_heads, scale, causal, window, sinks, w.a));
    if (!(keep >= 0.0f && keep <= 1.0f)) return set_error(CIH_ERR_ARG, "keep is not within [0, 1]");
    if (w.a.s.n_rows == 0 || w.a.s.n_seq == 0 || w.a.s.max_rows == 0) return CIH_OK;
    CIH_TRY(check_rows(q, "q", dtype, w.a.q));
    if (!lse || !weights) return set_error(CIH_ERR_ARG, "null %s", lse ? "weights" : "lse");
    if (!aligned(lse, 4) || !aligned(weights, 4)) return set_error(CIH_ERR_ARG, "lse and weights must be 4-byte aligned");
    w.a.lse = const_cast<float *>(lse);
    w.keep = keep;
    w.weights = weights;
    hipStream_t st = static_cast<hipStream_t>(stream);
    CIH_TRY(check_stream(st));
    const hipError_t e = launch_kv8_weigh(w, st);
    if (e != hipSuccess) return set_error(CIH_ERR_HIP, "weighing the cache failed: %s", hipGetErrorString(e));
    return CIH_OK;
}

int cih_kv8_evict_workspace(const cih_kv8_cache *cache, const cih_kv8_batch *batch, int32_t budget, size_t *bytes) {
    Kv8View c;
    Kv8Seqs s;
    if (!bytes) return set_error(CIH_ERR_ARG, "null bytes");
    CIH_TRY(check_cache(cache, c, false));
    CIH_TRY(check_batch(batch, s, false));
    CIH_TRY(check_budget(budget, 0, 0));
    CIH_TRY(check_evict_size(c, s, budget));
    *bytes = kv8_evict_bytes(c, s, budget);
    return CIH_OK;
}

int cih_kv8_evict(const cih_kv8_cache *cache, const cih_kv8_batch *batch, int32_t budget, int32_t first, int32_t recent,
                  const float *weights, float *weights_out, int32_t *lens_out, int32_t *shifts, int32_t *kept,
                  void *workspace, size_t workspace_bytes, void *stream) {
    Kv8Evict e{};
    CIH_TRY(check_cache(cache, e.c, true));
    if (!batch) return set_error(CIH_ERR_ARG, "null batch");
    cih_kv8_batch b = *batch;
    if (!b.cu_rows) b.cu_rows = b.lens;  // not read
    CIH_TRY(check_batch(&b, e.s, true));
    CIH_TRY(check_budget(budget, first, recent));
    CIH_TRY(check_evict_size(e.c, e.s, budget));
    if (e.s.n_seq == 0) return CIH_OK;
    if (!weights || !lens_out) return set_error(CIH_ERR_ARG, "null %s", weights ? "lens_out" : "weights");
    if (!aligned(weights, 4) || !aligned(weights_out, 4) || !aligned(lens_out, 4) || !aligned(shifts, 4) || !aligned(kept, 4))
        return set_error(CIH_ERR_ARG, "weights, lens_out, shifts and kept must be 4-byte aligned");
    const size_t need = kv8_evict_bytes(e.c, e.s, budget);
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < need)
        return set_error(CIH_ERR_CAPACITY, "the call needs a 16-byte aligned workspace of %zu bytes", need);
    e.budget = budget;
    e.first = first;
    e.recent = recent;
    e.weights = weights;
    e.weights_out = weights_out;
    e.lens_out = lens_out;
    e.shifts = shifts;
    e.kept = kept;
    hipStream_t st = static_cast<hipStream_t>(stream);
    CIH_TRY(check_stream(st));
    const hipError_t rc = launch_kv8_evict(e, workspace, st);
    if (rc != hipSuccess) return set_error(CIH_ERR_HIP, "eviction from the cache failed: %s", hipGetErrorString(rc));
    return CIH_OK;
}

int cih_token_logprobs_workspace(int32_t n_rows, int32_t vocab, int32_t top_k, size_t *bytes) {
    if (!bytes) return set_error(CIH_ERR_ARG, "null bytes");
    if (n_rows < 0 || n_rows > 1 << 30 || vocab < 1 || vocab > 1 << 30)
        return set_error(CIH_ERR_SHAPE, "%d rows of %d logits", n_rows, vocab);
    if (top_k < 0 || top_k > LOGPROBS_MAX_TOP) return set_error(CIH_ERR_SHAPE, "top_k %d outside [0, %d]", top_k, LOGPROBS_MAX_TOP);
    *bytes = token_logprobs_floats(n_rows, vocab, top_k) * sizeof(float);
    return CIH_OK;
}

int cih_token_logprobs(int32_t dtype, const void *logits, int64_t row_stride, int32_t n_rows, int32_t vocab,
                       const int32_t *targets, float *logprob, float *entropy, int32_t top_k, int32_t *top_ids,
                       float *top_logprobs, void *workspace, size_t workspace_bytes, void *stream) {
    size_t need = 0;
    CIH_TRY(check_float(dtype));
    CIH_TRY(cih_token_logprobs_workspace(n_rows, vocab, top_k, &need));
    if (n_rows == 0) return CIH_OK;
    if (!logits || (logprob && !targets) || (top_k > 0 && (!top_ids || !top_logprobs)))
        return set_error(CIH_ERR_ARG, "null argument");
    if (row_stride < vocab && n_rows > 1) return set_error(CIH_ERR_SHAPE, "rows of %d logits, %lld apart", vocab, (long long)row_stride);
    if (!aligned(logits, float_size(dtype)) || !aligned(targets, 4) || !aligned(logprob, 4) || !aligned(entropy, 4) ||
        !aligned(top_ids, 4) || !aligned(top_logprobs, 4))
        return set_error(CIH_ERR_ARG, "an argument is not aligned to its type");
    if (need > 0 && (!workspace || !aligned(workspace, 16) || workspace_bytes < need))
        return set_error(CIH_ERR_CAPACITY, "the call needs a 16-byte aligned workspace of %zu bytes", need);
    hipStream_t st = static_cast<hipStream_t>(stream);
    CIH_TRY(check_stream(st));
    const TokenLogprobs a{dtype, logits, n_rows > 1 ? row_stride : 0, n_rows, vocab, top_k, targets, logprob, entropy, top_ids, top_logprobs};
    const hipError_t e = launch_token_logprobs(a, static_cast<float *>(workspace), workspace_bytes / sizeof(float), st);
    if (e != hipSuccess) return set_error(CIH_ERR_HIP, "token log probabilities failed: %s", hipGetErrorString(e));
    return CIH_OK;
}

int cih_verify_drafts_workspace(int32_t n_seq, int32_t n_drafts, int32_t vocab, size_t *bytes) {
    if (!bytes) return set_error(CIH_ERR_ARG, "null bytes");
    if (n_seq < 0 || n_seq > 1 << 24 || n_drafts < 0 || n_drafts > 1 << 24 || vocab < 1 || vocab > 1 << 30)
        return set_error(CIH_ERR_SHAPE, "%d drafts of %d sequences over %d tokens", n_drafts, n_seq, vocab);
    *bytes = verify_drafts_bytes(n_seq, n_drafts, vocab);
    return CIH_OK;
}

int cih_verify_drafts(int32_t dtype, const void *logits, int64_t row_stride, const void *draft_logits,
                      int64_t draft_stride, int32_t n_seq, int32_t n_drafts, int32_t vocab, const int32_t *cu_drafts,
                      const int32_t *drafts, const float *accept_at, const float *sample_at, float temperature,
                      int32_t *accepted, int32_t *tokens, void *workspace, size_t workspace_bytes, void *stream) {
    size_t need = 0;
    CIH_TRY(check_float(dtype));
    CIH_TRY(cih_verify_drafts_workspace(n_seq, n_drafts, vocab, &need));
    if (!(temperature >= 0.0f) || !std::isfinite(temperature)) return set_error(CIH_ERR_ARG, "the temperature must be finite and not negative");
    if (n_seq == 0) return CIH_OK;
    const bool draws = temperature > 0.0f;
    if (!draws) draft_logits = nullptr;
    if (!logits || !cu_drafts || !accepted || !tokens || (n_drafts > 0 && !drafts) || (draws && !sample_at) ||
        (draws && n_drafts > 0 && !accept_at))
        return set_error(CIH_ERR_ARG, "null argument");
    const int64_t most = (int64_t)1 << 31;
    if ((row_stride < vocab && (int64_t)n_seq + n_drafts > 1) || row_stride > most)
        return set_error(CIH_ERR_SHAPE, "rows of %d logits, %lld apart", vocab, (long long)row_stride);
    if (draft_logits && n_drafts > 0 && ((draft_stride < vocab && n_drafts > 1) || draft_stride > most))
        return set_error(CIH_ERR_SHAPE, "draft rows of %d logits, %lld apart", vocab, (long long)draft_stride);
    if (!aligned(logits, float_size(dtype)) || !aligned(draft_logits, float_size(dtype)) || !aligned(cu_drafts, 4) ||
        !aligned(drafts, 4) || !aligned(accept_at, 4) || !aligned(sample_at, 4) || !aligned(accepted, 4) || !aligned(tokens, 4))
        return set_error(CIH_ERR_ARG, "an argument is not aligned to its type");
    if (need > 0 && (!workspace || !aligned(workspace, 16) || workspace_bytes < need))
        return set_error(CIH_ERR_CAPACITY, "the call needs a 16-byte aligned workspace of %zu bytes", need);
    hipStream_t st = static_cast<hipStream_t>(stream);
    CIH_TRY(check_stream(st));
    const VerifyDrafts v{dtype, logits, draft_logits, row_stride, draft_stride, n_seq, n_drafts, vocab, cu_drafts,
                         drafts, accept_at, sample_at, temperature, accepted, tokens};
    const hipError_t e = launch_verify_drafts(v, workspace, st);
    if (e != hipSuccess) return set_error(CIH_ERR_HIP, "the verification of drafts failed: %s", hipGetErrorString(e));
    return CIH_OK;
}

}  // extern "C"

// Internal launch interface of the 8-bit paged key/value cache and of the
// token log probabilities (not part of the C ABI).
#pragma once
#include <float.h>
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/codon_hip.h"

namespace cih {

constexpr int KV8_PAGE = 64;

// dims of a head as stored: what the matrix instructions' tiles need
__host__ __device__ constexpr int kv8_dims(int head_dim) { return head_dim == 24 ? 32 : head_dim; }

// K codes [page][head][64][dp], V codes [page][head][dp][64]: a lane of an int8
// matrix instruction reads 16 consecutive codes, along the dims for q k and
// along the tokens for p v.
struct Kv8View {
    signed char *k, *v;
    float2 *scales;  // [page][head]: of K, of V
    unsigned long long *bad;
    int n_pages, hk, d, dp;
};

struct Kv8Seqs {
    const int *cu, *lens, *table, *slots;
    int n_seq, n_rows, max_rows, table_rows, table_stride, max_pages;
};

struct RowsView {
    void *p;
    int64_t rs, hs;  // elements between rows, heads
};

// The largest v of the wave's lanes, in all of them, without LDS trips (permlane
// swaps of lane halves, then DPP: lanes ^ 32, 16, 8, 4, 2, 1).
template <int C, int BANK> __device__ __forceinline__ unsigned dpp_bits(unsigned old, unsigned v) {
    return (unsigned)__builtin_amdgcn_update_dpp((int)old, (int)v, C, 0xf, BANK, false);
}
__device__ __forceinline__ unsigned wave_max_bits(unsigned v) {
    unsigned w = v;
    asm volatile("" : "+v"(w));  // a register of its own
    const auto r = __builtin_amdgcn_permlane32_swap(v, w, false, false);
    const unsigned r0 = r[0], r1 = r[1];
    v = r0 > r1 ? r0 : r1;
    w = v;
    asm volatile("" : "+v"(w));
    const auto t = __builtin_amdgcn_permlane16_swap(v, w, false, false);
    const unsigned t0 = t[0], t1 = t[1];
    v = t0 > t1 ? t0 : t1;
    auto up = [&](unsigned o) { v = o > v ? o : v; };
    up(dpp_bits<0x128, 0xf>(v, v));
    up(dpp_bits<0x114, 0xa>(dpp_bits<0x104, 0x5>(v, v), v));
    up(dpp_bits<0x4E, 0xf>(v, v));
    up(dpp_bits<0xB1, 0xf>(v, v));
    return v;
}

// Rotary positions by value in the kernel arguments: turns per position.
struct RopeArg {
    int rot = 0, inter = 0;
    float gain = 1.0f;
    double turns[64] = {};
    const int *shift = nullptr;  // [n_seq]: added to a sequence's positions
};

// r (NULL: no rotary positions) for heads of head_dim as the kernels take it; an error code and message if it is refused.
int kv8_rope(const cih_rope *r, int head_dim, RopeArg &a);

// Workgroups of `threads` that one launch may have: its threads are counted in 32 bits.
inline bool kv8_grid(int64_t blocks, int threads) { return blocks > 0 && blocks <= INT32_MAX && blocks <= (int64_t)UINT32_MAX / threads; }

// A sequence of the batch as the kernels see it.
struct Kv8Seq {
    int r0, n;        // first row, rows
    int start, len;   // position of the first row (may be negative), tokens held (within the table)
    const int *table; // nullptr: no such slot
};
__device__ __forceinline__ Kv8Seq kv8_seq(const Kv8Seqs &s, int i) {
    Kv8Seq q;
    q.r0 = min(max(s.cu[i], 0), s.n_rows);
    q.n = min(min(max(s.cu[i + 1], q.r0), s.n_rows) - q.r0, s.max_rows);
    const int len = max(s.lens[i], 0);
    q.start = len - q.n;
    q.len = (int)min((int64_t)len, (int64_t)s.max_pages * KV8_PAGE);
    const int slot = s.slots ? s.slots[i] : i;
    q.table = slot >= 0 && slot < s.table_rows ? s.table + (int64_t)slot * s.table_stride : nullptr;
    return q;
}
// The page that holds tokens 64 pg ..; -1: none
__device__ __forceinline__ int kv8_page(const Kv8View &c, const Kv8Seq &q, int pg) {
    const int id = q.table ? q.table[pg] : -1;
    return id >= 0 && id < c.n_pages ? id : -1;
}

// The angle's position of token p of sequence i.
__device__ __forceinline__ int rope_position(const RopeArg &r, int i, int p) {
    if (!r.shift) return p;
    const int64_t x = (int64_t)p + r.shift[i];
    return (int)(x < INT32_MIN ? INT32_MIN : x > INT32_MAX - KV8_PAGE ? INT32_MAX - KV8_PAGE : x);
}
// cos and sin (times gain) of position p's angle at pair j.  The angle in
// turns is reduced in 64 bits: at position 1e6 a 32-bit product is off by
// 0.06 radians.
__device__ __forceinline__ void rope_cs(const RopeArg &r, int p, int j, float &c, float &s) {
    const double a = (double)p * r.turns[j];
    const float t = (float)(a - rint(a));
    sincospif(2.0f * t, &s, &c);
    c *= r.gain;
    s *= r.gain;
}

__device__ __forceinline__ int code8(float x, float inv) {
    return (int)fminf(fmaxf(rintf(x * inv), -127.0f), 127.0f) & 0xff;
}
// four codes scaled again
__device__ __forceinline__ unsigned recode4(unsigned w, float ratio) {
    unsigned o = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) o |= (unsigned)code8((float)(signed char)(w >> (8 * e)), ratio) << (8 * e);
    return o;
}

// A page's scales from the largest new |K| and |V| (as bits) and the kept
// tokens' (0 where none are kept): too small to be inverted, they are 0, and so are the codes.
__device__ __forceinline__ float2 kv8_scales(unsigned mk, unsigned mv, float2 old) {
    float2 sc = {__uint_as_float(mk) / 127.0f, __uint_as_float(mv) / 127.0f};
    if (!(sc.x >= FLT_MIN)) sc.x = 0.0f;
    if (!(sc.y >= FLT_MIN)) sc.y = 0.0f;
    return {fmaxf(sc.x, old.x), fmaxf(sc.y, old.y)};
}

// out_h2 (dtype F32 only): out is one matrix of f16-limb rows (x3.h) of hd
// q_heads columns, rs and hs unused.
struct Kv8Attention {
    Kv8View c;
    Kv8Seqs s;
    RowsView q, out;
    int dtype, heads, out_h2;
    float *lse;
    float scale;
    int causal, window, sinks;  // (sinks 0 without a window)
    int q16, out16;  // set by the launch: queries in 16-byte loads, output in stores of 4 dims
};

// A decoder's step (one FP32 row a sequence, no shared heads): append and
// attention in one launch.  The rows are qkv [n_rows][3 d] or, with part, the
// projection's sums over `splits` [splits][n_rows][3 d] plus bias.
struct Kv8Step {
    const float *qkv = nullptr, *part = nullptr, *bias = nullptr;
    int splits = 0;
    RopeArg rope;
};
hipError_t launch_kv8_step(const Kv8Attention &a, const Kv8Step &step, float *ws, size_t ws_floats, hipStream_t st);

hipError_t launch_kv8_append(const Kv8View &c, const Kv8Seqs &s, int dtype, const RowsView &k, const RowsView &v,
                             int heads, const RowsView &q, const RowsView &qo, const RopeArg &rope, hipStream_t st);
hipError_t launch_kv8_read(const Kv8View &c, const Kv8Seqs &s, int dtype, const RowsView &k, const RowsView &v,
                           hipStream_t st);
// ws_floats below kv8_attention_floats(...): the keys are split less
hipError_t launch_kv8_attention(const Kv8Attention &a, float *ws, size_t ws_floats, hipStream_t st);
size_t kv8_attention_floats(const Kv8View &c, const Kv8Seqs &s, int heads);

// The attention weight of each cached token over the rows of `a` (out unused, lse
// read) into weights [page][head][64]: a token before the rows keeps `keep` of what it had.
struct Kv8Weigh {
    Kv8Attention a;
    float keep;
    float *weights;
};
hipError_t launch_kv8_weigh(const Kv8Weigh &w, hipStream_t st);

// Eviction to `budget` tokens a sequence and head: the first `first`, the last
// `recent` and the best of the others by `weights`.
struct Kv8Evict {
    Kv8View c;
    Kv8Seqs s;
    int budget, first, recent;
    const float *weights;
    float *weights_out;
    int *lens_out, *shifts, *kept;  // shifts, kept: may be nullptr
    int room = 0;                   // set by the launch: tokens of the budget that a table has room for
};
bool kv8_evict_fits(const Kv8View &c, const Kv8Seqs &s, int budget);  // whether one launch may have that many workgroups
size_t kv8_evict_bytes(const Kv8View &c, const Kv8Seqs &s, int budget);
hipError_t launch_kv8_evict(const Kv8Evict &e, void *ws, hipStream_t st);

constexpr int LOGPROBS_MAX_TOP = 64;
struct TokenLogprobs {
    int dtype;
    const void *logits;
    int64_t stride;
    int n, vocab, top;
    const int *targets;
    float *logprob, *entropy;
    int *top_ids;
    float *top_lp;
};
size_t token_logprobs_floats(int n, int vocab, int top);
hipError_t launch_token_logprobs(const TokenLogprobs &a, float *ws, size_t ws_floats, hipStream_t st);

// Verification of drafted tokens: sequence i has drafts [cu[i], cu[i + 1]) and the
// target's rows from cu[i] + i on, one more.
struct VerifyDrafts {
    int dtype;
    const void *logits, *draft;  // draft nullptr: the drafted token is certain
    int64_t stride, draft_stride;
    int n_seq, n_drafts, vocab;
    const int *cu, *drafted;
    const float *accept_at, *sample_at;
    float temperature;
    int *accepted, *tokens;
};
size_t verify_drafts_bytes(int n_seq, int n_drafts, int vocab);
hipError_t launch_verify_drafts(const VerifyDrafts &v, void *ws, hipStream_t st);

// Element types of the row tensors.
enum { FT_F32 = 0, FT_F16 = 1, FT_BF16 = 2 };
template <class T> __device__ __forceinline__ float to_f32(T x) { return (float)x; }

}  // namespace cih

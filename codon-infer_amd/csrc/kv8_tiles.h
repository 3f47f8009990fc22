// Pieces of the kernels that read the 8-bit cache with matrix instructions: what a
// column of a tile sees, pages in registers, queries as bytes, scores.
#pragma once
#include <float.h>

#include "kernels.h"
#include "kv8.h"

namespace cih {

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

// max / sum over lanes l, l ^ 16, l ^ 32, l ^ 48 (the swaps exchange lane
// halves between two registers: w is v in a register of its own)
template <class OP> __device__ __forceinline__ float groups(float v, OP op) {
    float w = v;
    asm volatile("" : "+v"(w));
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(w), false, false);
    const unsigned r0 = r[0], r1 = r[1];
    v = op(__uint_as_float(r0), __uint_as_float(r1));
    w = v;
    asm volatile("" : "+v"(w));
    const auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(w), false, false);
    const unsigned t0 = t[0], t1 = t[1];
    return op(__uint_as_float(t0), __uint_as_float(t1));
}
__device__ __forceinline__ float groups_max(float v) {
    return groups(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float groups_sum(float v) {
    return groups(v, [](float a, float b) { return a + b; });
}

// What a column sees, and where it is.
struct Column {
    int row, head;   // row of the row tensors (-1: no such column)
    int begin, end;  // keys [begin, end)
};
__device__ __forceinline__ Column column(const Kv8Attention &a, const Kv8Seq &q, int kvh, int g, int f) {
    Column c;
    const int r = f / g;
    c.row = r < q.n ? q.r0 + r : -1;
    c.head = kvh * g + (f - r * g);
    const int pos = q.start + r;
    c.end = a.causal ? min(q.len, pos + 1) : q.len;
    c.begin = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    if (pos < 0 || c.row < 0) c.end = 0;
    if (c.begin > c.end) c.begin = c.end;
    return c;
}

// A value that all lanes read at the same address and nothing writes meanwhile: by a scalar load.
template <class V> __device__ __forceinline__ V uniform(const V *p) {
    return *(const __attribute__((address_space(4))) V *)(unsigned long long)p;
}
// A page's address, the same in all lanes, in scalar registers.
typedef const __attribute__((address_space(1))) signed char *page_ptr;
__device__ __forceinline__ page_ptr scalar_address(const signed char *p) {
    const unsigned long long u = (unsigned long long)p;
    const unsigned lo = __builtin_amdgcn_readfirstlane((int)u), hi = __builtin_amdgcn_readfirstlane((int)(u >> 32));
    return (page_ptr)((unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ i32x4 load16(page_ptr p) { return *(const __attribute__((address_space(1))) i32x4 *)p; }
__device__ __forceinline__ int page_id(const Kv8View &c, const Kv8Seq &q, int pg) {
    const int id = q.table ? uniform(q.table + pg) : -1;
    return __builtin_amdgcn_readfirstlane(id >= 0 && id < c.n_pages ? id : -1);
}

// The pages that columns with keys [begin, end) and the first `sinks` see, counted without
// those between the sinks and the window: page v of them is page at(v) of the sequence.  (The kernels' loops then
// run over one range, split as any: 64 rows behind a window of 4,096 of up to 16,384 tokens and 4 sinks, 32 heads over
// 8 of 128, read 538 MB in 113 us, 4.8 TB/s.)
struct SeenPages {
    int sink, skip, n;
    __device__ __forceinline__ SeenPages(int begin, int end, int sinks) {
        const int pg0 = begin / KV8_PAGE;
        sink = (min(sinks, end) + KV8_PAGE - 1) / KV8_PAGE;
        skip = max(pg0 - sink, 0);
        n = (end + KV8_PAGE - 1) / KV8_PAGE - skip;
    }
    __device__ __forceinline__ int at(int v) const { return v < sink ? v : v + skip; }
};

// Which of the 16 keys j0 .. are visible, as bits.
__device__ __forceinline__ unsigned visible16(int begin, int end, int j0) {
    const int lo = min(max(begin - j0, 0), 16), hi = min(max(end - j0, 0), 16);
    return ((1u << hi) - 1) & ~((1u << lo) - 1);
}

// A page of one head in registers: the A operands of both products.
template <int DP> struct Tile {
    static constexpr int KS = DP > 64 ? DP / 64 : 1;  // k steps of q k
    i32x4 k[4][KS], v[DP / 16];
    float sk, sv;
    unsigned long long bad;
};
// First of the 16 dims a lane reads of a key; dims past a narrow head's meet zeros of the query.
template <int DP> __device__ __forceinline__ int k_dim(int g4) { return (DP >= 64 ? g4 : g4 % (DP / 16)) * 16; }
template <int DP>
__device__ __forceinline__ void load_k(Tile<DP> &t, const Kv8View &c, int id, int kvh, int lane) {
    const int64_t ph = (int64_t)max(id, 0) * c.hk + kvh;
    const page_ptr k = scalar_address(c.k + ph * (KV8_PAGE * DP));
    const int i = lane & 15, g4 = lane >> 4;
    // the page's address in scalar registers, the lane's offset in one vector register
    const unsigned koff = ((i >> 2) * 16 + (i & 3)) * DP + k_dim<DP>(g4);
#pragma unroll
    for (int s = 0; s < Tile<DP>::KS; s++)
#pragma unroll
        for (int kt = 0; kt < 4; kt++) t.k[kt][s] = load16(k + koff + (kt * 4 * DP + s * 64));
    t.sk = uniform(&c.scales[ph].x);
    t.sv = uniform(&c.scales[ph].y);
    t.bad = uniform(c.bad + ph);
}
template <int DP>
__device__ __forceinline__ void load_v(Tile<DP> &t, const Kv8View &c, int id, int kvh, int lane) {
    const int64_t ph = (int64_t)max(id, 0) * c.hk + kvh;
    const page_ptr v = scalar_address(c.v + ph * (KV8_PAGE * DP));
    const unsigned voff = (lane & 15) * KV8_PAGE + (lane >> 4) * 16;
#pragma unroll
    for (int dt = 0; dt < DP / 16; dt++) t.v[dt] = load16(v + voff + dt * 16 * KV8_PAGE);
}

// A column's query, the 16 values of a lane of each k step.
template <int KS, class T>
__device__ __forceinline__ void load_query(const Kv8Attention &a, const Column &col, int g4, float (&x)[KS][16]) {
    constexpr int VL = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(VL)));
    const T *qp = static_cast<const T *>(a.q.p) + (col.row >= 0 ? col.row * a.q.rs + col.head * a.q.hs : 0);
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
        for (int e = 0; e < 16; e += VL) {  // a head has whole groups of VL dims
            const int i = s * 64 + g4 * 16 + e;
            const T *p = qp + (i < a.c.d ? i : 0);
            T w[VL];
            if (a.q16) {
                const vec y = *reinterpret_cast<const vec *>(p);
#pragma unroll
                for (int u = 0; u < VL; u++) w[u] = y[u];
            } else {
#pragma unroll
                for (int u = 0; u < VL; u++) w[u] = p[u];
            }
#pragma unroll
            for (int u = 0; u < VL; u++) {
                x[s][e + u] = col.row >= 0 && i < a.c.d ? to_f32(w[u]) : 0.0f;
            }
        }
}

// A column's query as QB bytes a value, ready as the second operand, and the
// factor that makes scores in units of log2 of its sums with a page's codes
// (times the K scale); NaN if the query is not finite.
template <int QB, int KS>
__device__ __forceinline__ float query_bytes(const float (&x)[KS][16], float scale, i32x4 (&ql)[QB][KS]) {
    constexpr int BITS = 8 * QB - 1, HALF = QB == 3 ? 0x8080 : 0x80;  // the lower bytes are + 128 at first
    constexpr float MOST = (1 << BITS) - 1 - HALF;
    unsigned top = 0;
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
        for (int e = 0; e < 16; e++) top = max(top, __float_as_uint(x[s][e]) & 0x7fffffffu);  // NaN above infinity above the rest
    float mx = __uint_as_float(top);
    const bool lost = groups_max(mx <= FLT_MAX ? 0.0f : 1.0f) > 0.0f;
    mx = groups_max(mx);
    int e = BITS - __builtin_amdgcn_frexp_expf(mx);
    if (ldexpf(mx, e) > MOST) e--;
    // a negative scale turns the query, so that the factor is never negative
    const float sign = lost ? 0.0f : scale < 0.0f ? -1.0f : 1.0f;
#pragma unroll
    for (int s = 0; s < KS; s++)
#pragma unroll
        for (int w = 0; w < 4; w++) {
            unsigned o[QB] = {};
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int v = (int)rintf(ldexpf(lost ? 0.0f : x[s][4 * w + u] * sign, e)) + HALF;
#pragma unroll
                for (int n = 0; n < QB; n++) o[n] |= (unsigned)(v >> (8 * (QB - 1 - n)) & 255) << (8 * u);
            }
#pragma unroll
            for (int n = 0; n < QB; n++) ql[n][s][w] = (int)(n == 0 ? o[n] : o[n] ^ 0x80808080u);
        }
    return lost ? NAN : ldexpf(fabsf(scale) * LOG2E, (QB == 3 ? 8 : 0) - e);
}

// Scores of 16 keys with one column, in the units of the last byte but (three bytes) one.
template <int QB, int KS>
__device__ __forceinline__ void score_tile(const i32x4 (&k)[KS], const i32x4 (&ql)[QB][KS], float (&s)[4]) {
    i32x4 d = {0, 0, 0, 0}, h = {0, 0, 0, 0};
    if (QB == 3) {
#pragma unroll
        for (int x = 0; x < KS; x++) d = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[x], ql[QB - 1][x], d, 0, 0, 0);
        d >>= 8;
    }
#pragma unroll
    for (int x = 0; x < KS; x++) h = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[x], ql[0][x], h, 0, 0, 0);
#pragma unroll
    for (int x = 0; x < KS; x++) d = __builtin_amdgcn_mfma_i32_16x16x64_i8(k[x], ql[1][x], d, 0, 0, 0);
#pragma unroll
    for (int r = 0; r < 4; r++) s[r] = (float)(h[r] * 256 + d[r]);  // below 2^30
}

}  // namespace

}  // namespace cih

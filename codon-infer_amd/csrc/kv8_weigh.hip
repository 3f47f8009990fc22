// The attention weight that cached tokens gather:
//   w_j <- keep w_j + sum over rows r that see j, heads h of the group: exp(scale q_rh k_j - lse_rh)
// with lse as the attention of the same rows gave it, so that the weights need no
// second pass over the keys.  A wave owns a page of one head: its 64 sums have one
// owner and a fixed order.
#include <stdlib.h>
#include <string.h>

#include <type_traits>

#include "kv8_tiles.h"
#include "x3.h"

namespace cih {

namespace {

// Sum over the 16 lanes of a row of lanes, value i of them to lane i: halves of the values are
// exchanged with lanes ^ 8, 4, 2, 1.
__device__ __forceinline__ float lanes_reduce(float (&x)[16], int c) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float keep = c & 8 ? x[i + 8] : x[i], give = c & 8 ? x[i] : x[i + 8];
        x[i] = keep + dpp_or<0x128, 0xf>(give, give);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float keep = c & 4 ? x[i + 4] : x[i], give = c & 4 ? x[i] : x[i + 4];
        x[i] = keep + dpp_or<0x114, 0xa>(dpp_or<0x104, 0x5>(give, give), give);
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const float keep = c & 2 ? x[i + 2] : x[i], give = c & 2 ? x[i] : x[i + 2];
        x[i] = keep + dpp_or<0x4E, 0xf>(give, give);
    }
    const float keep = c & 1 ? x[1] : x[0], give = c & 1 ? x[0] : x[1];
    return keep + dpp_or<0xB1, 0xf>(give, give);
}

// Rows [r0, r1) of a sequence that see any of keys [j0, j0 + keys).
struct SeenBy {
    int r0, r1;
    __device__ __forceinline__ SeenBy(const Kv8Attention &a, const Kv8Seq &q, int j0, int keys) {
        r0 = max(0, (a.causal ? max(j0, 0) : 0) - q.start);
        r1 = q.n;
        if (a.window > 0 && j0 >= a.sinks)
            r1 = (int)min((int64_t)q.n, max((int64_t)0, (int64_t)j0 + keys - 1 + a.window - q.start));
    }
};

// What a page's tokens gained, token `lane` of it in each lane.
__device__ __forceinline__ void gain(const Kv8Weigh &w, const Kv8Seq &q, int id, int kvh, int pg, int lane, float x) {
    const int j = pg * KV8_PAGE + lane;
    if (id < 0 || j >= q.len) return;
    float *p = w.weights + ((int64_t)id * w.a.c.hk + kvh) * KV8_PAGE + lane;
    if (w.keep != 0.0f && j < q.start) x = fmaf(w.keep, *p, x);
    *p = x;
}

constexpr int WEIGH_WAVES = 4;

// At most 16 columns: one workgroup per (sequence, kv head, pps pages), its waves take the pages
// in turn, the next page's keys under way; the query is an integer in three bytes, as in attention.  Bound by
// the bytes of K: 64 rows of 1,025 to 8,190 tokens, 8 heads of 128, 321 MB in 69 us, 4.6 TB/s.
// All pages of the sequence are read, also those that a window hides from every row.
template <int DP, class T>
__global__ __launch_bounds__(64 * WEIGH_WAVES) void k_kv8_weigh(Kv8Weigh w, int g, int pps) {
    constexpr int KS = Tile<DP>::KS;
    const Kv8Attention &a = w.a;
    // the same pages of all (sequence, kv head) pairs after each other: blocks go to the XCDs in turn, and
    // where a pair's own followed each other the XCDs of the last pages had none of the shorter sequences'
    // (64 sequences of 1025 to 8190 tokens 99 -> 74 us)
    const int pairs = a.c.hk * a.s.n_seq, group = blockIdx.x / pairs, pair = blockIdx.x % pairs;
    const int kvh = pair % a.c.hk;
    const Kv8Seq q = kv8_seq(a.s, pair / a.c.hk);
    if (q.n == 0) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g4 = lane >> 4;
    const int last = min((q.len + KV8_PAGE - 1) / KV8_PAGE, (group + 1) * pps);
    int pg = group * pps + wave;
    if (pg >= last) return;
    struct {
        i32x4 k[4][KS];
        float sk;
    } t;
    auto load = [&](int id) __attribute__((always_inline)) {
        const int64_t ph = (int64_t)max(id, 0) * a.c.hk + kvh;
        const page_ptr k = scalar_address(a.c.k + ph * (KV8_PAGE * DP));
        const unsigned koff = ((c >> 2) * 16 + (c & 3)) * DP + k_dim<DP>(g4);
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int kt = 0; kt < 4; kt++) t.k[kt][s] = load16(k + koff + (kt * 4 * DP + s * 64));
        t.sk = uniform(&a.c.scales[ph].x);
    };
    auto id_of = [&](int p) __attribute__((always_inline)) { return p < last ? page_id(a.c, q, p) : -1; };
    int id = id_of(pg), next = id_of(pg + WEIGH_WAVES);
    load(id);
    Column col = column(a, q, kvh, g, c);
    const float lse = col.row >= 0 ? a.lse[(int64_t)col.row * a.heads + col.head] : INFINITY;
    const bool fine = fabsf(lse) <= FLT_MAX;
    if (!fine) col.row = -1;  // its query is taken as zeros
    float x[KS][16];
    load_query<KS, T>(a, col, g4, x);
    i32x4 ql[3][KS];
    float f = query_bytes<3, KS>(x, a.scale, ql), off = lse * LOG2E;
    if (!fine || !(f <= FLT_MAX)) {
        f = 0.0f;
        off = INFINITY;
    }
    for (; pg < last; pg += WEIGH_WAVES) {
        const int j0 = pg * KV8_PAGE;
        float s[4][4];
#pragma unroll
        for (int kt = 0; kt < 4; kt++) score_tile<3, KS>(t.k[kt], ql, s[kt]);
        const float sk = t.sk, fk = fminf(f * sk, FLT_MAX);
        const int now = id;
        id = next;
        if (pg + WEIGH_WAVES < last) load(id);
        next = id_of(pg + 2 * WEIGH_WAVES);
        float sum[16] = {};
        if (now >= 0 && sk >= 0.0f && sk <= FLT_MAX) {
            unsigned see = visible16(col.begin, col.end, j0 + g4 * 16);
            if (a.sinks > 0) see |= visible16(0, min(a.sinks, col.end), j0 + g4 * 16);
#pragma unroll
            for (int u = 0; u < 16; u++) {
                const float e = __builtin_amdgcn_exp2f(fmaf(s[u / 4][u % 4], fk, -off));
                sum[u] = see >> u & 1 ? e : 0.0f;
            }
        }
        gain(w, q, now, kvh, pg, lane, lanes_reduce(sum, c));
    }
}

// Many columns.  The wave's page becomes f16 (bfloat16 rows: bfloat16) once, which holds the codes as
// they are, and stays in registers; the queries go by in LDS, 128 columns at a time for the eight waves, as they
// are (FP32 rows: two f16, hi + lo, under a power of two of the column's own).  sp pages a workgroup: with less than
// eight, the waves of a page share the columns among them.  Bound by issue: a weight costs a multiply-add, an exponential
// (four issue slots) and a sum, 55% of the clocks, the products 30%, and the two take turns: 2,047 rows of 16,000 tokens,
// 32 heads over 8 of 128, 324 us, 775 TFLOP/s (FP32 rows, two products a score, 474).  (One wave that reads its queries itself 588; exponentials
// between the next tile's products by hand 337.)
template <class T> struct Half {
    typedef _Float16 one;
    typedef _Float16 type __attribute__((ext_vector_type(8)));
    static constexpr int LIMBS = std::is_same<T, float>::value ? 2 : 1;
    static __device__ __forceinline__ type codes(int lo, int hi) { return quants_f16<1>(qu32x2_t{(unsigned)lo, (unsigned)hi}, 0); }
    static __device__ __forceinline__ f32x4 mfma(type a, type b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Half<__bf16> {
    typedef __bf16 one;
    typedef __bf16 type __attribute__((ext_vector_type(8)));
    static constexpr int LIMBS = 1;
    static __device__ __forceinline__ type codes(int lo, int hi) {
        type o;
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] = (__bf16)(float)(signed char)((e < 4 ? lo : hi) >> (8 * (e & 3)));
        return o;
    }
    static __device__ __forceinline__ f32x4 mfma(type a, type b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

// f / g by a product: m = ceil(2^(31 + l) / g) with g <= 2^l is exact for f < 2^31.
struct RowOf {
    unsigned m, shift;
    explicit RowOf(int g) {
        int l = 0;
        while ((1ll << l) < g) l++;
        m = (unsigned)(((1ull << (31 + l)) + g - 1) / g);
        shift = 31 + l;
    }
    __device__ __forceinline__ int row(int f) const { return (int)((unsigned long long)(unsigned)f * m >> shift); }
};

constexpr int MANY_WAVES = 8, MANY = 64 * MANY_WAVES, TILES = 8, COLS = 16 * TILES;  // of a turn
template <int DP, class T>
__global__ __launch_bounds__(MANY, 2) void k_kv8_weigh_prompt(Kv8Weigh w, int g, int sp, RowOf of) {
    typedef Half<T> H;
    typedef typename H::type half8;
    constexpr int KS = DP >= 64 ? DP / 32 : 1, L = H::LIMBS, PIECES = DP / 8;
    constexpr int IT = (COLS * PIECES + MANY - 1) / MANY;  // pieces of 8 dims a thread stages
    constexpr bool FULL = std::is_same<T, float>::value;
    const Kv8Attention &a = w.a;
    __shared__ half8 sq[2][L][TILES][KS][64];
    __shared__ float2 scol[2][COLS];  // of a column: lse in units of log2 (infinite: it adds nothing), the scores' factor
    __shared__ float red[MANY_WAVES][64];
    const int pairs = a.c.hk * a.s.n_seq, pair = blockIdx.x % pairs, group = blockIdx.x / pairs;
    const int kvh = pair % a.c.hk, tid = threadIdx.x;
    const Kv8Seq q = kv8_seq(a.s, pair / a.c.hk);
    const int np = (q.len + KV8_PAGE - 1) / KV8_PAGE;
    if (q.n == 0 || group * sp >= np) return;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, g4 = lane >> 4;
    const int pg = group * sp + wave % sp, id = pg < np ? page_id(a.c, q, pg) : -1;
    const int j0 = pg * KV8_PAGE;
    // the page's codes; of 16 and 32 dims a lane takes the 8 of its load that are its own
    half8 k[4][KS];
    float sk = 0.0f;
    {
        Tile<DP> t;
        load_k(t, a.c, id, kvh, lane);
        if (id >= 0) sk = t.sk;
#pragma unroll
        for (int kt = 0; kt < 4; kt++)
#pragma unroll
            for (int s = 0; s < KS; s++) {
                const i32x4 x = t.k[kt][s / 2];
                const bool up = DP >= 64 ? s & 1 : DP == 32 ? g4 >> 1 : g4 & 1;
                k[kt][s] = H::codes(up ? x[2] : x[0], up ? x[3] : x[1]);
            }
    }
    const bool there = id >= 0 && sk >= 0.0f && sk <= FLT_MAX;
    // columns that see any of the workgroup's keys, in turns
    const SeenBy by(a, q, group * sp * KV8_PAGE, sp * KV8_PAGE);
    const int c0 = (int64_t)by.r0 * g / COLS, c1 = by.r0 < by.r1 ? (int)(((int64_t)by.r1 * g + COLS - 1) / COLS) : c0;
    if (DP == 16)  // lanes whose dims there are none of
        for (int e = tid; e < 2 * L * TILES * 64; e += MANY)
            if (e % 64 >= 32) (&sq[0][0][0][0][0])[e] = half8{};

    // Pieces of the thread: 8 dims of a column, whose row and head follow from turn to turn without a
    // division.  Columns that are not there have a neighbour's query.
    constexpr int VL = 16 / sizeof(T), N = 8 / VL;
    typedef T vec __attribute__((ext_vector_type(VL)));
    vec held[IT][N];
    float held_lse = INFINITY;
    int row[IT], head[IT], lse_row = 0, lse_head = 0;  // (row of the sequence)
    const T *piece[IT];
#pragma unroll
    for (int it = 0; it < IT; it++) {
        const int e = tid + it * MANY, p = e % PIECES, f = c0 * COLS + e / PIECES;
        row[it] = of.row(f);
        head[it] = f - row[it] * g;
        piece[it] = static_cast<const T *>(a.q.p) + q.r0 * a.q.rs + kvh * g * a.q.hs + (p * 8 < a.c.d ? p * 8 : 0);
    }
    if (tid < COLS) {
        lse_row = of.row(c0 * COLS + tid);
        lse_head = c0 * COLS + tid - lse_row * g;
    }
    const int step_row = of.row(COLS), step_head = COLS - step_row * g;
    auto follow = [&](int &r, int &h) __attribute__((always_inline)) {
        const bool over = h + step_head >= g;
        r += step_row + (over ? 1 : 0);
        h += step_head - (over ? g : 0);
    };
    auto load = [&]() __attribute__((always_inline)) {  // and on to the next turn
#pragma unroll
        for (int it = 0; it < IT; it++) {
            const T *x = piece[it] + min(row[it], q.n - 1) * a.q.rs + head[it] * a.q.hs;
            if (a.q16) {
#pragma unroll
                for (int u = 0; u < N; u++) held[it][u] = *reinterpret_cast<const vec *>(x + u * VL);
            } else {
#pragma unroll
                for (int u = 0; u < 8; u++) held[it][u / VL][u % VL] = x[u];
            }
            if (DP == 32 && (tid + it * MANY) % PIECES * 8 >= a.c.d)
#pragma unroll
                for (int u = 0; u < N; u++) held[it][u] = vec{};
            follow(row[it], head[it]);
        }
        if (tid < COLS) {
            held_lse = lse_row < q.n && q.start + lse_row >= 0
                           ? a.lse[(int64_t)(q.r0 + lse_row) * a.heads + kvh * g + lse_head] : INFINITY;
            follow(lse_row, lse_head);
        }
    };
    // Powers of two of a column: FP32 rows as large as f16 takes; others only where their sums of
    // products (127 128 times as large) could leave FP32, or all of them are among the smallest numbers.  The
    // column's values are 0 where one is not finite.
    auto store = [&](int at) __attribute__((always_inline)) {
        constexpr bool F16 = std::is_same<T, _Float16>::value;
        constexpr unsigned MOST = FULL ? 0 : F16 ? 0x7c00u - 1 : 0x7800u, LEAST = F16 ? 0x0400u : 0x2000u;  // 2^113; 2^-14, 2^-63
#pragma unroll
        for (int it = 0; it < IT; it++) {
            const int e = tid + it * MANY, p = e % PIECES, col = e / PIECES;
            if (COLS * PIECES % MANY != 0 && col >= COLS) continue;  // (whole waves)
            // which k step and lanes have dims p * 8 ..; columns turned by p, so that the stores of a column meet no bank twice
            const int s = DP >= 64 ? p / 8 * 2 + (p & 1) : 0;
            const int gg = DP >= 64 ? p % 8 / 2 : DP == 32 ? (p & 1) * 2 + (p >> 1) : p;
            half8 *to = &sq[at][0][col / 16][s][gg * 16 + ((col ^ p) & 15)];
            float fac = a.scale * LOG2E;
            unsigned top = 0;
            if constexpr (!FULL) {
                typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
                const i32x4 bits = __builtin_bit_cast(i32x4, held[it][0]) & 0x7fff7fff;
                const u16x2 m = __builtin_elementwise_max(
                    __builtin_elementwise_max(__builtin_bit_cast(u16x2, (int)bits[0]), __builtin_bit_cast(u16x2, (int)bits[1])),
                    __builtin_elementwise_max(__builtin_bit_cast(u16x2, (int)bits[2]), __builtin_bit_cast(u16x2, (int)bits[3])));
                top = max((unsigned)m.x, (unsigned)m.y);
                *to = __builtin_bit_cast(half8, held[it][0]);
            }
            if (FULL || __ballot(top > MOST || (top > 0 && top < LEAST))) {
                float x[8], m = 0.0f;
                unsigned mb = 0;
#pragma unroll
                for (int u = 0; u < 8; u++) {
                    x[u] = to_f32(held[it][u / VL][u % VL]);
                    mb = max(mb, __float_as_uint(x[u]) & 0x7fffffffu);
                }
#pragma unroll
                for (int o = 1; o < PIECES; o <<= 1) mb = max(mb, (unsigned)__shfl_xor((int)mb, o));
                m = __uint_as_float(mb);
                int up = 0;
                if (FULL) up = 14 - __builtin_amdgcn_frexp_expf(m);
                else if (F16 && m < 0x1p-14f) up = -__builtin_amdgcn_frexp_expf(m);
                else if (!F16 && (m > 0x1p113f || m < 0x1p-63f)) up = (m > 1.0f ? 113 : 0) - __builtin_amdgcn_frexp_expf(m);
                const bool lost = !(m <= FLT_MAX);
                if (lost || m == 0.0f) up = 0;
                half8 hi, lo;
#pragma unroll
                for (int u = 0; u < 8; u++) {
                    x[u] = lost ? 0.0f : ldexpf(x[u], up);
                    hi[u] = (typename H::one)x[u];
                    lo[u] = (typename H::one)(x[u] - (float)hi[u]);
                }
                *to = hi;
                if (L == 2) *(to + (&sq[0][L - 1][0][0][0] - &sq[0][0][0][0][0])) = lo;
                fac = lost ? NAN : ldexpf(fac, -up);
            }
            if (p == 0) scol[at][col].y = fac;
        }
        if (tid < COLS) scol[at][tid].x = fabsf(held_lse) <= FLT_MAX ? held_lse * LOG2E : INFINITY;
    };
    float sum[16] = {};
    auto turn_of = [&](int turn, int at) __attribute__((always_inline)) {
        for (int tile = wave / sp; tile < TILES; tile += MANY_WAVES / sp) {
            // positions of the tile's first and last column
            const int f = turn * COLS + tile * 16, p0 = q.start + of.row(f), p1 = q.start + of.row(f + 15);
            const bool sink = j0 < a.sinks;
            if (f >= q.n * g || (a.causal && j0 > p1) || (a.window > 0 && !sink && (int64_t)p0 - a.window >= j0 + KV8_PAGE - 1)) continue;
            f32x4 s[4];
#pragma unroll
            for (int kt = 0; kt < 4; kt++) s[kt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int l = 0; l < L; l++)
#pragma unroll
                for (int u = 0; u < KS; u++) {
                    // the piece that lies there
                    const int p = DP >= 64 ? u / 2 * 8 + g4 * 2 + (u & 1) : DP == 32 ? (g4 & 1) * 2 + (g4 >> 1) : g4 & 1;
                    const half8 x = sq[at][l][tile][u][g4 * 16 + ((c ^ p) & 15)];
#pragma unroll
                    for (int kt = 0; kt < 4; kt++) s[kt] = H::mfma(k[kt][u], x, s[kt]);
                }
            const float2 of_col = scol[at][tile * 16 + c];
            float fk = of_col.y * sk, off = of_col.x;
            fk = fminf(fmaxf(fk, -FLT_MAX), FLT_MAX);
            if (of_col.y != of_col.y) off = INFINITY;  // a query that is not finite
            if (fk == 0.0f) fk = 0x1p-149f;            // so that what is hidden stays at -inf
            const bool all = (!a.causal || j0 + KV8_PAGE - 1 <= p0) &&
                             (a.window == 0 || j0 > (int64_t)p1 - a.window || j0 + KV8_PAGE <= a.sinks);
            if (!all) {
                const Column col = column(a, q, kvh, g, f + c);
                unsigned see = visible16(col.begin, col.end, j0 + g4 * 16);
                if (a.sinks > 0) see |= visible16(0, min(a.sinks, col.end), j0 + g4 * 16);
                const float never = fk > 0.0f ? -INFINITY : INFINITY;
#pragma unroll
                for (int u = 0; u < 16; u++) s[u / 4][u % 4] = see >> u & 1 ? s[u / 4][u % 4] : never;
            }
#pragma unroll
            for (int u = 0; u < 16; u++) sum[u] += __builtin_amdgcn_exp2f(fmaf(s[u / 4][u % 4], fk, -off));
        }
    };
    if (c0 < c1) {
        load();
        store(0);
        __syncthreads();
        for (int turn = c0; turn < c1; turn++) {
            const int at = (turn - c0) & 1;
            if (turn + 1 < c1) load();
            if (there) turn_of(turn, at);
            if (turn + 1 < c1) store(at ^ 1);
            __syncthreads();
        }
    }
    float x = lanes_reduce(sum, c);
    if (sp < MANY_WAVES) {
        red[wave][lane] = x;
        __syncthreads();
        if (wave >= sp) return;
        for (int v = wave + sp; v < MANY_WAVES; v += sp) x += red[v][lane];
    }
    if (pg < np) gain(w, q, id, kvh, pg, lane, x);
}

template <int DP, class T> hipError_t launch(const Kv8Weigh &w, hipStream_t st) {
    const int64_t pairs = (int64_t)w.a.s.n_seq * w.a.c.hk, mp = w.a.s.max_pages;
    const int g = w.a.heads / w.a.c.hk;
    const char *e = getenv("CIH_KV8_WEIGH");
    const bool many = (int64_t)w.a.s.max_rows * g > 16;
    if (many || (e && !strcmp(e, "1"))) {
        int sp = MANY_WAVES;
        while (sp > 1 && pairs * ((mp + sp - 1) / sp) < 256) sp /= 2;
        const int64_t blocks = pairs * ((mp + sp - 1) / sp);
        if (!kv8_grid(blocks, MANY)) return hipErrorInvalidValue;
        hipLaunchKernelGGL((k_kv8_weigh_prompt<DP, T>), dim3(blocks), dim3(MANY), 0, st, w, g, sp, RowOf(g));
    } else {
        // a page a wave at least (8 single tokens of 700, 20 heads of 64: 6.2 us, four pages 7.0)
        const int pps = (int)max((int64_t)4, min(mp * pairs / 2048, (int64_t)64)), groups = (int)((mp + pps - 1) / pps);
        if (!kv8_grid(pairs * groups, 64 * WEIGH_WAVES)) return hipErrorInvalidValue;
        hipLaunchKernelGGL((k_kv8_weigh<DP, T>), dim3(pairs * groups), dim3(64 * WEIGH_WAVES), 0, st, w, g, pps);
    }
    return hipGetLastError();
}

template <class T> hipError_t launch_dims(const Kv8Weigh &w, hipStream_t st) {
    switch (w.a.c.dp) {
        case 16: return launch<16, T>(w, st);
        case 32: return launch<32, T>(w, st);
        case 64: return launch<64, T>(w, st);
        case 128: return launch<128, T>(w, st);
    }
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_kv8_weigh(const Kv8Weigh &call, hipStream_t st) {
    if (call.a.s.n_rows == 0 || call.a.s.n_seq == 0 || call.a.s.max_rows == 0) return hipSuccess;
    Kv8Weigh w = call;
    const RowsView &q = w.a.q;
    const int64_t size = w.a.dtype == FT_F32 ? 4 : 2;
    w.a.q16 = (reinterpret_cast<uintptr_t>(q.p) | (uintptr_t)(q.rs * size) | (uintptr_t)(q.hs * size)) % 16 == 0;
    switch (w.a.dtype) {
        case FT_F32: return launch_dims<float>(w, st);
        case FT_F16: return launch_dims<_Float16>(w, st);
        case FT_BF16: return launch_dims<__bf16>(w, st);
    }
    return hipErrorInvalidValue;
}

}  // namespace cih

// Attention over the 8-bit paged key/value cache.
//
// q k runs on the int8 matrix instruction (16 x 16 x 64), which takes K's codes
// as they lie in the cache.  The query is an integer in signed bytes, q = 2^-e
// (256^2 q0 + 256 q1 + q2), so that the sums over the dims are exact and only
// the query rounds, to 2^-23 of its largest value; the sum with q2, without its
// last 8 bits, starts the one with q1, which leaves 2^-22 of an ordinary score.
// For 16-bit rows of prompts without sinks two bytes do: the scale is a power of 2, so that
// what is not below 2^-7 (float16: 2^-4) of the largest value is exact.  With sinks they have three
// as well: two left lse off by 10^-5 to 10^-4 for normal queries and by 10^-2 where one value is 100 times the
// others (2047 rows of 16000 keys behind a window of 4096, float16 259 -> 279 us, bfloat16 191 -> 214).
//
// Lanes.  S^T = K Q^T: keys are the rows of a tile, the 16 columns are (row, head
// of the group) pairs that share the kv head; row i of key tile t is key (i / 4)
// 16 + 4 t + i % 4 of the page, so a lane's 16 scores are those of 16
// consecutive keys, l / 16 * 16 .., of column l % 16, which is its share of the
// second operand of O^T = V^T P^T, for int8 and for f16: the weights never leave
// their lane.
//
// k_kv8_attend (few columns: single tokens).  Keys are split over waves and
// workgroups.  The weights are bytes as well, three of them, P = 127 256^2 at the
// largest of the page: p v is exact, and each page joins the running output with
// exp(max of the page - running max) times its V scale in FP32.  (Two bytes would do for
// bfloat16 rows, but what they round away shows in float16; the third costs 1% where the codes'
// bytes are the bound.)  Bound by reading the codes once: 64 sequences of 1025 to
// 8190 tokens, 32 heads over 8 of 128, bfloat16, 146 us (4.15 TB/s); one of 65003, 40 heads of
// 64, float16, 70 us (4.75 TB/s, what a copy reaches).  One row of 131 tokens, 20 heads of 16, takes
// 5.2 us, all latency.
//
// k_kv8_prompt (many columns).  V's codes become f16 and the weights f16 (FP32 and
// float16 rows: two f16, hi + lo; one has 11 bits, three more than a bfloat16 row
// keeps); a page's sums join the running output in FP32.  Bound by instruction
// issue, the exponentials and the weights' conversions: 2047 rows of 16000 keys, 32 heads over 8
// of 128, bfloat16, 600 us (837 TFLOP/s), float16 776; 131 to 512 rows of 8
// sequences, 20 heads of 64, FP32, 23 us.
#include <float.h>
#include <stdlib.h>
#include <string.h>

#include <type_traits>

#include "kernels.h"
#include "kv8.h"
#include "kv8_tiles.h"
#include "x3.h"

namespace cih {

namespace {

// A V scale as mant 2^exponent, the exponent NO_EXP for 0 (a page of zeros): outputs are kept
// in units of 2^unit that follow the pages' exponents, so that no FP32 scale is too
// large or too small for the sums.
constexpr int NO_EXP = -4096;
__device__ __forceinline__ int scale_exp(float s) { return s > 0.0f ? __builtin_amdgcn_frexp_expf(s) : NO_EXP; }

// Four dims i .. of one row (i % 4 == 0).
template <class T>
__device__ __forceinline__ void store_out4(const Kv8Attention &a, int row, int head, int i, f32x4 x) {
    typedef T vec __attribute__((ext_vector_type(4)));
    if (std::is_same<T, float>::value && a.out_h2) {
        h2_store4(static_cast<unsigned short *>(a.out.p), row, head * a.c.d + i, a.heads * a.c.d, make_float4(x[0], x[1], x[2], x[3]));
        return;
    }
    T *p = static_cast<T *>(a.out.p) + row * a.out.rs + head * a.out.hs + i;
    if (a.out16) *reinterpret_cast<vec *>(p) = vec{(T)x[0], (T)x[1], (T)x[2], (T)x[3]};
    else
#pragma unroll
        for (int r = 0; r < 4; r++) p[r] = (T)x[r];
}
template <class T>
__device__ __forceinline__ void store_out(const Kv8Attention &a, int row, int head, int i, float x) {
    if (std::is_same<T, float>::value && a.out_h2)
        h2_store(static_cast<unsigned short *>(a.out.p), row, head * a.c.d + i, a.heads * a.c.d, x);
    else
        static_cast<T *>(a.out.p)[row * a.out.rs + head * a.out.hs + i] = (T)x;
}

struct NoStep {};
template <bool STEP> using StepArg = typename std::conditional<STEP, Kv8Step, NoStep>::type;

// A row's query, key and value of one head: rotated, in LDS.
template <int DP, int W>
__device__ __forceinline__ void step_row(const Kv8Attention &a, const Kv8Step &step, int r, int h, int pos, bool kv,
                                         float (&row)[3][DP]) {
    const int hd = a.c.d, d = a.heads * hd, n = a.s.n_rows, pairs = step.rope.rot / 2, t = threadIdx.x;
    float c = 1.0f, s = 0.0f;
    if (t < pairs) rope_cs(step.rope, pos, t, c, s);
    for (int e = t; e < (kv ? 3 : 1) * hd; e += 64 * W) {
        const int which = e / hd, i = e - which * hd, col = which * d + h * hd + i;
        float v = 0.0f;
        if (step.part) {  // (fold_splits, in less code: a launch reads it anew)
            const float *p = step.part + (size_t)r * 3 * d + col;
            const int64_t stride = (int64_t)n * 3 * d;
            for (int s0 = 0; s0 < step.splits; s0 += 8) {
                float x[8];
#pragma unroll
                for (int u = 0; u < 8; u++) x[u] = p[min(s0 + u, step.splits - 1) * stride];
#pragma unroll
                for (int u = 0; u < 8; u++) v += s0 + u < step.splits ? x[u] : 0.0f;
            }
            v += step.bias[col];
        } else {
            v = step.qkv[(size_t)r * 3 * d + col];
        }
        row[which][i] = v;
    }
    __syncthreads();
    if (t < pairs) {
        const int i0 = step.rope.inter ? 2 * t : t, i1 = step.rope.inter ? i0 + 1 : t + pairs;
        const float q0 = row[0][i0], q1 = row[0][i1];
        row[0][i0] = q0 * c - q1 * s;
        row[0][i1] = q1 * c + q0 * s;
        if (kv) {
            const float k0 = row[1][i0], k1 = row[1][i1];
            row[1][i0] = k0 * c - k1 * s;
            row[1][i1] = k1 * c + k0 * s;
        }
    }
    __syncthreads();
}

// What a page's record is after a step's key and value went into it.  patch:
// the kept codes stayed, so that a wave that has the page from before puts
// the new codes in itself (from code[]) and no one waits for the stores.
struct Kv8Own {
    int pg, lo;
    bool patch;
    float2 sc;
    unsigned long long bad;
};
// Token `lo` of a page of one head, from rows in LDS (k_kv8_append's arithmetic); old, was_bad: the page's record.
template <int DP, int W>
__device__ __forceinline__ Kv8Own step_append(const Kv8View &c, int id, int h, int lo, float2 old,
                                              unsigned long long was_bad, const float (&k)[DP], const float (&v)[DP],
                                              unsigned char (&code)[2][DP]) {
    Kv8Own o{-1, lo, true, {0.0f, 0.0f}, 0};
    if (id < 0) return o;
    const int tid = threadIdx.x, lane = tid & 63;
    const int64_t ph = (int64_t)id * c.hk + h;
    if (lo == 0) old = {0.0f, 0.0f};
    unsigned mk = 0, mv = 0;
    for (int i = lane; i < c.d; i += 64) {
        mk = max(mk, __float_as_uint(k[i]) & 0x7fffffffu);
        mv = max(mv, __float_as_uint(v[i]) & 0x7fffffffu);
    }
    mk = wave_max_bits(mk);
    mv = wave_max_bits(mv);
    const bool lost = max(mk, mv) >= 0x7f800000u;
    o.sc = kv8_scales(lost ? 0 : mk, lost ? 0 : mv, old);
    o.bad = (was_bad & ((1ull << lo) - 1)) | (lost ? 1ull << lo : 0);
    const float ik = o.sc.x > 0.0f && !lost ? 1.0f / o.sc.x : 0.0f, iv = o.sc.y > 0.0f && !lost ? 1.0f / o.sc.y : 0.0f;
    signed char *kc = c.k + ph * (KV8_PAGE * DP), *vc = c.v + ph * (KV8_PAGE * DP);
    const float rk = lo > 0 && o.sc.x > 0.0f ? old.x / o.sc.x : lo > 0 ? 0.0f : 1.0f;
    const float rv = lo > 0 && o.sc.y > 0.0f ? old.y / o.sc.y : lo > 0 ? 0.0f : 1.0f;
    o.patch = __builtin_amdgcn_readfirstlane(rk == 1.0f && rv == 1.0f);
    for (int i = tid; i < 2 * DP; i += 64 * W) {
        const int j = i % DP;
        code[i / DP][j] = j < c.d && !lost ? code8(i < DP ? k[j] : v[j], i < DP ? ik : iv) : 0;
    }
    __syncthreads();  // every wave has the old record as well
    if (!o.patch) {  // a scale grew
        if (rk != 1.0f)
            for (int e = tid; e < lo * DP / 4; e += 64 * W) {
                unsigned *w = reinterpret_cast<unsigned *>(kc) + e;
                *w = recode4(*w, rk);
            }
        if (rv != 1.0f) {
            const int words = (lo + 3) / 4;
            for (int e = tid; e < c.d * words; e += 64 * W) {
                unsigned *w = reinterpret_cast<unsigned *>(vc + e / words * KV8_PAGE) + e % words;
                *w = recode4(*w, rv);
            }
        }
        __syncthreads();  // before the new codes, which share words with kept ones
    }
    if (tid == 0) {
        c.scales[ph] = o.sc;
        c.bad[ph] = o.bad;
    }
    for (int i = tid; i < DP; i += 64 * W) kc[lo * DP + i] = code[0][i];
    for (int i = tid; i < c.d; i += 64 * W) vc[i * KV8_PAGE + lo] = code[1][i];
    if (!o.patch) __syncthreads();  // the codes are written
    return o;
}
// The new key's codes in a tile that may not have them, and the new value's.
template <int DP>
__device__ __forceinline__ void patch_k(Tile<DP> &t, int lo, const unsigned char (&code)[DP], int lane) {
    const int c = lane & 15, g4 = lane >> 4;
    const bool mine = c == (lo >> 4) * 4 + (lo & 3);
#pragma unroll
    for (int s = 0; s < Tile<DP>::KS; s++) {
        const i32x4 x = *reinterpret_cast<const i32x4 *>(&code[k_dim<DP>(g4) + s * 64]);
#pragma unroll
        for (int kt = 0; kt < 4; kt++)
            if (kt == (lo >> 2 & 3))
#pragma unroll
                for (int w = 0; w < 4; w++) t.k[kt][s][w] = mine ? x[w] : t.k[kt][s][w];
    }
}
template <int DP>
__device__ __forceinline__ void patch_v(Tile<DP> &t, int lo, const unsigned char (&code)[DP], int lane) {
    const int c = lane & 15, g4 = lane >> 4, at = 8 * (lo & 3);
    const bool mine = g4 == lo >> 4;
#pragma unroll
    for (int dt = 0; dt < DP / 16; dt++) {
        const unsigned x = (unsigned)code[dt * 16 + c] << at;
#pragma unroll
        for (int w = 0; w < 4; w++)
            if (w == (lo >> 2 & 3)) t.v[dt][w] = mine ? (int)((t.v[dt][w] & ~(0xffu << at)) | x) : t.v[dt][w];
    }
}

// One workgroup of W waves per (sequence, kv head, 16 columns, split of the
// pages): with four waves a page's latency (1 us) is paid for four pages at once.  Its waves take the split's pages in turn and join their sums at the
// end.  splits > 1: results of the split's keys alone [row][head][split][DP + 2] in ws
// (output, maximum score, sum of 2^(score - maximum)).
//
// STEP (a decoder's row a sequence, FP32, no shared heads): the rows come as
// Q | K | V, or as the partial sums of their projection; the workgroup rotates its
// head's query, and the one that has the row's own page quantizes its key and value
// into it as k_kv8_append does: while the page's scale stays, the waves patch the
// new codes into the tile that they requested before, else they read the page anew.  The
// page has no other reader in the launch.  650M, one row at position 280: 11.4 us (append
// 2 and the projection's sums 1.5 of it), the attention alone 5.5.
template <int DP, class T, int W, bool STEP, bool SINK>
__global__ __launch_bounds__(64 * W, 2) void k_kv8_attend(Kv8Attention a, int g, int tiles, int splits, int pps,
                                                       float *__restrict__ ws, StepArg<STEP> step) {
    constexpr int KS = Tile<DP>::KS, DT = DP / 16;
    constexpr float P = 127.0f * 65536;
    __shared__ __attribute__((aligned(16))) float so[W][16][DP + 4];
    __shared__ float sml[W][3][16];  // maximum, sum, unit
    int b = blockIdx.x;
    const int split = b % splits;
    b /= splits;
    const int tile = b % tiles;
    b /= tiles;
    const int kvh = b % a.c.hk;
    const Kv8Seq q = kv8_seq(a.s, b / a.c.hk);
    if (tile * 16 >= q.n * g) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g4 = lane >> 4;
    const Column col = column(a, q, kvh, g, tile * 16 + c);
    // keys any column sees, and keys all of them see (rows ascend: the first and last columns that are there)
    const Column c0 = column(a, q, kvh, g, tile * 16), c1 = column(a, q, kvh, g, min(tile * 16 + 15, q.n * g - 1));
    const int any0 = __builtin_amdgcn_readfirstlane(c0.begin), any1 = __builtin_amdgcn_readfirstlane(c1.end);
    const int all0 = __builtin_amdgcn_readfirstlane(c1.begin), all1 = __builtin_amdgcn_readfirstlane(c0.end);
    // SINK: pages are counted without those between the sinks and the window
    const int sinks = SINK ? a.sinks : 0;
    const SeenPages seen(any0, any1, sinks);
    const int base_pg = SINK ? 0 : seen.skip, np = seen.n;
    const int first = base_pg + split * pps, last = base_pg + min(np, (split + 1) * pps);
    if (split > 0 && first >= last) return;  // the join knows
    auto page_of = [&](int pg) __attribute__((always_inline)) { return SINK ? seen.at(pg) : pg; };

    // the split's pages, dealt out to the waves
    auto id_of = [&](int pg) __attribute__((always_inline)) { return pg < last ? page_id(a.c, q, page_of(pg)) : -1; };
    Tile<DP> t;
    int pg = first + wave, id = id_of(pg);
    float x[KS][16];
    Kv8Own own;
    own.pg = -1;
    own.patch = false;
    __shared__ __attribute__((aligned(16))) unsigned char code[2][DP];  // the own token's (STEP)
    if constexpr (STEP) {
        const int pos = q.start, mine = pos / KV8_PAGE;
        const bool writes = mine >= first && mine < last;
        // the pages and the own page's record are on their way meanwhile
        if (pg < last) load_k(t, a.c, id, kvh, lane);
        const int own_id = writes ? page_id(a.c, q, mine) : -1;
        float2 old = {0.0f, 0.0f};
        unsigned long long was_bad = 0;
        if (own_id >= 0) {
            const int64_t ph = (int64_t)own_id * a.c.hk + kvh;
            old = a.c.scales[ph];
            was_bad = a.c.bad[ph];
        }
        __shared__ float row[3][DP];
        step_row<DP, W>(a, step, q.r0, kvh, pos, writes, row);
        if (writes) {
            own = step_append<DP, W>(a.c, own_id, kvh, pos % KV8_PAGE, old, was_bad, row[1], row[2], code);
            own.pg = mine;
        }
        if (pg < last && pg == mine && !own.patch) load_k(t, a.c, id, kvh, lane);
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int i = s * 64 + g4 * 16 + e;
                x[s][e] = c == 0 && i < a.c.d ? row[0][min(i, DP - 1)] : 0.0f;
            }
    } else {
        if (pg < last) load_k(t, a.c, id, kvh, lane);
        load_query<KS, T>(a, col, g4, x);
    }
    i32x4 ql[3][KS];
    const float f = query_bytes<3, KS>(x, a.scale, ql);

    float m = -INFINITY, l = 0.0f;
    int unit = NO_EXP;  // o is in units of 2^m 2^unit: at least what any page can have added, over 127
    float o[DT][4];
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int r = 0; r < 4; r++) o[dt][r] = 0.0f;

    auto page = [&](Tile<DP> &t, int id, int pg, int next) __attribute__((always_inline)) {
        const bool missing = id < 0;
        // scores in units of log2
        float s[4][4];
        const float fk = f * t.sk;
#pragma unroll
        for (int kt = 0; kt < 4; kt++) {
            score_tile<3, KS>(t.k[kt], ql, s[kt]);
#pragma unroll
            for (int r = 0; r < 4; r++) s[kt][r] *= fk;
        }
        float sv = t.sv;
        unsigned long long bad = t.bad;
        if (!(t.sk >= 0.0f && t.sk <= FLT_MAX && sv >= 0.0f && sv <= FLT_MAX)) {
            bad = ~0ull;
            sv = 0.0f;  // columns that do not see the page add nothing
        }
        if (pg + W < last) load_k(t, a.c, next, kvh, lane);
        const int j0 = page_of(pg) * KV8_PAGE;
        if ((j0 < all0 && !(SINK && j0 + KV8_PAGE <= sinks)) || j0 + KV8_PAGE > all1 || bad || missing) {
            unsigned see = missing ? 0 : visible16(col.begin, col.end, j0 + g4 * 16);
            if (SINK && !missing) see |= visible16(0, min(sinks, col.end), j0 + g4 * 16);
            const unsigned lost = (unsigned)(bad >> (g4 * 16)) & 0xffff;
            if (see & lost) l = NAN;
#pragma unroll
            for (int kt = 0; kt < 4; kt++)
#pragma unroll
                for (int r = 0; r < 4; r++) s[kt][r] = (see & ~lost) >> (kt * 4 + r) & 1 ? s[kt][r] : -INFINITY;
        }
        float mp = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < 4; kt++)
#pragma unroll
            for (int r = 0; r < 4; r++) mp = fmaxf(mp, s[kt][r]);
        mp = groups_max(mp);
        if (mp == INFINITY) l = NAN;
        const float base = mp == -INFINITY ? 0.0f : mp;
        // the page's weights as bytes; their sum before that rounding, which lse does not share
        i32x4 pl[3];
        float sum = 0.0f;
#pragma unroll
        for (int kt = 0; kt < 4; kt++) {
            unsigned v[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float e = __builtin_amdgcn_exp2f(s[kt][r] - base);
                v[r] = (unsigned)rintf(e * P);
                sum += e;
                v[r] += 0x8080;
            }
            const unsigned a01 = __builtin_amdgcn_perm(v[1], v[0], 0x05010602u);  // bytes 2 | bytes 1
            const unsigned a23 = __builtin_amdgcn_perm(v[3], v[2], 0x05010602u);
            const unsigned b01 = __builtin_amdgcn_perm(v[1], v[0], 0x0c0c0400u), b23 = __builtin_amdgcn_perm(v[3], v[2], 0x0c0c0400u);
            pl[0][kt] = (int)__builtin_amdgcn_perm(a23, a01, 0x05040100u);
            pl[1][kt] = (int)(__builtin_amdgcn_perm(a23, a01, 0x07060302u) ^ 0x80808080u);
            pl[2][kt] = (int)(__builtin_amdgcn_perm(b23, b01, 0x05040100u) ^ 0x80808080u);
        }
        const float mn = fmaxf(m, base == mp ? mp : m), mb = mn == -INFINITY ? 0.0f : mn;
        const float down = m - mb, below = mp - mb;  // -inf: nothing yet, nothing here
        l = fmaf(l, __builtin_amdgcn_exp2f(down), sum * __builtin_amdgcn_exp2f(below));
        m = mn;
        const int ex = scale_exp(sv), from = unit;
        unit = max(unit + (int)fmaxf(down, (float)NO_EXP), ex + (int)fmaxf(below, (float)NO_EXP));
        const float keep = __builtin_amdgcn_exp2f(down + (float)(from - unit));
        const float av = __builtin_amdgcn_exp2f(below + (float)(ex - unit)) * __builtin_amdgcn_frexp_mantf(sv) * (1.0f / P);
        if (STEP && pg == own.pg && own.patch && !missing) patch_v(t, own.lo, code[1], lane);
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
            i32x4 d[3];
#pragma unroll
            for (int n = 0; n < 3; n++)
                d[n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(t.v[dt], pl[n], i32x4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float hi = (float)(d[0][r] * 256 + d[1][r]);
                o[dt][r] = fmaf(o[dt][r], keep, fmaf(hi, 256.0f, (float)d[2][r]) * av);
            }
        }
    };

    for (; pg < last; pg += W) {
        if (STEP && pg == own.pg) {  // what was just written is not in the scalar cache
            t.sk = own.sc.x;
            t.sv = own.sc.y;
            t.bad = own.bad;
            if (own.patch && id >= 0) patch_k(t, own.lo, code[0], lane);
        }
        load_v(t, a.c, id, kvh, lane);
        const int next = id_of(pg + W);
        page(t, id, pg, next);
        id = next;
    }

    if (f != f && (any1 > any0 || (SINK && any1 > 0))) l = NAN;  // a query that is not finite
    if (col.begin >= col.end && !(SINK && col.end > 0)) l = 0.0f;
    l = groups_sum(l);
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
        *reinterpret_cast<float4 *>(&so[wave][c][dt * 16 + g4 * 4]) = make_float4(o[dt][0], o[dt][1], o[dt][2], o[dt][3]);
    if (g4 == 0) {
        sml[wave][0][c] = m;
        sml[wave][1][c] = l;
        sml[wave][2][c] = (float)unit;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 16 * DP; e += 64 * W) {
        const int cc = e / DP, i = e - cc * DP;
        const Column k = column(a, q, kvh, g, tile * 16 + cc);
        if (k.row < 0) continue;
        float mm = sml[0][0][cc];
#pragma unroll
        for (int w = 1; w < W; w++) mm = fmaxf(mm, sml[w][0][cc]);
        const float base = mm == -INFINITY ? 0.0f : mm;
        float u = 2.0f * NO_EXP;  // whole numbers
#pragma unroll
        for (int w = 0; w < W; w++) u = fmaxf(u, sml[w][2][cc] + truncf(fmaxf(sml[w][0][cc] - base, (float)NO_EXP)));
        float ll = 0.0f, oo = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float down = sml[w][0][cc] - base, x = __builtin_amdgcn_exp2f(down);
            ll += sml[w][1][cc] != sml[w][1][cc] ? NAN : sml[w][1][cc] * x;
            oo = fmaf(so[w][cc][i], __builtin_amdgcn_exp2f(down + (sml[w][2][cc] - u)), oo);
        }
        const float out = ll == 0.0f ? 0.0f : ldexpf(oo / ll, (int)u);
        if (splits > 1) {
            float *p = ws + (((int64_t)k.row * a.heads + k.head) * splits + split) * (DP + 2);
            p[i] = out;
            if (i == 0) {
                p[DP] = mm;
                p[DP + 1] = ll;
            }
            continue;
        }
        if (i < a.c.d) store_out<T>(a, k.row, k.head, i, out);
        if (i == 0 && a.lse) a.lse[(int64_t)k.row * a.heads + k.head] = ll == 0.0f ? -INFINITY : (mm + log2f(ll)) * LN2;
    }
}

// Joins a row's splits: a row of one head by W waves, the splits dealt out to
// them (W = 1: four rows a workgroup).  cols: columns whose pages were split together.
constexpr int JOIN_WAVES = 4;
template <int DP, class T, int W>
__global__ __launch_bounds__(64 * JOIN_WAVES) void k_kv8_join(Kv8Attention a, int g, int cols, int splits, int pps,
                                                              const float *__restrict__ ws) {
    constexpr int DL = DP > 64 ? DP / 64 : 1;  // dims a lane
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned at = W == 1 ? blockIdx.x * JOIN_WAVES + wave : blockIdx.x;  // (below 2^24)
    const unsigned b = at / (unsigned)a.heads;
    const int h = at - b * a.heads, seq = b / (unsigned)a.s.max_rows, r = b - seq * a.s.max_rows;
    if (seq >= a.s.n_seq) return;
    const Kv8Seq q = kv8_seq(a.s, seq);
    if (r >= q.n) return;
    // the splits of its columns that had pages
    const int kvh = h / g, f = r * g + (h - kvh * g), t0 = f / cols * cols;
    const Column c0 = column(a, q, kvh, g, t0), c1 = column(a, q, kvh, g, min(t0 + cols - 1, q.n * g - 1));
    const int np = SeenPages(c0.begin, c1.end, a.sinks).n;
    const int used = min(splits, max(1, (np + pps - 1) / pps));
    const int row = q.r0 + r;
    const float *p = ws + ((int64_t)row * a.heads + h) * splits * (DP + 2);
    float mm = -INFINITY, ll = 0.0f, oo[DL] = {};
    if constexpr (W == 1) {
        // four splits' values at a time, requested together; the maximum moves with them
        for (int s0 = 0; s0 < used; s0 += 4) {
            float m[4], l[4], o[4][DL];
#pragma unroll
            for (int s = 0; s < 4; s++) {
                const float *ps = p + min(s0 + s, used - 1) * (DP + 2);
                const float2 ml = *reinterpret_cast<const float2 *>(ps + DP);
                m[s] = s0 + s < used ? ml.x : -INFINITY;
                l[s] = ml.y;
#pragma unroll
                for (int u = 0; u < DL; u++) o[s][u] = ps[(DP >= 64 ? lane : lane % DP) + 64 * u];
            }
            const float mn = fmaxf(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), mm);
            const float base = mn == -INFINITY ? 0.0f : mn;
            ll *= __builtin_amdgcn_exp2f(mm - base);
            mm = mn;
            float x[4], sum = ll;
#pragma unroll
            for (int s = 0; s < 4; s++) {
                x[s] = s0 + s < used ? l[s] * __builtin_amdgcn_exp2f(m[s] - base) : 0.0f;  // (0 NaN is NaN)
                sum += x[s];
            }
            // oo is the mean so far, so that it is never larger than a value
            const float each = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
            for (int u = 0; u < DL; u++) oo[u] *= ll * each;
            ll = sum;
#pragma unroll
            for (int s = 0; s < 4; s++)
#pragma unroll
                for (int u = 0; u < DL; u++) oo[u] = s0 + s < used ? fmaf(o[s][u], x[s] * each, oo[u]) : oo[u];
        }
    } else {
        for (int s = lane; s < used; s += 64) mm = fmaxf(mm, p[s * (DP + 2) + DP]);
#pragma unroll
        for (int x = 32; x > 0; x >>= 1) mm = fmaxf(mm, __shfl_xor(mm, x));
        const float base = mm == -INFINITY ? 0.0f : mm;
        for (int s = lane; s < used; s += 64) ll += p[s * (DP + 2) + DP + 1] * __builtin_amdgcn_exp2f(p[s * (DP + 2) + DP] - base);
        ll = wave_butterfly(ll);
        const float each = ll == 0.0f ? 0.0f : 1.0f / ll;
#pragma unroll 4
        for (int s = wave; s < used; s += W) {
            const float *ps = p + s * (DP + 2);
            const float x = ps[DP + 1] * __builtin_amdgcn_exp2f(ps[DP] - base) * each;
#pragma unroll
            for (int u = 0; u < DL; u++)
                if (DP >= 64 || lane < DP) oo[u] = fmaf(ps[lane + 64 * u], x, oo[u]);
        }
        __shared__ float so[W][DP];
#pragma unroll
        for (int u = 0; u < DL; u++)
            if (DP >= 64 || lane < DP) so[wave][lane + 64 * u] = oo[u];
        __syncthreads();
        if (wave > 0) return;  // (behind the last barrier)
#pragma unroll
        for (int u = 0; u < DL; u++) {
            oo[u] = 0.0f;
            if (DP >= 64 || lane < DP)
#pragma unroll
                for (int w = 0; w < W; w++) oo[u] += so[w][lane + 64 * u];
        }
    }
#pragma unroll
    for (int u = 0; u < DL; u++)
        if (lane + 64 * u < a.c.d) store_out<T>(a, row, h, lane + 64 * u, oo[u]);
    if (a.lse && lane == 0) a.lse[(int64_t)row * a.heads + h] = ll == 0.0f ? -INFINITY : (mm + log2f(ll)) * LN2;
}

// Four waves of CT x 16 columns each, over the pages of a split that these see,
// with PL f16 a weight.  A column's weights are 2^8 at its reference w, a score, and its
// output is in units of 2^w 2^unit.  w moves when a score exceeds it by 2^5, or when all of a page
// that the column sees is more than 2^NEAR below it; unit (an exponent) when a page's V
// scale is not within 2^2 of it: f16 weights have room for that, and what rounds to 0 among
// them is below 2^(NEAR - 30) of the largest of its page (FP32 rows: 2^-26).  Both go down
// as well as up, as far as what the column already holds leaves room in
// FP32, so many small weights behind a large one keep their bits, V scales of the whole range of
// FP32 go together, and a column is not touched by a page that it does not see.
//
// SHARE (heads of 128): a page's V becomes f16 once for the four waves, in LDS, a
// page ahead.  Its conversion was a third of the instructions (2047 rows of 16000
// keys 656 -> 570 us); at narrower heads, with fewer columns and less to convert, the waves' waiting for each
// other costs as much (20 heads of 64: 2 x 512 rows 13.0, shared 14.8).
template <int DP, int QB, int PL, class T, int CT, bool SINK>
__global__ __launch_bounds__(256, 2) void k_kv8_prompt(Kv8Attention a, int g, int tiles, int splits, int pps,
                                                       float *__restrict__ ws) {
    constexpr int KS = Tile<DP>::KS, DT = DP / 16;
    constexpr bool SHARE = DP == 128;
    constexpr float SLACK = 5.0f, P0 = 8.0f, NEAR = PL == 2 ? 4.0f : 8.0f;
    constexpr int UNIT = 2;
    constexpr float ROOM = 60.0f;  // of a column's sums above 2^w (2^w 2^unit): what adds less than 2^-60 of them may be lost
    // The last rows, which see most keys, go first, over all (sequence, kv head)
    // pairs (a pair after the other left the longest to a quarter of the CUs:
    // prompts of 131 to 512 rows 28.4 -> 25.4 us; whole pairs to one XCD: no difference).
    const int split = blockIdx.x % splits, task = blockIdx.x / splits;
    const int pairs = a.c.hk * a.s.n_seq, pair = task % pairs, tile = tiles - 1 - task / pairs;
    const int kvh = pair % a.c.hk;
    const Kv8Seq q = kv8_seq(a.s, pair / a.c.hk);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g4 = lane >> 4;
    // columns of the workgroup, and the pages of the split that they see
    const int w0 = tile * 4 * CT * 16, w1 = min(w0 + 4 * CT * 16, q.n * g) - 1;
    if (w0 > w1) return;
    // SINK: pages are counted without those between the sinks and the window
    const int sinks = SINK ? a.sinks : 0;
    SeenPages seen(column(a, q, kvh, g, w0).begin, column(a, q, kvh, g, w1).end, sinks);
    seen.sink = __builtin_amdgcn_readfirstlane(seen.sink);
    seen.skip = __builtin_amdgcn_readfirstlane(seen.skip);
    const int base_pg = SINK ? 0 : seen.skip;
    int first = __builtin_amdgcn_readfirstlane(base_pg + split * pps);
    int last = __builtin_amdgcn_readfirstlane(base_pg + min(seen.n, (split + 1) * pps));
    if (split > 0 && first >= last) return;  // the join knows
    auto page_of = [&](int pg) __attribute__((always_inline)) { return SINK ? seen.at(pg) : pg; };
    // columns of the wave (none: it only helps with V)
    const int f0 = w0 + wave * CT * 16, f1 = min(f0 + CT * 16, q.n * g) - 1;
    const Column c0 = column(a, q, kvh, g, f0), c1 = column(a, q, kvh, g, max(f0, f1));
    const int any0 = __builtin_amdgcn_readfirstlane(c0.begin), any1 = __builtin_amdgcn_readfirstlane(f0 <= f1 ? c1.end : 0);
    const int all0 = __builtin_amdgcn_readfirstlane(c1.begin), all1 = __builtin_amdgcn_readfirstlane(c0.end);
    if (!SHARE) {  // the wave's own pages
        if (f0 > f1) return;
        if (!SINK) first = max(first, any0 / KV8_PAGE);
        last = min(last, (any1 + KV8_PAGE - 1) / KV8_PAGE - (SINK ? seen.skip : 0));
    }

    i32x4 ql[CT][QB][KS];
    float f[CT], w[CT], l[CT];
    float top[CT], most[CT];  // the largest score, the largest score + exponent of its page's V scale
    int begin[CT], end[CT], unit[CT];
    f32x4 o[CT][DT];
#pragma unroll
    for (int t = 0; t < CT; t++) {
        const Column col = column(a, q, kvh, g, f0 + t * 16 + c);
        float x[KS][16];
        load_query<KS, T>(a, col, g4, x);
        f[t] = query_bytes<QB, KS>(x, a.scale, ql[t]);
        begin[t] = col.begin;
        end[t] = col.end;
        w[t] = -FLT_MAX;  // below every score
        top[t] = most[t] = -INFINITY;
        unit[t] = 0;
        l[t] = f[t] != f[t] ? NAN : 0.0f;  // a query that is not finite
#pragma unroll
        for (int dt = 0; dt < DT; dt++) o[t][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    // SHARE: V's codes as f16, the operands of the page and of the next one; a wave converts a quarter
    constexpr int VN = SHARE ? DT / 4 : DT;  // of the wave's loads of V
    __shared__ f16x8 vs[SHARE ? 2 : 1][SHARE ? DT : 1][2][64];
    const int dt0 = SHARE ? wave * VN : 0;
    i32x4 kr[4][KS], vn[VN];
    float sk = 0.0f, sv = 0.0f, skn = 0.0f, svn = 0.0f;
    unsigned long long bad = 0, badn = 0;
    // the lane's offsets in a page: with the page's address in scalar registers a load takes one vector register
    const unsigned koff = ((c >> 2) * 16 + (c & 3)) * DP + k_dim<DP>(g4), voff = c * KV8_PAGE + g4 * 16;
    auto load_k = [&](int id) __attribute__((always_inline)) {
        const int64_t ph = (int64_t)max(id, 0) * a.c.hk + kvh;
        const page_ptr k = scalar_address(a.c.k + ph * (KV8_PAGE * DP));
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int kt = 0; kt < 4; kt++)
                kr[kt][s] = load16(k + koff + (kt * 4 * DP + s * 64));
        skn = uniform(&a.c.scales[ph].x);
        svn = uniform(&a.c.scales[ph].y);
        badn = uniform(a.c.bad + ph);
    };
    auto load_v = [&](int id) __attribute__((always_inline)) {
        const page_ptr v = scalar_address(a.c.v + ((int64_t)max(id, 0) * a.c.hk + kvh) * (KV8_PAGE * DP));
#pragma unroll
        for (int n = 0; n < VN; n++) vn[n] = load16(v + voff + (dt0 + n) * 16 * KV8_PAGE);
    };
    auto operand = [&](int n, int h) __attribute__((always_inline)) {
        return quants_f16<1>(qu32x2_t{(unsigned)vn[n][2 * h], (unsigned)vn[n][2 * h + 1]}, 0);
    };
    auto convert_v = [&](int at) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < VN; n++)
#pragma unroll
            for (int h = 0; h < 2; h++) vs[at][dt0 + n][h][lane] = operand(n, h);
    };
    // of a ballot, which columns: column c is lanes c, c + 16, c + 32, c + 48
    auto lanes = [](unsigned long long b) __attribute__((always_inline)) {
        b |= b >> 32;
        return (unsigned)(b | b >> 16) & 0xffff;
    };
    // LDS only: loads of K and V stay under way
    auto barrier = [&]() __attribute__((always_inline)) { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    // ids of the page and the next one, and the table's entry of the one after that
    auto entry = [&](int pg) __attribute__((always_inline)) { return q.table && pg < last ? uniform(q.table + page_of(pg)) : -1; };
    auto valid = [&](int e) __attribute__((always_inline)) {
        return __builtin_amdgcn_readfirstlane(e >= 0 && e < a.c.n_pages ? e : -1);
    };
    int id = valid(entry(first)), next = valid(entry(first + 1)), e2 = entry(first + 2);
    if (first < last) {
        load_k(id);
        if (SHARE) {
            load_v(id);
            convert_v(0);
            if (first + 1 < last) load_v(next);
        }
    }
    if (SHARE) barrier();
    for (int pg = first; pg < last; pg++) {
        const int at = SHARE ? (pg - first) & 1 : 0;
        sk = skn;
        sv = svn;
        bad = badn;
        const bool missing = id < 0;
        const int j0 = page_of(pg) * KV8_PAGE, next2 = valid(e2);
        if (!SHARE) {
            load_v(id);
        } else if (pg + 1 < last) {
            convert_v(at ^ 1);
            if (pg + 2 < last) load_v(next2);
        }
        e2 = entry(pg + 3);
        if (!SHARE || ((j0 + KV8_PAGE > any0 || (SINK && j0 < sinks)) && j0 < any1)) {
        float s[CT][4][4];
#pragma unroll
        for (int t = 0; t < CT; t++)
#pragma unroll
            for (int kt = 0; kt < 4; kt++) score_tile<QB, KS>(kr[kt], ql[t], s[t][kt]);
        if (pg + 1 < last) load_k(next);
        if (!(sk >= 0.0f && sk <= FLT_MAX && sv >= 0.0f && sv <= FLT_MAX)) {
            bad = ~0ull;
            sk = sv = 0.0f;  // columns that do not see the page add nothing
        }
        if ((j0 < all0 && !(SINK && j0 + KV8_PAGE <= sinks)) || j0 + KV8_PAGE > all1 || bad || missing) {  // hidden keys
#pragma unroll
            for (int t = 0; t < CT; t++) {
                unsigned see = missing ? 0 : visible16(begin[t], end[t], j0 + g4 * 16);
                if (SINK && !missing) see |= visible16(0, min(sinks, end[t]), j0 + g4 * 16);
                const unsigned lost = (unsigned)(bad >> (g4 * 16)) & 0xffff;
                l[t] = see & lost ? NAN : l[t];
                see &= ~lost;
#pragma unroll
                for (int kt = 0; kt < 4; kt++)
#pragma unroll
                    for (int r = 0; r < 4; r++) s[t][kt][r] = see >> (kt * 4 + r) & 1 ? s[t][kt][r] : -INFINITY;
            }
        }
        float fk[CT], x[CT];
        const int ex = scale_exp(sv);
        unsigned over = 0, near[CT], all = 0xffff;  // columns above their reference, and those that the reference suits
#pragma unroll
        for (int t = 0; t < CT; t++) {
            fk[t] = fmaxf(f[t] * sk, 0x1p-120f);  // above 0: what is hidden stays at -inf
            x[t] = -INFINITY;
#pragma unroll
            for (int kt = 0; kt < 4; kt++)
#pragma unroll
                for (int r = 0; r < 4; r++) x[t] = fmaxf(x[t], s[t][kt][r]);
            x[t] *= fk[t];
            over |= lanes(__ballot(x[t] > w[t] + SLACK));
            near[t] = lanes(__ballot(x[t] >= w[t] - NEAR && abs(ex - unit[t]) <= UNIT));
            all &= near[t];
        }
        unsigned move = over;
        if (all != 0xffff)  // (columns that see nothing of the page need no other)
#pragma unroll
            for (int t = 0; t < CT; t++) move |= lanes(__ballot(x[t] > -INFINITY)) & ~near[t];
        if (move) {
#pragma unroll
            for (int t = 0; t < CT; t++) {
                const float mp = ceilf(groups_max(x[t]));  // whole: sums are scaled by powers of two
                top[t] = fmaxf(top[t], mp);
                most[t] = fmaxf(most[t], mp + (float)ex);
                float wn = mp > w[t] + SLACK || mp <= w[t] - NEAR ? mp : w[t];
                wn = fmaxf(wn, top[t] - ROOM);
                const int un = max(ex, (int)fminf(fmaxf(most[t] - ROOM - wn, (float)NO_EXP), (float)-NO_EXP));
                const bool seen = mp > -INFINITY;
                const float d = seen ? w[t] - wn : 0.0f;
                const float y = __builtin_amdgcn_exp2f(d), z = __builtin_amdgcn_exp2f(d + (float)(seen ? unit[t] - un : 0));
                w[t] = seen ? wn : w[t];
                unit[t] = seen ? un : unit[t];
                l[t] *= y;
#pragma unroll
                for (int dt = 0; dt < DT; dt++) o[t][dt] *= z;
            }
        }
        const float up = P0 + (sv > 0.0f ? __builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(sv)) : 0.0f), down = __builtin_amdgcn_exp2f(-up);
        f16x8 p[CT][PL][2];
#pragma unroll
        for (int t = 0; t < CT; t++) {
            // (an exponent far below the unit: the weights are 0 in f16, their sum in FP32 is not)
            const int rel = min(max(ex - unit[t], -40), UNIT);
            const float off = up + (float)rel - w[t];
            float sum = 0.0f;
#pragma unroll
            for (int kt = 0; kt < 4; kt++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float e = __builtin_amdgcn_exp2f(fmaf(s[t][kt][r], fk[t], off));
                    sum += e;
                    const _Float16 hi = (_Float16)e;
                    p[t][0][kt / 2][kt % 2 * 4 + r] = hi;
                    if (PL == 2) p[t][PL - 1][kt / 2][kt % 2 * 4 + r] = (_Float16)(e - (float)hi);
                }
            l[t] = fmaf(sum, ldexpf(down, -rel), l[t]);
        }
        // The page's sums by themselves, then added: as one chain over 60,000 keys the
        // matrix instructions' roundings grow to 6e-5 of an output of one sign, this way to 1e-6.
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
            const f16x8 v0 = SHARE ? vs[at][SHARE ? dt : 0][0][lane] : operand(SHARE ? 0 : dt, 0);
            const f16x8 v1 = SHARE ? vs[at][SHARE ? dt : 0][1][lane] : operand(SHARE ? 0 : dt, 1);
#pragma unroll
            for (int t = 0; t < CT; t++) {
                f32x4 d = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int n = 0; n < PL; n++) {
                    d = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, p[t][n][0], d, 0, 0, 0);
                    d = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, p[t][n][1], d, 0, 0, 0);
                }
                o[t][dt] += d;
            }
        }
        } else if (pg + 1 < last) {
            load_k(next);
        }
        id = next;
        next = next2;
        if (SHARE && pg + 1 < last) barrier();
    }

#pragma unroll
    for (int t = 0; t < CT; t++) {
        const Column col = column(a, q, kvh, g, f0 + t * 16 + c);
        float sum = groups_sum(l[t]);
        if (begin[t] >= end[t] && !(SINK && end[t] > 0)) sum = 0.0f;
        if (col.row < 0) continue;
        const float x = __builtin_amdgcn_exp2f(-P0) / sum;
        float *p = ws + (((int64_t)col.row * a.heads + col.head) * splits + split) * (DP + 2);
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
            const int i = dt * 16 + g4 * 4;
            f32x4 y;
#pragma unroll
            for (int r = 0; r < 4; r++) y[r] = sum == 0.0f ? 0.0f : ldexpf(o[t][dt][r] * x, unit[t]);
            if (splits > 1) {
                *reinterpret_cast<float2 *>(p + i) = make_float2(y[0], y[1]);
                *reinterpret_cast<float2 *>(p + i + 2) = make_float2(y[2], y[3]);
            } else if (i < a.c.d) {
                store_out4<T>(a, col.row, col.head, i, y);
            }
        }
        if (splits > 1) {
            if (g4 == 0) *reinterpret_cast<float2 *>(p + DP) = make_float2(w[t], sum);
            continue;
        }
        if (g4 == 0 && a.lse)
            a.lse[(int64_t)col.row * a.heads + col.head] = sum == 0.0f ? -INFINITY : (w[t] + log2f(sum)) * LN2;
    }
}

// Columns of a prompt wave, / 16: heads of 128 share a wave's reads of V over 32
// (20 heads, 4096 rows, before the waves shared its conversion: bfloat16 238 -> 147 us, FP32 245 -> 215), narrower
// ones gain more from twice the waves (64 wide: 92 and 96, 20 -> 17; 32 wide 80
// and 79, 17 -> 15).
constexpr int prompt_tiles(int dp) { return dp == 128 ? 2 : 1; }

// Which kernel, and how the pages of a sequence are split.
struct Plan {
    bool prompt;
    int g, tiles, splits, pps;  // tiles of cols columns, a workgroup's
    int cols;
    int64_t blocks;
};
// Prompts: k_kv8_prompt where the columns alone fill the GPU, or are more than
// 64 and the keys long enough to be split (us, FP32 rows, 20 heads of 64, the one
// kernel and the other: 2 sequences of 512 rows 21.5 and 15.1, 256 rows of 4096 keys
// 35.3 and 33.7, but 512 of 1024 19.7 and 23.6, 64 of 1024 10.8 and 22.7).  Its
// pages are split until the workgroups are as many as run at once (two a CU for heads of
// 128, else four), not below 8 pages each (512 rows of 65536 keys, 32 over 8 heads
// of 128: FP32 2861 unsplit, 921; bfloat16 1945, 648), and only from 32 pages on (1000
// rows of 1000 keys, when that was measured: 18.1 unsplit, 29.8; now 23.7 unsplit).
//
// Few columns: splits of 16 to 64 pages, a wave's 4 to 16, so that there are some
// 2048 workgroups; shorter ones cost more in the join than they gain (8 single tokens of 700, 20
// heads of 64: 8.0 us, with 8 pages 12.1), and from 4096 tiles on none is split.
Plan plan(const Kv8View &c, const Kv8Seqs &s, int heads, int causal, int window, int sinks, bool step, size_t ws_floats) {
    Plan p;
    p.g = heads / c.hk;
    const int64_t columns = (int64_t)s.max_rows * p.g, pairs = (int64_t)s.n_seq * c.hk;
    const bool fits = pairs * ((columns + 15) / 16) >= 1024, split = s.max_pages >= 32;
    const char *e = getenv("CIH_KV8_PROMPT");
    p.prompt = step ? false : e ? !strcmp(e, "1") : columns > 16 && (fits || (columns > 64 && split));
    p.cols = p.prompt ? 64 * prompt_tiles(c.dp) : 16;
    p.tiles = (int)((columns + p.cols - 1) / p.cols);
    const int64_t tasks = pairs * p.tiles;
    // pages that the keys of a tile's columns touch at most
    int64_t pages = s.max_pages;
    if (window > 0)
        pages = min(pages, ((int64_t)window + (causal ? p.cols / p.g + 1 : s.max_rows) + KV8_PAGE - 2) / KV8_PAGE + 1 +
                               ((int64_t)sinks + KV8_PAGE - 1) / KV8_PAGE);
    const int64_t most = sinks > 0 ? pages : s.max_pages;
    int64_t pps = most;
    if (p.prompt && split) {
        const int64_t want = max((int64_t)1, (c.dp < 128 ? 1024 : 512) / tasks);
        pps = max((int64_t)8, (most + want - 1) / want);
    } else if (!p.prompt && tasks < 4096) {
        pps = max((int64_t)16, min(most * tasks / 2048, (int64_t)64));
    }
    const size_t each = (size_t)s.n_rows * heads * (c.dp + 2);  // floats of one split of all rows
    if (sinks > 0)  // as few pages a split as the workspace of the whole table allows
        pps = max(pps, (pages + (int64_t)(ws_floats / each) - 1) / max((int64_t)1, (int64_t)(ws_floats / each)));
    for (;; pps *= 2) {
        p.splits = (int)max((int64_t)1, (pages + pps - 1) / pps);
        if (p.splits == 1 || each * p.splits <= ws_floats) break;
    }
    p.pps = (int)(p.splits == 1 ? (int64_t)1 << 24 : pps);
    p.blocks = tasks * p.splits;
    return p;
}

template <int DP, class T>
hipError_t launch(const Kv8Attention &a, const Kv8Step *step, float *ws, size_t ws_floats, hipStream_t st) {
    constexpr bool full = std::is_same<T, float>::value;  // FP32 rows
    constexpr int CT = prompt_tiles(DP);
    const Plan p = plan(a.c, a.s, a.heads, a.causal, a.window, a.sinks, step != nullptr, ws_floats);
    const int64_t rows = (int64_t)a.s.n_seq * a.s.max_rows * a.heads;  // of the join
    if (!kv8_grid(p.blocks, 256) || (p.splits > 1 && !kv8_grid(rows, 64 * JOIN_WAVES))) return hipErrorInvalidValue;
    if constexpr (full)
        if (step)
            hipLaunchKernelGGL((k_kv8_attend<DP, T, 4, true, false>), dim3(p.blocks), dim3(256), 0, st, a, p.g, p.tiles,
                               p.splits, p.pps, ws, *step);
    constexpr int PL = std::is_same<T, __bf16>::value ? 1 : 2;
    auto prompt = [&](auto sink) {
        constexpr int QB = full || decltype(sink)::value ? 3 : 2;
        hipLaunchKernelGGL((k_kv8_prompt<DP, QB, PL, T, CT, decltype(sink)::value>), dim3(p.blocks), dim3(256), 0, st, a, p.g, p.tiles,
                           p.splits, p.pps, ws);
    };
    auto few = [&](auto sink) {
        hipLaunchKernelGGL((k_kv8_attend<DP, T, 4, false, decltype(sink)::value>), dim3(p.blocks), dim3(256), 0, st, a, p.g,
                           p.tiles, p.splits, p.pps, ws, NoStep{});
    };
    if (!step && p.prompt) a.sinks > 0 ? prompt(std::true_type{}) : prompt(std::false_type{});
    else if (!step) a.sinks > 0 ? few(std::true_type{}) : few(std::false_type{});
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    // A wave a row where the rows fill the GPU or the splits are few (20 heads of 64, 1024 rows
    // of 6100 keys: 107 us, by four waves 137), else four (6 rows of 16000 keys, 16 splits: 17.7, by one 18.6).
    if (p.splits <= 8 || rows >= 8192)
        hipLaunchKernelGGL((k_kv8_join<DP, T, 1>), dim3((rows + JOIN_WAVES - 1) / JOIN_WAVES), dim3(64 * JOIN_WAVES), 0, st, a,
                           p.g, p.cols, p.splits, p.pps, ws);
    else
        hipLaunchKernelGGL((k_kv8_join<DP, T, JOIN_WAVES>), dim3(rows), dim3(64 * JOIN_WAVES), 0, st, a, p.g, p.cols,
                           p.splits, p.pps, ws);
    return hipGetLastError();
}

template <class T>
hipError_t launch_dims(const Kv8Attention &a, const Kv8Step *step, float *ws, size_t ws_floats, hipStream_t st) {
    switch (a.c.dp) {
        case 16: return launch<16, T>(a, step, ws, ws_floats, st);
        case 32: return launch<32, T>(a, step, ws, ws_floats, st);
        case 64: return launch<64, T>(a, step, ws, ws_floats, st);
        case 128: return launch<128, T>(a, step, ws, ws_floats, st);
    }
    return hipErrorInvalidValue;
}

}  // namespace

size_t kv8_attention_floats(const Kv8View &c, const Kv8Seqs &s, int heads) {
    if (s.n_rows == 0 || s.n_seq == 0 || s.max_rows == 0) return 0;
    // a window leaves fewer pages at as many pages a split: what is enough without one is enough
    const Plan p = plan(c, s, heads, 1, 0, 0, false, SIZE_MAX);
    return p.splits == 1 ? 0 : (size_t)s.n_rows * heads * p.splits * (c.dp + 2);
}

hipError_t launch_kv8_attention(const Kv8Attention &call, float *ws, size_t ws_floats, hipStream_t st) {
    if (call.s.n_rows == 0 || call.s.n_seq == 0 || call.s.max_rows == 0) return hipSuccess;
    Kv8Attention a = call;
    const int64_t size = a.dtype == FT_F32 ? 4 : 2;
    auto aligned = [&](const RowsView &v, int64_t n) {
        return (reinterpret_cast<uintptr_t>(v.p) | (uintptr_t)(v.rs * size) | (uintptr_t)(v.hs * size)) % n == 0;
    };
    a.q16 = aligned(a.q, 16);
    a.out16 = aligned(a.out, 4 * size);
    switch (a.dtype) {
        case FT_F32: return launch_dims<float>(a, nullptr, ws, ws_floats, st);
        case FT_F16: return launch_dims<_Float16>(a, nullptr, ws, ws_floats, st);
        case FT_BF16: return launch_dims<__bf16>(a, nullptr, ws, ws_floats, st);
    }
    return hipErrorInvalidValue;
}

hipError_t launch_kv8_step(const Kv8Attention &call, const Kv8Step &step, float *ws, size_t ws_floats, hipStream_t st) {
    if (call.s.n_rows == 0 || call.s.n_seq == 0) return hipSuccess;
    if (call.dtype != FT_F32 || call.heads != call.c.hk || call.s.max_rows != 1 || call.s.n_rows != call.s.n_seq ||
        (step.part && (!step.bias || step.splits < 1)) || step.rope.rot > call.c.d)
        return hipErrorInvalidValue;
    Kv8Attention a = call;
    a.q16 = 0;
    a.out16 = 0;
    return launch_dims<float>(a, &step, ws, ws_floats, st);
}

}  // namespace cih

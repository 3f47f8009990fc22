// Attention over the 8-bit paged key/value cache.
//
// Both products run on the int8 matrix instruction (16 x 16 x 64), which takes
// the codes as they lie in the cache: nothing is converted.  The other operand
// is an integer in limbs of 7 bits,
//   q = (max |q| / M) (128^2 q0 + 128 q1 + q2),  M = 126 128^2
//   p = (1 / P) (128^2 p0 + 128 p1 + p2),        P = 127 128^2
// (FP32 rows; 16-bit rows take two limbs, M = 126 128, P = 127 128), so that the
// sums over dims and over a page's tokens are exact and only the limbs round: a
// query to 2^-21 of its largest value, a weight to 2^-21 of the largest of its
// page.  Each page has weights of its own, p = exp(s - max of the page), and joins the
// running output with exp(max of the page - running max) times the page's V
// scale, in FP32.
//
// Lanes.  S^T = K Q^T: keys are the rows of a tile, the 16 columns are (row, head
// of the group) pairs that share the kv head; row i of key tile t is key (i / 4)
// 16 + 4 t + i % 4 of the page, so a lane's 16 scores are those of 16
// consecutive keys, l / 16 * 16 .., of column l % 16: as bytes, just its
// operand of O^T = V^T P^T.  Nothing crosses lanes but the page's maximum.
#include <float.h>

#include <type_traits>

#include "kv8.h"
#include "x3.h"

namespace cih {

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

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

template <class T>
__device__ __forceinline__ void store_out(const Kv8Attention &a, int row, int head, int i, float x) {
    if (std::is_same<T, float>::value && a.out_h2)
        h2_store(static_cast<unsigned short *>(a.out.p), row, head * a.c.d + i, a.heads * a.c.d, x);
    else
        static_cast<T *>(a.out.p)[row * a.out.rs + head * a.out.hs + i] = (T)x;
}

// A page of one head in registers: the A operands of both products.
template <int DP> struct Tile {
    static constexpr int KS = DP > 64 ? DP / 64 : 1;  // k steps of q k
    i32x4 k[4][KS], v[DP / 16];
    float2 sc;
    unsigned long long bad;
};
template <int DP>
__device__ __forceinline__ void load_tile(Tile<DP> &t, const Kv8View &c, int id, int kvh, int lane) {
    const int64_t ph = (int64_t)max(id, 0) * c.hk + kvh;
    const signed char *k = c.k + ph * (KV8_PAGE * DP), *v = c.v + ph * (KV8_PAGE * DP);
    const int i = lane & 15, g4 = lane >> 4;
#pragma unroll
    for (int s = 0; s < Tile<DP>::KS; s++)
#pragma unroll
        for (int kt = 0; kt < 4; kt++) {
            const int key = (i >> 2) * 16 + kt * 4 + (i & 3);
            if (DP >= 64 || g4 < DP / 16) t.k[kt][s] = *reinterpret_cast<const i32x4 *>(k + key * DP + s * 64 + g4 * 16);
            else t.k[kt][s] = i32x4{0, 0, 0, 0};
        }
#pragma unroll
    for (int dt = 0; dt < DP / 16; dt++)
        t.v[dt] = *reinterpret_cast<const i32x4 *>(v + (dt * 16 + i) * KV8_PAGE + g4 * 16);
    t.sc = c.scales[ph];
    t.bad = c.bad[ph];
}

// One workgroup of W waves per (sequence, kv head, 16 columns, split of the
// pages); its waves take the split's pages in turn and join their sums at the
// end.  splits > 1: unnormalised results [row][head][split][DP + 2] in ws.
template <int DP, int NL, class T, int W>
__global__ __launch_bounds__(64 * W) void k_kv8_attend(Kv8Attention a, int g, int tiles, int splits, int pps,
                                                       float *__restrict__ ws) {
    constexpr int KS = Tile<DP>::KS, DT = DP / 16;
    constexpr float M = NL == 3 ? 126.0f * 16384 : 126.0f * 128, P = NL == 3 ? 127.0f * 16384 : 127.0f * 128;
    __shared__ __attribute__((aligned(16))) float so[W][16][DP + 4];
    __shared__ float sml[W][2][16];
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
    const int pg0 = any0 / KV8_PAGE, np = (any1 + KV8_PAGE - 1) / KV8_PAGE - pg0;  // pages
    const int first = pg0 + split * pps, last = pg0 + min(np, (split + 1) * pps);
    if (split > 0 && first >= last) return;  // the join knows

    // the query's limbs, as B operands, and its factor
    i32x4 ql[NL][KS];
    float f;
    {
        float x[KS][16];
        unsigned top = 0;
        const T *qp = static_cast<const T *>(a.q.p) + col.row * a.q.rs + col.head * a.q.hs;
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const int i = s * 64 + g4 * 16 + e;
                x[s][e] = col.row >= 0 && i < a.c.d ? to_f32(qp[i]) : 0.0f;
                top = max(top, __float_as_uint(x[s][e]) & 0x7fffffffu);  // NaN above infinity above the rest
            }
        float mx = __uint_as_float(top);
        const bool lost = groups_max(mx <= FLT_MAX ? 0.0f : 1.0f) > 0.0f;
        mx = groups_max(mx);
        const float up = mx < 0x1p-64f ? 0x1p64f : 1.0f;  // so that the reciprocal is finite
        mx *= up;
        const float inv = lost || mx < 0x1p-60f ? 0.0f : M / mx;
        f = lost ? NAN : mx / M / up * a.scale * LOG2E;
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int w = 0; w < 4; w++) {
                unsigned o[3] = {0, 0, 0};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    int v = lost ? 0 : (int)rintf(x[s][4 * w + e] * up * inv);
#pragma unroll
                    for (int n = NL - 1; n > 0; n--) {
                        const int r = ((v + 64) & 127) - 64;
                        o[n] |= (unsigned)(r & 255) << (8 * e);
                        v = (v - r) >> 7;
                    }
                    o[0] |= (unsigned)(v & 255) << (8 * e);
                }
#pragma unroll
                for (int n = 0; n < NL; n++) ql[n][s][w] = (int)o[n];
            }
    }

    float m = -INFINITY, l = 0.0f;
    float o[DT][4];
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int r = 0; r < 4; r++) o[dt][r] = 0.0f;

    auto page = [&](const Tile<DP> &t, int id, int pg) __attribute__((always_inline)) {
        if (id < 0) return;
        // scores in units of log2
        float s[4][4];
        const float fk = f * t.sc.x;
#pragma unroll
        for (int kt = 0; kt < 4; kt++) {
            i32x4 d[NL];
#pragma unroll
            for (int n = 0; n < NL; n++) {
                d[n] = i32x4{0, 0, 0, 0};
#pragma unroll
                for (int x = 0; x < KS; x++) d[n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(t.k[kt][x], ql[n][x], d[n], 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float hi = (float)(d[0][r] * 128 + d[1][r]);  // below 2^30
                s[kt][r] = (NL == 3 ? fmaf(hi, 128.0f, (float)d[NL - 1][r]) : hi) * fk;
            }
        }
        const int j0 = pg * KV8_PAGE;
        unsigned long long bad = t.bad;
        if (!(t.sc.x <= FLT_MAX && t.sc.y <= FLT_MAX)) bad = ~0ull;
        if (j0 < all0 || j0 + KV8_PAGE > all1 || bad) {
#pragma unroll
            for (int kt = 0; kt < 4; kt++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int k = g4 * 16 + kt * 4 + r, j = j0 + k;
                    const bool see = j >= col.begin && j < col.end, lost = bad >> k & 1;
                    if (see && lost) l = NAN;
                    if (!see || lost) s[kt][r] = -INFINITY;
                }
        }
        float mp = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < 4; kt++)
#pragma unroll
            for (int r = 0; r < 4; r++) mp = fmaxf(mp, s[kt][r]);
        mp = groups_max(mp);
        if (mp == INFINITY) l = NAN;
        const float base = mp == -INFINITY ? 0.0f : mp;
        // the page's weights, as B operands, and their sum (exact)
        i32x4 pl[NL];
        int sum = 0;
#pragma unroll
        for (int kt = 0; kt < 4; kt++) {
            unsigned w[3] = {0, 0, 0};
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const unsigned v = (unsigned)rintf(__builtin_amdgcn_exp2f(s[kt][r] - base) * P);
                sum += v;
                if (NL == 3) {
                    w[0] |= (v >> 14) << (8 * r);
                    w[1] |= (v >> 7 & 127) << (8 * r);
                    w[2] |= (v & 127) << (8 * r);
                } else {
                    w[0] |= (v >> 7) << (8 * r);
                    w[1] |= (v & 127) << (8 * r);
                }
            }
#pragma unroll
            for (int n = 0; n < NL; n++) pl[n][kt] = (int)w[n];
        }
        const float mn = fmaxf(m, base == mp ? mp : m);
        const float keep = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
        const float add = mp == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mp - mn) * (1.0f / P);
        l = fmaf(l, keep, (float)sum * add);
        m = mn;
        const float av = add * t.sc.y;
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
            i32x4 d[NL];
#pragma unroll
            for (int n = 0; n < NL; n++)
                d[n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(t.v[dt], pl[n], i32x4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float hi = (float)(d[0][r] * 128 + d[1][r]);
                o[dt][r] = fmaf(o[dt][r], keep, (NL == 3 ? fmaf(hi, 128.0f, (float)d[NL - 1][r]) : hi) * av);
            }
        }
    };

    // two pages in registers: the next one's loads are under way while one is worked on
    auto id_of = [&](int pg) __attribute__((always_inline)) { return pg < last ? kv8_page(a.c, q, pg) : -1; };
    Tile<DP> ta, tb;
    int pg = first + wave, ia = id_of(pg), ib = id_of(pg + W);
    if (pg < last) load_tile<DP>(ta, a.c, ia, kvh, lane);
    while (pg < last) {
        const int ic = id_of(pg + 2 * W);
        if (pg + W < last) load_tile<DP>(tb, a.c, ib, kvh, lane);
        page(ta, ia, pg);
        pg += W;
        if (pg >= last) break;
        const int id = id_of(pg + 2 * W);
        if (pg + W < last) load_tile<DP>(ta, a.c, ic, kvh, lane);
        page(tb, ib, pg);
        pg += W;
        ia = ic;
        ib = id;
    }

    if (f != f && any1 > any0) l = NAN;  // a query that is not finite
    if (col.begin >= col.end) l = 0.0f;
    l = groups_sum(l);
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
        *reinterpret_cast<float4 *>(&so[wave][c][dt * 16 + g4 * 4]) = make_float4(o[dt][0], o[dt][1], o[dt][2], o[dt][3]);
    if (g4 == 0) {
        sml[wave][0][c] = m;
        sml[wave][1][c] = l;
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
        float ll = 0.0f, oo = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float x = __builtin_amdgcn_exp2f(sml[w][0][cc] - base);
            ll += sml[w][1][cc] != sml[w][1][cc] ? NAN : sml[w][1][cc] * x;
            oo = fmaf(so[w][cc][i], x, oo);
        }
        if (splits > 1) {
            float *p = ws + (((int64_t)k.row * a.heads + k.head) * splits + split) * (DP + 2);
            p[i] = oo;
            if (i == 0) {
                p[DP] = mm;
                p[DP + 1] = ll;
            }
            continue;
        }
        if (i < a.c.d) store_out<T>(a, k.row, k.head, i, ll == 0.0f ? 0.0f : oo / ll);
        if (i == 0 && a.lse) a.lse[(int64_t)k.row * a.heads + k.head] = ll == 0.0f ? -INFINITY : (mm + log2f(ll)) * LN2;
    }
}

// Joins a row's splits: one wave per (row of a sequence, head).
template <int DP, class T>
__global__ __launch_bounds__(64) void k_kv8_join(Kv8Attention a, int g, int splits, int pps,
                                                 const float *__restrict__ ws) {
    const int h = blockIdx.x % a.heads, b = blockIdx.x / a.heads;
    const int r = b % a.s.max_rows, lane = threadIdx.x;
    const Kv8Seq q = kv8_seq(a.s, b / a.s.max_rows);
    if (r >= q.n) return;
    // the splits of its 16 columns that had pages
    const int kvh = h / g, f = r * g + (h - kvh * g), t0 = f / 16 * 16;
    const Column c0 = column(a, q, kvh, g, t0), c1 = column(a, q, kvh, g, min(t0 + 15, q.n * g - 1));
    const int pg0 = c0.begin / KV8_PAGE, np = (c1.end + KV8_PAGE - 1) / KV8_PAGE - pg0;
    const int used = min(splits, max(1, (np + pps - 1) / pps));
    const int row = q.r0 + r;
    const float *p = ws + ((int64_t)row * a.heads + h) * splits * (DP + 2);
    float mm = -INFINITY;
    for (int s = lane; s < used; s += 64) mm = fmaxf(mm, p[s * (DP + 2) + DP]);
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) mm = fmaxf(mm, __shfl_xor(mm, x));
    const float base = mm == -INFINITY ? 0.0f : mm;
    float ll = 0.0f, oo[(DP + 63) / 64] = {};
    for (int s = 0; s < used; s++) {
        const float *ps = p + s * (DP + 2);
        const float x = __builtin_amdgcn_exp2f(ps[DP] - base);
        ll += ps[DP + 1] != ps[DP + 1] ? NAN : ps[DP + 1] * x;
#pragma unroll
        for (int u = 0; u < (DP + 63) / 64; u++)
            if (lane + 64 * u < DP) oo[u] = fmaf(ps[lane + 64 * u], x, oo[u]);
    }
#pragma unroll
    for (int u = 0; u < (DP + 63) / 64; u++)
        if (lane + 64 * u < a.c.d) store_out<T>(a, row, h, lane + 64 * u, ll == 0.0f ? 0.0f : oo[u] / ll);
    if (a.lse && lane == 0) a.lse[(int64_t)row * a.heads + h] = ll == 0.0f ? -INFINITY : (mm + log2f(ll)) * LN2;
}

// Workgroups: how the pages of a sequence are split.
struct Plan {
    int g, tiles, splits, pps;
    int64_t blocks;
};
Plan plan(const Kv8View &c, const Kv8Seqs &s, int heads, int causal, int window) {
    Plan p;
    p.g = heads / c.hk;
    p.tiles = (int)(((int64_t)s.max_rows * p.g + 15) / 16);
    const int64_t tasks = (int64_t)s.n_seq * c.hk * p.tiles;
    int64_t pps = max((int64_t)16, min(s.max_pages * tasks / 2048, (int64_t)64));
    if (tasks >= 4096) pps = s.max_pages;
    // pages that the keys of 16 columns touch at most
    int64_t pages = s.max_pages;
    if (window > 0) pages = min(pages, ((int64_t)window + (causal ? 16 / p.g + 1 : s.max_rows) + KV8_PAGE - 2) / KV8_PAGE + 1);
    p.splits = (int)max((int64_t)1, (pages + pps - 1) / pps);
    p.pps = (int)(p.splits == 1 ? (int64_t)1 << 24 : pps);
    p.blocks = tasks * p.splits;
    return p;
}

template <int DP, class T> hipError_t launch(const Kv8Attention &a, float *ws, hipStream_t st) {
    constexpr int NL = std::is_same<T, float>::value ? 3 : 2;
    const Plan p = plan(a.c, a.s, a.heads, a.causal, a.window);
    if (p.blocks > INT32_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL((k_kv8_attend<DP, NL, T, 4>), dim3(p.blocks), dim3(256), 0, st, a, p.g, p.tiles, p.splits, p.pps, ws);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    const int64_t rows = (int64_t)a.s.n_seq * a.s.max_rows * a.heads;
    if (rows > INT32_MAX) return hipErrorInvalidValue;
    hipLaunchKernelGGL((k_kv8_join<DP, T>), dim3(rows), dim3(64), 0, st, a, p.g, p.splits, p.pps, ws);
    return hipGetLastError();
}

template <class T> hipError_t launch_dims(const Kv8Attention &a, float *ws, hipStream_t st) {
    switch (a.c.dp) {
        case 16: return launch<16, T>(a, ws, st);
        case 32: return launch<32, T>(a, ws, st);
        case 64: return launch<64, T>(a, ws, st);
        case 128: return launch<128, T>(a, ws, st);
    }
    return hipErrorInvalidValue;
}

}  // namespace

size_t kv8_attention_floats(const Kv8View &c, const Kv8Seqs &s, int heads) {
    if (s.n_rows == 0 || s.n_seq == 0 || s.max_rows == 0) return 0;
    // a window leaves fewer pages at as many pages a split: what is enough without one is enough
    const Plan p = plan(c, s, heads, 1, 0);
    return p.splits == 1 ? 0 : (size_t)s.n_rows * heads * p.splits * (c.dp + 2);
}

hipError_t launch_kv8_attention(const Kv8Attention &a, float *ws, hipStream_t st) {
    if (a.s.n_rows == 0 || a.s.n_seq == 0 || a.s.max_rows == 0) return hipSuccess;
    switch (a.dtype) {
        case FT_F32: return launch_dims<float>(a, ws, st);
        case FT_F16: return launch_dims<_Float16>(a, ws, st);
        case FT_BF16: return launch_dims<__bf16>(a, ws, st);
    }
    return hipErrorInvalidValue;
}

}  // namespace cih

// Log probabilities of given tokens, with entropy and the top alternatives.
//
// One pass over a row with the running maximum m: u = (x - m) log2 e, s = sum
// 2^u, t = sum 2^u u; then
//   log p(i) = x_i - m - ln 2 log2 s,  entropy = ln 2 (log2 s - t / s).
// A NaN or +inf anywhere makes s NaN.  Bound by reading the logits once, and close
// to it by the seven operations a logit: 512 rows of 131072 bfloat16 logits 26 us without
// alternatives, 31 with 20 (4.3 TB/s), 40 with 64; 8192 rows of 33, 7.4 us: eight waves a SIMD,
// each with as many steps of the count of better logits as there are logits.
#include <limits.h>

#include <algorithm>

#include "kernels.h"
#include "kv8.h"

namespace cih {

namespace {

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr float U_MIN = -200.0f;  // 2^u is 0 from there on: 0 * u instead of 0 * -inf

// v over the wave, the same in every lane (the steps of wave_butterfly)
template <class OP> __device__ __forceinline__ float wave_all(float v, OP op) {
    float w = v;
    asm volatile("" : "+v"(w));
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(w), false, false);
    const unsigned r0 = r[0], r1 = r[1];
    v = op(__uint_as_float(r0), __uint_as_float(r1));
    w = v;
    asm volatile("" : "+v"(w));
    const auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(w), false, false);
    const unsigned t0 = t[0], t1 = t[1];
    v = op(__uint_as_float(t0), __uint_as_float(t1));
    v = op(v, dpp_or<0x128, 0xf>(v, v));
    v = op(v, dpp_or<0x114, 0xa>(dpp_or<0x104, 0x5>(v, v), v));
    v = op(v, dpp_or<0x4E, 0xf>(v, v));
    v = op(v, dpp_or<0xB1, 0xf>(v, v));
    return v;
}
// the same of integers
template <class OP> __device__ __forceinline__ unsigned wave_bits(unsigned v, OP op) {
    return __builtin_amdgcn_readfirstlane((int)__float_as_uint(wave_all(__uint_as_float(v), [&](float a, float b) {
        return __uint_as_float(op(__float_as_uint(a), __float_as_uint(b)));
    })));
}
__device__ __forceinline__ float wave_max(float v) {
    return wave_all(v, [](float a, float b) { return fmaxf(a, b); });
}

// A logit and its place as one number: larger logits first, then earlier ones.
// -0 counts as 0; 0 is below every logit.
typedef unsigned long long u64;
__device__ __forceinline__ unsigned order32(float x) {
    const unsigned b = __float_as_uint(x + 0.0f);
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float order32_value(unsigned k) { return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k); }
__device__ __forceinline__ u64 place_key(float x, int i) { return (u64)order32(x) << 32 | (0xffffffffu - (unsigned)i); }
__device__ __forceinline__ float key_value(u64 k) { return order32_value((unsigned)(k >> 32)); }
__device__ __forceinline__ int key_index(u64 k) { return (int)(0xffffffffu - (unsigned)k); }

// Running sums of a part of a row: m = max, s = sum 2^u, t = sum 2^u u with u =
// (x - m) log2 e (the difference first: a row may hold the type's lowest value).
struct Sums {
    float m = -INFINITY, s = 0.0f, t = 0.0f;
    __device__ __forceinline__ void rebase(float mn) {
        if (mn > m) {
            const float d = fmaxf((m - mn) * LOG2E, U_MIN), a = __builtin_amdgcn_exp2f(d);
            t = a * fmaf(s, d, t);
            s *= a;  // a NaN stays
            m = mn;
        }
    }
    __device__ __forceinline__ void add(Sums o) {
        o.rebase(m);
        rebase(o.m);
        s += o.s;
        t += o.t;
    }
};
__device__ __forceinline__ Sums wave_sums(Sums v) {
    v.rebase(wave_max(v.m));
    v.s = wave_butterfly(v.s);
    v.t = wave_butterfly(v.t);
    return v;
}

// What the sums of a whole row say.
struct RowStats {
    float m, s, t, ls;
    bool lost, none;
    __device__ __forceinline__ RowStats(const Sums &v) : m(v.m), s(v.s), t(v.t), ls(__builtin_amdgcn_logf(v.s)) {
        lost = s != s || m == INFINITY;
        none = !lost && m == -INFINITY;
    }
    __device__ __forceinline__ float logprob(float x) const {
        return lost ? NAN : none || x == -INFINITY ? -INFINITY : fmaf(-ls, LN2, x - m);
    }
    __device__ __forceinline__ float entropy() const { return lost ? NAN : none ? 0.0f : (ls - t / s) * LN2; }
};
template <class T> __device__ __forceinline__ void store_row(const TokenLogprobs &a, int row, const RowStats &st) {
    if (a.logprob) {
        const int g = a.targets[row];
        const T *x = static_cast<const T *>(a.logits) + row * a.stride;
        a.logprob[row] = g < 0 ? 0.0f : g >= a.vocab ? NAN : st.logprob(to_f32(x[g]));
    }
    if (a.entropy) a.entropy[row] = st.entropy();
}
__device__ __forceinline__ void store_top(const TokenLogprobs &a, int row, int k, float x, int i, const RowStats &st) {
    const bool gone = st.lost || x == -INFINITY;
    a.top_ids[(int64_t)row * a.top + k] = gone ? -1 : i;
    a.top_lp[(int64_t)row * a.top + k] = st.lost ? NAN : st.logprob(x);
}

// At most 64 logits: a wave per row, a lane per logit; an alternative's place
// is the number of better ones.
constexpr int NARROW_ROWS = 4;
template <class T> __global__ __launch_bounds__(64 * NARROW_ROWS) void k_logprobs_narrow(TokenLogprobs a) {
    const int row = blockIdx.x * NARROW_ROWS + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (row >= a.n) return;
    const T *p = static_cast<const T *>(a.logits) + row * a.stride;
    const float x = lane < a.vocab ? to_f32(p[lane]) : -INFINITY;
    Sums v;
    v.m = wave_max(x);
    const float u = (x - (v.m == -INFINITY ? 0.0f : v.m)) * LOG2E, e = __builtin_amdgcn_exp2f(u);
    v.s = wave_butterfly(e);
    v.t = wave_butterfly(e * fmaxf(u, U_MIN));
    const RowStats st(v);
    if (lane == 0) store_row<T>(a, row, st);
    if (a.top == 0) return;
    int rank = 0;
    for (int j = 0; j < a.vocab; j++) {
        const float y = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), j));
        rank += y > x || (y == x && j < lane) ? 1 : 0;
    }
    if (st.lost || lane >= a.vocab) rank = lane;  // every place gets one of the marks
    if (rank < a.top) store_top(a, row, rank, x, lane, st);
}

template <class T> struct Vec {
    static constexpr int N = 16 / sizeof(T);
    // as aligned as its elements: rows of any stride
    typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// Logits of a thread in a tile, in 16-byte loads: 16 leave registers for 16
// waves a CU (512 rows of 131072 bfloat16 logits, with an earlier choice of the alternatives:
// 42.4 us, with 32 logits 43.6, with 8 47.8).
constexpr int LP_EACH = 16;
constexpr int LP_CAP = 768;  // list entries

// A key that between top and top + LP_SLACK of a wave's keys reach (1 where no
// more than that are above 0), bit by bit from the highest in which they differ: a ballot
// for each step and key.  Keys above 0 are distinct.
constexpr int LP_SLACK = 8;
template <int K> __device__ __forceinline__ u64 top_bound(const u64 (&key)[K], int top) {
    auto reach = [&](u64 t) __attribute__((always_inline)) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < K; i++) n += __popcll(__ballot(key[i] >= t));
        return n;
    };
    if (reach(1) <= top + LP_SLACK) return 1;
    u64 any = 0, all = ~0ull;  // of the keys above 0
#pragma unroll
    for (int i = 0; i < K; i++) {
        any |= key[i];
        all &= key[i] ? key[i] : ~0ull;
    }
    unsigned lo[2] = {(unsigned)(any >> 32), (unsigned)any}, hi[2] = {(unsigned)(all >> 32), (unsigned)all};
    u64 t = 0;
    int b = -1;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const unsigned o = wave_bits(lo[h], [](unsigned x, unsigned y) { return x | y; });
        const unsigned a = wave_bits(hi[h], [](unsigned x, unsigned y) { return x & y; });
        if (b < 0) {
            t |= (u64)(o & a) << (32 - 32 * h);
            if (o != a) {
                b = 63 - 32 * h - __builtin_clz(o ^ a);
                t &= ~0ull << b << 1;  // (b may be 63)
            }
        }
    }
    for (; b >= 0; b--) {
        const u64 up = t | 1ull << b;
        const int n = reach(up);
        if (n >= top) {
            t = up;
            if (n <= top + LP_SLACK) break;
        }
    }
    return t;
}

// The row (or the chunk blockIdx % chunks of its tiles) by NT threads.
//
// Alternatives.  In the pass a thread keeps only its largest logit and the
// 16-byte vector it came from.  Vectors are numbered in the logits' order, so
// (logit, vector) orders the threads' bests as the logits are ordered: what top_k
// of them reach, `least`, the row's top_k reach as well, and they all are among the vectors of the
// threads that reach it.  Those threads' vectors (some top_k / NT of the row, in L2 by then) are
// read again, and what reaches `least` goes to a list, about top_k logits.
template <class T, int NT>
__global__ __launch_bounds__(NT) void k_logprobs(TokenLogprobs a, int chunks, int tiles_per, float *__restrict__ ws) {
    constexpr int VL = Vec<T>::N, LP_VECS = LP_EACH / VL, TILE = NT * LP_EACH, NW = NT / 64;
    static_assert(64 * VL + LOGPROBS_MAX_TOP <= LP_CAP && NW * LOGPROBS_MAX_TOP <= LP_CAP, "the list holds a wave's vectors");
    __shared__ u64 list[LP_CAP], best[LOGPROBS_MAX_TOP];
    __shared__ int ranks[LP_CAP], owner[LOGPROBS_MAX_TOP + LP_SLACK], iw[NW], s_cnt, s_owners;
    __shared__ u64 s_least;
    __shared__ float sw[NW][3];
    const int row = blockIdx.x / chunks, chunk = blockIdx.x - row * chunks;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T *p = static_cast<const T *>(a.logits) + row * a.stride;
    const int top = a.top;
    const int begin = (int)((int64_t)chunk * tiles_per * TILE);
    const int end = (int)min((int64_t)a.vocab, (int64_t)begin + (int64_t)tiles_per * TILE);
    Sums v;
    float most = -INFINITY;
    int from = 0;  // its vector's number / NT

    auto add = [&](const float (&x)[LP_EACH], int tile) __attribute__((always_inline)) {
        float bm = -INFINITY;
#pragma unroll
        for (int u = 0; u < LP_VECS; u++) {
            float m = x[u * VL];
#pragma unroll
            for (int e = 1; e < VL; e++) m = fmaxf(m, x[u * VL + e]);
            if (m > most) {
                most = m;
                from = tile * LP_VECS + u;
            }
            bm = fmaxf(bm, m);
        }
        v.rebase(bm);
        const float off = v.m == -INFINITY ? 0.0f : v.m;
#pragma unroll
        for (int e = 0; e < LP_EACH; e++) {
            const float u = (x[e] - off) * LOG2E, y = __builtin_amdgcn_exp2f(u);
            v.s += y;
            v.t = fmaf(y, fmaxf(u, U_MIN), v.t);
        }
    };
    const int whole = (end - begin) / TILE;
    typename Vec<T>::type w[LP_VECS];  // the next tile's logits
    auto fetch = [&](int t) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < LP_VECS; u++)
            w[u] = *reinterpret_cast<const typename Vec<T>::type *>(p + begin + t * TILE + (u * NT + tid) * VL);
    };
    if (whole > 0) fetch(0);
    for (int t = 0; t < whole; t++) {
        float x[LP_EACH];
#pragma unroll
        for (int u = 0; u < LP_VECS; u++)
#pragma unroll
            for (int e = 0; e < VL; e++) x[u * VL + e] = to_f32(w[u][e]);
        if (t + 1 < whole) fetch(t + 1);
        add(x, t);
    }
    if (begin + whole * TILE < end) {
        float x[LP_EACH];
#pragma unroll
        for (int u = 0; u < LP_VECS; u++) {
            const int i = begin + whole * TILE + (u * NT + tid) * VL;
            if (i + VL <= end) {
                const typename Vec<T>::type w = *reinterpret_cast<const typename Vec<T>::type *>(p + i);
#pragma unroll
                for (int e = 0; e < VL; e++) x[u * VL + e] = to_f32(w[e]);
            } else {
#pragma unroll
                for (int e = 0; e < VL; e++) x[u * VL + e] = i + e < end ? to_f32(p[i + e]) : -INFINITY;
            }
        }
        add(x, whole);
    }
    v = wave_sums(v);
    if (lane == 0) {
        sw[wave][0] = v.m;
        sw[wave][1] = v.s;
        sw[wave][2] = v.t;
    }

    int cur = 0;  // list entries; uniform
    u64 bar = 0;  // the last of the top_k that a cut left
    if (top > 0) {
        // the list's best in order in best[] and at its front, cut to top; an
        // entry's place is the number of better ones, counted by NT / cur threads
        auto sort_list = [&]() {
            __syncthreads();
            for (int i = tid; i < cur; i += NT) ranks[i] = 0;
            __syncthreads();
            if (cur > 0) {
                const int parts = max(1, NT / cur), len = (cur + parts - 1) / parts;
                for (int x = tid; x < cur * parts; x += NT) {
                    const int part = x / cur, i = x - part * cur, j1 = min(cur, (part + 1) * len);
                    const u64 k = list[i];
                    int r = 0;
                    for (int j = part * len; j < j1; j++) r += list[j] > k ? 1 : 0;
                    atomicAdd(&ranks[i], r);
                }
            }
            __syncthreads();
            for (int i = tid; i < cur; i += NT)
                if (ranks[i] < top) best[ranks[i]] = list[i];
            __syncthreads();
            cur = min(cur, top);
            if (tid < cur) list[tid] = best[tid];
            if (tid == 0) s_cnt = cur;
            if (cur == top) bar = best[top - 1];
            __syncthreads();
        };
        // a count summed over the workgroup
        auto total = [&](int c) {
            int n = 0;
            c = (int)wave_butterfly((float)c);
            if (NW == 1) return c;
            __syncthreads();
            if (lane == 0) iw[wave] = c;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < NW; w++) n += iw[w];
            return n;
        };
        const u64 mine = most == -INFINITY ? 0 : (u64)order32(most) << 32 | (0xffffffffu - (unsigned)(from * NT + tid));
        if constexpr (NW > 1) {
            list[tid] = mine;
            __syncthreads();
            if (wave == 0) {
                u64 keys[NW];
#pragma unroll
                for (int w = 0; w < NW; w++) keys[w] = list[w * 64 + lane];
                const u64 t = top_bound(keys, top);
                if (lane == 0) s_least = t;
            }
        } else {
            const u64 keys[1] = {mine}, t = top_bound(keys, top);
            if (lane == 0) s_least = t;
        }
        if (tid == 0) s_cnt = s_owners = 0;
        __syncthreads();
        const u64 least = s_least;
        if (mine >= least) owner[atomicAdd(&s_owners, 1)] = tid;
        __syncthreads();
        const int owners = s_owners;
        const int vecs = ((end - begin) + NT * VL - 1) / (NT * VL);  // of a thread
        // Item w: VL logits from i on, of which those from i0 on are of the owner's vector n (a row's last
        // vector: its last VL logits; a row has more than 64).
        auto fetch_item = [&](int w, int &n, int &i, int &i0) __attribute__((always_inline)) {
            const int f = w / vecs;
            n = f < owners ? (w - f * vecs) * NT + owner[f] : 0;
            i0 = f < owners ? begin + n * VL : INT_MAX;
            i = min(f < owners ? i0 : begin, end - VL);
            return *reinterpret_cast<const typename Vec<T>::type *>(p + i);
        };
        auto reaches = [&](float x, int n) __attribute__((always_inline)) {
            return x > -INFINITY && ((u64)order32(x) << 32 | (0xffffffffu - (unsigned)n)) >= least;
        };
        for (int w0 = 0; w0 < owners * vecs; w0 += 2 * NT) {
            int n[2], i[2], i0[2];
            typename Vec<T>::type x[2];
#pragma unroll
            for (int u = 0; u < 2; u++) x[u] = fetch_item(w0 + u * NT + tid, n[u], i[u], i0[u]);
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int e = 0; e < VL; e++)
                    if (i[u] + e >= i0[u] && reaches(to_f32(x[u][e]), n[u])) {
                        const int at = atomicAdd(&s_cnt, 1);
                        if (at < LP_CAP) list[at] = place_key(to_f32(x[u][e]), i[u] + e);
                    }
        }
        __syncthreads();
        cur = s_cnt;
        if (cur > LP_CAP) {  // large logits side by side in the same threads: again, the list cut whenever it is full
            __syncthreads();
            cur = 0;
            if (tid == 0) s_cnt = 0;
            __syncthreads();
            for (int w0 = 0; w0 < owners * vecs; w0 += NT) {
                int n, i, i0;
                const typename Vec<T>::type x = fetch_item(w0 + tid, n, i, i0);
                auto counts = [&](int e) __attribute__((always_inline)) {
                    return i + e >= i0 && reaches(to_f32(x[e]), n) && place_key(to_f32(x[e]), i + e) > bar;
                };
                int c = 0;
#pragma unroll
                for (int e = 0; e < VL; e++) c += counts(e) ? 1 : 0;
                c = total(c);
                auto push = [&]() __attribute__((always_inline)) {
#pragma unroll
                    for (int e = 0; e < VL; e++)
                        if (counts(e)) list[atomicAdd(&s_cnt, 1)] = place_key(to_f32(x[e]), i + e);
                };
                if (cur + c <= LP_CAP) {
                    push();
                    cur += c;
                } else {  // wave by wave, each after a cut
                    for (int y = 0; y < NW; y++) {
                        sort_list();
                        if (wave == y) push();
                        __syncthreads();
                        cur = s_cnt;
                    }
                }
            }
        }
        sort_list();
    } else {
        __syncthreads();
    }

    v = Sums{sw[0][0], sw[0][1], sw[0][2]};
#pragma unroll
    for (int w = 1; w < NW; w++) v.add(Sums{sw[w][0], sw[w][1], sw[w][2]});
    if (chunks > 1) {
        float *o = ws + (int64_t)blockIdx.x * (4 + 2 * top);
        if (tid == 0) {
            o[0] = v.m;
            o[1] = v.s;
            o[2] = v.t;
        }
        for (int k = tid; k < top; k += NT) reinterpret_cast<u64 *>(o + 4)[k] = k < cur ? best[k] : 0;
        return;
    }
    const RowStats st(v);
    if (tid == 0) store_row<T>(a, row, st);
    for (int k = tid; k < top; k += NT)
        store_top(a, row, k, k < cur ? key_value(best[k]) : -INFINITY, k < cur ? key_index(best[k]) : -1, st);
}

// Joins a row's chunks: sums, and the places of the chunks' alternatives that
// reach the highest top_k-th of a chunk.
constexpr int JOIN_THREADS = 256, JOIN_MAX = 2048;
template <class T> __global__ __launch_bounds__(JOIN_THREADS) void k_logprobs_join(TokenLogprobs a, int chunks,
                                                                                   const float *__restrict__ ws) {
    __shared__ u64 list[JOIN_MAX];
    __shared__ int s_cnt;
    const int row = blockIdx.x, tid = threadIdx.x, top = a.top, step = 4 + 2 * top;
    const float *p = ws + (int64_t)row * chunks * step;
    Sums v;
    u64 floor = 1;  // 0: no alternative
    for (int c = tid & 63; c < chunks; c += 64) {
        v.add(Sums{p[c * step], p[c * step + 1], p[c * step + 2]});
        if (top > 0) floor = max(floor, reinterpret_cast<const u64 *>(p + c * step + 4)[top - 1]);
    }
    v = wave_sums(v);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) floor = max(floor, (u64)__shfl_xor(floor, o));
    if (tid == 0) s_cnt = 0;
    __syncthreads();
    for (int i = tid; i < chunks * top; i += JOIN_THREADS) {
        const u64 k = reinterpret_cast<const u64 *>(p + (i / top) * step + 4)[i % top];
        if (k >= floor) list[atomicAdd(&s_cnt, 1)] = k;
    }
    __syncthreads();
    const RowStats st(v);
    if (tid == 0) store_row<T>(a, row, st);
    const int n = s_cnt;
    for (int i = tid; i < n; i += JOIN_THREADS) {
        const u64 k = list[i];
        int rank = 0;
        for (int j = 0; j < n; j++) rank += list[j] > k ? 1 : 0;
        if (rank < top) store_top(a, row, rank, key_value(k), key_index(k), st);
    }
    for (int k = n + tid; k < top; k += JOIN_THREADS) store_top(a, row, k, -INFINITY, -1, st);
}

// Threads a row, chunks a row (bfloat16, us).  A workgroup's joins cost about as much as
// a thread's 64 logits, so a wave takes up to 4096 logits (4096 rows of 3000: 12, 256 threads 23)
// and 256 threads up to 65536 (4096 rows of 30000: 51, a wave 67, 512 threads 66).  A
// row is split where the rows leave CUs idle and it has 12 tiles or more, into
// chunks of at least four (one row of 131072: 15.7, in four 12.7, in 16 14.8; 64 rows of 30000:
// 10.3, in two 12.5; 200 rows of 131072: 18, in two 22).
struct LpPlan {
    int nt, chunks, tiles_per;
};
LpPlan lp_plan(int n, int vocab, int top) {
    LpPlan p;
    p.nt = vocab <= 4096 ? 64 : vocab <= 65536 ? 256 : 512;
    const int tiles = (vocab + p.nt * LP_EACH - 1) / (p.nt * LP_EACH);
    const int most = top > 0 ? JOIN_MAX / top : 64;
    p.chunks = tiles < 12 ? 1 : std::max(1, std::min(std::min(tiles / 4, most), 256 / n));
    p.tiles_per = (tiles + p.chunks - 1) / p.chunks;
    p.chunks = (tiles + p.tiles_per - 1) / p.tiles_per;
    return p;
}

template <class T> hipError_t launch_lp(const TokenLogprobs &a, float *ws, hipStream_t st) {
    if (a.vocab <= 64) {
        hipLaunchKernelGGL(k_logprobs_narrow<T>, dim3((a.n + NARROW_ROWS - 1) / NARROW_ROWS), dim3(64 * NARROW_ROWS), 0, st, a);
        return hipGetLastError();
    }
    const LpPlan p = lp_plan(a.n, a.vocab, a.top);
    if (!kv8_grid((int64_t)a.n * p.chunks, p.nt)) return hipErrorInvalidValue;
    const dim3 grid(a.n * p.chunks);
    if (p.nt == 64) hipLaunchKernelGGL((k_logprobs<T, 64>), grid, dim3(64), 0, st, a, p.chunks, p.tiles_per, ws);
    else if (p.nt == 256) hipLaunchKernelGGL((k_logprobs<T, 256>), grid, dim3(256), 0, st, a, p.chunks, p.tiles_per, ws);
    else hipLaunchKernelGGL((k_logprobs<T, 512>), grid, dim3(512), 0, st, a, p.chunks, p.tiles_per, ws);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.chunks == 1) return e;
    hipLaunchKernelGGL(k_logprobs_join<T>, dim3(a.n), dim3(JOIN_THREADS), 0, st, a, p.chunks, ws);
    return hipGetLastError();
}

}  // namespace

size_t token_logprobs_floats(int n, int vocab, int top) {
    if (n == 0 || vocab <= 64) return 0;
    const LpPlan p = lp_plan(n, vocab, top);
    return p.chunks > 1 ? (size_t)n * p.chunks * (4 + 2 * top) : 0;
}

// A launch counts its threads in 32 bits: this many rows have at most 2^31, and
// more of them go in several launches (rows are split into chunks only where they are few).
constexpr int LAUNCH_ROWS = 1 << 22;

hipError_t launch_token_logprobs(const TokenLogprobs &all, float *ws, size_t ws_floats, hipStream_t st) {
    if (token_logprobs_floats(all.n, all.vocab, all.top) > ws_floats) return hipErrorInvalidValue;
    for (int r0 = 0; r0 < all.n; r0 += LAUNCH_ROWS) {
        TokenLogprobs a = all;
        a.n = std::min(all.n - r0, LAUNCH_ROWS);
        a.logits = static_cast<const char *>(all.logits) + r0 * all.stride * (all.dtype == FT_F32 ? 4 : 2);
        if (all.targets) a.targets += r0;
        if (all.logprob) a.logprob += r0;
        if (all.entropy) a.entropy += r0;
        if (all.top > 0) {
            a.top_ids += (int64_t)r0 * all.top;
            a.top_lp += (int64_t)r0 * all.top;
        }
        hipError_t e = hipErrorInvalidValue;
        switch (a.dtype) {
            case FT_F32: e = launch_lp<float>(a, ws, st); break;
            case FT_F16: e = launch_lp<_Float16>(a, ws, st); break;
            case FT_BF16: e = launch_lp<__bf16>(a, ws, st); break;
        }
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace cih

// Log probabilities of given tokens, with entropy and the top alternatives.
//
// One pass over a row with the running maximum m: u = (x - m) log2 e, s = sum
// 2^u, t = sum 2^u u; then
//   log p(i) = x_i - m - ln 2 log2 s,  entropy = ln 2 (log2 s - t / s).
// A NaN or +inf anywhere makes s NaN.  Bound by reading the logits once; what
// the alternatives add is one comparison a thread and tile (see below).
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

constexpr int LP_VECS = 4;   // 16-byte loads of a thread in a tile
constexpr int LP_CAP = 768;  // candidates

// The row (or the chunk blockIdx % chunks of its tiles) by NT threads.
//
// Alternatives.  `bar` is a logit that top_k found ones reach.  A tile without
// a logit above it costs one comparison a thread; otherwise the logits above
// go to a list in LDS.  A tile with more than fit (the first, or one of a row
// that ascends) first raises the bar to the top_k-th largest of 64 threads'
// maxima, the best of the waves'; if that leaves too many (ties), the tile's
// top_k are taken one by one.  The list is put in order, and the bar raised to
// its top_k-th, when it is full and at the end.
template <class T, int NT>
__global__ __launch_bounds__(NT) void k_logprobs(TokenLogprobs a, int chunks, int tiles_per, float *__restrict__ ws) {
    constexpr int VL = Vec<T>::N, TILE = NT * LP_VECS * VL, NW = NT / 64;
    __shared__ u64 list[LP_CAP], best[LOGPROBS_MAX_TOP], kw[NW];
    __shared__ int ranks[LP_CAP], iw[NW], s_cnt;
    __shared__ float fw[NW], sw[NW][3];
    const int row = blockIdx.x / chunks, chunk = blockIdx.x - row * chunks;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T *p = static_cast<const T *>(a.logits) + row * a.stride;
    const int top = a.top;
    const int64_t begin = (int64_t)chunk * tiles_per * TILE;
    const int end = (int)min((int64_t)a.vocab, begin + (int64_t)tiles_per * TILE);
    Sums v;
    float bar = -INFINITY;
    int cur = 0;  // list entries; uniform
    if (tid == 0) s_cnt = 0;

    // a count summed over the workgroup (every thread calls it)
    auto total = [&](int c) {
        int n = 0;
        __syncthreads();
        c = (int)wave_butterfly((float)c);
        if (NW == 1) return c;
        if (lane == 0) iw[wave] = c;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NW; w++) n += iw[w];
        return n;
    };
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
        if (cur == top) bar = key_value(best[top - 1]);
        __syncthreads();
    };

    for (int base = (int)begin; base < end; base += TILE) {
        float x[LP_VECS * VL];
        int at[LP_VECS];
#pragma unroll
        for (int u = 0; u < LP_VECS; u++) {
            at[u] = base + (u * NT + tid) * VL;
            if (at[u] + VL <= end) {
                const typename Vec<T>::type w = *reinterpret_cast<const typename Vec<T>::type *>(p + at[u]);
#pragma unroll
                for (int e = 0; e < VL; e++) x[u * VL + e] = to_f32(w[e]);
            } else {
#pragma unroll
                for (int e = 0; e < VL; e++) x[u * VL + e] = at[u] + e < end ? to_f32(p[at[u] + e]) : -INFINITY;
            }
        }
        float bm = -INFINITY;
#pragma unroll
        for (int e = 0; e < LP_VECS * VL; e++) bm = fmaxf(bm, x[e]);
        v.rebase(bm);
        const float off = v.m == -INFINITY ? 0.0f : v.m;
#pragma unroll
        for (int e = 0; e < LP_VECS * VL; e++) {
            const float u = (x[e] - off) * LOG2E, y = __builtin_amdgcn_exp2f(u);
            v.s += y;
            v.t = fmaf(y, fmaxf(u, U_MIN), v.t);
        }
        if (top == 0) continue;
        if (!__syncthreads_or(bm > bar)) continue;
        // logits that count: above bar, and not below floor
        float floor = -INFINITY;
        auto count = [&]() {
            int c = 0;
#pragma unroll
            for (int e = 0; e < LP_VECS * VL; e++) c += x[e] > bar && x[e] >= floor ? 1 : 0;
            return total(c);
        };
        int n = count();
        if (cur + n > LP_CAP) {
            // the top-th largest of a wave's 64 maxima, bit by bit
            const unsigned key = order32(bm);
            unsigned k = 0;
#pragma unroll 1
            for (int bit = 31; bit >= 0; bit--) {
                const unsigned t = k | 1u << bit;
                if (__popcll(__ballot(key >= t)) >= top) k = t;
            }
            floor = k == 0 ? -INFINITY : order32_value(k);
            if (NW > 1) {
                __syncthreads();
                if (lane == 0) fw[wave] = floor;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < NW; w++) floor = fmaxf(floor, fw[w]);
            }
            sort_list();
            n = count();
        }
        if (cur + n <= LP_CAP) {
#pragma unroll
            for (int e = 0; e < LP_VECS * VL; e++)
                if (x[e] > bar && x[e] >= floor) list[atomicAdd(&s_cnt, 1)] = place_key(x[e], at[e / VL] + e % VL);
            cur += n;
        } else {
            u64 last = ~0ull;
            for (int k = 0; k < top; k++) {
                u64 y = 0;
#pragma unroll
                for (int e = 0; e < LP_VECS * VL; e++) {
                    const u64 z = place_key(x[e], at[e / VL] + e % VL);
                    if (x[e] > bar && z < last && z > y) y = z;
                }
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) y = max(y, (u64)__shfl_xor(y, o));
                __syncthreads();
                if (lane == 0) kw[wave] = y;
                __syncthreads();
                for (int w = 0; w < NW; w++) y = max(y, kw[w]);
                if (y == 0) break;
                last = y;
                if (tid == 0) list[cur] = y;
                cur++;
            }
            __syncthreads();
            if (tid == 0) s_cnt = cur;
        }
    }

    v = wave_sums(v);
    if (lane == 0) {
        sw[wave][0] = v.m;
        sw[wave][1] = v.s;
        sw[wave][2] = v.t;
    }
    if (top > 0) sort_list();
    else __syncthreads();
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

// Threads a row, chunks a row.
struct LpPlan {
    int nt, chunks, tiles_per;
};
LpPlan lp_plan(int n, int vocab, int top, int elem) {
    const int per = LP_VECS * 16 / elem;  // logits of a thread in a tile
    LpPlan p;
    p.nt = vocab <= 64 * per ? 64 : vocab <= 512 * per ? 256 : 512;
    const int tiles = (vocab + p.nt * per - 1) / (p.nt * per);
    const int most = top > 0 ? JOIN_MAX / top : 64;
    p.chunks = n >= 512 ? 1 : std::min(std::min(tiles, most), (767 + n) / n);
    p.tiles_per = (tiles + p.chunks - 1) / p.chunks;
    p.chunks = (tiles + p.tiles_per - 1) / p.tiles_per;
    return p;
}

template <class T> hipError_t launch_lp(const TokenLogprobs &a, float *ws, hipStream_t st) {
    if (a.vocab <= 64) {
        hipLaunchKernelGGL(k_logprobs_narrow<T>, dim3((a.n + NARROW_ROWS - 1) / NARROW_ROWS), dim3(64 * NARROW_ROWS), 0,
                           st, a);
        return hipGetLastError();
    }
    const LpPlan p = lp_plan(a.n, a.vocab, a.top, sizeof(T));
    if ((int64_t)a.n * p.chunks > INT32_MAX) return hipErrorInvalidValue;
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
    size_t most = 0;
    for (int elem = 2; elem <= 4; elem += 2) {
        const LpPlan p = lp_plan(n, vocab, top, elem);
        if (p.chunks > 1) most = std::max(most, (size_t)n * p.chunks * (4 + 2 * top));
    }
    return most;
}

hipError_t launch_token_logprobs(const TokenLogprobs &a, float *ws, hipStream_t st) {
    if (a.n == 0) return hipSuccess;
    switch (a.dtype) {
        case FT_F32: return launch_lp<float>(a, ws, st);
        case FT_F16: return launch_lp<_Float16>(a, ws, st);
        case FT_BF16: return launch_lp<__bf16>(a, ws, st);
    }
    return hipErrorInvalidValue;
}

}  // namespace cih

// Log probabilities of given tokens, with entropy and the top alternatives.
#include <limits.h>

#include "kv8.h"

namespace cih {

namespace {

constexpr int LP_THREADS = 256;

// a value and where it is; better: larger, or equal and earlier
struct Best {
    float x;
    int i;
};
__device__ __forceinline__ bool better(float x, int i, float y, int j) { return x > y || (x == y && i < j); }

template <class OP> __device__ __forceinline__ float block_all(float v, float *red, OP op) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < LP_THREADS / 64; w++) v = op(v, red[w]);
    return v;
}

// One workgroup per row: the maximum (NaN if there is one), the sums, then the
// alternatives one after the other, each the best below the one before.
template <class T> __global__ __launch_bounds__(LP_THREADS) void k_token_logprobs(TokenLogprobs a) {
    __shared__ float red[LP_THREADS / 64];
    __shared__ int redi[LP_THREADS / 64];
    const int r = blockIdx.x, V = a.vocab, tid = threadIdx.x;
    const T *x = static_cast<const T *>(a.logits) + r * a.stride;
    float m = -INFINITY;
    for (int i = tid; i < V; i += LP_THREADS) {
        const float v = to_f32(x[i]);
        m = v > m || v != v ? v : m;
    }
    m = block_all(m, red, [](float p, float q) { return q > p || q != q ? q : p; });
    float s = 0.0f, t = 0.0f;
    const float base = m == -INFINITY ? 0.0f : m;
    for (int i = tid; i < V; i += LP_THREADS) {
        const float v = to_f32(x[i]) - base, e = expf(v);
        s += e;
        t += e > 0.0f || e != e ? e * v : 0.0f;
    }
    auto add = [](float p, float q) { return p + q; };
    s = block_all(s, red, add);
    t = block_all(t, red, add);
    const bool none = m == -INFINITY, lost = !(m < INFINITY) || s != s;
    const float lse = lost ? NAN : none ? -INFINITY : base + logf(s);
    if (tid == 0) {
        if (a.logprob) {
            const int g = a.targets[r];
            float lp = 0.0f;
            if (g >= V || lost) lp = NAN;
            else if (g >= 0) lp = none ? -INFINITY : to_f32(x[g]) - lse;
            if (g < 0) lp = 0.0f;
            a.logprob[r] = lp;
        }
        if (a.entropy) a.entropy[r] = lost ? NAN : none ? 0.0f : logf(s) - t / s;
    }
    float px = INFINITY;
    int pi = -1;
    for (int k = 0; k < a.top; k++) {
        Best b = {-INFINITY, INT_MAX};
        if (!lost)
            for (int i = tid; i < V; i += LP_THREADS) {
                const float v = to_f32(x[i]);
                if (better(px, pi, v, i) && better(v, i, b.x, b.i)) b = {v, i};
            }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const float y = __shfl_xor(b.x, o);
            const int j = __shfl_xor(b.i, o);
            if (better(y, j, b.x, b.i)) b = {y, j};
        }
        __syncthreads();
        if ((tid & 63) == 0) {
            red[tid >> 6] = b.x;
            redi[tid >> 6] = b.i;
        }
        __syncthreads();
        for (int w = 0; w < LP_THREADS / 64; w++)
            if (better(red[w], redi[w], b.x, b.i)) b = {red[w], redi[w]};
        const bool end = b.x == -INFINITY;
        if (tid == 0) {
            a.top_ids[(int64_t)r * a.top + k] = end ? -1 : b.i;
            a.top_lp[(int64_t)r * a.top + k] = lost ? NAN : end ? -INFINITY : b.x - lse;
        }
        px = b.x;
        pi = b.i;
    }
}

}  // namespace

size_t token_logprobs_floats(int n, int vocab, int top) { return 0; }

hipError_t launch_token_logprobs(const TokenLogprobs &a, float *ws, hipStream_t st) {
    if (a.n == 0) return hipSuccess;
    const dim3 grid(a.n), block(LP_THREADS);
    switch (a.dtype) {
        case FT_F32: hipLaunchKernelGGL(k_token_logprobs<float>, grid, block, 0, st, a); break;
        case FT_F16: hipLaunchKernelGGL(k_token_logprobs<_Float16>, grid, block, 0, st, a); break;
        case FT_BF16: hipLaunchKernelGGL(k_token_logprobs<__bf16>, grid, block, 0, st, a); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace cih

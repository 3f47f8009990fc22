// Verification of drafted tokens (speculative sampling, Leviathan et al. 2023): with p =
// softmax(logits / T) and q = softmax(draft logits / T), draft x is taken if u q(x) < p(x).
// The token after the taken ones comes from max(p - q, 0) at the first refusal, from p
// after all drafts: the first whose running sum passes v times the whole.  T = 0: the largest logit.
// Sums and borders in 64 bits: in 32 a border moves across tokens.
#include <float.h>

#include "kernels.h"
#include "kv8.h"

namespace cih {

namespace {

constexpr int VERIFY_THREADS = 256;

template <class V, class OP> __device__ __forceinline__ V block_all(V v, OP op, V *red) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < VERIFY_THREADS / 64; w++) v = op(v, red[w]);
    return v;
}

// A row's largest logit and the sum of exp((x - largest) / T); lost: no distribution.
struct Dist {
    double m, z;
    bool lost;
    int best;
};
template <class T> __device__ Dist dist(const T *x, int vocab, double heat, double *red, int *ired) {
    Dist d;
    float m = -INFINITY;
    int best = 0x7fffffff;
    bool bad = false;
    for (int j = threadIdx.x; j < vocab; j += VERIFY_THREADS) {
        const float y = to_f32(x[j]);
        bad |= !(y < INFINITY);
        if (y > m) {
            m = y;
            best = j;
        }
    }
    const float all = (float)block_all((double)m, [](double a, double b) { return a > b ? a : b; }, red);
    d.best = block_all(m == all ? best : 0x7fffffff, [](int a, int b) { return min(a, b); }, ired);
    d.lost = block_all((int)bad, [](int a, int b) { return a | b; }, ired) || all == -INFINITY;
    d.m = all;
    d.z = 0.0;
    if (heat > 0.0 && !d.lost) {
        double z = 0.0;
        for (int j = threadIdx.x; j < vocab; j += VERIFY_THREADS) z += exp(((double)to_f32(x[j]) - d.m) / heat);
        d.z = block_all(z, [](double a, double b) { return a + b; }, red);
    }
    return d;
}
__device__ __forceinline__ double prob(const Dist &d, float x, double heat) { return exp(((double)x - d.m) / heat) / d.z; }

template <class T> __global__ __launch_bounds__(VERIFY_THREADS) void k_verify(VerifyDrafts v) {
    __shared__ double red[VERIFY_THREADS / 64], scan[VERIFY_THREADS];
    __shared__ int ired[VERIFY_THREADS / 64];
    const int i = blockIdx.x, tid = threadIdx.x;
    const int c0 = min(max(v.cu[i], 0), v.n_drafts), c1 = min(max(v.cu[i + 1], c0), v.n_drafts);
    const double heat = v.temperature;
    int taken = 0, token = -1;
    Dist p{}, q{};
    bool refused = false, lost = false;
    const T *pr = nullptr, *qr = nullptr;
    for (;; taken++) {
        pr = static_cast<const T *>(v.logits) + (int64_t)(c0 + i + taken) * v.stride;
        p = dist(pr, v.vocab, heat, red, ired);
        lost = p.lost;
        if (lost || c0 + taken >= c1) break;
        const int x = v.drafted[c0 + taken];
        const bool known = x >= 0 && x < v.vocab;
        if (heat == 0.0) {
            if (x != p.best) break;
            continue;
        }
        double qx = 1.0;
        if (v.draft) {
            qr = static_cast<const T *>(v.draft) + (int64_t)(c0 + taken) * v.draft_stride;
            q = dist(qr, v.vocab, heat, red, ired);
            lost = q.lost;
            if (lost) break;
            if (known) qx = prob(q, to_f32(qr[x]), heat);
        }
        refused = !(known && (double)v.accept_at[c0 + taken] * qx < prob(p, to_f32(pr[x]), heat));
        if (refused) break;
    }
    if (!lost && heat == 0.0) token = p.best;
    if (!lost && heat > 0.0) {
        const int x = refused ? v.drafted[c0 + taken] : -1;
        bool left = refused;
        auto weight = [&](int j) {
            double w = prob(p, to_f32(pr[j]), heat);
            if (left) w = v.draft ? fmax(w - prob(q, to_f32(qr[j]), heat), 0.0) : j == x ? 0.0 : w;
            return w;
        };
        double all = 0.0;
        for (int round = 0; round < 2; round++) {  // nothing left: from p itself
            all = 0.0;
            for (int j = tid; j < v.vocab; j += VERIFY_THREADS) all += weight(j);
            all = block_all(all, [](double a, double b) { return a + b; }, red);
            if (all > 0.0 || !left) break;
            left = false;
        }
        const double border = (double)v.sample_at[i] * all;
        double sum = 0.0;
        int last = -1, found = 0x7fffffff;
        for (int j0 = 0; j0 < v.vocab; j0 += VERIFY_THREADS) {
            const int j = j0 + tid;
            const double w = j < v.vocab ? weight(j) : 0.0;
            if (w > 0.0) last = j;
            __syncthreads();
            scan[tid] = w;
            __syncthreads();
            for (int o = 1; o < VERIFY_THREADS; o <<= 1) {
                const double y = tid >= o ? scan[tid - o] : 0.0;
                __syncthreads();
                scan[tid] += y;
                __syncthreads();
            }
            const int at = block_all(w > 0.0 && sum + scan[tid] > border ? j : 0x7fffffff, [](int a, int b) { return min(a, b); }, ired);
            if (at != 0x7fffffff) {
                found = at;
                break;
            }
            sum += scan[VERIFY_THREADS - 1];
        }
        last = block_all(last, [](int a, int b) { return max(a, b); }, ired);
        token = found != 0x7fffffff ? found : last;
    }
    if (tid == 0) {
        v.accepted[i] = taken;
        v.tokens[i] = token;
    }
}

}  // namespace

size_t verify_drafts_bytes(int n_seq, int n_drafts, int vocab) { return 0; }

hipError_t launch_verify_drafts(const VerifyDrafts &v, void *ws, hipStream_t st) {
    if (v.n_seq == 0) return hipSuccess;
    if (!kv8_grid(v.n_seq, VERIFY_THREADS)) return hipErrorInvalidValue;
    switch (v.dtype) {
        case FT_F32: hipLaunchKernelGGL(k_verify<float>, dim3(v.n_seq), dim3(VERIFY_THREADS), 0, st, v); break;
        case FT_F16: hipLaunchKernelGGL(k_verify<_Float16>, dim3(v.n_seq), dim3(VERIFY_THREADS), 0, st, v); break;
        case FT_BF16: hipLaunchKernelGGL(k_verify<__bf16>, dim3(v.n_seq), dim3(VERIFY_THREADS), 0, st, v); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace cih

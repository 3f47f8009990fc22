// Attention over the 8-bit paged key/value cache.
#include "kv8.h"
#include "x3.h"

namespace cih {

namespace {

// One wave per (row, head): a lane per key of a page for the scores, a lane per
// dim for the values, one pass over the pages with a running maximum and sum.
template <class T>
__global__ __launch_bounds__(64) void k_kv8_attend_row(Kv8Attention a) {
    __shared__ float qs[128], ps[KV8_PAGE];
    const int r = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, d = a.c.d;
    // the row's sequence: the last one that starts at or before it
    int lo = 0, hi = a.s.n_seq;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.s.cu[mid] <= r) lo = mid;
        else hi = mid;
    }
    const Kv8Seq q = kv8_seq(a.s, lo);
    if (r < q.r0 || r >= q.r0 + q.n) return;
    const int pos = q.start + (r - q.r0), kv = h / (a.heads / a.c.hk);
    const int end = a.causal ? min(q.len, pos + 1) : q.len;
    const int begin = a.window > 0 ? max(0, pos - a.window + 1) : 0;
    const T *qp = static_cast<const T *>(a.q.p) + r * a.q.rs + h * a.q.hs;
    for (int i = lane; i < d; i += 64) qs[i] = to_f32(qp[i]);
    float m = -INFINITY, l = 0.0f, o[2] = {0.0f, 0.0f};
    for (int pg = begin / KV8_PAGE; pg * KV8_PAGE < end && pos >= 0; pg++) {
        const int id = kv8_page(a.c, q, pg);
        if (id < 0) continue;
        const int64_t ph = (int64_t)id * a.c.hk + kv;
        const float2 sc = a.c.scales[ph];
        const unsigned long long bad = a.c.bad[ph];
        __syncthreads();
        const int j = pg * KV8_PAGE + lane;
        float s = 0.0f;
        const signed char *kc = a.c.k + ph * (KV8_PAGE * a.c.dp) + lane * a.c.dp;
        for (int i = 0; i < d; i++) s += qs[i] * (float)kc[i];
        s = bad >> lane & 1 ? NAN : s * (sc.x * a.scale);
        if (j < begin || j >= end) s = -INFINITY;
        float mx = s;
        for (int x = 32; x > 0; x >>= 1) {
            const float y = __shfl_xor(mx, x);
            mx = y > mx || y != y ? y : mx;
        }
        const float mn = mx > m || mx != mx ? mx : m, base = mn == -INFINITY ? 0.0f : mn;
        const float p = expf(s - base), al = expf(m - base);
        float sum = p;
        for (int x = 32; x > 0; x >>= 1) sum += __shfl_xor(sum, x);
        l = l * al + sum;
        m = mn;
        ps[lane] = p;
        __syncthreads();
        for (int u = 0; u < 2; u++) {
            const int i = lane + 64 * u;
            if (i >= d) break;
            const signed char *vc = a.c.v + ph * (KV8_PAGE * a.c.dp) + i * KV8_PAGE;
            float t = 0.0f;
            for (int k = 0; k < KV8_PAGE; k++) t += ps[k] * (float)vc[k];
            o[u] = o[u] * al + t * sc.y;
        }
    }
    T *op = static_cast<T *>(a.out.p) + r * a.out.rs + h * a.out.hs;
    for (int u = 0; u < 2; u++) {
        const int i = lane + 64 * u;
        if (i >= d) break;
        const float x = l == 0.0f ? 0.0f : o[u] / l;
        if (a.out_h2) h2_store(static_cast<unsigned short *>(a.out.p), r, h * d + i, a.heads * d, x);
        else op[i] = (T)x;
    }
    if (a.lse && lane == 0) a.lse[(int64_t)r * a.heads + h] = l == 0.0f ? -INFINITY : m + logf(l);
}

}  // namespace

size_t kv8_attention_floats(const Kv8View &c, const Kv8Seqs &s, int heads) { return 0; }

hipError_t launch_kv8_attention(const Kv8Attention &a, float *ws, hipStream_t st) {
    if (a.s.n_rows == 0 || a.s.n_seq == 0) return hipSuccess;
    const dim3 grid(a.s.n_rows, a.heads), block(64);
    switch (a.dtype) {
        case FT_F32: hipLaunchKernelGGL(k_kv8_attend_row<float>, grid, block, 0, st, a); break;
        case FT_F16: hipLaunchKernelGGL(k_kv8_attend_row<_Float16>, grid, block, 0, st, a); break;
        case FT_BF16: hipLaunchKernelGGL(k_kv8_attend_row<__bf16>, grid, block, 0, st, a); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace cih

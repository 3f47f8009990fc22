// Eviction from the 8-bit cache by accumulated attention weight.  Each kv head of a
// sequence of more than `budget` tokens keeps its first `first` tokens, its last `recent`
// ones and the `budget - first - recent` of the others with the largest weights (ties: the
// earlier token); what is kept moves to the sequence's first `budget` places, in order.
//
// k_kv8_choose (a workgroup per sequence and head) finds the kept tokens' ids and what becomes of
// their pages' records; k_kv8_move moves the codes.  A page's new scale is the largest of the
// pages that its tokens come from, so codes are rounded again only where their page's scale
// grows: a token that moves many times is not rounded each time.
#include "kernels.h"
#include "kv8.h"

namespace cih {

namespace {

constexpr int CHOOSE_THREADS = 1024, MOVE_THREADS = 256;

// Of each (sequence, head), in the workspace.
struct Work {
    int *list;                 // [budget]: the kept tokens
    float2 *ratio;             // [budget]: by which their codes are scaled, K and V
    float *weight;             // [budget]
    float2 *scales;            // [pages]
    unsigned long long *bad;   // [pages]
    int *state;                // {tokens kept, 1 if they move}
    int pages, tokens;
};
__host__ __device__ inline size_t work_size(int budget) {  // a multiple of 16 bytes
    const size_t pages = (budget + KV8_PAGE - 1) / KV8_PAGE, tokens = pages * KV8_PAGE;
    return tokens * (sizeof(int) + sizeof(float2) + sizeof(float)) + pages * (sizeof(float2) + sizeof(unsigned long long)) + 16;
}
__device__ __forceinline__ Work work_of(void *ws, int budget, int64_t pair) {
    char *p = static_cast<char *>(ws) + pair * work_size(budget);
    Work w;
    w.pages = (budget + KV8_PAGE - 1) / KV8_PAGE;
    w.tokens = w.pages * KV8_PAGE;
    w.state = reinterpret_cast<int *>(p);
    w.ratio = reinterpret_cast<float2 *>(p + 16);
    w.scales = reinterpret_cast<float2 *>(w.ratio + w.tokens);
    w.bad = reinterpret_cast<unsigned long long *>(w.scales + w.pages);
    w.list = reinterpret_cast<int *>(w.bad + w.pages);
    w.weight = reinterpret_cast<float *>(w.list + w.tokens);
    return w;
}

// Larger weights have larger keys; -0 counts as 0, NaN is below every other.
__device__ __forceinline__ unsigned weight_key(float x) {
    const unsigned b = __float_as_uint(x + 0.0f);
    return x != x ? 0 : b >> 31 ? ~b : b | 0x80000000u;
}

// Tokens a sequence holds and its row of the table.
struct Held {
    int n;
    const int *table;
};
__device__ __forceinline__ Held held(const Kv8Seqs &s, int i) {
    const int slot = s.slots ? s.slots[i] : i;
    return {(int)min((int64_t)max(s.lens[i], 0), (int64_t)s.max_pages * KV8_PAGE),
            slot >= 0 && slot < s.table_rows ? s.table + (int64_t)slot * s.table_stride : nullptr};
}

__global__ __launch_bounds__(CHOOSE_THREADS) void k_kv8_choose(Kv8Evict e, void *ws) {
    __shared__ int total, part[CHOOSE_THREADS / 64][2];
    const int h = blockIdx.x % e.c.hk, i = blockIdx.x / e.c.hk;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Held q = held(e.s, i);
    const Work w = work_of(ws, e.budget, blockIdx.x);
    int *kept = e.kept ? e.kept + (int64_t)blockIdx.x * e.budget : nullptr;
    const int pages = (q.n + KV8_PAGE - 1) / KV8_PAGE;
    // every page has to be there
    if (tid == 0) total = 0;
    __syncthreads();
    int gone = q.table == nullptr && q.n > 0;
    for (int p = tid; !gone && p < pages; p += CHOOSE_THREADS) {
        const int id = q.table[p];
        gone |= id < 0 || id >= e.c.n_pages;
    }
    if (gone) atomicOr(&total, 1);
    __syncthreads();
    const bool lost = total != 0;
    auto weight = [&](int j) { return e.weights[((int64_t)q.table[j / KV8_PAGE] * e.c.hk + h) * KV8_PAGE + j % KV8_PAGE]; };
    if (lost || q.n <= e.budget) {  // stays as it is
        const int n = lost ? 0 : q.n;
        for (int m = tid; kept && m < e.budget; m += CHOOSE_THREADS) kept[m] = m < n ? m : -1;
        for (int m = tid; m < n; m += CHOOSE_THREADS) {
            w.list[m] = m;
            w.weight[m] = weight(m);
        }
        if (tid == 0) {
            w.state[0] = n;
            w.state[1] = 0;
        }
        return;
    }
    const int lo = e.first, hi = q.n - e.recent, need = e.budget - e.first - e.recent;  // of tokens [lo, hi), fewer than those
    auto count = [&](unsigned least) {  // tokens with a key of at least that
        __syncthreads();
        if (tid == 0) total = 0;
        __syncthreads();
        int n = 0;
        for (int j = lo + tid; j < hi; j += CHOOSE_THREADS) n += weight_key(weight(j)) >= least;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o);
        if (lane == 0) atomicAdd(&total, n);
        __syncthreads();
        return total;
    };
    // the smallest key that is kept, from its highest bit on
    unsigned border = 0;
    for (int bit = 31; bit >= 0; bit--)
        if (count(border | 1u << bit) >= need) border |= 1u << bit;
    int equal = need;
    if (border != 0xffffffffu) equal -= count(border + 1);
    // in order: all above the border, the first of those at it
    int before = 0, ties = 0;
    for (int j0 = 0; j0 < q.n; j0 += CHOOSE_THREADS) {
        const int j = j0 + tid;
        const unsigned key = j >= lo && j < hi ? weight_key(weight(j)) : 0;
        const bool mid = j >= lo && j < hi, at = mid && key == border;
        const bool sure = j < q.n && (!mid || key > border);
        const unsigned long long below = (1ull << lane) - 1, a = __ballot(at), b = __ballot(sure);
        __syncthreads();
        if (lane == 0) {
            part[wave][0] = __popcll(a);
            part[wave][1] = __popcll(b);
        }
        __syncthreads();
        int at_before = ties + __popcll(a & below), sure_before = before + __popcll(b & below), at_all = 0, sure_all = 0;
        for (int x = 0; x < CHOOSE_THREADS / 64; x++) {
            if (x < wave) {
                at_before += part[x][0];
                sure_before += part[x][1];
            }
            at_all += part[x][0];
            sure_all += part[x][1];
        }
        if (sure || (at && at_before < equal)) {
            const int m = sure_before + min(at_before, equal);
            w.list[m] = j;
            w.weight[m] = weight(j);
            if (kept) kept[m] = j;
        }
        ties += at_all;
        before += sure_all;
    }
    __syncthreads();
    // the pages' records, a wave a page
    for (int p = wave; p < w.pages; p += CHOOSE_THREADS / 64) {
        const int m = p * KV8_PAGE + lane;
        const bool there = m < e.budget;
        const int j = there ? w.list[m] : 0;
        const int64_t ph = (int64_t)q.table[j / KV8_PAGE] * e.c.hk + h;
        const float2 old = there ? e.c.scales[ph] : float2{0.0f, 0.0f};
        float2 now = old;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            now.x = fmaxf(now.x, __shfl_xor(now.x, o));
            now.y = fmaxf(now.y, __shfl_xor(now.y, o));
        }
        const unsigned long long bits = __ballot(there && e.c.bad[ph] >> (j % KV8_PAGE) & 1);
        w.ratio[m] = {now.x > 0.0f ? old.x / now.x : 0.0f, now.y > 0.0f ? old.y / now.y : 0.0f};
        if (lane == 0) {
            w.scales[p] = now;
            w.bad[p] = bits;
        }
    }
    if (tid == 0) {
        w.state[0] = e.budget;
        w.state[1] = 1;
    }
}

// One workgroup per (sequence, head) and K or V: page after page, its codes read before they
// are written.  Token m of the kept ones comes from place m or a later one, so what is written has been read.
__global__ __launch_bounds__(MOVE_THREADS) void k_kv8_move(Kv8Evict e, void *ws) {
    const int which = blockIdx.x & 1, pair = blockIdx.x >> 1, h = pair % e.c.hk, i = pair / e.c.hk, tid = threadIdx.x;
    const Held q = held(e.s, i);
    const Work w = work_of(ws, e.budget, pair);
    const int n = w.state[0], dp = e.c.dp;
    if (which == 0 && h == 0 && tid == 0) {
        const int len = w.state[1] ? e.budget : e.s.lens[i];
        if (w.state[1] && e.shifts) e.shifts[i] += q.n - e.budget;
        w.state[2] = len;
    }
    if (which == 0 && e.weights_out)
        for (int m = tid; m < n; m += MOVE_THREADS)
            e.weights_out[((int64_t)q.table[m / KV8_PAGE] * e.c.hk + h) * KV8_PAGE + m % KV8_PAGE] = w.weight[m];
    if (!w.state[1]) return;
    for (int p = 0; p < w.pages; p++) {
        const int64_t to = (int64_t)q.table[p] * e.c.hk + h;
        const int held_here = min(KV8_PAGE, n - p * KV8_PAGE);
        unsigned x[8][4];
#pragma unroll
        for (int it = 0; it < 8; it++) {
            const int at = tid + it * MOVE_THREADS;
            if (which == 0) {  // 16 dims of a token
                const int per = dp / 16, m = at / per, d = at % per * 16;
                if (m >= held_here) continue;
                const int j = w.list[p * KV8_PAGE + m];
                const float r = w.ratio[p * KV8_PAGE + m].x;
                const uint4 y = *reinterpret_cast<const uint4 *>(
                    e.c.k + (((int64_t)q.table[j / KV8_PAGE] * e.c.hk + h) * KV8_PAGE + j % KV8_PAGE) * dp + d);
                x[it][0] = recode4(y.x, r);
                x[it][1] = recode4(y.y, r);
                x[it][2] = recode4(y.z, r);
                x[it][3] = recode4(y.w, r);
            } else {  // four tokens of a dim
                const int d = at / 16, m0 = at % 16 * 4;
                if (d >= dp || m0 >= held_here) continue;
                unsigned o = 0;
                for (int u = 0; u < 4 && m0 + u < held_here; u++) {
                    const int j = w.list[p * KV8_PAGE + m0 + u];
                    const signed char y = e.c.v[(((int64_t)q.table[j / KV8_PAGE] * e.c.hk + h) * dp + d) * KV8_PAGE + j % KV8_PAGE];
                    o |= (unsigned)code8((float)y, w.ratio[p * KV8_PAGE + m0 + u].y) << (8 * u);
                }
                x[it][0] = o;
            }
        }
        __syncthreads();
#pragma unroll
        for (int it = 0; it < 8; it++) {
            const int at = tid + it * MOVE_THREADS;
            if (which == 0) {
                const int per = dp / 16, m = at / per, d = at % per * 16;
                if (m < held_here)
                    *reinterpret_cast<uint4 *>(e.c.k + (to * KV8_PAGE + m) * dp + d) = make_uint4(x[it][0], x[it][1], x[it][2], x[it][3]);
            } else {
                const int d = at / 16, m0 = at % 16 * 4;
                signed char *y = e.c.v + (to * dp + d) * KV8_PAGE + m0;
                if (d < dp && m0 + 4 <= held_here) *reinterpret_cast<unsigned *>(y) = x[it][0];
                else if (d < dp)
                    for (int u = 0; m0 + u < held_here; u++) y[u] = (signed char)(x[it][0] >> (8 * u));
            }
        }
        if (which == 0 && tid == 0) {
            e.c.scales[to] = w.scales[p];
            e.c.bad[to] = w.bad[p];
        }
        __syncthreads();
    }
}

// Last, for lens_out may be lens.
__global__ void k_kv8_lens(Kv8Evict e, void *ws) {
    const int i = blockIdx.x * 64 + threadIdx.x;
    if (i < e.s.n_seq) e.lens_out[i] = work_of(ws, e.budget, (int64_t)i * e.c.hk).state[2];
}

}  // namespace

size_t kv8_evict_bytes(const Kv8View &c, const Kv8Seqs &s, int budget) {
    return (size_t)s.n_seq * c.hk * work_size(budget);
}

hipError_t launch_kv8_evict(const Kv8Evict &e, void *ws, hipStream_t st) {
    const int64_t pairs = (int64_t)e.s.n_seq * e.c.hk;
    if (pairs == 0) return hipSuccess;
    if (!kv8_grid(pairs, CHOOSE_THREADS) || !kv8_grid(2 * pairs, MOVE_THREADS)) return hipErrorInvalidValue;
    hipLaunchKernelGGL(k_kv8_choose, dim3(pairs), dim3(CHOOSE_THREADS), 0, st, e, ws);
    hipLaunchKernelGGL(k_kv8_move, dim3(2 * pairs), dim3(MOVE_THREADS), 0, st, e, ws);
    if (e.lens_out) hipLaunchKernelGGL(k_kv8_lens, dim3((e.s.n_seq + 63) / 64), dim3(64), 0, st, e, ws);
    return hipGetLastError();
}

}  // namespace cih

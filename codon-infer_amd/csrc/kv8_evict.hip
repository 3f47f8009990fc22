// Eviction from the 8-bit cache by accumulated attention weight.  Each kv head of a
// sequence of more than `budget` tokens keeps its first `first` tokens, its last `recent`
// ones and the `budget - first - recent` of the others with the largest weights (ties: the
// earlier token); what is kept moves to the sequence's first `budget` places, in order.
//
// k_kv8_choose (a workgroup per sequence and head) finds the kept tokens' places; k_kv8_move moves their
// codes and makes the new pages' records.  A page's new scale is the largest of the
// pages that its tokens come from, so codes are rounded again only where their page's scale
// grows: a token that moves many times is not rounded each time.
#include "kernels.h"
#include "kv8.h"

namespace cih {

namespace {

constexpr int MOVE_THREADS = 256;

// Of each (sequence, head), in the workspace.
struct Work {
    int4 *state;    // tokens held, tokens kept, whether they move, the next page to move
    int2 *list;     // [tokens]: the kept ones, place and page
    float *weight;  // [tokens]
    int *read;      // [pages]: whether this page's tokens have been read
    int *rank;      // [pages + 1]: how many kept tokens come from pages before this one
    int pages;
};
__host__ __device__ inline size_t work_size(int budget) {  // a multiple of 16 bytes
    const size_t pages = (budget + KV8_PAGE - 1) / KV8_PAGE, tokens = pages * KV8_PAGE;
    return sizeof(int4) + tokens * (sizeof(int2) + sizeof(float)) + ((2 * pages + 1) * sizeof(int) + 15) / 16 * 16;
}
__device__ __forceinline__ Work work_of(void *ws, int budget, int64_t pair) {
    char *p = static_cast<char *>(ws) + pair * work_size(budget);
    Work w;
    w.pages = (budget + KV8_PAGE - 1) / KV8_PAGE;
    w.state = reinterpret_cast<int4 *>(p);
    w.list = reinterpret_cast<int2 *>(w.state + 1);
    w.weight = reinterpret_cast<float *>(w.list + (int64_t)w.pages * KV8_PAGE);
    w.read = reinterpret_cast<int *>(w.weight + (int64_t)w.pages * KV8_PAGE);
    w.rank = w.read + w.pages;
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

// Sum of v over the threads before this one, and over all.
template <int NT> __device__ __forceinline__ int block_scan(int v, int *part, int &all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();  // part was read
    if (lane == 63) part[wave] = x;
    __syncthreads();
    int before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; w++) {
        if (w < wave) before += part[w];
        all += part[w];
    }
    return before + x - v;
}

// NT threads; a wave owns a run of pages, token `lane` of each in a lane.  The smallest key that
// is kept is found by its digits from the highest on (12, 12 and 8 bits), each from a
// histogram of the keys that have the digits before it.  A wave keeps the weights of its first NK pages in
// registers and of the next NL in LDS; those behind are read again for each digit.
constexpr int RUN = 8;
template <int NT, int NK, int NL> __global__ __launch_bounds__(NT) void k_kv8_choose(Kv8Evict e, void *ws) {
    constexpr int BINS = 4096, PER = BINS / NT, NW = NT / 64;
    __shared__ int hist[BINS], part[NW], found[2], count[2][NW];
    __shared__ float in_lds[NL > 0 ? NW * NL * KV8_PAGE : 1];
    const int h = blockIdx.x % e.c.hk, i = blockIdx.x / e.c.hk;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Held q = held(e.s, i);
    const Work w = work_of(ws, e.budget, blockIdx.x);
    int *kept = e.kept ? e.kept + (int64_t)blockIdx.x * e.budget : nullptr;
    const int pages = (q.n + KV8_PAGE - 1) / KV8_PAGE;
    const int own = (pages + NW - 1) / NW;  // pages of a wave
    const int first = min(wave * own, pages), last = min(first + own, pages);
    auto there = [&](int id) __attribute__((always_inline)) { return id >= 0 && id < e.c.n_pages; };
    // (0: no such page of the wave)
    auto id_of = [&](int p) __attribute__((always_inline)) { return p < last ? __builtin_amdgcn_readfirstlane(q.table[p]) : 0; };
    auto weight_at = [&](int id, int p) __attribute__((always_inline)) {
        return p < last && there(id) && p * KV8_PAGE + lane < q.n ? e.weights[((int64_t)id * e.c.hk + h) * KV8_PAGE + lane] : 0.0f;
    };
    if (tid == 0) found[0] = 0;
#pragma unroll
    for (int k = 0; k < PER; k++) hist[k * NT + tid] = 0;
    __syncthreads();
    const int lo = e.first, hi = q.n - e.recent, need = e.budget - e.first - e.recent;
    auto top = [&](int j, float y) __attribute__((always_inline)) {  // the first digit
        if (j >= lo && j < hi) atomicAdd(&hist[weight_key(y) >> 20], 1);
    };
    // Every page has to be there: a wave's first pages, then runs of those behind.
    float x[NK];
    int id[NK];
    bool gone = q.table == nullptr;
    if (!gone) {
#pragma unroll
        for (int k = 0; k < NK; k++) id[k] = id_of(first + k);
#pragma unroll
        for (int k = 0; k < NK; k++) {
            gone |= !there(id[k]);
            x[k] = weight_at(id[k], first + k);
        }
#pragma unroll
        for (int k = 0; k < NK; k++)
            if (first + k < last) top((first + k) * KV8_PAGE + lane, x[k]);
        for (int p = first + NK; p < last; p += RUN) {
            int is[RUN];
            float y[RUN];
#pragma unroll
            for (int k = 0; k < RUN; k++) is[k] = id_of(p + k);
#pragma unroll
            for (int k = 0; k < RUN; k++) {
                gone |= !there(is[k]);
                y[k] = weight_at(is[k], p + k);
            }
#pragma unroll
            for (int k = 0; k < RUN; k++)
                if (p + k < last) {
                    top((p + k) * KV8_PAGE + lane, y[k]);
                    const int at = p + k - first - NK;
                    if (at < NL) in_lds[(wave * NL + at) * KV8_PAGE + lane] = y[k];
                }
        }
    }
    if (gone && q.n > 0) found[0] = 1;
    __syncthreads();
    const int n = found[0] != 0 ? 0 : q.n;
    // f(token, weight, page id) for each token of the lane, in order
    auto tokens = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < NK; k++)
            if (first + k < last) f((first + k) * KV8_PAGE + lane, x[k], id[k]);
        for (int p = first + NK; p < last; p += RUN) {
            int is[RUN];
            float y[RUN];
            const bool near = p + RUN <= first + NK + NL;
#pragma unroll
            for (int k = 0; k < RUN; k++) is[k] = id_of(p + k);
#pragma unroll
            for (int k = 0; k < RUN; k++)
                y[k] = near ? in_lds[(wave * NL + p + k - first - NK) * KV8_PAGE + lane] : weight_at(is[k], p + k);
#pragma unroll
            for (int k = 0; k < RUN; k++)
                if (p + k < last) f((p + k) * KV8_PAGE + lane, y[k], is[k]);
        }
    };
    if (tid == 0) *w.state = make_int4(q.n, min(n, e.budget), n > e.budget, 0);
    if (n <= e.budget) {  // stays as it is
        for (int m = tid; kept && m < e.budget; m += NT) kept[m] = m < n ? m : -1;
        if (n > 0)
            tokens([&](int j, float y, int) __attribute__((always_inline)) {
                if (j < n) w.weight[j] = y;
            });
        return;
    }
    for (int p = tid; p < w.pages; p += NT) w.read[p] = 0;
    // of tokens [lo, hi) fewer are kept than there are
    unsigned border = 0xffffffffu;  // (need 0: above all keys)
    int equal = need;               // kept of those at the border
    if (need > 0) {
        border = 0;
        for (int pass = 0; pass < 3; pass++) {
            const int shift = pass == 0 ? 20 : pass == 1 ? 8 : 0, mask = pass < 2 ? 4095 : 255;
            if (pass > 0) {
                const int known = pass == 1 ? 20 : 8;
#pragma unroll
                for (int k = 0; k < PER; k++) hist[k * NT + tid] = 0;
                __syncthreads();
                tokens([&](int j, float y, int) __attribute__((always_inline)) {
                    const unsigned key = weight_key(y);
                    if (j >= lo && j < hi && key >> known == border >> known) atomicAdd(&hist[key >> shift & mask], 1);
                });
                __syncthreads();
            }
            // the largest first: thread t has bins BINS - 1 - PER t and below
            int mine[PER], sum = 0, all;
#pragma unroll
            for (int k = 0; k < PER; k++) sum += mine[k] = hist[BINS - 1 - PER * tid - k];
            int before = block_scan<NT>(sum, part, all);
            if (before < equal && before + sum >= equal)
#pragma unroll
                for (int k = 0; k < PER; k++) {
                    if (before < equal && before + mine[k] >= equal) {
                        found[0] = BINS - 1 - PER * tid - k;
                        found[1] = equal - before;
                    }
                    before += mine[k];
                }
            __syncthreads();
            border |= (unsigned)found[0] << shift;
            equal = found[1];
            __syncthreads();
        }
    }
    auto sure_of = [&](int j, float y) __attribute__((always_inline)) { return j < n && (j < lo || j >= hi || weight_key(y) > border); };
    auto at_of = [&](int j, float y) __attribute__((always_inline)) { return j >= lo && j < hi && weight_key(y) == border; };
    // in order: all above the border, the first of those at it
    int sure = 0, ties = 0;
    tokens([&](int j, float y, int) __attribute__((always_inline)) {
        sure += __popcll(__ballot(sure_of(j, y)));
        ties += __popcll(__ballot(at_of(j, y)));
    });
    if (lane == 0) {
        count[0][wave] = sure;
        count[1][wave] = ties;
    }
    __syncthreads();
    sure = ties = 0;
    for (int u = 0; u < wave; u++) {
        sure += count[0][u];
        ties += count[1][u];
    }
    tokens([&](int j, float y, int id) __attribute__((always_inline)) {
        const unsigned long long below = (1ull << lane) - 1, a = __ballot(at_of(j, y)), b = __ballot(sure_of(j, y));
        const int t = ties + __popcll(a & below), m = sure + __popcll(b & below) + min(t, equal);
        if (lane == 0 && j / KV8_PAGE <= w.pages) w.rank[j / KV8_PAGE] = m;
        if (b >> lane & 1 || (a >> lane & 1 && t < equal)) {
            w.list[m] = make_int2(j, id);
            w.weight[m] = y;
            if (kept) kept[m] = j;
        }
        sure += __popcll(b);
        ties += __popcll(a);
    });
    if (tid == 0 && pages <= w.pages) w.rank[pages] = e.budget;
}

// Four codes scaled by r <= 1: u - 128 is the code, the fused product is rounded
// once, as code r is, and 1.5 2^23 rounds it to a whole number in the low bits.
__device__ __forceinline__ unsigned shrink4(unsigned w, float r) {
    const unsigned u = w ^ 0x80808080u;
    unsigned o[4];
#pragma unroll
    for (int b = 0; b < 4; b++) {
        const float x = fmaf((float)(u >> (8 * b) & 0xff), r, -128.0f * r);
        o[b] = __float_as_uint(x + 12582912.0f);
    }
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(o[3], o[2], 0x0c0c0400u), __builtin_amdgcn_perm(o[1], o[0], 0x0c0c0400u), 0x05040100u);
}

// One workgroup per (sequence, head, page that is filled).  Token m of the kept ones comes from
// place m or a later one, so a page and its record may be written once the pages before it that take tokens from it
// have read them.  A workgroup draws its page's number when it starts: those that it waits for have
// started before it, and say that they have read before they wait themselves.
template <int DP> __global__ __launch_bounds__(MOVE_THREADS) void k_kv8_move(Kv8Evict e, void *ws, int pages) {
    constexpr int KP = (DP / 16 * KV8_PAGE + MOVE_THREADS - 1) / MOVE_THREADS, VP = DP * 16 / MOVE_THREADS;
    __shared__ int spage;
    __shared__ float2 sratio[KV8_PAGE];
    const int64_t pair = blockIdx.x / pages;
    const int h = pair % e.c.hk, i = pair / e.c.hk, tid = threadIdx.x, lane = tid & 63;
    const Work w = work_of(ws, e.budget, pair);
    int p = blockIdx.x % pages;
    if (tid == 0) spage = atomicAdd(&w.state->w, 1);
    const int slot = e.s.slots ? e.s.slots[i] : i;  // (sequences of slots that are not there have nothing to move)
    const int *table = e.s.table + (int64_t)slot * e.s.table_stride;
    const int held = w.state->x, n = w.state->y;
    const bool moves = w.state->z != 0;
    if (p == 0 && h == 0 && tid == 0) {
        // (a sequence that is left alone keeps its length, also one that is not there)
        if (moves) e.lens_out[i] = e.budget;
        else if (e.lens_out != e.s.lens) e.lens_out[i] = e.s.lens[i];
        if (moves && e.shifts) e.shifts[i] += held - e.budget;
    }
    __syncthreads();
    if (moves) p = spage;
    const int m0 = p * KV8_PAGE, here = min(KV8_PAGE, n - m0);
    if (here <= 0) return;
    const int64_t to = (int64_t)table[p] * e.c.hk + h;
    if (tid < here && e.weights_out) e.weights_out[to * KV8_PAGE + tid] = w.weight[m0 + tid];
    if (!moves) return;
    auto source = [&](int m) __attribute__((always_inline)) { return w.list[m0 + min(m, here - 1)]; };
    const int2 mine = source(lane);
    const int r0 = w.rank[p], r1 = w.rank[p + 1];
    // (the last token in its own place: so are all, and the record is what it was)
    const bool stays = here == KV8_PAGE && __shfl(mine.x, KV8_PAGE - 1) == m0 + KV8_PAGE - 1;
    uint4 k[KP];
    unsigned v[VP];
    float2 now = {0.0f, 0.0f};
    unsigned long long bad = 0;
    if (!stays) {
        // K: 16 dims of a token; V: four tokens of a dim
#pragma unroll
        for (int it = 0; it < KP; it++) {
            const int at = tid + it * MOVE_THREADS;
            const int2 s = source(at / (DP / 16));
            k[it] = *reinterpret_cast<const uint4 *>(
                e.c.k + (((int64_t)s.y * e.c.hk + h) * KV8_PAGE + s.x % KV8_PAGE) * DP + at % (DP / 16) * 16);
        }
        const int vm = tid % 16 * 4;
        unsigned char b[VP][4];
        const signed char *src[4];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int2 s = source(vm + u);
            src[u] = e.c.v + (((int64_t)s.y * e.c.hk + h) * DP + tid / 16) * KV8_PAGE + s.x % KV8_PAGE;
        }
#pragma unroll
        for (int it = 0; it < VP; it++)
#pragma unroll
            for (int u = 0; u < 4; u++) b[it][u] = (unsigned char)src[u][it * (MOVE_THREADS / 16) * KV8_PAGE];
        // the new record: the largest scales, the tokens' bad bits (each wave for itself)
        const int64_t ph = (int64_t)mine.y * e.c.hk + h;
        const float2 old = e.c.scales[ph];
        bad = __ballot(lane < here && e.c.bad[ph] >> (mine.x % KV8_PAGE) & 1);
        // (not negative: as bits they compare alike)
        now = {__uint_as_float(wave_max_bits(__float_as_uint(old.x))), __uint_as_float(wave_max_bits(__float_as_uint(old.y)))};
        if (tid < KV8_PAGE) sratio[tid] = {now.x > 0.0f ? old.x / now.x : 0.0f, now.y > 0.0f ? old.y / now.y : 0.0f};
        __syncthreads();
#pragma unroll
        for (int it = 0; it < KP; it++) {
            const float r = sratio[(tid + it * MOVE_THREADS) / (DP / 16) % KV8_PAGE].x;
            k[it] = make_uint4(shrink4(k[it].x, r), shrink4(k[it].y, r), shrink4(k[it].z, r), shrink4(k[it].w, r));
        }
        float r[4];
#pragma unroll
        for (int u = 0; u < 4; u++) r[u] = sratio[vm + u].y;
#pragma unroll
        for (int it = 0; it < VP; it++) {
            unsigned o[4];
#pragma unroll
            for (int u = 0; u < 4; u++)
                o[u] = __float_as_uint(fmaf((float)(b[it][u] ^ 0x80), r[u], -128.0f * r[u]) + 12582912.0f);
            v[it] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(o[3], o[2], 0x0c0c0400u), __builtin_amdgcn_perm(o[1], o[0], 0x0c0c0400u), 0x05040100u);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // every wave's loads have come back
    __syncthreads();
    if (tid == 0) __hip_atomic_store(&w.read[p], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (stays) return;
    // pages that take tokens from this one: 64 tokens go to two at most
    if (r0 < r1) {
        const int q = r0 / KV8_PAGE + tid;
        if (q <= (r1 - 1) / KV8_PAGE && q < p)
            while (!__hip_atomic_load(&w.read[q], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) __builtin_amdgcn_s_sleep(1);
    }
    __syncthreads();
#pragma unroll
    for (int it = 0; it < KP; it++) {
        const int at = tid + it * MOVE_THREADS, m = at / (DP / 16);
        if (m < here) *reinterpret_cast<uint4 *>(e.c.k + (to * KV8_PAGE + m) * DP + at % (DP / 16) * 16) = k[it];
    }
    const int vm = tid % 16 * 4;
#pragma unroll
    for (int it = 0; it < VP; it++) {
        signed char *y = e.c.v + (to * DP + tid / 16 + it * (MOVE_THREADS / 16)) * KV8_PAGE + vm;
        if (vm + 4 <= here) *reinterpret_cast<unsigned *>(y) = v[it];
        else
            for (int u = 0; vm + u < here; u++) y[u] = (signed char)(v[it] >> (8 * u));
    }
    if (tid == 0) {
        e.c.scales[to] = now;
        e.c.bad[to] = bad;
    }
}

}  // namespace

size_t kv8_evict_bytes(const Kv8View &c, const Kv8Seqs &s, int budget) {
    return (size_t)s.n_seq * c.hk * work_size(budget);
}

hipError_t launch_kv8_evict(const Kv8Evict &e, void *ws, hipStream_t st) {
    const int64_t pairs = (int64_t)e.s.n_seq * e.c.hk, most = (int64_t)e.s.max_pages * KV8_PAGE;
    if (pairs == 0) return hipSuccess;
    const int pages = (int)min((int64_t)(e.budget + KV8_PAGE - 1) / KV8_PAGE, (int64_t)e.s.max_pages);
    if (!kv8_grid(pairs, 1024) || !kv8_grid(pairs * pages, MOVE_THREADS)) return hipErrorInvalidValue;
    if (most <= 2048) hipLaunchKernelGGL((k_kv8_choose<256, 8, 0>), dim3(pairs), dim3(256), 0, st, e, ws);
    else if (most <= 8192) hipLaunchKernelGGL((k_kv8_choose<1024, 8, 0>), dim3(pairs), dim3(1024), 0, st, e, ws);
    else hipLaunchKernelGGL((k_kv8_choose<1024, 32, 32>), dim3(pairs), dim3(1024), 0, st, e, ws);
    const dim3 grid(pairs * pages), threads(MOVE_THREADS);
    switch (e.c.dp) {
        case 16: hipLaunchKernelGGL(k_kv8_move<16>, grid, threads, 0, st, e, ws, pages); break;
        case 32: hipLaunchKernelGGL(k_kv8_move<32>, grid, threads, 0, st, e, ws, pages); break;
        case 64: hipLaunchKernelGGL(k_kv8_move<64>, grid, threads, 0, st, e, ws, pages); break;
        case 128: hipLaunchKernelGGL(k_kv8_move<128>, grid, threads, 0, st, e, ws, pages); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace cih

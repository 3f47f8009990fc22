// Eviction from the 8-bit cache by accumulated attention weight.  Each kv head of a
// sequence of more than `budget` tokens keeps its first `first` tokens, its last `recent`
// ones and the `budget - first - recent` of the others with the largest weights (ties: the
// earlier token); what is kept moves to the sequence's first `budget` places, in order.
//
// k_kv8_choose (a workgroup per sequence and head) finds the kept tokens' places; k_kv8_move moves their
// codes and makes the new pages' records.  A page's new scale is the largest of the
// pages that its tokens come from, so codes are rounded again only where their page's scale
// grows: a token that moves many times is not rounded each time.
#include <stdlib.h>

#include <type_traits>

#include "kernels.h"
#include "kv8.h"

namespace cih {

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// Of each (sequence, head), in the workspace.
struct Work {
    int4 *state;    // the sequence's length, tokens kept, whether they move, the next run of pages to move
    int2 *list;     // [tokens]: the kept ones, place and page
    float *weight;  // [tokens]
    int *read;      // [pages]: whether this page's tokens have been read
    int *rank;      // [pages + 1]: how many kept tokens come from pages before this one
    int pages;
};
__host__ __device__ inline size_t work_size(int room) {  // a multiple of 16 bytes
    const size_t pages = ((size_t)room + KV8_PAGE - 1) / KV8_PAGE, tokens = pages * KV8_PAGE;
    return sizeof(int4) + tokens * (sizeof(int2) + sizeof(float)) +
           ((2 * pages + 1) * sizeof(int) + 15) / 16 * 16;
}
__device__ __forceinline__ Work work_of(const Kv8Evict &e, void *ws, int64_t pair) {
    char *p = static_cast<char *>(ws) + pair * work_size(e.room);
    Work w;
    w.pages = (e.room + KV8_PAGE - 1) / KV8_PAGE;
    w.state = reinterpret_cast<int4 *>(p);
    w.list = reinterpret_cast<int2 *>(w.state + 1);
    w.weight = reinterpret_cast<float *>(w.list + (int64_t)w.pages * KV8_PAGE);
    w.read = reinterpret_cast<int *>(w.weight + (int64_t)w.pages * KV8_PAGE);
    w.rank = w.read + w.pages;
    return w;
}

// Larger weights have larger keys, all between NAN_KEY and SURE; -0 counts as 0, NaN is below every other.
constexpr unsigned NO_KEY = 0, NAN_KEY = 1, ZERO_KEY = 0x80000000u, SURE = 0xffffffffu;
__device__ __forceinline__ unsigned weight_key(float x) {
    const unsigned b = __float_as_uint(x + 0.0f);
    return x != x ? NAN_KEY : b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_weight(unsigned k) { return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k); }

// Whether weights of sequences that stay as they are go anywhere.
__device__ __forceinline__ bool copies(const Kv8Evict &e) { return e.weights_out && e.weights_out != e.weights; }

// Tokens a sequence holds (of its length those that the table has room for), its row of the table, its length.
struct Held {
    int n;
    const int *table;
    int len;
};
__device__ __forceinline__ Held held(const Kv8Seqs &s, int i) {
    const int slot = s.slots ? s.slots[i] : i;
    return {(int)min((int64_t)max(s.lens[i], 0), (int64_t)s.max_pages * KV8_PAGE),
            slot >= 0 && slot < s.table_rows ? s.table + (int64_t)slot * s.table_stride : nullptr, s.lens[i]};
}

// Tokens of a sequence and head as a wave sees them: a page's token `lane` in a lane.
struct Tokens {
    const Kv8Evict &e;
    Held q;
    int h, lane;
    __device__ __forceinline__ bool there(int id) const { return id >= 0 && id < e.c.n_pages; }
    __device__ __forceinline__ int id(int p, int last) const { return p < last ? __builtin_amdgcn_readfirstlane(q.table[p]) : 0; }
    __device__ __forceinline__ float weight(int id, int p, int last) const {
        return p < last && there(id) && p * KV8_PAGE + lane < q.n ? e.weights[((int64_t)id * e.c.hk + h) * KV8_PAGE + lane] : 0.0f;
    }
    // kept for sure, not there, or by its weight
    __device__ __forceinline__ unsigned key(int p, float y) const {
        const int j = p * KV8_PAGE + lane;
        const unsigned k = j < e.first || j >= q.n - e.recent ? SURE : weight_key(y);
        return j < q.n ? k : NO_KEY;
    }
};
// A sequence that stays as it is has no weights looked at, only whether its pages are there.
__device__ __forceinline__ Held looked_at(const Kv8Evict &e, const Held &q) { return {q.n > e.budget ? q.n : 0, q.table, q.len}; }
__device__ __forceinline__ bool chosen(unsigned key) { return key - 1 < SURE - 1; }  // by its weight
// A kept token's weight (a key of 0 or NaN does not have all of it).
__device__ __forceinline__ bool has_weight(unsigned key) { return key != SURE && key != NAN_KEY && key != ZERO_KEY; }

// Where bin i of the histogram stands, so that threads that read runs of 4 or 16 bins meet no bank twice.
__device__ __forceinline__ int bin(int i) { return i ^ (i >> 5 & 31); }

// Running sum over the wave's lanes (shifts within rows of 16 lanes, then their last lanes' sums to the rows behind).
template <int C, int ROWS> __device__ __forceinline__ int dpp_or_0(int v) { return __builtin_amdgcn_update_dpp(0, v, C, ROWS, 0xf, false); }
__device__ __forceinline__ int wave_scan(int v) {
    v += dpp_or_0<0x111, 0xf>(v);
    v += dpp_or_0<0x112, 0xf>(v);
    v += dpp_or_0<0x114, 0xf>(v);
    v += dpp_or_0<0x118, 0xf>(v);
    v += dpp_or_0<0x142, 0xa>(v);
    v += dpp_or_0<0x143, 0xc>(v);
    return v;
}
// Sum of v over the threads before this one.
template <int NT> __device__ __forceinline__ int block_scan(int v, int *part) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int x = wave_scan(v);
    if (lane == 63) part[wave] = x;
    __syncthreads();
    int before = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; w++)
        if (w < wave) before += part[w];
    return before + x - v;
}

// The bin in which the `want` largest end, and how many of it are among them, of a histogram whose bins BINS - 1 - PER
// t and below thread t has in `mine`.
constexpr int BINS = 4096;
template <int NT> __device__ __forceinline__ int2 bin_of(const int (&mine)[BINS / NT], int want, int *part, int *found) {
    constexpr int PER = BINS / NT;
    int sum = 0;
#pragma unroll
    for (int k = 0; k < PER; k++) sum += mine[k];
    int before = block_scan<NT>(sum, part);
    if (before < want && before + sum >= want)
#pragma unroll
        for (int k = 0; k < PER; k++) {
            if (before < want && before + mine[k] >= want) {
                found[0] = BINS - 1 - PER * (int)threadIdx.x - k;
                found[1] = want - before;
            }
            before += mine[k];
        }
    __syncthreads();
    return make_int2(found[0], found[1]);  // (next written behind block_scan's barrier)
}
// The same of a histogram in LDS, which is cleared.
template <int NT> __device__ __forceinline__ int2 bin_of_hist(int *hist, int want, int *part, int *found) {
    constexpr int PER = BINS / NT;
    int mine[PER];
#pragma unroll
    for (int k = 0; k < PER; k++) {
        int &c = hist[bin(BINS - 1 - PER * (int)threadIdx.x - k)];
        mine[k] = c;
        c = 0;
    }
    return bin_of<NT>(mine, want, part, found);
}

// NT threads; a wave owns a run of pages, token `lane` of each in a lane.  The smallest key that
// is kept is found by its digits from the highest on (12, 12 and 8 bits), each from a
// histogram of the keys that have the digits before it.  A wave keeps the keys of its first NK pages in
// registers and of the next NL in LDS; those behind are read again for each digit.  Bound by its chain of loads, scans
// and barriers: 8 sequences of 577 tokens, 20 heads, 9 us (bins that share a bank 13), 32 of 1,900 to 6,000, 8 heads, 15.
constexpr int RUN = 8;
template <int NT, int NK, int NL> __global__ __launch_bounds__(NT) void k_kv8_choose(Kv8Evict e, void *ws) {
    constexpr int PER = BINS / NT, NW = NT / 64;
    __shared__ int hist[BINS], part[NW], found[2], count[2][NW];
    __shared__ unsigned in_lds[NL > 0 ? NW * NL * KV8_PAGE : 1];
    const int h = blockIdx.x % e.c.hk, i = blockIdx.x / e.c.hk;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Held q = held(e.s, i);
    const Work w = work_of(e, ws, blockIdx.x);
    int *kept = e.kept ? e.kept + (int64_t)blockIdx.x * e.budget : nullptr;
    const int pages = (q.n + KV8_PAGE - 1) / KV8_PAGE;
    const int own = (pages + NW - 1) / NW;  // pages of a wave
    const int first = min(wave * own, pages), last = min(first + own, pages);
    const Tokens z{e, q, h, lane}, look{e, looked_at(e, q), h, lane};
    if (tid == 0) found[0] = 0;
#pragma unroll
    for (int k = 0; k < PER; k++) hist[k * NT + tid] = 0;
    __syncthreads();
    const int need = e.budget - e.first - e.recent;
    auto top = [&](unsigned key) __attribute__((always_inline)) {  // the first digit
        if (chosen(key)) atomicAdd(&hist[bin(key >> 20)], 1);
    };
    // Every page has to be there: a wave's first pages, then runs of those behind.
    unsigned x[NK];
    int id[NK];
    bool gone = q.table == nullptr;
    if (!gone) {
#pragma unroll
        for (int k = 0; k < NK; k++) id[k] = z.id(first + k, last);
        float y[NK];
#pragma unroll
        for (int k = 0; k < NK; k++) {
            gone |= !z.there(id[k]);
            y[k] = look.weight(id[k], first + k, last);
        }
#pragma unroll
        for (int k = 0; k < NK; k++) {
            x[k] = first + k < last ? look.key(first + k, y[k]) : NO_KEY;
            top(x[k]);
        }
        for (int p = first + NK; p < last; p += RUN) {
            int is[RUN];
            float y[RUN];
#pragma unroll
            for (int k = 0; k < RUN; k++) is[k] = z.id(p + k, last);
#pragma unroll
            for (int k = 0; k < RUN; k++) {
                gone |= !z.there(is[k]);
                y[k] = look.weight(is[k], p + k, last);
            }
#pragma unroll
            for (int k = 0; k < RUN; k++)
                if (p + k < last) {
                    const unsigned key = look.key(p + k, y[k]);
                    top(key);
                    const int at = p + k - first - NK;
                    if (at < NL) in_lds[(wave * NL + at) * KV8_PAGE + lane] = key;
                }
        }
    }
    if (gone && q.n > 0) found[0] = 1;
    __syncthreads();
    const int n = found[0] != 0 ? 0 : q.n;
    // f(page, key, page id) for the wave's pages, in order
    auto tokens = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < NK; k++)
            if (first + k < last) f(first + k, x[k], id[k]);
        for (int p = first + NK; p < last; p += RUN) {
            int is[RUN];
            unsigned y[RUN];
            const bool near = p + RUN <= first + NK + NL;
#pragma unroll
            for (int k = 0; k < RUN; k++) is[k] = z.id(p + k, last);
#pragma unroll
            for (int k = 0; k < RUN; k++)
                y[k] = near ? in_lds[(wave * NL + p + k - first - NK) * KV8_PAGE + lane]
                            : z.key(p + k, z.weight(is[k], p + k, last));
#pragma unroll
            for (int k = 0; k < RUN; k++)
                if (p + k < last) f(p + k, y[k], is[k]);
        }
    };
    if (tid == 0) *w.state = make_int4(q.len, min(n, e.budget), n > e.budget, 0);
    if (n <= e.budget) {  // stays as it is
        for (int m = tid; kept && m < e.budget; m += NT) kept[m] = m < n ? m : -1;
        if (n > 0 && copies(e))
            tokens([&](int p, unsigned, int id) __attribute__((always_inline)) {
                if (p * KV8_PAGE + lane < n) w.weight[p * KV8_PAGE + lane] = z.weight(id, p, last);
            });
        return;
    }
    for (int p = tid; p < w.pages; p += NT) w.read[p] = 0;
    // of tokens [lo, hi) fewer are kept than there are
    unsigned border = SURE - 1;  // (need 0: above all keys)
    int equal = need;            // kept of those at the border
    if (need > 0) {
        border = 0;
        for (int pass = 0; pass < 3; pass++) {
            const int shift = pass == 0 ? 20 : pass == 1 ? 8 : 0, mask = pass < 2 ? 4095 : 255;
            if (pass > 0) {
                const int known = pass == 1 ? 20 : 8;
                tokens([&](int, unsigned key, int) __attribute__((always_inline)) {
                    if (key >> known == border >> known && chosen(key)) atomicAdd(&hist[bin(key >> shift & mask)], 1);
                });
                __syncthreads();
            }
            const int2 bin = bin_of_hist<NT>(hist, equal, part, found);
            border |= (unsigned)bin.x << shift;
            equal = bin.y;
        }
    }
    // in order: all above the border, the first of those at it
    int sure = 0, ties = 0;
    tokens([&](int, unsigned key, int) __attribute__((always_inline)) {
        sure += __popcll(__ballot(key > border));
        ties += __popcll(__ballot(key == border));
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
    tokens([&](int p, unsigned key, int id) __attribute__((always_inline)) {
        const unsigned long long below = (1ull << lane) - 1, a = __ballot(key == border), b = __ballot(key > border);
        const int t = ties + __popcll(a & below), m = sure + __popcll(b & below) + min(t, equal);
        if (lane == 0 && p <= w.pages) w.rank[p] = m;
        if (key > border || (key == border && t < equal)) {
            w.list[m] = make_int2(p * KV8_PAGE + lane, id);
            w.weight[m] = has_weight(key) ? key_weight(key) : z.weight(id, p, last);
            if (kept) kept[m] = p * KV8_PAGE + lane;
        }
        sure += __popcll(b);
        ties += __popcll(a);
    });
    if (tid == 0 && pages <= w.pages) w.rank[pages] = e.budget;
}

// The same for a long table and few heads, by several workgroups (parts) of each sequence and head in three launches: each
// part's histogram of the first digit; its tokens of the border's bin, when all parts' histograms are summed; the list, when all those
// tokens' other digits are looked at.  40 heads of 65,003 tokens: 8 + 13 + 17 us, one workgroup of each 84 (it is bound by the instructions
// of one CU), a launch for each of four digits of 8 bits and one for the list 74, 12 parts in two turns 9 + 24 + 23.  Each launch waits
// for what others wrote: loads that do not depend on each other are all under way together.
constexpr int PART_THREADS = 1024, PART_WAVES = PART_THREADS / 64, MOST_PARTS = 8;  // (one for a wave of the list's workgroups at most)
struct Parts {
    int2 *top;       // the border's first digit, and how many are kept of those that have it
    int *above;      // [MOST_PARTS]: a part's tokens chosen for a larger first digit
    int *near;       // [MOST_PARTS]: those with the border's
    int *gone;       // [MOST_PARTS]: whether a page of the part is not there
    int *hist;       // [parts][BINS]
    unsigned *keys;  // [tokens of the table]: from a part's first token on, the keys of those with the border's first digit
};
inline size_t parts_size(int n, int max_pages) {
    return (4 + 3 * MOST_PARTS + (size_t)n * BINS + (size_t)max_pages * KV8_PAGE) * sizeof(int);  // a multiple of 16 bytes
}
struct Part {
    int64_t pair;
    int own, first, last, begin;  // part; pages of this wave; the part's first page
    int *hist;
    Parts t;
};
__device__ __forceinline__ Part part_of(const Kv8Evict &e, char *ws, int parts, int64_t size, const Held &q, int64_t pair) {
    Part a;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int pages = (q.n + KV8_PAGE - 1) / KV8_PAGE, each = (pages + parts * PART_WAVES - 1) / (parts * PART_WAVES);
    a.pair = pair;
    a.own = blockIdx.x % parts;
    a.begin = min(a.own * PART_WAVES * each, pages);
    a.first = min(a.begin + wave * each, pages);
    a.last = min(a.first + each, pages);
    a.t.top = reinterpret_cast<int2 *>(ws + pair * size);
    a.t.above = reinterpret_cast<int *>(a.t.top + 2);
    a.t.near = a.t.above + MOST_PARTS;
    a.t.gone = a.t.near + MOST_PARTS;
    a.t.hist = a.t.gone + MOST_PARTS;
    a.t.keys = reinterpret_cast<unsigned *>(a.t.hist + parts * BINS);
    return a;
}
// f(page, key, page id, weight) for a wave's pages, in order.
template <class F> __device__ __forceinline__ void each_page(const Tokens &z, const Part &a, F f) {
    for (int p = a.first; p < a.last; p += RUN) {
        int id[RUN];
        float y[RUN];
#pragma unroll
        for (int k = 0; k < RUN; k++) id[k] = z.id(p + k, a.last);
#pragma unroll
        for (int k = 0; k < RUN; k++) y[k] = z.weight(id[k], p + k, a.last);
#pragma unroll
        for (int k = 0; k < RUN; k++)
            if (p + k < a.last) f(p + k, z.key(p + k, y[k]), id[k], y[k]);
    }
}
__global__ __launch_bounds__(PART_THREADS) void k_kv8_part(Kv8Evict e, char *ws, int parts, int64_t size) {
    constexpr int PER = BINS / PART_THREADS;
    __shared__ int hist[BINS], gone;
    const int64_t pair = blockIdx.x / parts;
    const int tid = threadIdx.x;
    const Held q = held(e.s, pair / e.c.hk);
    const Tokens z{e, looked_at(e, q), (int)(pair % e.c.hk), tid & 63};
    const Part a = part_of(e, ws, parts, size, q, pair);
    if (tid == 0) gone = 0;
#pragma unroll
    for (int k = 0; k < PER; k++) hist[k * PART_THREADS + tid] = 0;
    __syncthreads();
    bool missing = q.table == nullptr;
    if (!missing)
        each_page(z, a, [&](int, unsigned key, int id, float) __attribute__((always_inline)) {
            missing |= !z.there(id);
            if (chosen(key)) atomicAdd(&hist[bin(key >> 20)], 1);
        });
    if (missing && q.n > 0) gone = 1;
    __syncthreads();
    int4 c;
    c.x = hist[bin(PER * tid)];
    c.y = hist[bin(PER * tid + 1)];
    c.z = hist[bin(PER * tid + 2)];
    c.w = hist[bin(PER * tid + 3)];
    reinterpret_cast<int4 *>(a.t.hist + a.own * BINS)[tid] = c;
    if (tid == 0) a.t.gone[a.own] = gone;
}
__global__ __launch_bounds__(PART_THREADS) void k_kv8_near(Kv8Evict e, char *ws, int parts, int64_t size) {
    constexpr int PER = BINS / PART_THREADS;
    __shared__ int part[PART_WAVES], found[2], above, near;
    const int64_t pair = blockIdx.x / parts;
    const int tid = threadIdx.x, lane = tid & 63;
    const Held q = held(e.s, pair / e.c.hk);
    const Tokens z{e, q, (int)(pair % e.c.hk), lane};
    const Part a = part_of(e, ws, parts, size, q, pair);
    const int need = e.budget - e.first - e.recent;
    if (q.table == nullptr || q.n <= e.budget || need == 0) return;
    if (tid < 2) found[tid] = 0;
    if (tid == 0) above = near = 0;
    int4 c[MOST_PARTS];
#pragma unroll
    for (int k = 0; k < MOST_PARTS; k++)
        c[k] = reinterpret_cast<const int4 *>(a.t.hist + min(k, parts - 1) * BINS)[BINS / PER - 1 - tid];
    int sum[PER] = {}, mine[PER] = {};
#pragma unroll
    for (int k = 0; k < MOST_PARTS; k++) {
        const int v[PER] = {c[k].w, c[k].z, c[k].y, c[k].x};
#pragma unroll
        for (int u = 0; u < PER; u++) {
            sum[u] += k < parts ? v[u] : 0;
            mine[u] = k == a.own ? v[u] : mine[u];
        }
    }
    const int2 top = bin_of<PART_THREADS>(sum, need, part, found);
    int larger = 0;
#pragma unroll
    for (int u = 0; u < PER; u++) larger += BINS - 1 - PER * tid - u > top.x ? mine[u] : 0;
    if (larger > 0) atomicAdd(&above, larger);
    if (a.own == 0 && tid == 0) *a.t.top = top;
    // (in any order)
    unsigned *keys = a.t.keys + (int64_t)a.begin * KV8_PAGE;
    each_page(z, a, [&](int, unsigned key, int, float) __attribute__((always_inline)) {
        if (chosen(key) && (int)(key >> 20) == top.x) keys[atomicAdd(&near, 1)] = key;
    });
    __syncthreads();
    if (tid == 0) {
        a.t.above[a.own] = above;
        a.t.near[a.own] = near;
    }
}
__global__ __launch_bounds__(PART_THREADS) void k_kv8_list(Kv8Evict e, void *ws, char *parts_ws, int parts, int64_t size) {
    constexpr int NK = 8;
    __shared__ int hist[BINS], part[PART_WAVES], found[2], count[2][PART_WAVES], before[2];
    const int64_t pair = blockIdx.x / parts;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Held q = held(e.s, pair / e.c.hk);
    const Tokens z{e, q, (int)(pair % e.c.hk), lane};
    const Work w = work_of(e, ws, pair);
    const Part a = part_of(e, parts_ws, parts, size, q, pair);
    int *kept = e.kept ? e.kept + pair * e.budget : nullptr;
    const int need = e.budget - e.first - e.recent;
    const int pages = (q.n + KV8_PAGE - 1) / KV8_PAGE;
    const int n = __ballot(lane < parts && a.t.gone[min(lane, parts - 1)] != 0) ? 0 : q.n;
    if (a.own == 0 && tid == 0) *w.state = make_int4(q.len, min(n, e.budget), n > e.budget, 0);
    if (n <= e.budget) {  // stays as it is
        for (int m = a.own * PART_THREADS + tid; kept && m < e.budget; m += parts * PART_THREADS) kept[m] = m < n ? m : -1;
        if (n > 0 && copies(e))
            each_page(z, a, [&](int p, unsigned, int, float y) __attribute__((always_inline)) {
                if (p * KV8_PAGE + lane < n) w.weight[p * KV8_PAGE + lane] = y;
            });
        return;
    }
    for (int p = a.own * PART_THREADS + tid; p < w.pages; p += parts * PART_THREADS) w.read[p] = 0;
    unsigned border = SURE - 1;  // (need 0: above all keys)
    int equal = 0;
    if (tid < 2) before[tid] = 0;
    if (need > 0) {
        // wave k has part k's keys of the border's bin: the first NK of a lane in registers
        const int near = wave < parts ? a.t.near[wave] : 0, over = wave < a.own ? a.t.above[wave] : 0;
        const int each = (pages + parts * PART_WAVES - 1) / (parts * PART_WAVES);
        const unsigned *keys = a.t.keys + (int64_t)min(wave * PART_WAVES * each, pages) * KV8_PAGE;
        const int2 top = *a.t.top;
        unsigned x[NK];
#pragma unroll
        for (int k = 0; k < NK; k++) x[k] = k * 64 + lane < near ? keys[k * 64 + lane] : NO_KEY;
        auto others = [&](auto f) __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < NK; k++) f(x[k]);
            for (int k = NK * 64; k < near; k += 64) f(k + lane < near ? keys[k + lane] : NO_KEY);
        };
#pragma unroll
        for (int k = 0; k < BINS / PART_THREADS; k++) hist[k * PART_THREADS + tid] = 0;
        if (tid < 2) found[tid] = 0;
        __syncthreads();
        others([&](unsigned key) __attribute__((always_inline)) {
            if (key != NO_KEY) atomicAdd(&hist[bin(key >> 8 & 4095)], 1);
        });
        __syncthreads();
        int2 b = bin_of_hist<PART_THREADS>(hist, top.y, part, found);
        border = (unsigned)top.x << 20 | (unsigned)b.x << 8;
        others([&](unsigned key) __attribute__((always_inline)) {
            if (key != NO_KEY && key >> 8 == border >> 8) atomicAdd(&hist[bin(key & 255)], 1);
        });
        __syncthreads();
        b = bin_of_hist<PART_THREADS>(hist, b.y, part, found);
        border |= b.x;
        equal = b.y;
        // of the parts before this one
        if (wave < a.own) {
            int sure = 0, ties = 0;
            others([&](unsigned key) __attribute__((always_inline)) {
                sure += __popcll(__ballot(key > border));
                ties += __popcll(__ballot(key == border));
            });
            if (lane == 0) {
                atomicAdd(&before[0], sure + over);
                atomicAdd(&before[1], ties);
            }
        }
    }
    // (those that are kept for sure: the first, and the recent if this part begins among them)
    const int start = a.begin * KV8_PAGE;
    const int fixed = min(start, e.first) + max(min(start, q.n) - (q.n - e.recent), 0);
    int sure = 0, ties = 0;
    each_page(z, a, [&](int, unsigned key, int, float) __attribute__((always_inline)) {
        sure += __popcll(__ballot(key > border));
        ties += __popcll(__ballot(key == border));
    });
    if (lane == 0) {
        count[0][wave] = sure;
        count[1][wave] = ties;
    }
    __syncthreads();
    sure = before[0] + fixed;
    ties = before[1];
    for (int u = 0; u < wave; u++) {
        sure += count[0][u];
        ties += count[1][u];
    }
    each_page(z, a, [&](int p, unsigned key, int id, float y) __attribute__((always_inline)) {
        const unsigned long long below = (1ull << lane) - 1, at = __ballot(key == border), over = __ballot(key > border);
        const int tie = ties + __popcll(at & below), m = sure + __popcll(over & below) + min(tie, equal);
        if (lane == 0 && p <= w.pages) w.rank[p] = m;
        if (key > border || (key == border && tie < equal)) {
            w.list[m] = make_int2(p * KV8_PAGE + lane, id);
            w.weight[m] = y;
            if (kept) kept[m] = p * KV8_PAGE + lane;
        }
        sure += __popcll(over);
        ties += __popcll(at);
    });
    if (a.own == 0 && tid == 0 && pages <= w.pages) w.rank[pages] = e.budget;
}

// A code scaled by r <= 1, in the low byte: the product is rounded to FP32, as code r is, and 1.5 2^23 rounds it to a
// whole number (not fused: that would round once).
__device__ __forceinline__ unsigned shrink(int code, float r) {
#pragma clang fp contract(off)
    const float z = (float)code * r;
    return __float_as_uint(z + 12582912.0f);
}
// Four codes of a word: byte - 128 is the code (of the word ^ 0x80808080), and the fused product is code r, rounded.
template <int B> __device__ __forceinline__ unsigned shrink_byte(unsigned u, float r) {
    return __float_as_uint(fmaf((float)(u >> (8 * B) & 0xff), r, -128.0f * r) + 12582912.0f);
}
__device__ __forceinline__ unsigned shrink4(unsigned w, float r) {
    const unsigned u = w ^ 0x80808080u;
    const unsigned lo = __builtin_amdgcn_perm(shrink_byte<1>(u, r), shrink_byte<0>(u, r), 0x0c0c0400u);
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(shrink_byte<3>(u, r), shrink_byte<2>(u, r), 0x0c0c0400u), lo, 0x05040100u);
}

// One workgroup per (sequence, head, run of pages that are filled).  Token m of the kept ones comes from
// place m or a later one, so a page and its record may be written once the pages before it that take tokens from it
// have read them.  A workgroup draws its run's number when it starts: those that it waits for have
// started before it, and say that they have read before they wait themselves.  (Draws of one sequence and head follow
// each other in memory, so a run is as long as a workgroup's waves allow.)
//
// V: the codes of a dim's kept tokens are a product with a matrix that has one 1 in each column, exact on the int8
// matrix instruction: A has a row for each of 16 places of the new page (its token's place in the source page, or none), B
// the source page's codes as they lie there, 16 tokens of a dim a lane; what comes out, four places of a dim a
// lane, is a word of the new page but for its scale.  Source pages add up.  (Other ways for 32 sequences to 2,048 tokens, 8 heads
// of 128: a load from memory for each byte keeps the address unit busy, 107 us; rows through LDS and bytes there, a dim a
// lane, 103; this way 90: the 252 MB that it cannot do without at 2.8 TB/s.)  K: 16 dims of a token a lane.  Bound by the chain of
// ticket, list, codes and flag, which two workgroups of 88 registers on a CU do not hide; 80 registers spill (115), 16 dims a wave (52 registers) double the workgroups and draws (118), 1,024 threads are no better (101).
constexpr int MOST_POLLS = 1 << 20;
constexpr int MOVE_THREADS = 512;
constexpr int move_waves(int dp) { return dp > 32 ? dp / 32 : 1; }  // of a page
template <int DP> struct Move {
    static constexpr int WAVES = move_waves(DP);
    static constexpr int TILES = DP / 16 / WAVES;          // of 16 dims, a wave's; pieces of K, a lane's
    static constexpr int RUN = 8 / WAVES, THREADS = MOVE_THREADS;
};
inline int64_t move_runs(int pages, int dp) {  // of a sequence and head
    const int run = 8 / move_waves(dp);
    return (pages + run - 1) / run;
}
template <int DP> __global__ __launch_bounds__(Move<DP>::THREADS) void k_kv8_move(Kv8Evict e, void *ws, int polls) {
    constexpr int TILES = Move<DP>::TILES, RUN = Move<DP>::RUN, UNIT = 64 * Move<DP>::WAVES;
    __shared__ int srun, late[RUN];
    // runs of a pair start apart, on XCDs in turn (one after the other: 107 us for 99, all on one XCD 148)
    const int pairs = e.s.n_seq * e.c.hk;
    const int64_t pair = (blockIdx.x % pairs + blockIdx.x / pairs) % pairs;
    const int h = pair % e.c.hk, i = pair / e.c.hk;
    const int unit = __builtin_amdgcn_readfirstlane(threadIdx.x / UNIT), tid = threadIdx.x % UNIT, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Work w = work_of(e, ws, pair);
    int run = blockIdx.x / pairs;
    const int slot = e.s.slots ? e.s.slots[i] : i;  // (sequences of slots that are not there have nothing to move)
    const int *table = e.s.table + (int64_t)slot * e.s.table_stride;
    const int len = w.state->x, n = w.state->y;
    const bool moves = w.state->z != 0;
    // (behind the state, so that those of sequences that stay draw nothing: 64 sequences of 4,000 tokens within a budget of
    // 4,096, 8 heads, 39 -> 23 us in all, and the moves 99 -> 92)
    if (moves && threadIdx.x == 0) srun = atomicAdd(&w.state->w, 1);
    if (threadIdx.x < RUN) late[threadIdx.x] = 0;
    if (run == 0 && h == 0 && threadIdx.x == 0) {
        // (a sequence that is left alone keeps its length, also one that is not there)
        if (moves) e.lens_out[i] = e.budget;
        else if (e.lens_out != e.s.lens) e.lens_out[i] = e.s.lens[i];
        if (moves && e.shifts) e.shifts[i] += len - e.budget;  // (positions go on behind it)
    }
    if (!moves && !copies(e)) return;
    __syncthreads();
    if (moves) run = __builtin_amdgcn_readfirstlane(srun);
    const int p = run * RUN + unit, m0 = p * KV8_PAGE, here = min(KV8_PAGE, n - m0);
    if (run * RUN * KV8_PAGE >= n) return;
    const int64_t to = here > 0 ? (int64_t)table[p] * e.c.hk + h : 0;
    if (tid < here && e.weights_out) e.weights_out[to * KV8_PAGE + tid] = w.weight[m0 + tid];
    if (!moves) return;
    int r0 = 0, r1 = 0;
    const int g4 = lane >> 4;
    uint4 k[TILES], v[TILES];
    float2 now = {0.0f, 0.0f};
    unsigned long long bad = 0;
    bool stays = true;
    if (here > 0) {
        const int2 mine = w.list[m0 + min(lane, here - 1)];  // token `lane` of the page
        r0 = w.rank[p];
        r1 = w.rank[p + 1];
        // (the last token in its own place: so are all, and the record is what it was)
        stays = here == KV8_PAGE && __builtin_amdgcn_readlane(mine.x, KV8_PAGE - 1) == m0 + KV8_PAGE - 1;
        if (!stays) {
#pragma unroll
            for (int it = 0; it < TILES; it++) {
                const int at = tid + it * UNIT;
                const int2 s = w.list[m0 + min(at / (DP / 16), here - 1)];
                k[it] = *reinterpret_cast<const uint4 *>(
                    e.c.k + (((int64_t)s.y * e.c.hk + h) * KV8_PAGE + s.x % KV8_PAGE) * DP + at % (DP / 16) * 16);
            }
            // the tokens of source pages in turn; the next page's codes under way
            i32x4 x[TILES], y[TILES];
            int from = 0, next = 0;  // the first token of the page in x, in y
            auto load = [&](i32x4 (&o)[TILES], int first) __attribute__((always_inline)) {
                const int64_t ph = (int64_t)__builtin_amdgcn_readlane(mine.y, first) * e.c.hk + h;
#pragma unroll
                for (int t = 0; t < TILES; t++)
                    o[t] = *reinterpret_cast<const i32x4 *>(e.c.v + (ph * DP + (wave * TILES + t) * 16 + (lane & 15)) * KV8_PAGE + g4 * 16);
                // behind the last of its tokens
                return first + __popcll(__ballot(lane >= first && lane < here && mine.x / KV8_PAGE == __builtin_amdgcn_readlane(mine.x, first) / KV8_PAGE));
            };
            next = load(x, 0);
            // the new record: the largest scales (not negative: as bits they compare alike), the tokens' bad bits
            const int64_t ph = (int64_t)mine.y * e.c.hk + h;
            const float2 old = e.c.scales[ph];
            bad = __ballot(lane < here && e.c.bad[ph] >> (mine.x % KV8_PAGE) & 1);
            i32x4 sum[TILES][4];
            int place[4];  // in its source page, of token 16 m + lane % 16
#pragma unroll
            for (int m = 0; m < 4; m++) {
                place[m] = __shfl(mine.x, m * 16 + (lane & 15)) % KV8_PAGE;
#pragma unroll
                for (int t = 0; t < TILES; t++) sum[t][m] = i32x4{0, 0, 0, 0};
            }
            for (;;) {
                int behind = next;
                if (next < here) behind = load(y, next);
#pragma unroll
                for (int m = 0; m < 4; m++) {
                    if (next <= m * 16 || from >= m * 16 + 16) continue;
                    const int at = m * 16 + (lane & 15), q = place[m] - g4 * 16;
                    const int one = at >= from && at < next && q >= 0 && q < 16 ? 1 << 8 * (q & 3) : 0;
                    i32x4 a;
#pragma unroll
                    for (int u = 0; u < 4; u++) a[u] = q >> 2 == u ? one : 0;
#pragma unroll
                    for (int t = 0; t < TILES; t++) sum[t][m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a, x[t], sum[t][m], 0, 0, 0);
                }
                if (next >= here) break;
                from = next;
                next = behind;
#pragma unroll
                for (int t = 0; t < TILES; t++) x[t] = y[t];
            }
            now = {__uint_as_float(wave_max_bits(__float_as_uint(old.x))), __uint_as_float(wave_max_bits(__float_as_uint(old.y)))};
            const float rk = now.x > 0.0f ? old.x / now.x : 0.0f, rv = now.y > 0.0f ? old.y / now.y : 0.0f;
#pragma unroll
            for (int it = 0; it < TILES; it++) {
                const float r = __shfl(rk, (tid + it * UNIT) / (DP / 16) % KV8_PAGE);
                k[it] = make_uint4(shrink4(k[it].x, r), shrink4(k[it].y, r), shrink4(k[it].z, r), shrink4(k[it].w, r));
            }
            unsigned o[TILES][4];  // tokens 16 m + 4 g4 ..
#pragma unroll
            for (int m = 0; m < 4; m++) {
                float r[4];
#pragma unroll
                for (int u = 0; u < 4; u++) r[u] = __shfl(rv, m * 16 + g4 * 4 + u);
#pragma unroll
                for (int t = 0; t < TILES; t++) {
                    unsigned c[4];
#pragma unroll
                    for (int u = 0; u < 4; u++) c[u] = shrink(sum[t][m][u], r[u]);
                    o[t][m] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(c[3], c[2], 0x0c0c0400u),
                                                    __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u), 0x05040100u);
                }
            }
            // word m of lanes 16 g .. to word g of lanes 16 m ..: tokens 16 g4 .. in a lane
#pragma unroll
            for (int t = 0; t < TILES; t++) {
                auto a = __builtin_amdgcn_permlane32_swap(o[t][0], o[t][2], false, false);
                auto b = __builtin_amdgcn_permlane32_swap(o[t][1], o[t][3], false, false);
                const unsigned a0 = a[0], a1 = a[1], b0 = b[0], b1 = b[1];
                a = __builtin_amdgcn_permlane16_swap(a0, b0, false, false);
                b = __builtin_amdgcn_permlane16_swap(a1, b1, false, false);
                v[t] = make_uint4(a[0], a[1], b[0], b[1]);
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // every wave's loads have come back
    __syncthreads();
    if (tid == 0 && here > 0) __hip_atomic_store(&w.read[p], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // pages of runs before this one that take tokens from a page: 64 tokens go to two at most
    if (!stays && r0 < r1) {
        const int q = r0 / KV8_PAGE + tid;
        if (q <= (r1 - 1) / KV8_PAGE && q < run * RUN) {
            // (microseconds; bounded for calls at the same time that share a workspace against the rule)
            int n = polls;
            for (; n > 0 && !__hip_atomic_load(&w.read[q], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); n--) __builtin_amdgcn_s_sleep(1);
            if (n == 0) late[unit] = 1;
        }
    }
    __syncthreads();
    if (stays) return;
    // not read by all in time: left as it is, for them, and all its tokens bad, for everyone else
    if (late[unit]) {
        if (tid == 0) e.c.bad[to] = ~0ull;
        return;
    }
#pragma unroll
    for (int it = 0; it < TILES; it++) {
        const int at = tid + it * UNIT, m = at / (DP / 16);
        if (m < here) *reinterpret_cast<uint4 *>(e.c.k + (to * KV8_PAGE + m) * DP + at % (DP / 16) * 16) = k[it];
    }
    if (tid == 0) {
        e.c.scales[to] = now;
        e.c.bad[to] = bad;
    }
#pragma unroll
    for (int t = 0; t < TILES; t++) {
        signed char *z = e.c.v + (to * DP + (wave * TILES + t) * 16 + (lane & 15)) * KV8_PAGE + g4 * 16;
        const unsigned word[4] = {v[t].x, v[t].y, v[t].z, v[t].w};
        if (g4 * 16 + 16 <= here) *reinterpret_cast<uint4 *>(z) = v[t];
        else
#pragma unroll
            for (int u = 0; u < 16; u++)
                if (g4 * 16 + u < here) z[u] = (signed char)(word[u / 4] >> (8 * (u & 3)));
    }
}

}  // namespace

// How many workgroups choose for a sequence and head (0: one, in one launch), so that one of 1,024 threads is on each CU.  Whole
// evictions of one sequence to 4,000 tokens, one workgroup / several: 8 heads of 9,000 tokens 34 / 30 us, of 65,000 95 / 42; 40 heads 102 /
// 57; 128 heads 130 / 122, 192 heads 156 / 195 (in two turns).
static int choose_parts(const Kv8Seqs &s, int hk) {
    const int64_t pairs = (int64_t)s.n_seq * hk, most = (int64_t)s.max_pages * KV8_PAGE;
    return most <= 8192 || pairs > 128 ? 0 : (int)min((int64_t)MOST_PARTS, 256 / pairs);
}
// (a table holds no more)
static int room_of(const Kv8Seqs &s, int budget) { return (int)min((int64_t)budget, (int64_t)s.max_pages * KV8_PAGE); }

// Threads of the workgroups that choose in one launch.
static int choose_threads(const Kv8Seqs &s) { return (int64_t)s.max_pages * KV8_PAGE <= 2048 ? 256 : 1024; }
static int pages_of(int room) { return (room + KV8_PAGE - 1) / KV8_PAGE; }

bool kv8_evict_fits(const Kv8View &c, const Kv8Seqs &s, int budget) {
    const int64_t pairs = (int64_t)s.n_seq * c.hk;  // (with several parts each, 1,024 workgroups at most)
    return pairs == 0 || (kv8_grid(pairs, choose_threads(s)) && kv8_grid(pairs * move_runs(pages_of(room_of(s, budget)), c.dp), MOVE_THREADS));
}
size_t kv8_evict_bytes(const Kv8View &c, const Kv8Seqs &s, int budget) {
    const int parts = choose_parts(s, c.hk);
    return (size_t)s.n_seq * c.hk * (work_size(room_of(s, budget)) + (parts ? parts_size(parts, s.max_pages) : 0));
}

hipError_t launch_kv8_evict(const Kv8Evict &call, void *ws, hipStream_t st) {
    Kv8Evict e = call;
    e.room = room_of(e.s, e.budget);
    const int64_t pairs = (int64_t)e.s.n_seq * e.c.hk, most = (int64_t)e.s.max_pages * KV8_PAGE;
    if (pairs == 0) return hipSuccess;
    if (!kv8_evict_fits(e.c, e.s, e.budget)) return hipErrorInvalidValue;
    if (choose_threads(e.s) == 256) hipLaunchKernelGGL((k_kv8_choose<256, 8, 0>), dim3(pairs), dim3(256), 0, st, e, ws);
    else if (most <= 8192) hipLaunchKernelGGL((k_kv8_choose<1024, 8, 0>), dim3(pairs), dim3(1024), 0, st, e, ws);
    else if (const int parts = choose_parts(e.s, e.c.hk); !parts)
        hipLaunchKernelGGL((k_kv8_choose<1024, 32, 32>), dim3(pairs), dim3(1024), 0, st, e, ws);
    else {
        char *more = static_cast<char *>(ws) + pairs * work_size(e.room);
        const int64_t size = parts_size(parts, e.s.max_pages);
        hipLaunchKernelGGL(k_kv8_part, dim3(pairs * parts), dim3(PART_THREADS), 0, st, e, more, parts, size);
        if (const hipError_t rc = hipGetLastError(); rc != hipSuccess) return rc;
        hipLaunchKernelGGL(k_kv8_near, dim3(pairs * parts), dim3(PART_THREADS), 0, st, e, more, parts, size);
        if (const hipError_t rc = hipGetLastError(); rc != hipSuccess) return rc;
        hipLaunchKernelGGL(k_kv8_list, dim3(pairs * parts), dim3(PART_THREADS), 0, st, e, ws, more, parts, size);
    }
    // (the moves wait for one another by what the choice has cleared)
    if (const hipError_t rc = hipGetLastError(); rc != hipSuccess) return rc;
    const char *p = getenv("CIH_KV8_EVICT_POLLS");
    const int polls = p ? (int)min(max(strtol(p, nullptr, 10), 0l), (long)MOST_POLLS) : MOST_POLLS;
    auto move = [&](auto dp) {
        constexpr int DP = decltype(dp)::value;
        const int runs = (int)move_runs(pages_of(e.room), DP);
        hipLaunchKernelGGL(k_kv8_move<DP>, dim3(pairs * runs), dim3(Move<DP>::THREADS), 0, st, e, ws, polls);
    };
    switch (e.c.dp) {
        case 16: move(std::integral_constant<int, 16>{}); break;
        case 32: move(std::integral_constant<int, 32>{}); break;
        case 64: move(std::integral_constant<int, 64>{}); break;
        case 128: move(std::integral_constant<int, 128>{}); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace cih

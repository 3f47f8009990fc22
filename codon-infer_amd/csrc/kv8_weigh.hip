// The attention weight that cached tokens gather:
//   w_j <- keep w_j + sum over rows r that see j, heads h of the group: exp(scale q_rh k_j - lse_rh)
// with lse as the attention of the same rows gave it, so that the weights need no
// second pass over the keys.  A wave owns a page of one head: its 64 sums have one
// owner and a fixed order.
#include "kv8_tiles.h"

namespace cih {

namespace {

// Sum over the 16 lanes of a row of lanes, value i of them to lane i: halves of the values are
// exchanged with lanes ^ 8, 4, 2, 1.
__device__ __forceinline__ float lanes_reduce(float (&x)[16], int c) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float keep = c & 8 ? x[i + 8] : x[i], give = c & 8 ? x[i] : x[i + 8];
        x[i] = keep + dpp_or<0x128, 0xf>(give, give);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float keep = c & 4 ? x[i + 4] : x[i], give = c & 4 ? x[i] : x[i + 4];
        x[i] = keep + dpp_or<0x114, 0xa>(dpp_or<0x104, 0x5>(give, give), give);
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const float keep = c & 2 ? x[i + 2] : x[i], give = c & 2 ? x[i] : x[i + 2];
        x[i] = keep + dpp_or<0x4E, 0xf>(give, give);
    }
    const float keep = c & 1 ? x[1] : x[0], give = c & 1 ? x[0] : x[1];
    return keep + dpp_or<0xB1, 0xf>(give, give);
}

// Rows [r0, r1) of a sequence that see any of keys [j0, j0 + keys).
struct SeenBy {
    int r0, r1;
    __device__ __forceinline__ SeenBy(const Kv8Attention &a, const Kv8Seq &q, int j0, int keys) {
        r0 = max(0, (a.causal ? max(j0, 0) : 0) - q.start);
        r1 = q.n;
        if (a.window > 0 && j0 >= a.sinks)
            r1 = (int)min((int64_t)q.n, max((int64_t)0, (int64_t)j0 + keys - 1 + a.window - q.start));
    }
};

// What a page's tokens gained, token `lane` of it in each lane.
__device__ __forceinline__ void gain(const Kv8Weigh &w, const Kv8Seq &q, int id, int kvh, int pg, int lane, float x) {
    const int j = pg * KV8_PAGE + lane;
    if (id < 0 || j >= q.len) return;
    float *p = w.weights + ((int64_t)id * w.a.c.hk + kvh) * KV8_PAGE + lane;
    if (w.keep != 0.0f && j < q.start) x = fmaf(w.keep, *p, x);
    *p = x;
}

constexpr int WEIGH_WAVES = 4;

// One workgroup per (sequence, kv head, pps pages); its waves take the pages in turn.
template <int DP, class T>
__global__ __launch_bounds__(64 * WEIGH_WAVES) void k_kv8_weigh(Kv8Weigh w, int g, int groups, int pps) {
    constexpr int KS = Tile<DP>::KS;
    const Kv8Attention &a = w.a;
    int b = blockIdx.x;
    const int group = b % groups;
    b /= groups;
    const int kvh = b % a.c.hk;
    const Kv8Seq q = kv8_seq(a.s, b / a.c.hk);
    if (q.n == 0) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g4 = lane >> 4;
    const int last = min((q.len + KV8_PAGE - 1) / KV8_PAGE, (group + 1) * pps);
    i32x4 ql[3][KS];
    float f = 0.0f, off = INFINITY;
    Column col{};
    int held = -1;  // the tile of columns in ql
    for (int pg = group * pps + wave; pg < last; pg += WEIGH_WAVES) {
        const int id = page_id(a.c, q, pg);
        if (id < 0) continue;
        const int j0 = pg * KV8_PAGE;
        float sum[16] = {};
        const SeenBy by(a, q, j0, KV8_PAGE);
        const int64_t ph = (int64_t)id * a.c.hk + kvh;
        const float sk = uniform(&a.c.scales[ph].x);
        if (by.r0 < by.r1 && sk >= 0.0f && sk <= FLT_MAX) {
            Tile<DP> t;
            load_k(t, a.c, id, kvh, lane);
            const int t1 = (by.r1 * g + 15) / 16;
            for (int tile = by.r0 * g / 16; tile < t1; tile++) {
                if (tile != held) {
                    held = tile;
                    col = column(a, q, kvh, g, tile * 16 + c);
                    const float lse = col.row >= 0 ? a.lse[(int64_t)col.row * a.heads + col.head] : INFINITY;
                    const bool fine = fabsf(lse) <= FLT_MAX;
                    if (!fine) col.row = -1;  // its query is taken as zeros
                    off = lse * LOG2E;
                    float x[KS][16];
                    load_query<KS, T>(a, col, g4, x);
                    f = query_bytes<3, KS>(x, a.scale, ql);
                    if (!fine || !(f <= FLT_MAX)) {
                        f = 0.0f;
                        off = INFINITY;
                    }
                }
                unsigned see = visible16(col.begin, col.end, j0 + g4 * 16);
                if (a.sinks > 0) see |= visible16(0, min(a.sinks, col.end), j0 + g4 * 16);
                const float fk = fminf(f * sk, FLT_MAX);
#pragma unroll
                for (int kt = 0; kt < 4; kt++) {
                    float s[4];
                    score_tile<3, KS>(t.k[kt], ql, s);
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float e = __builtin_amdgcn_exp2f(fmaf(s[r], fk, -off));
                        sum[kt * 4 + r] += see >> (kt * 4 + r) & 1 ? e : 0.0f;
                    }
                }
            }
        }
        gain(w, q, id, kvh, pg, lane, lanes_reduce(sum, c));
    }
}

template <int DP, class T> hipError_t launch(const Kv8Weigh &w, hipStream_t st) {
    const int64_t pairs = (int64_t)w.a.s.n_seq * w.a.c.hk;
    const int g = w.a.heads / w.a.c.hk, pps = 16, groups = (w.a.s.max_pages + pps - 1) / pps;
    if (!kv8_grid(pairs * groups, 64 * WEIGH_WAVES)) return hipErrorInvalidValue;
    hipLaunchKernelGGL((k_kv8_weigh<DP, T>), dim3(pairs * groups), dim3(64 * WEIGH_WAVES), 0, st, w, g, groups, pps);
    return hipGetLastError();
}

template <class T> hipError_t launch_dims(const Kv8Weigh &w, hipStream_t st) {
    switch (w.a.c.dp) {
        case 16: return launch<16, T>(w, st);
        case 32: return launch<32, T>(w, st);
        case 64: return launch<64, T>(w, st);
        case 128: return launch<128, T>(w, st);
    }
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_kv8_weigh(const Kv8Weigh &call, hipStream_t st) {
    if (call.a.s.n_rows == 0 || call.a.s.n_seq == 0 || call.a.s.max_rows == 0) return hipSuccess;
    Kv8Weigh w = call;
    const RowsView &q = w.a.q;
    const int64_t size = w.a.dtype == FT_F32 ? 4 : 2;
    w.a.q16 = (reinterpret_cast<uintptr_t>(q.p) | (uintptr_t)(q.rs * size) | (uintptr_t)(q.hs * size)) % 16 == 0;
    switch (w.a.dtype) {
        case FT_F32: return launch_dims<float>(w, st);
        case FT_F16: return launch_dims<_Float16>(w, st);
        case FT_BF16: return launch_dims<__bf16>(w, st);
    }
    return hipErrorInvalidValue;
}

}  // namespace cih

// The 8-bit paged key/value cache: rows of K and V rotated, quantized and
// written into their pages, and read back.
//
// A workgroup owns one (page, head) that its sequence's new rows touch, so the
// page's scale, its kept codes and its new ones change under one owner:
//   s = max(s_old where tokens are kept, max |new| / 127)
//   kept codes  q <- rint(q s_old / s)   only where s grew
//   new codes   q  = rint(x / s)
//
// Bound by the rows' bytes for many of them: 12,300 bfloat16 rows of 32 + 8 heads of
// 128, append 70 us (4.3 TB/s with the rotated queries) and read 19 us; by latency for
// few: one FP32 row of 8 sequences, 20 heads of 64, 6.1 and 4.5 us.
#include <float.h>

#include "kv8.h"

namespace cih {

namespace {

constexpr int KV_THREADS = 256;
constexpr int VQ = KV8_PAGE + 4;  // bytes of a dim's codes in LDS

// The two dims of pair j of a head: rotated pairs first, then neighbours.
__device__ __forceinline__ void pair_dims(const RopeArg &r, int j, int &i0, int &i1) {
    const int half = r.rot / 2;
    if (j >= half || r.inter) {
        i0 = 2 * j;
        i1 = i0 + 1;
    } else {
        i0 = j;
        i1 = j + half;
    }
}

// Which (sequence, page, head) a workgroup owns, and the page's new tokens
// [lo, hi) (in the page).  Pages a sequence's rows can touch: per_seq.
struct PageTask {
    Kv8Seq q;
    int h, pg, lo, hi;
};
__device__ __forceinline__ bool page_task(const Kv8View &c, const Kv8Seqs &s, int per_seq, PageTask &t) {
    const int b = blockIdx.x, rest = b / c.hk;
    t.h = b - rest * c.hk;
    const int i = rest / per_seq;
    t.q = kv8_seq(s, i);
    const int first = max(t.q.start, 0);
    if (first >= t.q.len) return false;
    t.pg = first / KV8_PAGE + (rest - i * per_seq);
    t.lo = max(first - t.pg * KV8_PAGE, 0);
    t.hi = min(t.q.len - t.pg * KV8_PAGE, KV8_PAGE);
    return t.lo < t.hi;
}

template <class T>
__global__ __launch_bounds__(KV_THREADS) void k_kv8_append(Kv8View c, Kv8Seqs s, RowsView k, RowsView v, RowsView q,
                                                           RowsView qo, int g, int per_seq, RopeArg rope) {
    extern __shared__ float sm[];
    __shared__ float red[2][KV_THREADS / 64];
    __shared__ unsigned long long sbad;
    PageTask t;
    if (!page_task(c, s, per_seq, t)) return;
    const int nt = t.hi - t.lo, d = c.d, tid = threadIdx.x, half = d / 2;
    const int p0 = t.pg * KV8_PAGE + t.lo;          // position of the first new token
    const int64_t row0 = t.q.r0 + (p0 - t.q.start);  // and its row
    float *kf = sm;                                  // [nt][d]: K, rotated
    unsigned char *vq = reinterpret_cast<unsigned char *>(sm + nt * d);  // [d][VQ]: V's codes, by dim
    if (tid == 0) sbad = 0;
    __syncthreads();
    const T *kp = static_cast<const T *>(k.p) + t.h * k.hs, *vp = static_cast<const T *>(v.p) + t.h * v.hs;
    for (int e = tid; e < nt * half; e += KV_THREADS) {
        const int n = e / half, j = e - n * half;
        int i0, i1;
        pair_dims(rope, j, i0, i1);
        const T *kr = kp + (row0 + n) * k.rs, *vr = vp + (row0 + n) * v.rs;
        float x0 = to_f32(kr[i0]), x1 = to_f32(kr[i1]);
        const float v0 = to_f32(vr[i0]), v1 = to_f32(vr[i1]);
        float cs = 1.0f, sn = 0.0f;
        const bool turn = 2 * j < rope.rot;
        if (turn) {
            rope_cs(rope, p0 + n, j, cs, sn);
            const float y0 = x0 * cs - x1 * sn;
            x1 = x1 * cs + x0 * sn;
            x0 = y0;
        }
        if (!(fabsf(x0) <= FLT_MAX && fabsf(x1) <= FLT_MAX && fabsf(v0) <= FLT_MAX && fabsf(v1) <= FLT_MAX))
            atomicOr(&sbad, 1ull << (t.lo + n));
        kf[n * d + i0] = x0;
        kf[n * d + i1] = x1;
        if (q.p) {
            for (int hq = t.h * g; hq < (t.h + 1) * g; hq++) {
                const T *qr = static_cast<const T *>(q.p) + (row0 + n) * q.rs + hq * q.hs;
                T *qw = static_cast<T *>(qo.p) + (row0 + n) * qo.rs + hq * qo.hs;
                const float a = to_f32(qr[i0]), b = to_f32(qr[i1]);
                qw[i0] = (T)(turn ? a * cs - b * sn : a);
                qw[i1] = (T)(turn ? b * cs + a * sn : b);
            }
        }
    }
    const int id = kv8_page(c, t.q, t.pg);
    if (id < 0) return;
    __syncthreads();
    const unsigned long long bad = sbad;
    float mk = 0.0f, mv = 0.0f;
    for (int e = tid; e < nt * d; e += KV_THREADS) {
        const int n = e / d;
        if (!(bad >> (t.lo + n) & 1)) {
            mk = fmaxf(mk, fabsf(kf[e]));
            mv = fmaxf(mv, fabsf(to_f32(vp[(row0 + n) * v.rs + (e - n * d)])));
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        mk = fmaxf(mk, __shfl_xor(mk, o));
        mv = fmaxf(mv, __shfl_xor(mv, o));
    }
    if ((tid & 63) == 0) {
        red[0][tid >> 6] = mk;
        red[1][tid >> 6] = mv;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < KV_THREADS / 64; w++) {
        mk = fmaxf(mk, red[0][w]);
        mv = fmaxf(mv, red[1][w]);
    }
    const int64_t ph = (int64_t)id * c.hk + t.h;
    float2 old = {0.0f, 0.0f};
    unsigned long long kept_bad = 0;
    if (t.lo > 0) {
        old = c.scales[ph];
        kept_bad = c.bad[ph] & ((1ull << t.lo) - 1);
    }
    const float2 sc = kv8_scales(__float_as_uint(mk), __float_as_uint(mv), old);
    __syncthreads();  // the old scales are read before they are replaced
    if (tid == 0) {
        c.scales[ph] = sc;
        c.bad[ph] = kept_bad | bad;
    }
    const float ik = sc.x > 0.0f ? 1.0f / sc.x : 0.0f, iv = sc.y > 0.0f ? 1.0f / sc.y : 0.0f;
    const float rk = sc.x > 0.0f ? old.x / sc.x : 0.0f, rv = sc.y > 0.0f ? old.y / sc.y : 0.0f;
    signed char *kc = c.k + ph * (KV8_PAGE * c.dp), *vc = c.v + ph * (KV8_PAGE * c.dp);
    const int dq = c.dp / 4;
    if (t.lo > 0 && rk != 1.0f)  // kept keys
        for (int e = tid; e < t.lo * dq; e += KV_THREADS) {
            unsigned *w = reinterpret_cast<unsigned *>(kc) + e;
            *w = recode4(*w, rk);
        }
    for (int e = tid; e < nt * dq; e += KV_THREADS) {
        const int n = e / dq, i = 4 * (e - n * dq);
        unsigned w = 0;
        if (!(bad >> (t.lo + n) & 1))
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (i + u < d) w |= (unsigned)code8(kf[n * d + i + u], ik) << (8 * u);
        *reinterpret_cast<unsigned *>(kc + (t.lo + n) * c.dp + i) = w;
    }
    for (int e = tid; e < nt * d; e += KV_THREADS) {
        const int n = e / d, i = e - n * d;
        vq[i * VQ + t.lo + n] =
            bad >> (t.lo + n) & 1 ? 0 : (unsigned char)code8(to_f32(vp[(row0 + n) * v.rs + i]), iv);
    }
    __syncthreads();
    // values: four tokens of a dim at a time, from the first that changes
    const int q0 = t.lo > 0 && rv != 1.0f ? 0 : t.lo / 4, nq = (t.hi + 3) / 4 - q0;
    for (int e = tid; e < c.dp * nq; e += KV_THREADS) {
        const int i = e / nq, n4 = 4 * (q0 + e - i * nq);
        unsigned *w = reinterpret_cast<unsigned *>(vc + i * KV8_PAGE + n4), o = 0;
        if (n4 < t.lo) o = recode4(*w, rv);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int n = n4 + u;
            if (n < t.lo) continue;
            o &= ~(0xffu << (8 * u));
            if (n < t.hi && i < d) o |= (unsigned)vq[i * VQ + n] << (8 * u);
        }
        *w = o;
    }
}

// A dword of four tokens' codes of one dim.
__device__ __forceinline__ unsigned pack4(const float (&x)[4], float inv) {
    unsigned o = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) o |= (unsigned)code8(x[e], inv) << (8 * e);
    return o;
}
__device__ __forceinline__ unsigned abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }  // NaN > inf > the rest
template <class T> struct Chunk {
    static constexpr int N = 16 / sizeof(T);
    typedef T type __attribute__((ext_vector_type(16 / sizeof(T))));
};
template <class T> __device__ __forceinline__ void load_chunk(const T *p, float (&x)[Chunk<T>::N]) {
    const auto w = *reinterpret_cast<const typename Chunk<T>::type *>(p);
#pragma unroll
    for (int e = 0; e < Chunk<T>::N; e++) x[e] = to_f32(w[e]);
}
template <class T> __device__ __forceinline__ void store_chunk(T *p, const float (&x)[Chunk<T>::N]) {
    typename Chunk<T>::type w;
#pragma unroll
    for (int e = 0; e < Chunk<T>::N; e++) w[e] = (T)x[e];
    *reinterpret_cast<typename Chunk<T>::type *>(p) = w;
}

// The same in 16-byte pieces (VL values), K and V kept in registers between
// the maximum and the codes.  K and Q: a thread takes two pieces of a token
// that hold VL whole pairs (neighbouring ones, or half the rotated dims apart).  V:
// a thread takes one piece of four tokens, whose codes of a dim are one word
// of the page.  Bound by the rows' bytes; NT = 64 for at most 4 rows a
// sequence, where a page's 256 threads would mostly idle (a row each of 512 sequences, 20 heads of 64: append
// and read 85 us, with 256 threads 118; of 8 sequences no difference).
template <class T, int NT>
__global__ __launch_bounds__(NT) void k_kv8_append_vec(Kv8View c, Kv8Seqs s, RowsView k, RowsView v, RowsView q,
                                                       RowsView qo, int g, int per_seq, RopeArg rope) {
    constexpr int VL = Chunk<T>::N, NW = NT / 64;
    constexpr int KIT = NT == 64 ? 1 : 16 / VL, VIT = NT == 64 ? 1 : 8 / VL;  // pieces of a thread at 64 x 128
    __shared__ unsigned red[2][NW];
    __shared__ unsigned long long sbad;
    PageTask t;
    if (!page_task(c, s, per_seq, t)) return;
    const int nt = t.hi - t.lo, d = c.d, tid = threadIdx.x;
    const int p0 = t.pg * KV8_PAGE + t.lo;
    const int64_t row0 = t.q.r0 + (p0 - t.q.start);
    const int id = kv8_page(c, t.q, t.pg);
    const int64_t ph = (int64_t)max(id, 0) * c.hk + t.h;
    float2 old = {0.0f, 0.0f};
    unsigned long long kept_bad = 0;
    if (t.lo > 0 && id >= 0) {
        old = c.scales[ph];
        kept_bad = c.bad[ph] & ((1ull << t.lo) - 1);
    }
    // V: pieces of four tokens n4 .., aligned to the page's words
    const T *vp = static_cast<const T *>(v.p) + t.h * v.hs;
    const int q0 = t.lo / 4, nq = (t.hi + 3) / 4 - q0, chunks = d / VL;
    // (loads without branches, at the nearest row there is, so that all are under way at once)
    float vx[VIT][4][VL], kx[KIT][2][VL];
    unsigned mv = 0, mk = 0;
    const int items = d / (2 * VL), turned = rope.rot / (2 * VL);
#pragma unroll
    for (int it = 0; it < VIT; it++) {
        if (it * NT >= chunks * nq) continue;
        const int x = tid + it * NT, ch = x / nq, n4 = 4 * (q0 + x - ch * nq);
#pragma unroll
        for (int u = 0; u < 4; u++)
            load_chunk<T>(vp + (row0 + min(max(n4 + u, t.lo), t.hi - 1) - t.lo) * v.rs + min(ch, chunks - 1) * VL, vx[it][u]);
    }
    // K and Q: items of two pieces
    const T *kp = static_cast<const T *>(k.p) + t.h * k.hs;
#pragma unroll
    for (int it = 0; it < KIT; it++) {
        if (it * NT >= nt * items) continue;
        const int x = tid + it * NT, n = min(x / items, nt - 1), i = x % items;
        const bool turn = i < turned;
        const int da = turn && !rope.inter ? i * VL : i * 2 * VL, db = turn && !rope.inter ? da + rope.rot / 2 : da + VL;
        load_chunk<T>(kp + (row0 + n) * k.rs + da, kx[it][0]);
        load_chunk<T>(kp + (row0 + n) * k.rs + db, kx[it][1]);
    }
#pragma unroll
    for (int it = 0; it < KIT; it++) {
        if (it * NT >= nt * items) {
#pragma unroll
            for (int e = 0; e < VL; e++) kx[it][0][e] = kx[it][1][e] = 0.0f;
            continue;
        }
        const int x = tid + it * NT, n = x / items, i = x - n * items;
        const bool live = n < nt, turn = i < turned;
        const int da = turn && !rope.inter ? i * VL : i * 2 * VL, db = turn && !rope.inter ? da + rope.rot / 2 : da + VL;
        auto rotate = [&](float (&a)[VL], float (&b)[VL], const float (&cs)[VL], const float (&sn)[VL])
                          __attribute__((always_inline)) {
            if (!rope.inter) {
#pragma unroll
                for (int e = 0; e < VL; e++) {
                    const float y = a[e] * cs[e] - b[e] * sn[e];
                    b[e] = b[e] * cs[e] + a[e] * sn[e];
                    a[e] = y;
                }
            } else {
#pragma unroll
                for (int e = 0; e < VL; e += 2) {
                    float y = a[e] * cs[e / 2] - a[e + 1] * sn[e / 2];
                    a[e + 1] = a[e + 1] * cs[e / 2] + a[e] * sn[e / 2];
                    a[e] = y;
                    y = b[e] * cs[(VL + e) / 2] - b[e + 1] * sn[(VL + e) / 2];
                    b[e + 1] = b[e + 1] * cs[(VL + e) / 2] + b[e] * sn[(VL + e) / 2];
                    b[e] = y;
                }
            }
        };
        if (live) {
            const T *qr = static_cast<const T *>(q.p) + (row0 + n) * q.rs + t.h * g * q.hs;
            T *qw = static_cast<T *>(qo.p) + (row0 + n) * qo.rs + t.h * g * qo.hs;
            float qa[VL], qb[VL];  // the next head's
            if (q.p) {
                load_chunk<T>(qr + da, qa);
                load_chunk<T>(qr + db, qb);
            }
            float cs[VL], sn[VL];
            if (turn) {
#pragma unroll
                for (int e = 0; e < VL; e++) rope_cs(rope, p0 + n, (rope.inter ? da / 2 : da) + e, cs[e], sn[e]);
                rotate(kx[it][0], kx[it][1], cs, sn);
            }
            if (q.p)
                for (int hq = 0; hq < g; hq++) {
                    float a[VL], b[VL];
#pragma unroll
                    for (int e = 0; e < VL; e++) {
                        a[e] = qa[e];
                        b[e] = qb[e];
                    }
                    if (hq + 1 < g) {
                        load_chunk<T>(qr + (hq + 1) * q.hs + da, qa);
                        load_chunk<T>(qr + (hq + 1) * q.hs + db, qb);
                    }
                    if (turn) rotate(a, b, cs, sn);
                    store_chunk<T>(qw + hq * qo.hs + da, a);
                    store_chunk<T>(qw + hq * qo.hs + db, b);
                }
        }
#pragma unroll
        for (int e = 0; e < VL; e++) {
            kx[it][0][e] = live ? kx[it][0][e] : 0.0f;
            kx[it][1][e] = live ? kx[it][1][e] : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < VL; e++) mk = max(mk, max(abs_bits(kx[it][0][e]), abs_bits(kx[it][1][e])));
    }
    if (id < 0) return;
#pragma unroll
    for (int it = 0; it < VIT; it++) {
        if (it * NT >= chunks * nq) {
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int e = 0; e < VL; e++) vx[it][u][e] = 0.0f;
            continue;
        }
        const int x = tid + it * NT, ch = x / nq, n4 = 4 * (q0 + x - ch * nq);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const bool live = ch < chunks && n4 + u >= t.lo && n4 + u < t.hi;
#pragma unroll
            for (int e = 0; e < VL; e++) {
                vx[it][u][e] = live ? vx[it][u][e] : 0.0f;
                mv = max(mv, abs_bits(vx[it][u][e]));
            }
        }
    }
    auto all = [&]() {  // mk and mv over the workgroup
        mk = wave_max_bits(mk);
        mv = wave_max_bits(mv);
        if (NW == 1) return;
        __syncthreads();
        if ((tid & 63) == 0) {
            red[0][tid >> 6] = mk;
            red[1][tid >> 6] = mv;
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NW; w++) {
            mk = max(mk, red[0][w]);
            mv = max(mv, red[1][w]);
        }
    };
    all();
    unsigned long long bad = 0;
    if (max(mk, mv) >= 0x7f800000u) {  // a value that is not finite: its tokens' codes are 0
        if (tid == 0) sbad = 0;
        __syncthreads();
#pragma unroll
        for (int it = 0; it < VIT; it++)
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int e = 0; e < VL; e++)
                    if (abs_bits(vx[it][u][e]) >= 0x7f800000u) {
                        const int x = tid + it * NT;
                        atomicOr(&sbad, 1ull << (4 * (q0 + x % nq) + u));
                    }
#pragma unroll
        for (int it = 0; it < KIT; it++)
#pragma unroll
            for (int e = 0; e < VL; e++)
                if (max(abs_bits(kx[it][0][e]), abs_bits(kx[it][1][e])) >= 0x7f800000u)
                    atomicOr(&sbad, 1ull << (t.lo + (tid + it * NT) / items));
        __syncthreads();
        bad = sbad;
        mk = mv = 0;
#pragma unroll
        for (int it = 0; it < VIT; it++)
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const bool lost = bad >> (4 * (q0 + (tid + it * NT) % nq) + u) & 1;
#pragma unroll
                for (int e = 0; e < VL; e++) {
                    if (lost) vx[it][u][e] = 0.0f;
                    mv = max(mv, abs_bits(vx[it][u][e]));
                }
            }
#pragma unroll
        for (int it = 0; it < KIT; it++) {
            const int n = (tid + it * NT) / items;
            const bool lost = n < nt && bad >> (t.lo + n) & 1;
#pragma unroll
            for (int e = 0; e < VL; e++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if (lost) kx[it][h][e] = 0.0f;
                    mk = max(mk, abs_bits(kx[it][h][e]));
                }
        }
        all();
    }
    const float2 sc = kv8_scales(mk, mv, old);
    if (NW > 1) __syncthreads();  // the old scales are read before they are replaced
    if (tid == 0) {
        c.scales[ph] = sc;
        c.bad[ph] = kept_bad | bad;
    }
    const float ik = sc.x > 0.0f ? 1.0f / sc.x : 0.0f, iv = sc.y > 0.0f ? 1.0f / sc.y : 0.0f;
    signed char *kc = c.k + ph * (KV8_PAGE * c.dp), *vc = c.v + ph * (KV8_PAGE * c.dp);
    const float rv = t.lo > 0 && sc.y > 0.0f ? old.y / sc.y : 0.0f;
    if (t.lo > 0) {  // kept codes whose scale grew
        const float rk = sc.x > 0.0f ? old.x / sc.x : 0.0f;
        if (rk != 1.0f)
            for (int e = tid; e < t.lo * c.dp / 4; e += NT) {
                unsigned *w = reinterpret_cast<unsigned *>(kc) + e;
                *w = recode4(*w, rk);
            }
        if (rv != 1.0f)
            for (int e = tid; e < d * q0; e += NT) {
                unsigned *w = reinterpret_cast<unsigned *>(vc + e / q0 * KV8_PAGE) + e % q0;
                *w = recode4(*w, rv);
            }
    }
#pragma unroll
    for (int it = 0; it < KIT; it++) {
        const int x = tid + it * NT, n = x / items, i = x - n * items;
        if (n >= nt) break;
        const bool turn = i < turned;
        const int da = turn && !rope.inter ? i * VL : i * 2 * VL, db = turn && !rope.inter ? da + rope.rot / 2 : da + VL;
        signed char *kr = kc + (t.lo + n) * c.dp;
#pragma unroll
        for (int e = 0; e < VL; e += 4) {
            const float a[4] = {kx[it][0][e], kx[it][0][e + 1], kx[it][0][e + 2], kx[it][0][e + 3]};
            const float b[4] = {kx[it][1][e], kx[it][1][e + 1], kx[it][1][e + 2], kx[it][1][e + 3]};
            *reinterpret_cast<unsigned *>(kr + da + e) = pack4(a, ik);
            *reinterpret_cast<unsigned *>(kr + db + e) = pack4(b, ik);
        }
    }
#pragma unroll
    for (int it = 0; it < VIT; it++) {
        const int x = tid + it * NT, ch = x / nq, n4 = 4 * (q0 + x - ch * nq);
        if (ch >= chunks) break;
        const int keep = max(t.lo - n4, 0);  // kept tokens in the word
#pragma unroll
        for (int e = 0; e < VL; e++) {
            unsigned *w = reinterpret_cast<unsigned *>(vc + (ch * VL + e) * KV8_PAGE + n4);
            const float y[4] = {vx[it][0][e], vx[it][1][e], vx[it][2][e], vx[it][3][e]};
            unsigned o = pack4(y, iv);
            if (keep > 0) {
                const unsigned m = (1u << (8 * keep)) - 1, was = rv == 1.0f ? *w : recode4(*w, rv);
                o = (o & ~m) | (was & m);
            }
            *w = o;
        }
    }
    // dims past a head of 24
    if (c.dp > d) {
        for (int e = tid; e < nt * (c.dp - d) / 4; e += NT) {
            const int per = (c.dp - d) / 4, n = e / per;
            *reinterpret_cast<unsigned *>(kc + (t.lo + n) * c.dp + d + 4 * (e - n * per)) = 0;
        }
        for (int e = tid; e < nq * (c.dp - d); e += NT)
            *reinterpret_cast<unsigned *>(vc + (d + e / nq) * KV8_PAGE + 4 * (q0 + e % nq)) = 0;
    }
}

template <class T>
__global__ __launch_bounds__(KV_THREADS) void k_kv8_read(Kv8View c, Kv8Seqs s, RowsView k, RowsView v, int per_seq) {
    __shared__ unsigned vs[128 * 17];  // [dims][16 + 1] words of four tokens
    PageTask t;
    if (!page_task(c, s, per_seq, t)) return;
    const int id = kv8_page(c, t.q, t.pg);
    if (id < 0) return;
    const int nt = t.hi - t.lo, d = c.d, tid = threadIdx.x;
    const int64_t row0 = t.q.r0 + (t.pg * KV8_PAGE + t.lo - t.q.start), ph = (int64_t)id * c.hk + t.h;
    const float2 sc = c.scales[ph];
    const unsigned long long bad = c.bad[ph];
    const signed char *kc = c.k + ph * (KV8_PAGE * c.dp), *vc = c.v + ph * (KV8_PAGE * c.dp);
    for (int e = tid; e < d * 16; e += KV_THREADS) vs[(e >> 4) * 17 + (e & 15)] = reinterpret_cast<const unsigned *>(vc)[e];
    __syncthreads();
    T *kp = static_cast<T *>(k.p) + t.h * k.hs, *vp = static_cast<T *>(v.p) + t.h * v.hs;
    for (int e = tid; e < nt * d; e += KV_THREADS) {
        const int n = e / d, i = e - n * d, tok = t.lo + n;
        const bool lost = bad >> tok & 1;
        kp[(row0 + n) * k.rs + i] = (T)(lost ? NAN : (float)kc[tok * c.dp + i] * sc.x);
        vp[(row0 + n) * v.rs + i] =
            (T)(lost ? NAN : (float)(signed char)(vs[i * 17 + (tok >> 2)] >> (8 * (tok & 3))) * sc.y);
    }
}

// The same in 16-byte pieces: K a piece of a token, V a piece of four tokens
// from the words of its dims.
template <class T>
__global__ __launch_bounds__(KV_THREADS) void k_kv8_read_vec(Kv8View c, Kv8Seqs s, RowsView k, RowsView v, int per_seq) {
    constexpr int VL = Chunk<T>::N;
    PageTask t;
    if (!page_task(c, s, per_seq, t)) return;
    const int id = kv8_page(c, t.q, t.pg);
    if (id < 0) return;
    const int nt = t.hi - t.lo, chunks = c.d / VL, tid = threadIdx.x;
    const int64_t row0 = t.q.r0 + (t.pg * KV8_PAGE + t.lo - t.q.start), ph = (int64_t)id * c.hk + t.h;
    const float2 sc = c.scales[ph];
    const unsigned long long bad = c.bad[ph];
    const signed char *kc = c.k + ph * (KV8_PAGE * c.dp), *vc = c.v + ph * (KV8_PAGE * c.dp);
    T *kp = static_cast<T *>(k.p) + t.h * k.hs, *vp = static_cast<T *>(v.p) + t.h * v.hs;
    for (int x = tid; x < nt * chunks; x += KV_THREADS) {
        const int n = x / chunks, ch = x - n * chunks, tok = t.lo + n;
        const bool lost = bad >> tok & 1;
        float y[VL];
#pragma unroll
        for (int e = 0; e < VL; e += 4) {
            const unsigned w = *reinterpret_cast<const unsigned *>(kc + tok * c.dp + ch * VL + e);
#pragma unroll
            for (int u = 0; u < 4; u++) y[e + u] = lost ? NAN : (float)(signed char)(w >> (8 * u)) * sc.x;
        }
        store_chunk<T>(kp + (row0 + n) * k.rs + ch * VL, y);
    }
    const int q0 = t.lo / 4, nq = (t.hi + 3) / 4 - q0;
    for (int x = tid; x < nq * chunks; x += KV_THREADS) {
        const int ch = x / nq, n4 = 4 * (q0 + x - ch * nq);
        unsigned w[VL];
#pragma unroll
        for (int e = 0; e < VL; e++) w[e] = *reinterpret_cast<const unsigned *>(vc + (ch * VL + e) * KV8_PAGE + n4);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int tok = n4 + u;
            if (tok < t.lo || tok >= t.hi) continue;
            const bool lost = bad >> tok & 1;
            float y[VL];
#pragma unroll
            for (int e = 0; e < VL; e++) y[e] = lost ? NAN : (float)(signed char)(w[e] >> (8 * u)) * sc.y;
            store_chunk<T>(vp + (row0 + tok - t.lo) * v.rs + ch * VL, y);
        }
    }
}

// pages that max_rows consecutive tokens can touch
int pages_per_seq(int max_rows) { return (max_rows + KV8_PAGE - 2) / KV8_PAGE + 1; }

// every row and head begins at a multiple of 16 bytes
bool pieces(const RowsView &v, int64_t size) {
    return (reinterpret_cast<uintptr_t>(v.p) | (uintptr_t)(v.rs * size) | (uintptr_t)(v.hs * size)) % 16 == 0;
}

template <class T>
hipError_t launch_append(const Kv8View &c, const Kv8Seqs &s, const RowsView &k, const RowsView &v, int g,
                         const RowsView &q, const RowsView &qo, const RopeArg &rope, int per, int64_t blocks,
                         hipStream_t st) {
    constexpr int VL = Chunk<T>::N;
    // In 16-byte pieces where the rows are aligned to them and a pair's halves
    // lie in the same two pieces: 12,300 bfloat16 rows of 32 + 8 heads of 128,
    // half of them rotated, 70 us, value by value 223.
    const bool vec = pieces(k, sizeof(T)) && pieces(v, sizeof(T)) && pieces(q, sizeof(T)) && pieces(qo, sizeof(T)) &&
                     c.d % (2 * VL) == 0 && rope.rot % (2 * VL) == 0;
    if (vec && s.max_rows <= 4)
        hipLaunchKernelGGL((k_kv8_append_vec<T, 64>), dim3(blocks), dim3(64), 0, st, c, s, k, v, q, qo, g, per, rope);
    else if (vec)
        hipLaunchKernelGGL((k_kv8_append_vec<T, 256>), dim3(blocks), dim3(256), 0, st, c, s, k, v, q, qo, g, per, rope);
    else {
        const size_t lds = sizeof(float) * (size_t)(s.max_rows < KV8_PAGE ? s.max_rows : KV8_PAGE) * c.d + (size_t)VQ * c.d;
        hipLaunchKernelGGL(k_kv8_append<T>, dim3(blocks), dim3(KV_THREADS), lds, st, c, s, k, v, q, qo, g, per, rope);
    }
    return hipGetLastError();
}

template <class T>
hipError_t launch_read(const Kv8View &c, const Kv8Seqs &s, const RowsView &k, const RowsView &v, int per, int64_t blocks,
                       hipStream_t st) {
    if (pieces(k, sizeof(T)) && pieces(v, sizeof(T)))  // a head has whole pieces
        hipLaunchKernelGGL(k_kv8_read_vec<T>, dim3(blocks), dim3(KV_THREADS), 0, st, c, s, k, v, per);
    else hipLaunchKernelGGL(k_kv8_read<T>, dim3(blocks), dim3(KV_THREADS), 0, st, c, s, k, v, per);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_kv8_append(const Kv8View &c, const Kv8Seqs &s, int dtype, const RowsView &k, const RowsView &v,
                             int heads, const RowsView &q, const RowsView &qo, const RopeArg &rope, hipStream_t st) {
    const int per = pages_per_seq(s.max_rows), g = heads / c.hk;
    const int64_t blocks = (int64_t)s.n_seq * per * c.hk;
    if (blocks == 0) return hipSuccess;
    if (!kv8_grid(blocks, KV_THREADS)) return hipErrorInvalidValue;
    switch (dtype) {
        case FT_F32: return launch_append<float>(c, s, k, v, g, q, qo, rope, per, blocks, st);
        case FT_F16: return launch_append<_Float16>(c, s, k, v, g, q, qo, rope, per, blocks, st);
        case FT_BF16: return launch_append<__bf16>(c, s, k, v, g, q, qo, rope, per, blocks, st);
    }
    return hipErrorInvalidValue;
}

hipError_t launch_kv8_read(const Kv8View &c, const Kv8Seqs &s, int dtype, const RowsView &k, const RowsView &v,
                           hipStream_t st) {
    const int per = pages_per_seq(s.max_rows);
    const int64_t blocks = (int64_t)s.n_seq * per * c.hk;
    if (blocks == 0) return hipSuccess;
    if (!kv8_grid(blocks, KV_THREADS)) return hipErrorInvalidValue;
    switch (dtype) {
        case FT_F32: return launch_read<float>(c, s, k, v, per, blocks, st);
        case FT_F16: return launch_read<_Float16>(c, s, k, v, per, blocks, st);
        case FT_BF16: return launch_read<__bf16>(c, s, k, v, per, blocks, st);
    }
    return hipErrorInvalidValue;
}

}  // namespace cih

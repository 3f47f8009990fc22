// The 8-bit paged key/value cache: rows of K and V rotated, quantized and
// written into their pages, and read back.
//
// A workgroup owns one (page, head) that its sequence's new rows touch, so the
// page's scale, its kept codes and its new ones change under one owner:
//   s = max(s_old where tokens are kept, max |new| / 127)
//   kept codes  q <- rint(q s_old / s)   only where s grew
//   new codes   q  = rint(x / s)
#include <float.h>

#include "kv8.h"

namespace cih {

namespace {

constexpr int KV_THREADS = 256;
constexpr int VQ = KV8_PAGE + 4;  // bytes of a dim's codes in LDS

// cos and sin (times gain) of position p's angle at pair j.  The angle in
// turns is reduced in 64 bits: at position 1e6 a 32-bit product is off by
// 0.06 radians.
__device__ __forceinline__ void rope_cs(const RopeArg &r, int p, int j, float &c, float &s) {
    const double a = (double)p * r.turns[j];
    const float t = (float)(a - rint(a));
    sincospif(2.0f * t, &s, &c);
    c *= r.gain;
    s *= r.gain;
}

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

__device__ __forceinline__ int code8(float x, float inv) {
    return (int)fminf(fmaxf(rintf(x * inv), -127.0f), 127.0f) & 0xff;
}
// four codes scaled again
__device__ __forceinline__ unsigned recode4(unsigned w, float ratio) {
    unsigned o = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) o |= (unsigned)code8((float)(signed char)(w >> (8 * e)), ratio) << (8 * e);
    return o;
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
    // scales too small to be inverted are 0, and so are their codes
    float2 sc = {mk / 127.0f, mv / 127.0f};
    if (!(sc.x >= FLT_MIN)) sc.x = 0.0f;
    if (!(sc.y >= FLT_MIN)) sc.y = 0.0f;
    const int64_t ph = (int64_t)id * c.hk + t.h;
    float2 old = {0.0f, 0.0f};
    unsigned long long kept_bad = 0;
    if (t.lo > 0) {
        old = c.scales[ph];
        kept_bad = c.bad[ph] & ((1ull << t.lo) - 1);
        sc.x = fmaxf(sc.x, old.x);
        sc.y = fmaxf(sc.y, old.y);
    }
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

// pages that max_rows consecutive tokens can touch
int pages_per_seq(int max_rows) { return (max_rows + KV8_PAGE - 2) / KV8_PAGE + 1; }

}  // namespace

hipError_t launch_kv8_append(const Kv8View &c, const Kv8Seqs &s, int dtype, const RowsView &k, const RowsView &v,
                             int heads, const RowsView &q, const RowsView &qo, const RopeArg &rope, hipStream_t st) {
    const int per = pages_per_seq(s.max_rows);
    const int64_t blocks = (int64_t)s.n_seq * per * c.hk;
    if (blocks == 0) return hipSuccess;
    if (blocks > INT32_MAX) return hipErrorInvalidValue;
    const size_t lds = sizeof(float) * (size_t)(s.max_rows < KV8_PAGE ? s.max_rows : KV8_PAGE) * c.d + (size_t)VQ * c.d;
    const int g = heads / c.hk;
    switch (dtype) {
        case FT_F32:
            hipLaunchKernelGGL(k_kv8_append<float>, dim3(blocks), dim3(KV_THREADS), lds, st, c, s, k, v, q, qo, g, per, rope);
            break;
        case FT_F16:
            hipLaunchKernelGGL(k_kv8_append<_Float16>, dim3(blocks), dim3(KV_THREADS), lds, st, c, s, k, v, q, qo, g, per, rope);
            break;
        case FT_BF16:
            hipLaunchKernelGGL(k_kv8_append<__bf16>, dim3(blocks), dim3(KV_THREADS), lds, st, c, s, k, v, q, qo, g, per, rope);
            break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t launch_kv8_read(const Kv8View &c, const Kv8Seqs &s, int dtype, const RowsView &k, const RowsView &v,
                           hipStream_t st) {
    const int per = pages_per_seq(s.max_rows);
    const int64_t blocks = (int64_t)s.n_seq * per * c.hk;
    if (blocks == 0) return hipSuccess;
    if (blocks > INT32_MAX) return hipErrorInvalidValue;
    switch (dtype) {
        case FT_F32: hipLaunchKernelGGL(k_kv8_read<float>, dim3(blocks), dim3(KV_THREADS), 0, st, c, s, k, v, per); break;
        case FT_F16: hipLaunchKernelGGL(k_kv8_read<_Float16>, dim3(blocks), dim3(KV_THREADS), 0, st, c, s, k, v, per); break;
        case FT_BF16: hipLaunchKernelGGL(k_kv8_read<__bf16>, dim3(blocks), dim3(KV_THREADS), 0, st, c, s, k, v, per); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace cih

// Verification of drafted tokens (speculative sampling, Leviathan et al. 2023): with p =
// softmax(logits / T) and q = softmax(draft logits / T), draft x is taken if u q(x) < p(x).
// The token after the taken ones comes from max(p - q, 0) at the first refusal, from p
// after all drafts: the first whose running sum passes v times the whole.  T = 0: the largest logit.
//
// Whether a draft is taken asks for two sums of a row, whose FP32 exponentials' errors (10^-7) decide
// as rarely as the random numbers' own 24 bits do.  A drawn token lies between two running sums of
// as many terms as there are tokens, and errors of 10^-7 of the whole would move it to a neighbour in one
// draw of a hundred (131,072 tokens): what is drawn from is summed in 64 bits, and only that row.
//
// k_verify_rows: (largest, sum) of parts of all rows.  k_verify_finish, a workgroup a part of the
// drawn row of a sequence: where its drafts end, then 64-bit sums of pieces of the part; the last workgroup of a sequence
// draws.  k_verify_narrow does it all for vocabularies of up to 256 tokens, a workgroup a sequence.
//
// One pass sums what is left of p, max(e_p - r e_q, 0) with r = Z_p / Z_q, before r is known in 64 bits: the tokens that count
// are those with e_p / e_q > r, and with r from the FP32 sums they are the same ones unless a token's ratio lies
// between the two.  The pass keeps the sums of e_p and e_q over them, and how near to r the nearest ratio is; where the 64-bit r
// turns out to be further away than that, the last workgroup sums the row again: of FP32 rows of 131,072 tokens one in a hundred where
// the draft's logits are 1 off the target's, a tenth at 0.03 to 0.1, a third at 0.01 (16-bit rows, whose ratios lie apart: none in a hundred).
// That one workgroup needs 200 us (finish of 64 FP32 sequences 37 -> 240).
//
// 64 sequences of 3 to 7 drafts over 131,072 tokens (bfloat16): rows 29 us, bound by bytes (168 MB at 5.7 TB/s, a part from the
// last-level cache), finish 34, bound by the 64-bit exponentials of 64 rows of p and q and three turns of dependent
// loads; 8 drafted streams over 33 tokens (narrow) 4.3, a chain of loads and sums.
#include <float.h>

#include <type_traits>

#include "kernels.h"
#include "kv8.h"

namespace cih {

namespace {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr int NONE = 0x7fffffff;
constexpr int VERIFY_THREADS = 256, VERIFY_WAVES = VERIFY_THREADS / 64;
constexpr int NARROW = 256;  // tokens
constexpr int FINE = 512;    // tokens of a piece of a part, of which the sums are kept

// Values of other lanes without LDS trips, word by word: f(word) gives each word's.
template <class V, class F> __device__ __forceinline__ V words(V v, F f) {
    constexpr int N = sizeof(V) / 4;
    struct {
        unsigned w[N];
    } x = __builtin_bit_cast(decltype(x), v);
#pragma unroll
    for (int k = 0; k < N; k++) x.w[k] = f(x.w[k]);
    return __builtin_bit_cast(V, x);
}
template <int C, int ROWS, class V> __device__ __forceinline__ V dpp_of(V v) {  // 0 where there is no such lane
    return words(v, [](unsigned x) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, C, ROWS, 0xf, false); });
}
template <class V> __device__ __forceinline__ V across(V v, bool far) {  // lane ^ 32, or ^ 16
    return words(v, [&](unsigned x) {
        unsigned y = x;
        asm volatile("" : "+v"(y));  // a register of its own
        const auto r = far ? __builtin_amdgcn_permlane32_swap(x, y, false, false) : __builtin_amdgcn_permlane16_swap(x, y, false, false);
        const unsigned r0 = r[0], r1 = r[1];
        return threadIdx.x & (far ? 32 : 16) ? r0 : r1;
    });
}
// op over the wave, the same in all lanes: neighbours, quads, halves of a row's 16 lanes, rows.
template <class V, class OP> __device__ __forceinline__ V wave_all(V v, OP op) {
    v = op(v, dpp_of<0xB1, 0xf>(v));
    v = op(v, dpp_of<0x4E, 0xf>(v));
    v = op(v, dpp_of<0x141, 0xf>(v));
    v = op(v, dpp_of<0x140, 0xf>(v));
    v = op(v, across(v, false));
    return op(v, across(v, true));
}
// Running sum over the wave's lanes: within rows of 16, then the rows before.
__device__ __forceinline__ double running(double c) {
    c += dpp_of<0x111, 0xf>(c);
    c += dpp_of<0x112, 0xf>(c);
    c += dpp_of<0x114, 0xf>(c);
    c += dpp_of<0x118, 0xf>(c);
    c += dpp_of<0x142, 0xa>(c);
    c += dpp_of<0x143, 0xc>(c);
    return c;
}
template <int W = VERIFY_WAVES, class V, class OP> __device__ __forceinline__ V block_all(V v, OP op, V *red) {
    v = wave_all(v, op);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int w = 1; w < W; w++) v = op(v, red[w]);
    return v;
}
struct Plus {
    template <class V> __device__ __forceinline__ V operator()(V a, V b) const { return a + b; }
};
struct Less {
    template <class V> __device__ __forceinline__ V operator()(V a, V b) const { return b < a ? b : a; }
};
struct More {
    template <class V> __device__ __forceinline__ V operator()(V a, V b) const { return b > a ? b : a; }
};

// A row's largest logit (NaN: one is NaN or +inf), where it first stands, sum of exp((x - largest) / T).
struct Stats {
    float m, s;
    int at;
};
__device__ __forceinline__ bool no_dist(float m) { return !(m <= FLT_MAX && m > -INFINITY); }

// 2^t for t <= 0, to 4 10^-16 of itself (0 from t = -1000 on): t = k + f with |f| <= 1/2, 2^f by the polynomial
// of degree 10 that meets it at the 11 Chebyshev nodes, k into the exponent.  Half the clocks of the library's
// exp, which the sums of a drawn row wait for.
__device__ __forceinline__ double pow2(double t) {
    constexpr double WHOLE = 6755399441055744.0;  // 1.5 2^52: its sum with a number has that rounded in its low bits
    const double near = fmax(t, -1000.0), kd = near + WHOLE, f = near - (kd - WHOLE);
    double e = 7.072585949269223e-09;
    e = fma(e, f, 1.0208690299958306e-07);
    e = fma(e, f, 1.321544258792169e-06);
    e = fma(e, f, 1.5252657260200837e-05);
    e = fma(e, f, 0.0001540353044173605);
    e = fma(e, f, 0.0013333558230164974);
    e = fma(e, f, 0.009618129107606888);
    e = fma(e, f, 0.05550410866444772);
    e = fma(e, f, 0.24022650695910097);
    e = fma(e, f, 0.69314718055995);
    e = fma(e, f, 1.0);
    const double o = __hiloint2double(__double2hiint(e) + (__double2loint(kd) << 20), __double2loint(e));
    return t > -1000.0 ? o : 0.0;
}

// exp((x - m) / T) as FP32 and in 64 bits (for x <= m).
struct Heat {
    float scale;  // log2 e / T
    double over;  // the same
    // (a finite scale above 0: at the edges of FP32 0 and -inf differences keep their exponentials)
    __device__ __forceinline__ explicit Heat(float t)
        : scale(t > 0.0f ? fminf(fmaxf(LOG2E / t, FLT_MIN), FLT_MAX) : 0.0f), over(t > 0.0f ? 1.4426950408889634074 / (double)t : 0.0) {}
    __device__ __forceinline__ float e32(float x, float m) const { return __builtin_amdgcn_exp2f((x - m) * scale); }
    __device__ __forceinline__ double e64(float x, float m) const { return pow2(((double)x - (double)m) * over); }
};

// What a sequence's drafts are.
struct Drafts {
    int c0, c1;
    __device__ __forceinline__ Drafts(const VerifyDrafts &v, int i) {
        c0 = min(max(v.cu[i], 0), v.n_drafts);
        c1 = min(max(v.cu[i + 1], c0), v.n_drafts);
    }
};
template <class T> __device__ __forceinline__ const T *target_row(const VerifyDrafts &v, int64_t r) { return static_cast<const T *>(v.logits) + r * v.stride; }
template <class T> __device__ __forceinline__ const T *draft_row(const VerifyDrafts &v, int64_t r) { return static_cast<const T *>(v.draft) + r * v.draft_stride; }

// A draft of the target's row, with its logits (qrow nullptr: it is certain).
struct Draft {
    int x;
    float at, lp, lq;
    bool certain, known;
    Draft() = default;
    template <class T>
    __device__ __forceinline__ Draft(const VerifyDrafts &v, const Heat &h, int d, const T *prow, const T *qrow) : x(v.drafted[d]), at(0.0f), lp(0.0f), lq(0.0f) {
        known = x >= 0 && x < v.vocab;
        certain = qrow == nullptr;
        if (h.over > 0.0) {
            at = v.accept_at[d];
            lp = to_f32(prow[known ? x : 0]);
            lq = certain ? 0.0f : to_f32(qrow[known ? x : 0]);
        }
    }
    // whether it is taken, p and q the rows' stats
    __device__ __forceinline__ bool taken(const Heat &h, const Stats &p, const Stats &q) const {
        if (h.over == 0.0) return x == p.at;
        const double px = h.e64(lp, p.m) / (double)p.s, qx = certain ? 1.0 : h.e64(lq, q.m) / (double)q.s;
        return known && (double)at * qx < px;
    }
};

// ---- narrow vocabularies: a workgroup a sequence, its waves take the rows in turn -----------------

// A row of at most 64 NK tokens: token 64 k + lane.
template <class T, int NK> struct NarrowRow {
    float x[NK];
    __device__ __forceinline__ void load(const T *row, int vocab, int lane) {
#pragma unroll
        for (int k = 0; k < NK; k++) x[k] = 64 * k + lane < vocab ? to_f32(row[64 * k + lane]) : -INFINITY;
    }
    __device__ __forceinline__ Stats stats(const Heat &h, int vocab, int lane) const {
        float m = -INFINITY;
        int at = NONE;
        bool bad = false;
#pragma unroll
        for (int k = 0; k < NK; k++) {
            bad |= !(x[k] < INFINITY);
            if (x[k] > m) {
                m = x[k];
                at = 64 * k + lane;
            }
        }
        const float all = wave_all(m, More());
        Stats s{all, 0.0f, wave_all(m == all ? at : NONE, Less())};
        if (__ballot(bad)) s.m = NAN;
        if (no_dist(s.m)) return s;
        if (h.over > 0.0) {
#pragma unroll
            for (int k = 0; k < NK; k++)
                if (64 * k < vocab) s.s += h.e32(x[k], all);
            s.s = wave_all(s.s, Plus());
        }
        return s;
    }
};

template <class T, int NK> __global__ __launch_bounds__(VERIFY_THREADS) void k_verify_narrow(VerifyDrafts v) {
    __shared__ int stops[VERIFY_WAVES];
    const int i = blockIdx.x, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Drafts d(v, i);
    const Heat h(v.temperature);
    const int n = d.c1 - d.c0;
    // rows 0 .. n, a wave each, until one is not taken (row n never is)
    int stop = NONE;
    Stats p{}, q{};
    NarrowRow<T, NK> pr, qr;
    bool lost = false;
    for (int r0 = 0;; r0 += VERIFY_WAVES) {
        const int r = r0 + wave;
        stop = NONE;
        if (r <= n) {
            const T *prow = target_row<T>(v, d.c0 + i + r), *qrow = v.draft && r < n ? draft_row<T>(v, d.c0 + r) : nullptr;
            pr.load(prow, v.vocab, lane);
            if (qrow) qr.load(qrow, v.vocab, lane);
            Draft draft;
            if (r < n) draft = Draft(v, h, d.c0 + r, prow, qrow);
            p = pr.stats(h, v.vocab, lane);
            lost = no_dist(p.m);
            if (qrow) {
                q = qr.stats(h, v.vocab, lane);
                lost |= no_dist(q.m);
            }
            if (lost || r == n || !draft.taken(h, p, q)) stop = r;
        }
        if (lane == 0) stops[wave] = stop;
        __syncthreads();
        int first = stops[0];
#pragma unroll
        for (int w = 1; w < VERIFY_WAVES; w++) first = min(first, stops[w]);
        if (first != NONE) {
            if (stop != first) return;  // (another wave's row, behind the last barrier)
            break;
        }
        __syncthreads();
    }
    int token = -1;
    if (!lost && h.over == 0.0) token = p.at;
    if (!lost && h.over > 0.0) {
        const bool refused = stop < n;
        const int x = refused ? v.drafted[d.c0 + stop] : -1;
        // the sums of both in 64 bits, then what is drawn from
        double w[NK], zp = 0.0, zq = 0.0, all = 0.0;
#pragma unroll
        for (int k = 0; k < NK; k++) {
            w[k] = 0.0;
            if (64 * k < v.vocab) {
                w[k] = h.e64(pr.x[k], p.m);
                zp += w[k];
                if (refused && v.draft) zq += h.e64(qr.x[k], q.m);
            }
        }
        zp = wave_all(zp, Plus());
        if (refused) {
            double left[NK];
            const double rq = v.draft ? zp / wave_all(zq, Plus()) : 0.0;
#pragma unroll
            for (int k = 0; k < NK; k++) {
                left[k] = 0.0;
                if (64 * k < v.vocab) left[k] = v.draft ? fmax(w[k] - h.e64(qr.x[k], q.m) * rq, 0.0) : 64 * k + lane == x ? 0.0 : w[k];
                all += left[k];
            }
            all = wave_all(all, Plus());
            if (all > 0.0) {
#pragma unroll
                for (int k = 0; k < NK; k++) w[k] = left[k];
            }
        }
        if (!(all > 0.0)) all = zp;
        const double border = (double)v.sample_at[i] * all;
        double sum = 0.0;
        int found = NONE, last = -1;
#pragma unroll
        for (int k = 0; k < NK; k++) {
            if (64 * k >= v.vocab || found != NONE) continue;
            const double c = running(w[k]);
            const unsigned long long past = __ballot(w[k] > 0.0 && sum + c > border), some = __ballot(w[k] > 0.0);
            if (past) found = 64 * k + __builtin_ctzll(past);
            if (some) last = 64 * k + 63 - __builtin_clzll(some);
            sum += __shfl(c, 63);
        }
        token = found != NONE ? found : last;
    }
    if (lane == 0) {
        v.accepted[i] = stop;
        v.tokens[i] = token;
    }
}

// ---- wide vocabularies ------------------------------------------------------------------------

// Parts of a row, of whole pieces: 8 to 32 pieces, so that all rows make some 2048 workgroups, and at most
// 256 parts.
struct Cut {
    int parts, size;
    Cut(int n_seq, int n_drafts, int vocab) {
        const int64_t rows = (int64_t)n_seq + 2 * (int64_t)n_drafts, pieces = ((int64_t)vocab + FINE - 1) / FINE;
        const int64_t want = pieces * rows / 2048, least = (pieces + 255) / 256;
        const int64_t each = want < 8 ? 8 : want > 32 ? 32 : want;
        size = (int)(each > least ? each : least) * FINE;
        parts = (int)(((int64_t)vocab + size - 1) / size);
    }
};
// Sums over a piece: e_p and e_q of the tokens that are left, and of all.
struct Piece {
    double left_p, left_q, p, q;
};
struct Space {
    Stats *stats;   // [rows of the target, then the draft][parts]
    int *done;      // [n_seq]: parts that have their sums
    double *near;   // [n_seq][parts]: of the ratios that decide what is left, how near the nearest is (log2)
    Piece *pieces;  // [n_seq][parts][fine]
    int rows, parts, size, fine;
    size_t bytes;
    Space(int n_seq, int n_drafts, int vocab, void *ws) {
        auto up32 = [](size_t n) { return (n + 31) / 32 * 32; };
        const Cut c(n_seq, n_drafts, vocab);
        rows = n_seq + n_drafts;
        parts = c.parts;
        size = c.size;
        fine = size / FINE;
        const size_t all = up32(((size_t)rows + n_drafts) * parts * sizeof(Stats)), own = up32((size_t)n_seq * sizeof(int));
        const size_t cut = (size_t)n_seq * parts;
        char *p = static_cast<char *>(ws);
        stats = reinterpret_cast<Stats *>(p);
        done = reinterpret_cast<int *>(p + all);
        near = reinterpret_cast<double *>(p + all + own);
        pieces = reinterpret_cast<Piece *>(p + all + own + up32(cut * sizeof(double)));
        bytes = all + own + up32(cut * sizeof(double)) + cut * fine * sizeof(Piece);
    }
};

// 16 bytes of a row's tokens j .. as FP32, -inf from `end` on.
template <class T, bool VEC> __device__ __forceinline__ void load16(const T *row, int j, int end, float (&x)[16 / sizeof(T)]) {
    constexpr int VL = 16 / sizeof(T);
    typedef T vec __attribute__((ext_vector_type(VL)));
    if (VEC && j + VL <= end) {
        const vec y = *reinterpret_cast<const vec *>(row + j);
#pragma unroll
        for (int u = 0; u < VL; u++) x[u] = to_f32(y[u]);
    } else {
#pragma unroll
        for (int u = 0; u < VL; u++) x[u] = j + u < end ? to_f32(row[j + u]) : -INFINITY;
    }
}

// A part of a row: one pass with the largest logit so far.
template <class T, bool VEC> __global__ __launch_bounds__(VERIFY_THREADS) void k_verify_rows(VerifyDrafts v, Space s) {
    constexpr int VL = 16 / sizeof(T), RUN = 4, STEP = VERIFY_THREADS * VL;
    __shared__ float fred[VERIFY_WAVES];
    __shared__ int ired[VERIFY_WAVES];
    const int part = blockIdx.x % s.parts, r = blockIdx.x / s.parts;
    const T *row = r < s.rows ? target_row<T>(v, r) : draft_row<T>(v, r - s.rows);
    const Heat h(v.temperature);
    const int first = part * s.size, end = (int)min((int64_t)first + s.size, (int64_t)v.vocab);
    float m = -INFINITY, sum = 0.0f;
    int at = NONE;
    bool bad = false;
    for (int j0 = first + threadIdx.x * VL; j0 < end; j0 += RUN * STEP) {
        float x[RUN][VL];
#pragma unroll
        for (int k = 0; k < RUN; k++) {
            if (j0 + k * STEP < end) load16<T, VEC>(row, j0 + k * STEP, end, x[k]);
            else
#pragma unroll
                for (int u = 0; u < VL; u++) x[k][u] = -INFINITY;
        }
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < RUN; k++)
#pragma unroll
            for (int u = 0; u < VL; u++) {
                bad |= !(x[k][u] < INFINITY);
                top = fmaxf(top, x[k][u]);
            }
        if (top > m) {
            if (h.over == 0.0) {  // where it stands
#pragma unroll
                for (int k = RUN - 1; k >= 0; k--)
#pragma unroll
                    for (int u = VL - 1; u >= 0; u--)
                        if (x[k][u] == top) at = j0 + k * STEP + u;
            }
            sum *= h.e32(m, top);  // (0 at first)
            m = top;
        }
        if (h.over > 0.0 && m > -INFINITY)
#pragma unroll
            for (int k = 0; k < RUN; k++)
#pragma unroll
                for (int u = 0; u < VL; u++) sum += h.e32(x[k][u], m);
    }
    const float all = block_all(m, More(), fred);
    if (m > -INFINITY) sum *= h.e32(m, all);
    sum = block_all(sum, Plus(), fred);
    if (h.over == 0.0) at = block_all(m == all ? at : NONE, Less(), ired);
    const bool lost = __syncthreads_or(bad);
    if (threadIdx.x == 0) {
        s.stats[blockIdx.x] = {lost ? NAN : all, sum, at};
        if (part == 0 && r < v.n_seq) s.done[r] = 0;
    }
}

// The parts of a row joined, by a wave.
__device__ __forceinline__ Stats join(const Stats *s, int parts, const Heat &h, int lane) {
    Stats o{-INFINITY, 0.0f, NONE};
    bool bad = false;
    for (int k = lane; k < parts; k += 64) {
        const Stats x = s[k];
        bad |= x.m != x.m;
        const float m = fmaxf(o.m, x.m);
        if (m > -INFINITY) {
            o.s = o.s * (o.m > -INFINITY ? h.e32(o.m, m) : 0.0f) + x.s * (x.m > -INFINITY ? h.e32(x.m, m) : 0.0f);
            if (x.m > o.m) o.at = x.at;
            o.m = m;
        }
    }
    const float m = wave_all(o.m, More());
    o.s = wave_all(o.m > -INFINITY ? o.s * h.e32(o.m, m) : 0.0f, Plus());
    o.at = wave_all(o.m == m ? o.at : NONE, Less());
    o.m = __ballot(bad) ? NAN : m;
    return o;
}

// What is drawn from, in units of 1 / Z_p: max(p - q, 0) (left) and p.
template <class T> struct Weights {
    const T *prow, *qrow;
    Heat h;
    float pm, qm;
    double rq;  // Z_p / Z_q
    int x;      // a certain draft that was refused, else -1
    bool refused;
    __device__ __forceinline__ void of(float p, float q, int j, double &left, double &all) const {
        all = h.e64(p, pm);
        left = qrow ? fmax(all - h.e64(q, qm) * rq, 0.0) : j == x ? 0.0 : all;
    }
};


// Numbers that another workgroup of the launch reads: past the XCDs' caches, without writing those back, as a fence would
// (64 sequences of 8 workgroups: 120 us, so 39).
__device__ __forceinline__ void share(double *p, double x) { __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ double shared(const double *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

constexpr int FINISH_THREADS = 512, FINISH_WAVES = FINISH_THREADS / 64;  // (a token of a piece a thread)

// The token, by the last workgroup of sequence i: the piece in which the border lies, by every wave, then a thread a token.
template <class T, class SUM> __device__ __forceinline__ int drawn(const VerifyDrafts &v, const Weights<T> &w, int i, int which, SUM sum_of, double *part, int *ired) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int pieces = (v.vocab + FINE - 1) / FINE;
    double all = 0.0;
    for (int f = lane; f < pieces; f += 64) all += sum_of(f, which);
    all = wave_all(all, Plus());
    if (which == 0 && !(all > 0.0)) {  // nothing left: from p itself
        which = 1;
        all = 0.0;
        for (int f = lane; f < pieces; f += 64) all += sum_of(f, which);
        all = wave_all(all, Plus());
    }
    const double border = (double)v.sample_at[i] * all;
    // the first piece whose running sum passes the border; else the last one with a weight
    double sum = 0.0, start = 0.0, last_start = 0.0;
    int piece = NONE, last = 0;
    for (int f0 = 0; f0 < pieces && piece == NONE; f0 += 64) {
        const double x = f0 + lane < pieces ? sum_of(f0 + lane, which) : 0.0, c = running(x);
        const unsigned long long past = __ballot(x > 0.0 && sum + c > border), some = __ballot(x > 0.0);
        if (past) {
            const int at = __builtin_ctzll(past);
            piece = f0 + at;
            start = sum + __shfl(c - x, at);
        }
        if (some) {
            const int at = 63 - __builtin_clzll(some);
            last = f0 + at;
            last_start = sum + __shfl(c - x, at);
        }
        sum += __shfl(c, 63);
    }
    if (piece == NONE) {
        piece = last;
        start = last_start;
    }
    const int j = piece * FINE + threadIdx.x;
    double x = 0.0;
    if (j < v.vocab) {
        double left, p;
        w.of(to_f32(w.prow[j]), w.qrow ? to_f32(w.qrow[j]) : 0.0f, j, left, p);
        x = which == 1 ? p : left;
    }
    double c = running(x);
    __syncthreads();  // part was read
    if (lane == 63) part[wave] = c;
    __syncthreads();
    c += start;
    for (int u = 0; u < wave; u++) c += part[u];
    const int found = block_all<FINISH_WAVES>(x > 0.0 && c > border ? j : NONE, Less(), ired);
    const int behind = block_all<FINISH_WAVES>(x > 0.0 ? j : -1, More(), ired);
    return found != NONE ? found : behind;
}

// Where a sequence's drafts end, found by every workgroup of it (a wave a row: eight, so that up to seven drafts take one
// round); then a part's sums, a wave a piece; the last workgroup draws.
template <class T, bool VEC> __global__ __launch_bounds__(FINISH_THREADS) void k_verify_finish(VerifyDrafts v, Space s) {
    constexpr int VL = 16 / sizeof(T);
    struct Turn {
        int taken, lost, refused, at;
        Stats p, q;
    };
    __shared__ Turn turns[FINISH_WAVES];
    __shared__ double dred[FINISH_WAVES];
    __shared__ int ired[FINISH_WAVES];
    const int part = blockIdx.x % s.parts, i = blockIdx.x / s.parts;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Drafts d(v, i);
    const Heat h(v.temperature);
    const int n = d.c1 - d.c0;
    Turn t{};
    for (int r0 = 0;; r0 += FINISH_WAVES) {
        const int r = r0 + wave;
        t.taken = NONE;
        if (r <= n) {
            const bool drafted = v.draft && r < n;
            Draft draft;
            if (r < n)
                draft = Draft(v, h, d.c0 + r, target_row<T>(v, d.c0 + i + r), drafted ? draft_row<T>(v, d.c0 + r) : nullptr);
            const Stats p = join(s.stats + (int64_t)(d.c0 + i + r) * s.parts, s.parts, h, lane);
            const Stats q = drafted ? join(s.stats + (int64_t)(s.rows + d.c0 + r) * s.parts, s.parts, h, lane) : Stats{};
            const bool lost = no_dist(p.m) || (drafted && no_dist(q.m));
            if (lost || r == n || !draft.taken(h, p, q)) t = {r, lost, r < n, p.at, p, q};
        }
        if (lane == 0) turns[wave] = t;
        __syncthreads();
        int first = 0;
#pragma unroll
        for (int w = 1; w < FINISH_WAVES; w++)
            if (turns[w].taken < turns[first].taken) first = w;
        t = turns[first];
        if (t.taken != NONE) break;
        __syncthreads();
    }
    if (t.lost || h.over == 0.0) {
        if (part == 0 && threadIdx.x == 0) {
            v.accepted[i] = t.taken;
            v.tokens[i] = t.lost ? -1 : t.at;
        }
        return;
    }
    const bool draft = t.refused && v.draft;
    Weights<T> w{target_row<T>(v, d.c0 + i + t.taken), draft ? draft_row<T>(v, d.c0 + t.taken) : nullptr, h, t.p.m, t.q.m, 0.0,
                 t.refused && !v.draft ? v.drafted[d.c0 + t.taken] : -1, t.refused != 0};
    // log2 of the ratio that decides what is left, from the FP32 sums
    const double about = draft ? log2((double)t.p.s / (double)t.q.s) : 0.0;
    const int end = (int)min((int64_t)(part + 1) * s.size, (int64_t)v.vocab);
    double near = INFINITY;
    for (int f = wave; f < s.fine; f += FINISH_WAVES) {
        const int first = part * s.size + f * FINE, last = min(first + FINE, end);
        Piece o{0.0, 0.0, 0.0, 0.0};
        for (int j = first + lane * VL; j < last; j += 64 * VL) {
            float x[VL], y[VL];
            load16<T, VEC>(w.prow, j, last, x);
            if (draft) {
                load16<T, VEC>(w.qrow, j, last, y);
#pragma unroll
                for (int u = 0; u < VL; u++) {
                    const double tp = ((double)x[u] - (double)w.pm) * h.over, tq = ((double)y[u] - (double)w.qm) * h.over;
                    const double ep = pow2(tp), eq = pow2(tq), over = tp - tq - about;  // (NaN where both are -inf)
                    near = fmin(near, fabs(over));
                    o.p += ep;
                    o.q += eq;
                    o.left_p += over > 0.0 ? ep : 0.0;
                    o.left_q += over > 0.0 ? eq : 0.0;
                }
            } else {
#pragma unroll
                for (int u = 0; u < VL; u++) {
                    const double ep = h.e64(x[u], w.pm);
                    o.p += ep;
                    o.left_p += j + u == w.x ? 0.0 : ep;
                }
            }
        }
        o.p = wave_all(o.p, Plus());
        o.left_p = wave_all(o.left_p, Plus());
        if (draft) {
            o.q = wave_all(o.q, Plus());
            o.left_q = wave_all(o.left_q, Plus());
        }
        if (lane == 0) {
            Piece *to = s.pieces + ((int64_t)i * s.parts + part) * s.fine + f;
            share(&to->left_p, o.left_p);
            share(&to->left_q, o.left_q);
            share(&to->p, o.p);
            share(&to->q, o.q);
        }
    }
    near = block_all<FINISH_WAVES>(near, Less(), dred);
    if (threadIdx.x == 0) share(&s.near[(int64_t)i * s.parts + part], near);
    // the last workgroup of the sequence sees the others' sums: they are written before it is counted
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) ired[0] = atomicAdd(&s.done[i], 1);
    __syncthreads();
    if (ired[0] != s.parts - 1) return;
    Piece *own = s.pieces + (int64_t)i * s.parts * s.fine;
    const int pieces = (v.vocab + FINE - 1) / FINE;  // (parts are whole pieces: piece f of the row is own[f])
    int which = t.refused ? 0 : 1;
    if (draft) {
        double zp = 0.0, zq = 0.0;
        near = INFINITY;
        for (int f = lane; f < pieces; f += 64) {
            zp += shared(&own[f].p);
            zq += shared(&own[f].q);
        }
        for (int k = lane; k < s.parts; k += 64) near = fmin(near, shared(&s.near[(int64_t)i * s.parts + k]));
        zp = wave_all(zp, Plus());
        zq = wave_all(zq, Plus());
        near = wave_all(near, Less());
        w.rq = zp / zq;
        // (1e-10: the exponents' roundings, 1000 2^-53)
        if (!(fabs(log2(w.rq) - about) < near - 1e-10)) {
            __syncthreads();  // every wave has its sums
            for (int f = wave; f < pieces; f += FINISH_WAVES) {
                double sum = 0.0;
                for (int j = f * FINE + lane; j < min((f + 1) * FINE, v.vocab); j += 64) {
                    double left, p;
                    w.of(to_f32(w.prow[j]), to_f32(w.qrow[j]), j, left, p);
                    sum += left;
                }
                sum = wave_all(sum, Plus());
                if (lane == 0) {
                    share(&own[f].left_p, sum);
                    share(&own[f].left_q, 0.0);
                }
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
        }
    }
    auto sum_of = [&](int f, int which) __attribute__((always_inline)) {
        return which == 1 ? shared(&own[f].p) : draft ? fmax(shared(&own[f].left_p) - w.rq * shared(&own[f].left_q), 0.0) : shared(&own[f].left_p);
    };
    const int token = drawn<T>(v, w, i, which, sum_of, dred, ired);
    if (threadIdx.x == 0) {
        v.accepted[i] = t.taken;
        v.tokens[i] = token;
    }
}

template <class T> hipError_t launch(const VerifyDrafts &v, void *ws, hipStream_t st) {
    if (v.vocab <= NARROW) {
        if (!kv8_grid(v.n_seq, VERIFY_THREADS)) return hipErrorInvalidValue;
        if (v.vocab <= 64) hipLaunchKernelGGL((k_verify_narrow<T, 1>), dim3(v.n_seq), dim3(VERIFY_THREADS), 0, st, v);
        else hipLaunchKernelGGL((k_verify_narrow<T, NARROW / 64>), dim3(v.n_seq), dim3(VERIFY_THREADS), 0, st, v);
        return hipGetLastError();
    }
    const Space s(v.n_seq, v.n_drafts, v.vocab, ws);
    const int64_t rows = (int64_t)v.n_seq + v.n_drafts + (v.draft ? v.n_drafts : 0), own = (int64_t)v.n_seq * s.parts;
    if (!kv8_grid(rows * s.parts, VERIFY_THREADS) || !kv8_grid(own, VERIFY_THREADS)) return hipErrorInvalidValue;
    if (!kv8_grid(own, FINISH_THREADS)) return hipErrorInvalidValue;
    auto aligned = [](const void *p, int64_t stride) { return (reinterpret_cast<uintptr_t>(p) | (uintptr_t)(stride * sizeof(T))) % 16 == 0; };
    auto go = [&](auto vec) -> hipError_t {
        constexpr bool VEC = decltype(vec)::value;
        hipLaunchKernelGGL((k_verify_rows<T, VEC>), dim3(rows * s.parts), dim3(VERIFY_THREADS), 0, st, v, s);
        if (const hipError_t rc = hipGetLastError(); rc != hipSuccess) return rc;
        hipLaunchKernelGGL((k_verify_finish<T, VEC>), dim3(own), dim3(FINISH_THREADS), 0, st, v, s);
        return hipGetLastError();
    };
    return aligned(v.logits, v.stride) && (!v.draft || aligned(v.draft, v.draft_stride)) ? go(std::true_type{}) : go(std::false_type{});
}

}  // namespace

size_t verify_drafts_bytes(int n_seq, int n_drafts, int vocab) {
    return vocab <= NARROW || n_seq == 0 ? 0 : Space(n_seq, n_drafts, vocab, nullptr).bytes;
}

hipError_t launch_verify_drafts(const VerifyDrafts &v, void *ws, hipStream_t st) {
    if (v.n_seq == 0) return hipSuccess;
    switch (v.dtype) {
        case FT_F32: return launch<float>(v, ws, st);
        case FT_F16: return launch<_Float16>(v, ws, st);
        case FT_BF16: return launch<__bf16>(v, ws, st);
    }
    return hipErrorInvalidValue;
}

}  // namespace cih

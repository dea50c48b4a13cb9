// dlr_losses.hip -- softmax losses on gfx950: log-probabilities of given
// classes and their gradient, the paired logistic (preference) loss, the
// clipped policy loss with a KL term, and log-probabilities straight from
// hidden states and the output layer's weights.
//
// Mathematics used throughout, for a row of logits z and a temperature tau:
//   lse     = log sum_j exp(z_j / tau)
//   logprob = z_y / tau - lse
//   d logprob / d z_j = (1[j = y] - exp(z_j / tau - lse)) / tau
// A row's statistics are its maximum m (exact: a logit) and
// s = sum_j 2^((z_j - m) k), k = log2(e) / tau, in 32 bits; the difference
// z_j - m is taken first because it is exact or nearly so for the terms that
// count, where z_j k - m k would lose bits to |m|.  lse = m / tau + ln s and
// everything after it is done once per row in 64 bits: a sequence's sum of
// log-probabilities nearly cancels against the reference model's, and the
// policy loss's gradient jumps at the clip's border.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <tuple>

#include "dlr_losses.h"

namespace dlr {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// Rows may start at any element: 16-byte accesses at an element's alignment.
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

#define NEG_INF (-__builtin_inff())

__device__ inline float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// k = hi + lo of the row statistics and of the gradients.  One float for k is
// off by up to 2^-23 (rounded down), always to the same side: lse would be off
// by that share of the mean |d| (1e-7 for logits of a trained model, as much as
// float32's own rounding), a gradient's probabilities by that share of their
// own |d| (1.7e-6 in the mean of 50,257 at temperature 0.7).
// The other roundings are of either sign and average out over a row; so does
// v_exp_f32's (mean -3e-9, at most 8e-8, measured over [-24, 0]).
// hi is k rounded down and lo > 0, so that d = -inf gives -inf twice.
struct ExpScale {
    float hi, lo;
};
__host__ __device__ inline ExpScale two_floats(double k) {  // k > 0
    float hi = (float)k;
    if ((double)hi > k) hi = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, hi) - 1u);  // one step down
    const float lo = (float)(k - (double)hi);
    return {hi, lo > 0.f ? lo : 1e-30f};
}
constexpr double kLog2e = 1.44269504088896340736;
__host__ __device__ inline ExpScale exp_scale(double temperature) { return two_floats(kLog2e / temperature); }
__device__ inline float exp2_scaled(float d, ExpScale k) { return exp2_hw(__builtin_fmaf(d, k.hi, d * k.lo)); }

// 16 bytes of a row: N elements.
template <typename T>
struct Pack;
template <>
struct Pack<float> {
    static constexpr int N = 4;
    static __device__ float get(const u32x4 &v, int i) { return __uint_as_float(v[i]); }
    static __device__ u32x4 put(const float *f) {
        u32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __float_as_uint(f[i]);
        return v;
    }
};
template <>
struct Pack<__bf16> {
    static constexpr int N = 8;
    static __device__ float get(const u32x4 &v, int i) {
        const uint32_t w = v[i >> 1];
        return __uint_as_float((i & 1) ? (w & 0xffff0000u) : (w << 16));
    }
    static __device__ u32x4 put(const float *f) {
        union {
            __bf16 h[8];
            u32x4 v;
        } u;
#pragma unroll
        for (int i = 0; i < 8; ++i) u.h[i] = (__bf16)f[i];  // round to nearest even
        return u.v;
    }
};
template <>
struct Pack<_Float16> {
    static constexpr int N = 8;
    static __device__ float get(const u32x4 &v, int i) {
        union {
            u32x4 v;
            _Float16 h[8];
        } u;
        u.v = v;
        return (float)u.h[i];
    }
    static __device__ u32x4 put(const float *f) {
        union {
            _Float16 h[8];
            u32x4 v;
        } u;
#pragma unroll
        for (int i = 0; i < 8; ++i) u.h[i] = (_Float16)f[i];
        return u.v;
    }
};

// A pack of a row.  `once`: past the caches, for logits that are more than
// they hold (the flag is the launch's; see kOnceBytes).
template <typename T>
__device__ inline u32x4 load_pack(const T *row, int64_t p, bool once) {
    const u32x4_any *at = reinterpret_cast<const u32x4_any *>(row + p * Pack<T>::N);
    return once ? __builtin_nontemporal_load(at) : *at;
}
// Gradients are written past the caches: 4,096 x 131,072 bf16 467 -> 454 us,
// 1,021 x 50,257 f32 91 -> 76 us.
template <typename T>
__device__ inline void store_pack(T *row, int64_t p, const u32x4 &v) {
    __builtin_nontemporal_store(v, reinterpret_cast<u32x4_any *>(row + p * Pack<T>::N));
}

__device__ inline int64_t load_target(const void *target, int bits, int64_t t) {
    return bits == 64 ? static_cast<const int64_t *>(target)[t] : static_cast<const int32_t *>(target)[t];
}

// ------------------------------------------------------------ row statistics

struct RowStat {
    float m;  // maximum (-inf: nothing yet)
    float s;  // sum of 2^((z - m) k)
};

// Joins b into a.  A side that is empty (m = -inf, s = 0) adds nothing; NaN
// and +inf anywhere make s NaN.
__device__ inline RowStat join(RowStat a, RowStat b, ExpScale k) {
    const float m = fmaxf(a.m, b.m);
    const float r = m == NEG_INF ? 0.f : m;
    return {m, a.s * exp2_scaled(a.m - r, k) + b.s * exp2_scaled(b.m - r, k)};
}

// The block's maximum and sum, in every thread.  The maximum first: each
// thread's sum is then scaled once, and the scaled sums are added in 64 bits.
// Joining pairs level by level would round the last levels' few numbers again
// and again: 1e-7 in lse, several times what the thread sums leave.
struct BlockStat {
    float m;
    double s;
};

template <int NT>
struct BlockLds {
    float m[NT / 64];
    double s[NT / 64];
};

template <int NT>
__device__ inline BlockStat join_block(RowStat a, ExpScale k, BlockLds<NT> &lds) {
    const int wave = threadIdx.x >> 6;
    float m = a.m;
#pragma unroll
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if ((threadIdx.x & 63) == 0) lds.m[wave] = m;
    __syncthreads();
    m = lds.m[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) m = fmaxf(m, lds.m[w]);
    const float r = m == NEG_INF ? 0.f : m;
    double s = (double)a.s * (double)exp2_scaled(a.m - r, k);
#pragma unroll
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) lds.s[wave] = s;
    __syncthreads();
    s = lds.s[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) s += lds.s[w];
    return {m, s};
}

// Terms are added to each other before they reach the running sum: one by
// one, those below half its last bit would all be lost, and a vocabulary's
// tail is many of them (3e-7 in lse at 131,072 classes).
template <int N>
__device__ inline float tree_sum(const float (&e)[N]) {
    float t[N];
#pragma unroll
    for (int i = 0; i < N; ++i) t[i] = e[i];
#pragma unroll
    for (int w = N / 2; w; w >>= 1)
#pragma unroll
        for (int i = 0; i < w; ++i) t[i] += t[i + w];
    return t[0];
}

// One pass over a row: U packs a thread in flight, one rescaling of the
// running sum per U packs.
template <typename T, int NT, int U>
__device__ inline RowStat row_stat(const T *row, int vocab, ExpScale k, bool once) {
    using PK = Pack<T>;
    constexpr int N = PK::N;
    const int packs = vocab / N;
    RowStat a{NEG_INF, 0.f};
    for (int base = threadIdx.x; base < packs; base += NT * U) {
        u32x4 v[U];
        bool have[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int p = base + u * NT;
            have[u] = p < packs;
            if (have[u]) v[u] = load_pack(row, p, once);
        }
        float m = a.m;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (have[u]) {
#pragma unroll
                for (int i = 0; i < N; ++i) m = fmaxf(m, PK::get(v[u], i));
            }
        const float r = m == NEG_INF ? 0.f : m;
        float s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            s[u] = 0.f;
            if (have[u]) {
                float e[N];
#pragma unroll
                for (int i = 0; i < N; ++i) e[i] = exp2_scaled(PK::get(v[u], i) - r, k);
                s[u] = tree_sum(e);
            }
        }
        a.s = a.s * exp2_scaled(a.m - r, k) + tree_sum(s);
        a.m = m;
    }
    const int tail = packs * N + threadIdx.x;
    if (tail < vocab) {
        const float z = (float)row[tail];
        a = join(a, RowStat{z, z == z ? 1.f : z}, k);
    }
    return a;
}

// The difference to the maximum first: lse itself cannot hold ln s where the
// logits are huge (a row masked with the type's lowest value).
__device__ inline double target_logprob(float zy, float m, double ln_s, double tau) {
    return ((double)zy - (double)m) / tau - ln_s;
}

// ----------------------------------------------------- token log-probabilities

// One row a workgroup, one read.  Bound by memory: 4,096 x 131,072 bf16, a
// quarter of the rows out, 141 us, 5.7 TB/s of what is read (the exponentials
// alone would take 55 us); short and few rows by the row's ends.
template <typename T, int NT>
__global__ __launch_bounds__(NT) void k_token_logprob(const T *logits, int64_t stride, int vocab, const void *target,
                                                      int target_bits, ExpScale k, double tau, bool once, float *logprob,
                                                      float *lse) {
    __shared__ BlockLds<NT> lds;
    const int64_t t = blockIdx.x;
    const int64_t y = load_target(target, target_bits, t);
    if (y < 0) {  // ignored: the row is not read
        if (threadIdx.x == 0) {
            logprob[t] = 0.f;
            lse[t] = 0.f;
        }
        return;
    }
    const T *row = logits + t * stride;
    const float zy = y < vocab ? (float)row[y] : __builtin_nanf("");
    const BlockStat a = join_block<NT>(row_stat<T, NT, 4>(row, vocab, k, once), k, lds);
    if (threadIdx.x == 0) {
        const double ln = log(a.s);
        lse[t] = (float)(a.m / tau + ln);
        logprob[t] = (float)target_logprob(zy, a.m, ln, tau);
    }
}

// ---- few long rows: a row's chunks by several workgroups
//
// A CU alone reads a long row slowly.  Up to 128 rows of 8,192 packs and more
// go by chunks: their statistics to scratch memory (and the target's logit,
// which the gradient may then overwrite), a second launch joins them.  1 x
// 131,072 bf16: 5.9 us, 10.9 by one workgroup; the policy loss 8.6, 18.8.  From
// about 160 rows on a workgroup a row is as fast (129 rows, logprob and policy
// loss: 13.5 and 28.5 by chunks, 14.1 and 29.5 by rows; 160: 14.2 and 31.9, 15.0
// and 30.8; 255: 18.3 and 43.1, 16.6 and 36.9).
struct RowPart {
    double s;
    float m;
    float pad;
};
struct RowParts {
    RowPart *part;  // rows x chunks
    float *zy;      // rows
    int chunks, span;
};

template <typename T, int NT>
__global__ __launch_bounds__(NT) void k_row_part(const T *logits, int64_t stride, int vocab, const void *target,
                                                 int target_bits, const float *weight, ExpScale k, RowParts w) {
    __shared__ BlockLds<NT> lds;
    const int64_t t = blockIdx.x / w.chunks;
    const int begin = (int)(blockIdx.x % w.chunks) * w.span, here = vocab - begin < w.span ? vocab - begin : w.span;
    const int64_t y = load_target(target, target_bits, t);
    if (y < 0 || (weight && weight[t] == 0.f)) return;
    const T *row = logits + t * stride;
    const BlockStat a = join_block<NT>(row_stat<T, NT, 4>(row + begin, here, k, false), k, lds);
    if (threadIdx.x == 0) {
        w.part[blockIdx.x] = {a.s, a.m, 0.f};
        if (y >= begin && y < begin + here) w.zy[t] = (float)row[y];
    }
}

// A row's chunks (at most 64) joined by one wave, in every lane.
__device__ inline BlockStat join_parts(const RowParts &w, int64_t t, ExpScale k) {
    const int lane = threadIdx.x & 63;
    RowPart q{0.0, NEG_INF, 0.f};
    if (lane < w.chunks) q = w.part[t * w.chunks + lane];
    float m = q.m;
#pragma unroll
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    double s = q.s * (double)exp2_scaled(q.m - (m == NEG_INF ? 0.f : m), k);
#pragma unroll
    for (int o = 32; o; o >>= 1) s += __shfl_xor(s, o);
    return {m, s};
}

__global__ __launch_bounds__(64) void k_token_finish(const void *target, int target_bits, int vocab, ExpScale k,
                                                     double tau, RowParts w, float *logprob, float *lse) {
    const int64_t t = blockIdx.x;
    const int64_t y = load_target(target, target_bits, t);
    if (y < 0) {
        if (threadIdx.x == 0) logprob[t] = lse[t] = 0.f;
        return;
    }
    const BlockStat a = join_parts(w, t, k);
    if (threadIdx.x == 0) {
        const double ln = log(a.s);
        lse[t] = (float)(a.m / tau + ln);
        logprob[t] = (float)target_logprob(y < vocab ? w.zy[t] : __builtin_nanf(""), a.m, ln, tau);
    }
}

// Writes `out`'s row of zeros.
template <typename T, int NT>
__device__ inline void zero_row(T *out, int vocab) {
    constexpr int N = Pack<T>::N;
    const int packs = vocab / N;
    const u32x4 z = {0u, 0u, 0u, 0u};
    for (int p = threadIdx.x; p < packs; p += NT) store_pack(out, p, z);
    const int tail = packs * N + threadIdx.x;
    if (tail < vocab) out[tail] = (T)0.f;
}

// out_j = (j = y ? c : 0) + prob(z_j), prob the probability times -c: the
// softmax residual.  Each thread reads a pack before it writes it, so out may
// be the row itself.
template <typename T, int NT, int U, typename F>
__device__ inline void residual_row(const T *row, T *out, int vocab, int64_t y, float c, F prob, bool once) {
    using PK = Pack<T>;
    constexpr int N = PK::N;
    const int packs = vocab / N;
    for (int base = threadIdx.x; base < packs; base += NT * U) {
        u32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int p = base + u * NT;
            if (p < packs) v[u] = load_pack(row, p, once);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int p = base + u * NT;
            if (p >= packs) continue;
            float f[N];
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] = prob(PK::get(v[u], i));
            const int64_t at = y - (int64_t)p * N;
            if (at >= 0 && at < N) {
#pragma unroll
                for (int i = 0; i < N; ++i) f[i] += i == at ? c : 0.f;
            }
            store_pack(out, p, PK::put(f));
        }
    }
    const int tail = packs * N + threadIdx.x;
    if (tail < vocab) out[tail] = (T)(prob((float)row[tail]) + (tail == y ? c : 0.f));
}

// 32 bits of lse are a relative error of |lse| 2^-24 in every probability:
// below 1e-5 up to here.  Rows beyond (logits in the hundreds, rows masked
// with the type's lowest value) take their statistics again.
constexpr float kLseExact = 128.f;

// What 2^((z - m) k) is multiplied by to give exp(z / tau - l): 1 / s where the l
// given is the row's own lse as far as 32 bits show (another rounding of it
// included), less where it is of more classes than these, as a caller has it
// who holds only some of them.
__device__ inline double share_of_lse(BlockStat a, double tau, float l) {
    if (a.s == 0.0 && l != NEG_INF) return 0.0;  // these classes have probability 0, others may not
    const double own = a.m / tau + log(a.s), off = own - (double)l;
    if ((float)own == l || fabs(off) <= 0x1p-23 * fabs(own)) return 1.0 / a.s;
    return exp(off) / a.s;
}

// One row a workgroup, one read and one write.  Bound by memory: 4,096 x
// 131,072 bf16 379 us (5.7 TB/s), 2,048 x 50,257 f16 with odd rows 71 us (5.1).
template <typename T, int NT>
__global__ __launch_bounds__(NT) void k_token_logprob_grad(const T *logits, int64_t stride, int vocab,
                                                           const void *target, int target_bits, ExpScale k, double tau,
                                                           bool once, const float *lse, const float *grad, T *out,
                                                           int64_t out_stride, int chunks, int span) {
    const int64_t t = blockIdx.x / chunks;
    const int begin = (int)(blockIdx.x % chunks) * span, here = vocab - begin < span ? vocab - begin : span;
    const int64_t y = load_target(target, target_bits, t);
    T *o = out + t * out_stride + begin;
    const float g = y < 0 ? 0.f : grad[t];
    if (g == 0.f) {  // ignored, or nothing flows back: the row is not read
        zero_row<T, NT>(o, here);
        return;
    }
    const T *row = logits + t * stride;
    const float c = y < vocab ? (float)(g / tau) : __builtin_nanf("");
    const float l = lse[t];
    if (fabsf(l) > kLseExact) {
        __shared__ BlockLds<NT> lds;
        const BlockStat a = join_block<NT>(row_stat<T, NT, 4>(row, vocab, k, false), k, lds);
        const float neg = (float)(-c * share_of_lse(a, tau, l)), m = a.s == 0.0 && l != NEG_INF ? 0.f : a.m;
        residual_row<T, NT, 4>(row + begin, o, here, y - begin, c,
                               [=](float z) { return neg * exp2_scaled(z - m, k); }, once);
        return;
    }
    // z / tau - l, rounded once, times log2(e); what the first floats of 1 / tau
    // and log2(e) leave out goes in before the second rounding
    const ExpScale it = two_floats(1.0 / tau), e = two_floats(kLog2e);
    const float it_lo = it.lo * e.hi;
    residual_row<T, NT, 4>(
        row + begin, o, here, y - begin, c,
        [=](float z) {
            const float x = __builtin_fmaf(z, it.hi, -l);
            return -c * exp2_hw(__builtin_fmaf(x, e.hi, __builtin_fmaf(x, e.lo, z * it_lo)));
        },
        once);
}

// ---------------------------------------------------------------- policy loss

struct PolicyOut {
    float *loss, *logprob, *kl;
    uint8_t *clipped;
};

// One row's loss from its log-probability, in 64 bits.  Returns d loss /
// d logprob times the weight; `write`: this caller writes the row's results.
__device__ inline double policy_token(double lp, const dlr_policy &p, int64_t t, double w, const PolicyOut &o,
                                      bool write) {
    const double adv = p.advantage[t];
    const double ratio = exp(lp - (double)p.old_logprob[t]);
    const double lo = 1.0 - p.clip_low, hi = 1.0 + p.clip_high;
    // min(ratio A, clip(ratio) A): the clip holds back gains above hi and
    // losses below lo; A = 0 has no surrogate (0 * inf otherwise)
    const bool held = (adv > 0.0 && ratio > hi) || (adv < 0.0 && ratio < lo);
    const double surrogate = adv == 0.0 ? 0.0 : (held ? (adv > 0.0 ? hi : lo) : ratio) * adv;
    double kl = 0.0, slope = held || adv == 0.0 ? 0.0 : -ratio * adv;
    double loss = -surrogate;
    if (p.ref_logprob) {
        const double gap = (double)p.ref_logprob[t] - lp;
        const double e = expm1(gap);
        kl = e - (e == __builtin_inf() ? 0.0 : gap);  // a class of probability 0: inf, not inf - inf
        if (p.kl_coef != 0.0) {
            loss += p.kl_coef * kl;
            slope -= p.kl_coef * e;
        }
    }
    if (ratio != ratio) loss = slope = ratio;  // NaN log-probabilities stay visible
    if (write) {
        o.loss[t] = (float)loss;
        o.logprob[t] = (float)lp;
        o.kl[t] = (float)kl;
        o.clipped[t] = held;
    }
    return slope * w;
}

__device__ inline void policy_nothing(int64_t t, const PolicyOut &o) {
    o.loss[t] = o.logprob[t] = o.kl[t] = 0.f;
    o.clipped[t] = 0;
}

// The second launch over a row's chunks: each joins the statistics and writes
// its part of the gradient, the first also the row's results.
template <typename T, int NT>
__global__ __launch_bounds__(NT) void k_policy_finish(const T *logits, int64_t stride, int vocab, const void *target,
                                                      int target_bits, ExpScale k, double tau, dlr_policy p,
                                                      PolicyOut po, T *out, int64_t out_stride, RowParts w) {
    __shared__ float coef;
    const int64_t t = blockIdx.x / w.chunks;
    const int begin = (int)(blockIdx.x % w.chunks) * w.span, here = vocab - begin < w.span ? vocab - begin : w.span;
    if (begin && !out) return;
    const int64_t y = load_target(target, target_bits, t);
    const float weight = p.weight ? p.weight[t] : 1.f;
    T *o = out + t * out_stride + begin;
    if (y < 0 || weight == 0.f) {
        if (begin == 0 && threadIdx.x == 0) policy_nothing(t, po);
        if (out) zero_row<T, NT>(o, here);
        return;
    }
    const BlockStat a = join_parts(w, t, k);
    if (threadIdx.x == 0) {
        const float zy = y < vocab ? w.zy[t] : __builtin_nanf("");
        const double lp = target_logprob(zy, a.m, log(a.s), tau);
        coef = (float)(policy_token(lp, p, t, weight, po, begin == 0) / tau);
    }
    if (!out) return;
    __syncthreads();
    const float c = coef, neg = (float)(-c / a.s), m = a.m;
    residual_row<T, NT, 4>(logits + t * stride + begin, o, here, y - begin, c,
                           [=](float z) { return neg * exp2_scaled(z - m, k); }, false);
}

// A row held by its workgroup: R packs a thread in registers, Q in LDS, pack i
// of thread x at i NT + x, and the element of the tail that is this thread's.
template <typename T, int NT, int R, int Q>
struct HeldRow {
    using PK = Pack<T>;
    u32x4 v[R];
    float tail;
    u32x4 *lds;  // [Q][NT], a thread touches its own

    __device__ void load(const T *row, int vocab, bool once) {
        const int packs = vocab / PK::N;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int p = i * NT + threadIdx.x;
            if (p < packs) v[i] = load_pack(row, p, once);
        }
        const int at = packs * PK::N + threadIdx.x;
        tail = at < vocab ? (float)row[at] : NEG_INF;
        constexpr int G = 3;
#pragma unroll
        for (int i = 0; i < Q; i += G) {
            u32x4 w[G];
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const int p = (R + i + g) * NT + threadIdx.x;
                if (i + g < Q && p < packs) w[g] = load_pack(row, p, once);
            }
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const int p = (R + i + g) * NT + threadIdx.x;
                if (i + g < Q && p < packs) lds[(i + g) * NT + threadIdx.x] = w[g];
            }
        }
    }
    __device__ RowStat stat(int vocab, ExpScale k) const {
        const int packs = vocab / PK::N;
        float m = tail;
#pragma unroll
        for (int i = 0; i < R; ++i)
            if (i * NT + (int)threadIdx.x < packs) {
#pragma unroll
                for (int e = 0; e < PK::N; ++e) m = fmaxf(m, PK::get(v[i], e));
            }
#pragma unroll
        for (int i = 0; i < Q; ++i)
            if ((R + i) * NT + (int)threadIdx.x < packs) {
                const u32x4 w = lds[i * NT + threadIdx.x];
#pragma unroll
                for (int e = 0; e < PK::N; ++e) m = fmaxf(m, PK::get(w, e));
            }
        const float r = m == NEG_INF ? 0.f : m;
        float s[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            s[i] = 0.f;
            if (i * NT + (int)threadIdx.x < packs) {
                float x[PK::N];
#pragma unroll
                for (int e = 0; e < PK::N; ++e) x[e] = exp2_scaled(PK::get(v[i], e) - r, k);
                s[i] = tree_sum(x);
            }
        }
        float total = tree_sum(s) + exp2_scaled(tail - r, k);
        for (int i = 0; i < Q; ++i)
            if ((R + i) * NT + (int)threadIdx.x < packs) {
                const u32x4 w = lds[i * NT + threadIdx.x];
                float x[PK::N];
#pragma unroll
                for (int e = 0; e < PK::N; ++e) x[e] = exp2_scaled(PK::get(w, e) - r, k);
                total += tree_sum(x);
            }
        return {m, total};
    }
    template <typename F>
    static __device__ void write(T *out, int p, const u32x4 &v, int64_t y, float c, F prob) {
        float f[PK::N];
#pragma unroll
        for (int e = 0; e < PK::N; ++e) f[e] = prob(PK::get(v, e));
        const int64_t at = y - (int64_t)p * PK::N;
        if (at >= 0 && at < PK::N) {
#pragma unroll
            for (int e = 0; e < PK::N; ++e) f[e] += e == at ? c : 0.f;
        }
        store_pack(out, p, PK::put(f));
    }
    template <typename F>
    __device__ void residual(T *out, int vocab, int64_t y, float c, F prob) const {
        const int packs = vocab / PK::N;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int p = i * NT + threadIdx.x;
            if (p < packs) write(out, p, v[i], y, c, prob);
        }
        for (int i = 0; i < Q; ++i) {
            const int p = (R + i) * NT + threadIdx.x;
            if (p < packs) write(out, p, lds[i * NT + threadIdx.x], y, c, prob);
        }
        const int at = packs * PK::N + threadIdx.x;
        if (at < vocab) out[at] = (T)(prob(tail) + (at == y ? c : 0.f));
    }
};

// Logits to gradient with one read: a row's coefficient needs the whole row's
// statistics, so the row stays on the CU until they are known.  REST: rows
// longer than (R + Q) NT packs; what does not fit is read again, from the
// Infinity Cache.
// Bound by memory: 4,096 x 131,072 bf16 419 us (5.1 TB/s; reading all of the
// row a second time instead of holding it 547), 1,021 x 50,257 f32 86 us.  The
// exponentials of a row's two passes take two thirds of its time, so another
// row has to be on the CU beside it.  Loading the next row into the registers
// that the gradient frees spilled them (882 us).
template <typename T, int NT, int R, int Q, bool REST>
__global__ __launch_bounds__(NT) void k_policy_loss(const T *logits, int64_t stride, int vocab, const void *target,
                                                    int target_bits, ExpScale k, double tau, bool once, dlr_policy p,
                                                    PolicyOut po, T *out, int64_t out_stride) {
    __shared__ BlockLds<NT> lds;
    __shared__ float coef;
    const int64_t t = blockIdx.x;
    const int64_t y = load_target(target, target_bits, t);
    const float w = p.weight ? p.weight[t] : 1.f;
    if (y < 0 || w == 0.f) {
        if (threadIdx.x == 0) policy_nothing(t, po);
        if (out) zero_row<T, NT>(out + t * out_stride, vocab);
        return;
    }
    constexpr int kHeld = (R + Q) * NT * Pack<T>::N;
    __shared__ u32x4 stash[Q ? Q * NT : 1];
    const int here = REST ? kHeld : vocab;
    const T *row = logits + t * stride;
    HeldRow<T, NT, R, Q> held;
    held.lds = stash;
    held.load(row, here, once);
    const float zy = y < vocab ? (float)row[y] : __builtin_nanf("");
    RowStat own = held.stat(here, k);
    if constexpr (REST) own = join(own, row_stat<T, NT, 4>(row + kHeld, vocab - kHeld, k, false), k);
    const BlockStat a = join_block<NT>(own, k, lds);
    if (threadIdx.x == 0) {
        const double lp = target_logprob(zy, a.m, log(a.s), tau);
        coef = (float)(policy_token(lp, p, t, w, po, true) / tau);
    }
    if (!out) return;
    __syncthreads();
    const float c = coef, neg = (float)(-c / a.s), m = a.m;
    auto prob = [=](float z) { return neg * exp2_scaled(z - m, k); };
    T *o = out + t * out_stride;
    held.residual(o, here, y, c, prob);
    if constexpr (REST) residual_row<T, NT, 4>(row + kHeld, o + kHeld, vocab - kHeld, y - kHeld, c, prob, once);
}

// ------------------------------------------------------------ preference loss

struct PairOut {
    float *loss, *chosen, *rejected, *grad;
};

// softplus(-u) = -log sigma(u), without overflow on either side
__device__ inline double softplus(double x) { return fmax(x, 0.0) + log1p(exp(-fabs(x))); }

typedef f32x4 f32x4_any __attribute__((aligned(4)));
typedef uint32_t u32_any __attribute__((aligned(1)));

// Whether offsets[from .. to] descend between two neighbours that this thread
// looks at.
template <int NT>
__device__ inline bool descend(const int64_t *offsets, int64_t from, int64_t to) {
    bool falls = false;
#pragma unroll 4
    for (int64_t i = from + threadIdx.x; i < to; i += NT) falls |= offsets[i + 1] < offsets[i];
    return falls;
}

// One pair a workgroup, half of it for each sequence: the sums of log ratios
// in 64 bits (they nearly cancel), the logistic loss of their difference, and
// the pair's one slope written over its tokens.  4 tokens a thread and step,
// loaded whether the mask counts them or not: a load that waits for its mask
// costs a second trip to memory.  Bound by latency, three dependent trips and
// the logarithms: 1,024 pairs of 1.5M tokens 13.5 us (19.6 a token at a time
// behind its mask), two pairs 4.  One workgroup a pair also where the
// sequences are very long (1 x 400,000 tokens 55 us): the logits of such a
// pair take a thousand times as long.
//
// Offsets that descend anywhere make sequences overlap, and which workgroup
// would write a shared token's gradient last is nobody's to say: then every pair
// and token is NaN.  `look`: each workgroup looks through the offsets for itself (1
// of the 13.5 us); else k_preference_order does, behind this launch.
template <int NT>
__global__ __launch_bounds__(NT) void k_preference_loss(dlr_preference p, PairOut o, bool look) {
    constexpr int H = NT / 2, W = NT / 64;
    __shared__ double sums[W];
    __shared__ int64_t counts[W];
    __shared__ int descends[W];
    const int64_t P = p.pairs, T = p.tokens;
    // tokens [b, e) of the gradient, by all workgroups
    auto fill = [&](int64_t b, int64_t e, float v) {
        for (int64_t i = b + (int64_t)blockIdx.x * NT + threadIdx.x; i < e; i += (int64_t)gridDim.x * NT) o.grad[i] = v;
    };
    if (!P) {
        if (o.grad) fill(0, T, 0.f);
        return;
    }
    const int64_t from = p.offsets[0], to = p.offsets[2 * P];
    const int64_t pair = blockIdx.x;
    const int q = threadIdx.x / H, at = threadIdx.x % H;
    int64_t first[2], last[2];
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        first[i] = p.offsets[pair + i * P];
        last[i] = p.offsets[pair + i * P + 1];
        // No range of the tokens: what lies within them gets the pair's NaN, so
        // that every token's gradient is written.
        if (first[i] < 0 || last[i] < first[i] || last[i] > T) bad = true;
        first[i] = first[i] < 0 ? 0 : first[i] > T ? T : first[i];
        last[i] = last[i] < first[i] ? first[i] : last[i] > T ? T : last[i];
    }
    const int64_t b = q ? first[1] : first[0], e = q ? last[1] : last[0];
    auto mask4 = [&](int64_t i) { return p.mask ? *reinterpret_cast<const u32_any *>(p.mask + i) : 0x01010101u; };
    const int64_t packs = (e - b) / 4, tail = b + packs * 4 + at;
    const bool wave_falls = look && __any(descend<NT>(p.offsets, 0, 2 * P));
    double sum = 0.0;
    int64_t count = 0;
#pragma unroll 4
    for (int64_t v = at; v < packs; v += H) {
        const int64_t i = b + 4 * v;
        const uint32_t m = mask4(i);
        const f32x4 l = *reinterpret_cast<const f32x4_any *>(p.logprob + i);
        f32x4 r = {};
        if (p.ref_logprob) r = *reinterpret_cast<const f32x4_any *>(p.ref_logprob + i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool on = (m >> (8 * j)) & 0xff;
            sum += on ? (double)l[j] - (double)r[j] : 0.0;
            count += on;
        }
    }
    const bool tail_on = tail < e && (!p.mask || p.mask[tail]);
    if (tail_on) {
        sum += (double)p.logprob[tail] - (p.ref_logprob ? (double)p.ref_logprob[tail] : 0.0);
        count += 1;
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        sum += __shfl_xor(sum, d);
        count += __shfl_xor(count, d);
    }
    if ((threadIdx.x & 63) == 0) {
        sums[threadIdx.x >> 6] = sum;
        counts[threadIdx.x >> 6] = count;
        descends[threadIdx.x >> 6] = wave_falls;
    }
    __syncthreads();
    bool falls = false;
#pragma unroll
    for (int w = 0; w < W; ++w) falls |= descends[w] != 0;
    double reward[2], scale[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        double s = 0.0;
        int64_t n = 0;
#pragma unroll
        for (int w = 0; w < W / 2; ++w) {
            s += sums[i * W / 2 + w];
            n += counts[i * W / 2 + w];
        }
        scale[i] = p.average ? p.beta / (double)(n > 1 ? n : 1) : p.beta;
        reward[i] = scale[i] * s;
    }
    const double eps = p.label_smoothing;
    double u = reward[0] - reward[1] - p.margin;
    if (bad || falls) u = reward[0] = reward[1] = __builtin_nan("");
    const double w = p.weight ? (double)p.weight[pair] : 1.0;
    if (threadIdx.x == 0) {
        // a side without weight adds nothing, also where it is infinite
        o.loss[pair] = (float)((eps < 1.0 ? (1.0 - eps) * softplus(-u) : 0.0) + (eps > 0.0 ? eps * softplus(u) : 0.0));
        o.chosen[pair] = (float)reward[0];
        o.rejected[pair] = (float)reward[1];
    }
    if (!o.grad) return;
    if (falls) {
        fill(0, T, __builtin_nanf(""));
        return;
    }
    // tokens of no sequence: before the first, behind the last
    fill(0, from < T ? from : T, 0.f);
    fill(to < 0 ? 0 : to < T ? to : T, T, 0.f);
    // d loss / d u = sigma(u) - (1 - eps)
    const double slope = w == 0.0 && !bad ? 0.0 : w * (eps / (1.0 + exp(-u)) - (1.0 - eps) / (1.0 + exp(u)));
    const float g = (float)(q ? -slope * scale[1] : slope * scale[0]);
#pragma unroll 4
    for (int64_t v = at; v < packs; v += H) {
        const uint32_t m = mask4(b + 4 * v);
        f32x4 d;
#pragma unroll
        for (int j = 0; j < 4; ++j) d[j] = (m >> (8 * j)) & 0xff ? g : 0.f;
        *reinterpret_cast<f32x4_any *>(o.grad + b + 4 * v) = d;
    }
    if (tail < e) o.grad[tail] = tail_on ? g : 0.f;
}

// Behind k_preference_loss: a workgroup that finds its part of the offsets to
// descend writes NaN over everything (all that do write the same).
__global__ __launch_bounds__(1024) void k_preference_order(dlr_preference p, PairOut o, int64_t part) {
    const int64_t from = blockIdx.x * part, to = from + part < 2 * p.pairs ? from + part : 2 * p.pairs;
    if (!__syncthreads_or(descend<1024>(p.offsets, from, to))) return;
    const float nan = __builtin_nanf("");
    for (int64_t i = threadIdx.x; i < p.pairs; i += 1024) o.loss[i] = o.chosen[i] = o.rejected[i] = nan;
    if (!o.grad) return;
    for (int64_t i = threadIdx.x; i < p.tokens; i += 1024) o.grad[i] = nan;
}

// -------------------------------------------------- head log-probabilities

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ inline f32x4 mfma(const u32x4 &a, const u32x4 &b, f32x4 c, __bf16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
}
__device__ inline f32x4 mfma(const u32x4 &a, const u32x4 &b, f32x4 c, _Float16) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
}

// 8 elements of row `r` from element k on; what lies outside [0, rows) x
// [0, dim) is 0 and not read.
__device__ inline u32x4 load8(const uint16_t *base, int64_t stride, int64_t r, int64_t rows, int k, int dim) {
    u32x4 v = {0u, 0u, 0u, 0u};
    if (r >= rows) return v;
    const uint16_t *s = base + r * stride + k;
    if (k + 8 <= dim) return *reinterpret_cast<const u32x4_any *>(s);
    union {
        uint16_t h[8];
        u32x4 v;
    } u;
    u.v = v;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (k + i < dim) u.h[i] = s[i];
    return u.v;
}

constexpr int kTileV = 128, kTileT = 128, kTileK = 64, kLdsRow = kTileK + 8;

// One tile of kTileV classes x kTileT tokens: logits = head . hidden^T by
// MFMA in 32 bits, never written; per token the tile's (maximum, sum) goes
// to part[tile][token], and the target's logit to zy[token].  Classes lie
// along the MFMA's rows, so a token's values sit in one lane column.
// For rows that the DMA cannot take.  Bound by its stages, fetched through
// registers between two barriers with nothing to multiply meanwhile: 333 x 1535
// x 50257 bf16 200 us, 68 at dim 1536 by DMA; 1 x 4095 x 131072 475, 180.
template <typename T>
__global__ __launch_bounds__(256) void k_head_tile(dlr_head h, float2 *part, float *zy) {
    __shared__ __attribute__((aligned(16))) uint16_t sw[kTileV * kLdsRow];
    __shared__ __attribute__((aligned(16))) uint16_t sx[kTileT * kLdsRow];
    __shared__ RowStat st[2][kTileT];
    const uint16_t *head = static_cast<const uint16_t *>(h.head), *hidden = static_cast<const uint16_t *>(h.hidden);
    const int64_t vtiles = (h.vocab + kTileV - 1) / kTileV, vt = blockIdx.x % vtiles;
    const int64_t v0 = vt * kTileV, t0 = blockIdx.x / vtiles * kTileT;
    const int dim = (int)h.dim;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wv = wave >> 1, wt = wave & 1;
    f32x4 acc[4][4] = {};
    for (int k0 = 0; k0 < dim; k0 += kTileK) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = tid + i * 256, r = c >> 3, kk = (c & 7) * 8;
            *reinterpret_cast<u32x4 *>(&sw[r * kLdsRow + kk]) = load8(head, h.head_stride, v0 + r, h.vocab, k0 + kk, dim);
            *reinterpret_cast<u32x4 *>(&sx[r * kLdsRow + kk]) =
                load8(hidden, h.hidden_stride, t0 + r, h.rows, k0 + kk, dim);
        }
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < kTileK; kk += 32) {
            u32x4 a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                a[i] = *reinterpret_cast<u32x4 *>(&sw[(wv * 64 + i * 16 + (lane & 15)) * kLdsRow + kk + (lane >> 4) * 8]);
                b[i] = *reinterpret_cast<u32x4 *>(&sx[(wt * 64 + i * 16 + (lane & 15)) * kLdsRow + kk + (lane >> 4) * 8]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = mfma(a[i], b[j], acc[i][j], T());
        }
    }
    const ExpScale k = exp_scale(h.temperature);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int64_t t = t0 + wt * 64 + j * 16 + (lane & 15);
        const int64_t y = t < h.rows ? load_target(h.target, h.target_bits, t) : -1;
        RowStat a{NEG_INF, 0.f};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int64_t v = v0 + wv * 64 + i * 16 + (lane >> 4) * 4 + e;
                if (v < h.vocab) {
                    const float z = acc[i][j][e];
                    a = join(a, RowStat{z, z == z ? 1.f : z}, k);
                    if (v == y) zy[t] = z;
                }
            }
        a = join(a, RowStat{__shfl_xor(a.m, 16), __shfl_xor(a.s, 16)}, k);
        a = join(a, RowStat{__shfl_xor(a.m, 32), __shfl_xor(a.s, 32)}, k);
        if (lane < 16) st[wv][wt * 64 + j * 16 + lane] = a;
    }
    __syncthreads();
    if (tid < kTileT && t0 + tid < h.rows) {
        const RowStat a = join(st[0][tid], st[1][tid], k);
        part[vt * h.rows + t0 + tid] = make_float2(a.m, a.s);
    }
}

// ---- aligned rows: both operands through LDS by DMA
//
// Classes v_first .. h.vocab - 1, `part` from the first of their tiles on.
// A workgroup of WV x WT waves takes TV = WV * 16 * MV classes x TT = WT * 16
// * MT tokens, 64 of the dimension (a stage) at a time, S stages in LDS.
// Rows of a stage are 128 bytes, classes first; the 16-byte chunk c of row r
// sits at slot c ^ (r & 7), so that a wave's fragment reads (16 rows, one
// chunk) meet no bank twice although the DMA writes linearly: the lane that
// fills slot s of row r fetches chunk s ^ (r & 7).
__device__ const u32x4 kZero16 = {0u, 0u, 0u, 0u};

// 64 lanes x 16 bytes, memory to LDS: lane i's at lds + 16 i.
__device__ inline void lds_dma16(const void *src, void *lds) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)src,
                                     (__attribute__((address_space(3))) void *)lds, 16, 0, 0);
}

// The rows that take part, in order, where they are picked first (row not
// null): row[0 .. *count).
struct HeadPick {
    const int32_t *row;
    const int64_t *count;
};

// Picks them, one workgroup; the others' results are written here.
__global__ __launch_bounds__(1024) void k_head_pick(const void *target, int target_bits, int64_t rows, int32_t *row,
                                                    int64_t *count, float *logprob, float *lse) {
    __shared__ int found[16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t total = 0;
    for (int64_t base = 0; base < rows; base += 1024) {
        const int64_t t = base + threadIdx.x;
        const bool on = t < rows && load_target(target, target_bits, t) >= 0;
        const uint64_t mask = __ballot(on);
        if (lane == 0) found[wave] = __popcll(mask);
        __syncthreads();
        int64_t at = total + __popcll(mask & ((UINT64_C(1) << lane) - 1));
        for (int w = 0; w < 16; ++w) {
            if (w < wave) at += found[w];
            total += found[w];
        }
        if (on) {
            row[at] = (int32_t)t;
        } else if (t < rows) {
            logprob[t] = 0.f;
            lse[t] = 0.f;
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) *count = total;
}

// One scheduling group: N instructions of a kind (8: MFMA, 32: memory reads,
// 256: LDS reads), in program order with the groups around it.
#define SCHED_MFMA(n) __builtin_amdgcn_sched_group_barrier(8, n, 0)
#define SCHED_DMA(n) __builtin_amdgcn_sched_group_barrier(32, n, 0)
#define SCHED_LDS(n) __builtin_amdgcn_sched_group_barrier(256, n, 0)

// Measured (bf16): 256 x 256 tiles, 8 waves of 128 x 64, 4096 x 4096 x 65536
// 1.57 to 1.60 ms once the clock has settled (the first ten launches after a pause
// up to 2.1), 1,380 TFLOP/s, softmax included, where the library's product alone
// takes 1.46 to 1.54; the matrix cores are busy 72 to 75% of the cycles, at the 1.8
// GHz that they leave of the clock.  A tile's ends (filling the stages, the softmax,
// nothing else on the CU) are 9 to 10 us beside 1.4 a stage: 4096 x 512 x 131072 676
// us, 813 TFLOP/s.  4 waves of 128 x 128 read a third less from LDS, but
// the compiler then moves accumulators between register files (994 TFLOP/s);
// 32 x 32 products meet LDS banks twice in this layout (1,109); a workgroup
// that goes on to its next tile and fetches it under this one's end spills
// (1,105).  The groups' order below was the best of eleven (1,310 .. 1,380).
// Few rows: bound by the head's bytes, 1 x 4096 x 131072 178 us (6.0 TB/s).
template <typename T, int WV, int WT, int MV, int MT, int S>
__global__ __launch_bounds__(WV *WT * 64) void k_head_dma(dlr_head h, int64_t v_first, HeadPick pick, float2 *part,
                                                          float *zy) {
    constexpr int NW = WV * WT, TV = WV * MV * 16, TT = WT * MT * 16, kRow = 128;
    constexpr int kLoads = (TV + TT) / 8, L = (kLoads + NW - 1) / NW;  // DMA loads of 8 rows: all, a wave's
    static_assert(TV % 8 == 0 && TT % 8 == 0 && S >= 2 && L * (S - 1) < 64, "whole loads, a wait that can be written");
    __shared__ __attribute__((aligned(256))) char sm[S][(TV + TT) * kRow];
    RowStat *stat = reinterpret_cast<RowStat *>(sm[0]);  // [WV][TT], behind the products
    static_assert(sizeof(RowStat) * WV * TT <= sizeof sm, "they fit");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wv = wave / WT, wt = wave % WT;
    const int64_t used = pick.row ? *pick.count : h.rows;
    const int64_t vtiles = (h.vocab - v_first + TV - 1) / TV, ttiles = (used + TT - 1) / TT, tiles = vtiles * ttiles;
    if (blockIdx.x >= tiles) return;  // the launch counts all rows
    // XCD x takes a contiguous piece of the tile order, in which up to 8 token
    // tiles of one class tile follow each other: an XCD's 32 running workgroups
    // share 8 token and 4 class tiles in its L2.
    const int64_t q8 = tiles / 8, rem = tiles % 8, x8 = blockIdx.x % 8;
    const int64_t tile = x8 * q8 + (x8 < rem ? x8 : rem) + blockIdx.x / 8;
    const int64_t group = vtiles * 8, g = tile / group;  // tiles of 8 token tiles' group
    const int in_g = ttiles - g * 8 < 8 ? (int)(ttiles - g * 8) : 8;
    const int64_t rest = tile - g * group;
    // the same in every lane, which the divisions do not show: scalar registers
    const int64_t vt = __builtin_amdgcn_readfirstlane((int)(rest / in_g)), v0 = v_first + vt * TV;
    const int64_t t0 = (int64_t)__builtin_amdgcn_readfirstlane((int)(g * 8 + rest % in_g)) * TT;
    const int dim = (int)h.dim, full = dim / 64, steps = (dim + 63) / 64;
    const bool picked = pick.row && used < h.rows;  // all of them: in their places, without a trip to the list
    auto token = [&](int64_t t) { return picked ? (int64_t)pick.row[t] : t; };

    // This lane's places in the wave's DMA loads.  Rows outside repeat the last
    // one; a wave without an L-th load repeats the last load (every wave then
    // has L of them in flight per stage).
    const char *src[L];  // of the stage to be filled next
    // The whole stages in a circle, then the short one: class tiles begin a stage
    // apart, or, where rows lie a power of two apart, all workgroups would read
    // from few memory channels at a time (128 x 4096 x 65536 149 us from the same
    // stage, 115; 256 x 4096 x 65536 174, 145).  Not up to 16 tokens, whose two
    // workgroups a CU drift apart by themselves (1 x 4096 x 131072 178, 183).
    constexpr bool kCircle = TT > 16;
    const int start = kCircle && full > 0 ? (int)(vt % full) : 0;
    int at_stage = start, left = full;
    const int chunk = (lane & 7) ^ (lane >> 3);
    auto load_no = [&](int q) {
        const int n = wave * L + q;
        return n < kLoads ? n : kLoads - 1;
    };
#pragma unroll
    for (int q = 0; q < L; ++q) {
        const int n = load_no(q);
        const bool x = n >= TV / 8;
        const int r = (x ? n - TV / 8 : n) * 8 + (lane >> 3);
        const int64_t first = x ? t0 : v0, last = (x ? used : h.vocab) - 1;
        int64_t at = first + r < last ? first + r : last;
        if (x) at = token(at);
        src[q] = static_cast<const char *>(x ? h.hidden : h.head) + at * (x ? h.hidden_stride : h.head_stride) * 2 +
                 chunk * 16 + start * 128;
    }
    auto step_on = [&]() {  // bytes to the next stage
        if constexpr (!kCircle) return (int64_t)128;
        int next = at_stage + 1 < full ? at_stage + 1 : 0;
        if (--left == 0) next = full;
        const int64_t by = (int64_t)(next - at_stage) * 128;
        at_stage = next;
        return by;
    };
    auto fill = [&](int buf) {
        const int64_t by = step_on();
#pragma unroll
        for (int q = 0; q < L; ++q) {
            lds_dma16(src[q], sm[buf] + load_no(q) * 1024);
            src[q] += by;
        }
    };
    auto fill_last = [&](int step, int buf) {  // a stage that may be short (dim is a multiple of 8): zeros behind it
        const bool in = step < full || step * 64 + chunk * 8 < dim;
        const int64_t by = step_on();
#pragma unroll
        for (int q = 0; q < L; ++q) {
            lds_dma16(in ? src[q] : (const char *)&kZero16, sm[buf] + load_no(q) * 1024);
            src[q] += by;
        }
    };
    struct Frag {
        u32x4 a[MV], b[MT];
    };
    const int at_v = (wv * MV * 16 + (lane & 15)) * kRow, at_t = TV * kRow + (wt * MT * 16 + (lane & 15)) * kRow;
    auto read = [&](Frag &f, int buf, int half) {
        const int slot = ((half * 4 + (lane >> 4)) ^ (lane & 7)) * 16;
#pragma unroll
        for (int j = 0; j < MT; ++j) f.b[j] = *reinterpret_cast<const u32x4 *>(sm[buf] + at_t + j * 16 * kRow + slot);
#pragma unroll
        for (int i = 0; i < MV; ++i) f.a[i] = *reinterpret_cast<const u32x4 *>(sm[buf] + at_v + i * 16 * kRow + slot);
    };
    f32x4 acc[MV][MT] = {};
    auto multiply = [&](const Frag &f) {
#pragma unroll
        for (int i = 0; i < MV; ++i)
#pragma unroll
            for (int j = 0; j < MT; ++j) acc[i][j] = mfma(f.a[i], f.b[j], acc[i][j], T());
    };
    // The first half's fragments of a stage are read while the second half
    // of the stage before is multiplied, the second half's while the first
    // is: the matrix cores wait for LDS nowhere.  One barrier a stage, in its
    // middle: then the next stage has landed (each wave waits for its own
    // part first; `later` loads of the stages behind it stay in flight) and
    // nobody reads this one any more.
#define MEET(later)                                                                                \
    do {                                                                                           \
        __builtin_amdgcn_sched_barrier(0);                                                         \
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(later) : "memory");                    \
        __builtin_amdgcn_s_barrier();                                                              \
        asm volatile("" ::: "memory");                                                             \
    } while (0)
    Frag f0, f1;
    if (full >= S) {
#pragma unroll
        for (int p = 0; p < S; ++p) fill(p);
    } else {
#pragma unroll
        for (int p = 0; p < S; ++p)
            if (p < steps) fill_last(p, p);
    }
    if (steps >= S)
        MEET(L *(S - 1));  // the first stage has landed
    else
        MEET(0);
    read(f0, 0, 0);
    int step = 0, buf = 0;
    for (; step + S < full; ++step) {
        const int next = buf + 1 < S ? buf + 1 : 0;
        read(f1, buf, 1);
        multiply(f0);
#pragma unroll
        for (int i = 0; i < MV + MT; ++i) {
            SCHED_LDS(1);
            SCHED_MFMA(2);
        }
        MEET(L *(S - 2));
        fill(buf);
        read(f0, next, 0);
        multiply(f1);
#pragma unroll
        for (int i = 0; i < L; ++i) {
            SCHED_DMA(1);
            SCHED_MFMA(2);
        }
#pragma unroll
        for (int i = 0; i < MV + MT; ++i) {
            SCHED_LDS(1);
            SCHED_MFMA(1);
        }
        __builtin_amdgcn_sched_barrier(0);
        buf = next;
    }
    for (; step < steps; ++step) {
        const int next = buf + 1 < S ? buf + 1 : 0;
        read(f1, buf, 1);
        multiply(f0);
        MEET(0);
        if (step + S < steps) fill_last(step + S, buf);
        if (step + 1 < steps) read(f0, next, 0);
        multiply(f1);
        buf = next;
    }
    __syncthreads();  // sm is free
    // per token (a lane column) over this wave's classes, then over the waves
    const ExpScale k = exp_scale(h.temperature);
    const int classes = h.vocab - v0 < TV ? (int)(h.vocab - v0) : TV, base = wv * MV * 16 + (lane >> 4) * 4;
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        const int64_t t = t0 + wt * MT * 16 + j * 16 + (lane & 15);
        const int64_t row = t < used ? token(t) : -1;
        const int64_t y = (row >= 0 ? load_target(h.target, h.target_bits, row) : -1) - v0;
        const int target = y >= 0 && y < TV ? (int)y : -1;  // in the tile
        float m = NEG_INF;
#pragma unroll
        for (int i = 0; i < MV; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (classes < TV && base + i * 16 + e >= classes) acc[i][j][e] = NEG_INF;
                if (base + i * 16 + e == target) zy[row] = acc[i][j][e];
                m = fmaxf(m, acc[i][j][e]);
            }
        m = fmaxf(m, __shfl_xor(m, 16));
        m = fmaxf(m, __shfl_xor(m, 32));
        const float r = m == NEG_INF ? 0.f : m;
        float s[MV];
#pragma unroll
        for (int i = 0; i < MV; ++i) {
            float e4[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) e4[e] = exp2_scaled(acc[i][j][e] - r, k);
            s[i] = tree_sum(e4);
        }
        float sum = tree_sum(s);
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        if (lane < 16) stat[wv * TT + wt * MT * 16 + j * 16 + lane] = {m, sum};
    }
    __syncthreads();
    for (int i = tid; i < TT; i += NW * 64)
        if (t0 + i < used) {
            RowStat a = stat[i];
#pragma unroll
            for (int w = 1; w < WV; ++w) a = join(a, stat[w * TT + i], k);
            part[vt * h.rows + t0 + i] = make_float2(a.m, a.s);
        }
}

// ---- small tiles: the dimension split over a workgroup's four waves
//
// A tile of TV = MV * 16 classes x TT = MT * 16 tokens keeps one wave too little
// busy to hide a stage's barrier and LDS trips, and few classes leave most CUs
// without a tile.  So the four waves take every fourth stage each, from LDS
// rings of their own: no barrier until their products are added, in a fixed
// order.
template <typename T, int MV, int MT, int S>
__global__ __launch_bounds__(256) void k_head_waves(dlr_head h, int64_t v_first, HeadPick pick, float2 *part,
                                                    float *zy) {
    constexpr int TV = MV * 16, TT = MT * 16, kRow = 128, L = (TV + TT) / 8, B = MV * MT / 4;
    static_assert(MV == 4 && (MT == 1 || MT == 4) && S >= 2 && L * (S - 1) < 64, "a wave's share of the blocks");
    __shared__ __attribute__((aligned(256))) char sm[4][S][(TV + TT) * kRow];
    __shared__ RowStat stat[4][TT];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t used = pick.row ? *pick.count : h.rows;
    const int64_t vtiles = (h.vocab - v_first + TV - 1) / TV, ttiles = (used + TT - 1) / TT;
    if (blockIdx.x >= vtiles * ttiles) return;  // the launch counts all rows
    const int64_t vt = __builtin_amdgcn_readfirstlane((int)(blockIdx.x / ttiles)), v0 = v_first + vt * TV;
    const int64_t t0 = (int64_t)__builtin_amdgcn_readfirstlane((int)(blockIdx.x % ttiles)) * TT;
    const int dim = (int)h.dim, steps = (dim + 63) / 64;
    auto token = [&](int64_t t) { return pick.row ? (int64_t)pick.row[t] : t; };

    const char *src[L];  // this lane's places in the wave's DMA loads, of the wave's next stage
    const int chunk = (lane & 7) ^ (lane >> 3);
#pragma unroll
    for (int q = 0; q < L; ++q) {
        const bool x = q >= TV / 8;
        const int r = (x ? q - TV / 8 : q) * 8 + (lane >> 3);
        const int64_t first = x ? t0 : v0, last = (x ? used : h.vocab) - 1;
        int64_t at = first + r < last ? first + r : last;
        if (x) at = token(at);
        src[q] = static_cast<const char *>(x ? h.hidden : h.head) + at * (x ? h.hidden_stride : h.head_stride) * 2 +
                 chunk * 16 + wave * 128;
    }
    auto fill = [&](int step, int buf) {  // dim is a multiple of 8: zeros behind it
        const bool in = step * 64 + chunk * 8 < dim;
#pragma unroll
        for (int q = 0; q < L; ++q) {
            lds_dma16(in ? src[q] : (const char *)&kZero16, sm[wave][buf] + q * 1024);
            src[q] += 4 * 128;
        }
    };
    const int at = (lane & 15) * kRow;
    f32x4 acc[MV][MT] = {};
    int buf = 0;
#pragma unroll
    for (int p = 0; p < S; ++p)
        if (wave + 4 * p < steps) fill(wave + 4 * p, p);
    for (int step = wave; step < steps; step += 4) {
        // this stage has landed; the ring's others stay in flight
        if (step + 4 * (S - 1) < steps)
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(L *(S - 1)) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const char *sv = sm[wave][buf] + at, *sx = sv + TV * kRow;
        u32x4 a[2][MV], b[2][MT];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int slot = ((half * 4 + (lane >> 4)) ^ (lane & 7)) * 16;
#pragma unroll
            for (int j = 0; j < MT; ++j) b[half][j] = *reinterpret_cast<const u32x4 *>(sx + j * 16 * kRow + slot);
#pragma unroll
            for (int i = 0; i < MV; ++i) a[half][i] = *reinterpret_cast<const u32x4 *>(sv + i * 16 * kRow + slot);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read: the slot is free
        if (step + 4 * S < steps) fill(step + 4 * S, buf);
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int i = 0; i < MV; ++i)
#pragma unroll
                for (int j = 0; j < MT; ++j) acc[i][j] = mfma(a[half][i], b[half][j], acc[i][j], T());
        buf = buf + 1 < S ? buf + 1 : 0;
    }
    // the waves' products added; wave w then has blocks w B .. w B + B - 1 of
    // the tile's MV x MT, counted along the classes
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    f32x4 *sum = reinterpret_cast<f32x4 *>(sm);  // [4][MV * MT][64]
    static_assert(sizeof(f32x4) * 4 * MV * MT * 64 <= sizeof sm, "they fit");
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
        for (int i = 0; i < MV; ++i) sum[(wave * MV * MT + j * MV + i) * 64 + lane] = acc[i][j];
    __syncthreads();
    const ExpScale k = exp_scale(h.temperature);
    const int classes = h.vocab - v0 < TV ? (int)(h.vocab - v0) : TV;
    const int first = wave * B, j = first / MV;
    const int64_t t = t0 + j * 16 + (lane & 15);
    const int64_t row = t < used ? token(t) : -1;
    const int64_t y = (row >= 0 ? load_target(h.target, h.target_bits, row) : -1) - v0;
    const int target = y >= 0 && y < TV ? (int)y : -1;  // in the tile
    f32x4 z[B];
    float m = NEG_INF;
#pragma unroll
    for (int n = 0; n < B; ++n) {
        z[n] = sum[(first + n) * 64 + lane];
#pragma unroll
        for (int w = 1; w < 4; ++w) z[n] += sum[(w * MV * MT + first + n) * 64 + lane];
        const int base = ((first + n) % MV) * 16 + (lane >> 4) * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (base + e >= classes) z[n][e] = NEG_INF;
            if (base + e == target) zy[row] = z[n][e];
            m = fmaxf(m, z[n][e]);
        }
    }
    m = fmaxf(m, __shfl_xor(m, 16));
    m = fmaxf(m, __shfl_xor(m, 32));
    const float r = m == NEG_INF ? 0.f : m;
    float s[B];
#pragma unroll
    for (int n = 0; n < B; ++n) {
        float e4[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) e4[e] = exp2_scaled(z[n][e] - r, k);
        s[n] = tree_sum(e4);
    }
    float total = tree_sum(s);
    total += __shfl_xor(total, 16);
    total += __shfl_xor(total, 32);
    constexpr int W = B >= MV ? 1 : 4;  // waves that share a token
    if (lane < 16) stat[W == 1 ? 0 : wave][j * 16 + lane] = {m, total};
    __syncthreads();
    const int i = threadIdx.x;
    if (i < TT && t0 + i < used) {
        RowStat q = stat[0][i];
#pragma unroll
        for (int w = 1; w < W; ++w) q = join(q, stat[w][i], k);
        part[vt * h.rows + t0 + i] = make_float2(q.m, q.s);
    }
}

// The tiles' statistics, joined: RT tokens a workgroup (their statistics lie
// side by side), NT / RT threads each.  The maximum first, then the scaled
// sums in 64 bits (as join_block); a thread keeps its first 16 tiles.  Bound by
// its trips to memory, 5 to 7 us up to 1,000 tokens.
template <int RT, int NT>
__global__ __launch_bounds__(NT) void k_head_join(dlr_head h, HeadPick pick, int64_t tiles, const float2 *part,
                                                  const float *zy, float *logprob, float *lse) {
    constexpr int G = NT / RT, K = 16, W = NT / 64;
    __shared__ float lm[W][RT];
    __shared__ double ls[W][RT];
    const int tok = threadIdx.x % RT, first = threadIdx.x / RT, wave = threadIdx.x >> 6;
    const int64_t t = (int64_t)blockIdx.x * RT + tok, used = pick.row ? *pick.count : h.rows;
    const bool in = t < used;
    const int64_t row = !in ? 0 : pick.row ? (int64_t)pick.row[t] : t;
    const int64_t y = in ? load_target(h.target, h.target_bits, row) : -1;
    const ExpScale k = exp_scale(h.temperature);
    const float2 *p = part + (in ? t : 0);
    if (!in) tiles = 0;
    float2 q[K];
#pragma unroll
    for (int i = 0; i < K; ++i) {
        const int64_t n = first + i * G;
        q[i] = n < tiles ? p[n * h.rows] : make_float2(NEG_INF, 0.f);
    }
    const float z = y >= 0 && y < h.vocab ? zy[row] : __builtin_nanf("");
    float m = NEG_INF;
#pragma unroll
    for (int i = 0; i < K; ++i) m = fmaxf(m, q[i].x);
#pragma unroll 4
    for (int64_t n = first + K * G; n < tiles; n += G) m = fmaxf(m, p[n * h.rows].x);
#pragma unroll
    for (int o = RT; o < 64; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
    if ((threadIdx.x & 63) < RT) lm[wave][tok] = m;
    __syncthreads();
    m = lm[0][tok];
#pragma unroll
    for (int w = 1; w < W; ++w) m = fmaxf(m, lm[w][tok]);
    const float r = m == NEG_INF ? 0.f : m;
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < K; ++i) s += (double)q[i].y * (double)exp2_scaled(q[i].x - r, k);
#pragma unroll 4
    for (int64_t n = first + K * G; n < tiles; n += G) {
        const float2 v = p[n * h.rows];
        s += (double)v.y * (double)exp2_scaled(v.x - r, k);
    }
#pragma unroll
    for (int o = RT; o < 64; o <<= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) < RT) ls[wave][tok] = s;
    __syncthreads();
    if (first || !in) return;
    s = ls[0][tok];
#pragma unroll
    for (int w = 1; w < W; ++w) s += ls[w][tok];
    const double tau = h.temperature, ln = log(s);
    lse[row] = y < 0 ? 0.f : (float)(m / tau + ln);
    logprob[row] = y < 0 ? 0.f : (float)target_logprob(z, m, ln, tau);
}

}  // namespace

// A launch's own error: the runtime's last error may be an earlier call's.
template <typename... P, typename... A>
static hipError_t launch(void (*kernel)(P...), int64_t blocks, int threads, hipStream_t st, const A &...a) {
    static_assert(sizeof...(P) == sizeof...(A), "every argument");
    std::tuple<P...> values(static_cast<P>(a)...);
    return std::apply(
        [&](auto &...v) {
            void *args[] = {const_cast<void *>(static_cast<const void *>(&v))...};
            const hipError_t e = hipLaunchKernel(reinterpret_cast<const void *>(kernel), dim3((unsigned)blocks),
                                                 dim3((unsigned)threads), args, 0, st);
            if (e != hipSuccess) (void)hipGetLastError();  // reported here, not by the caller's next call
            return e;
        },
        values);
}

template <typename F>
static hipError_t by_dtype(int dtype, F f) {
    switch (dtype) {
        case DLR_DTYPE_F32: return f(float());
        case DLR_DTYPE_BF16: return f(__bf16());
        default: return f(_Float16());
    }
}

constexpr int64_t kCus = 256;

// A launch has fewer than 2^32 threads: more rows than this go by several
// launches of about as many (never by a few: row_parts' workspace is the whole
// call's).
constexpr int64_t kLaunchRows = INT64_C(1) << 21;

// f(rows at .. of `x`, at), slice by slice; at least one row.
template <typename X, typename F>
static hipError_t by_rows(const X &x, int64_t most, F f) {
    const int64_t slices = (x.rows + most - 1) / most, each = (x.rows + slices - 1) / slices;
    hipError_t e = hipSuccess;
    for (int64_t at = 0; at < x.rows && e == hipSuccess; at += each) {
        X part = x;
        part.target = static_cast<const char *>(x.target) + at * (x.target_bits / 8);
        part.rows = x.rows - at < each ? x.rows - at : each;
        e = f(part, at);
    }
    return e;
}

// The same with the logits' type as f's first argument.
template <typename F>
static hipError_t by_logits(const dlr_logits &whole, F f) {
    return by_rows(whole, kLaunchRows, [&](dlr_logits &x, int64_t at) {
        return by_dtype(x.dtype, [&](auto e) {
            x.data = static_cast<const decltype(e) *>(x.data) + at * x.row_stride;
            return f(e, x, at);
        });
    });
}

// Logits of more bytes than the 256 MB Infinity Cache cannot be there when the
// call begins, nor will a second read find them: they are read past it.
constexpr int64_t kOnceBytes = INT64_C(1) << 28;
static bool read_once(const dlr_logits &x) {
    return x.rows * x.vocab * (x.dtype == DLR_DTYPE_F32 ? 4 : 2) > kOnceBytes;
}

// The chunks of a row: 1, or for few long rows (see RowParts) about two
// workgroups a CU in all, of 2,048 packs and more.
static RowParts row_parts(int64_t rows, int64_t vocab, int pack, void *workspace) {
    const int64_t packs = vocab / pack;
    int64_t chunks = 1, span = packs;
    if (rows >= 1 && rows <= 128 && packs >= 8192) {
        chunks = 2 * kCus / rows < packs / 2048 ? 2 * kCus / rows : packs / 2048;
        if (chunks > 63) chunks = 63;  // one more where a tail is left over
        span = (packs + chunks - 1) / chunks;
        chunks = (vocab + span * pack - 1) / (span * pack);
    }
    RowPart *part = static_cast<RowPart *>(workspace);
    return {part, reinterpret_cast<float *>(part + rows * chunks), (int)chunks, (int)(span * pack)};
}

int64_t logits_workspace(int64_t rows, int64_t vocab, int32_t dtype) {
    const RowParts w = row_parts(rows, vocab, dtype == DLR_DTYPE_F32 ? 4 : 8, nullptr);
    return w.chunks == 1 ? 0 : rows * w.chunks * (int64_t)sizeof(RowPart) + rows * (int64_t)sizeof(float);
}

template <typename T>
static hipError_t launch_parts(hipStream_t st, const dlr_logits &x, const float *weight, const RowParts &w) {
    return launch(k_row_part<T, 512>, x.rows * w.chunks, 512, st, static_cast<const T *>(x.data), x.row_stride,
                  (int)x.vocab, x.target, x.target_bits, weight, exp_scale(x.temperature), w);
}

// A row's threads.  Short rows: as few as keep a few packs each, for the
// rows' ends (joining, the logarithm) are what costs (8,000 x 1,000 bf16: 7.8
// us with 64 threads, 20 with 512).  Long rows: enough loads in flight
// (1 x 32,000: 4.9 us with 512, 12.8 with 64; 4,096 x 131,072: 189 against
// 195).
template <typename T, int NT>
static hipError_t launch_logprob(hipStream_t st, const dlr_logits &x, float *logprob, float *lse) {
    return launch(k_token_logprob<T, NT>, x.rows, NT, st, static_cast<const T *>(x.data), x.row_stride, (int)x.vocab,
                  x.target, x.target_bits, exp_scale(x.temperature), x.temperature, read_once(x), logprob, lse);
}

hipError_t launch_token_logprob(hipStream_t st, const dlr_logits &all, void *workspace, float *logprobs, float *lses) {
    return by_logits(all, [&](auto e, const dlr_logits &x, int64_t at) {
        using T = decltype(e);
        float *logprob = logprobs + at, *lse = lses + at;
        const RowParts w = row_parts(x.rows, x.vocab, Pack<T>::N, workspace);
        if (w.chunks > 1) {
            const hipError_t r = launch_parts<T>(st, x, nullptr, w);
            return r != hipSuccess ? r : launch(k_token_finish, x.rows, 64, st, x.target, x.target_bits, (int)x.vocab,
                                                exp_scale(x.temperature), x.temperature, w, logprob, lse);
        }
        const int64_t packs = x.vocab / Pack<T>::N;
        if (packs <= 256) return launch_logprob<T, 64>(st, x, logprob, lse);
        if (packs <= 1024) return launch_logprob<T, 128>(st, x, logprob, lse);
        return launch_logprob<T, 512>(st, x, logprob, lse);
    });
}

template <typename T, int NT>
static hipError_t launch_grad(hipStream_t st, const dlr_logits &x, const float *lse, const float *grad, void *out,
                              int64_t out_stride, int chunks = 1, int span = 1 << 30) {
    return launch(k_token_logprob_grad<T, NT>, x.rows * chunks, NT, st, static_cast<const T *>(x.data), x.row_stride,
                  (int)x.vocab, x.target, x.target_bits, exp_scale(x.temperature), x.temperature, read_once(x), lse,
                  grad, static_cast<T *>(out), out_stride, chunks, span);
}

// As above; rows of 2,048 to 16,384 packs gain from fewer of them in flight
// at once (8,192 x 32,000 bf16 191 -> 174 us with 1,024 threads a row), longer
// ones lose (4,096 x 131,072 f32 810 -> 864).
hipError_t launch_token_logprob_grad(hipStream_t st, const dlr_logits &all, const float *lses, const float *grads,
                                     void *outs, int64_t out_stride) {
    return by_logits(all, [&](auto e, const dlr_logits &x, int64_t at) {
        using T = decltype(e);
        const float *lse = lses + at, *grad = grads + at;
        T *out = static_cast<T *>(outs) + at * out_stride;
        const int64_t packs = x.vocab / Pack<T>::N;
        // Few long rows by chunks of 1,024 packs and more, four workgroups a CU
        // in all (1 x 131,072 bf16: 2.9 us, 10.6 by one workgroup); not over
        // the logits, which a chunk may have to read again as a whole.
        if (x.rows <= kCus && packs >= 2048 && out != x.data) {
            const int64_t most = 4 * kCus / x.rows < packs / 1024 ? 4 * kCus / x.rows : packs / 1024;
            const int64_t span = (packs + most - 1) / most * Pack<T>::N, chunks = (x.vocab + span - 1) / span;
            return launch_grad<T, 512>(st, x, lse, grad, out, out_stride, (int)chunks, (int)span);
        }
        if (packs <= 256) return launch_grad<T, 64>(st, x, lse, grad, out, out_stride);
        if (packs <= 1024) return launch_grad<T, 128>(st, x, lse, grad, out, out_stride);
        if (packs <= 2048 || packs > 16384) return launch_grad<T, 512>(st, x, lse, grad, out, out_stride);
        return launch_grad<T, 1024>(st, x, lse, grad, out, out_stride);
    });
}

template <typename T, int NT, int R, int Q = 0, bool REST = false>
static hipError_t launch_policy(hipStream_t st, const dlr_logits &x, const dlr_policy &p, const PolicyOut &po,
                                void *out, int64_t out_stride) {
    return launch(k_policy_loss<T, NT, R, Q, REST>, x.rows, NT, st, static_cast<const T *>(x.data), x.row_stride,
                  (int)x.vocab, x.target, x.target_bits, exp_scale(x.temperature), x.temperature, read_once(x), p, po,
                  static_cast<T *>(out), out_stride);
}

// The smallest workgroup that holds a row: the more of them on a CU, the more of
// a row's two passes overlap with other rows' memory (bf16, us, the row held by
// 512 / 1,024 threads: 4,096 x 65,536 204 / 254, 8,192 x 32,000 186 / 189;
// 8,000 x 1,000 by 128 / 256: 14 / 18).  Longer rows: two workgroups a CU that
// hold 136 KB each, in registers and LDS, and read what is left again beat one
// that holds all in 16 bits, whose passes compute twice as much per byte (4,096
// x 131,072 415 / 463, 1,024 x 200,000 177 / 192), not in 32 (921 / 900).
hipError_t launch_policy_loss(hipStream_t st, const dlr_logits &all, const dlr_policy &policy, void *workspace,
                              float *loss, float *logprob, float *kl, uint8_t *clipped, void *outs,
                              int64_t out_stride) {
    return by_logits(all, [&](auto e, const dlr_logits &x, int64_t at) {
        using T = decltype(e);
        dlr_policy p = policy;
        p.old_logprob += at;
        p.advantage += at;
        if (p.ref_logprob) p.ref_logprob += at;
        if (p.weight) p.weight += at;
        const PolicyOut po{loss + at, logprob + at, kl + at, clipped + at};
        T *out = outs ? static_cast<T *>(outs) + at * out_stride : nullptr;
        const RowParts w = row_parts(x.rows, x.vocab, Pack<T>::N, workspace);
        if (w.chunks > 1) {
            const hipError_t r = launch_parts<T>(st, x, p.weight, w);
            return r != hipSuccess ? r : launch(k_policy_finish<T, 512>, x.rows * w.chunks, 512, st,
                                                static_cast<const T *>(x.data), x.row_stride, (int)x.vocab, x.target,
                                                x.target_bits, exp_scale(x.temperature), x.temperature, p, po,
                                                static_cast<T *>(out), out_stride, w);
        }
        const int64_t packs = x.vocab / Pack<T>::N;
        if (packs <= 512) return launch_policy<T, 128, 4>(st, x, p, po, out, out_stride);
        if (packs <= 1024) return launch_policy<T, 256, 4>(st, x, p, po, out, out_stride);
        if (packs <= 4096) return launch_policy<T, 512, 8>(st, x, p, po, out, out_stride);
        if constexpr (sizeof(T) == 2) {
            if (packs <= 17 * 512) return launch_policy<T, 512, 16, 1>(st, x, p, po, out, out_stride);
            return launch_policy<T, 512, 8, 9, true>(st, x, p, po, out, out_stride);
        } else {
            if (packs <= 8192) return launch_policy<T, 512, 16>(st, x, p, po, out, out_stride);
            if (packs <= 16384) return launch_policy<T, 1024, 16>(st, x, p, po, out, out_stride);
            return launch_policy<T, 1024, 16, 0, true>(st, x, p, po, out, out_stride);
        }
    });
}

// Up to here a workgroup looks through all offsets itself, beyond a second launch
// does (pairs of 146 tokens, us a call: 2,048 pairs 11.9 against 13.7, 4,096 22.6
// against 15.3; 11.9 and 12.7 without looking).
constexpr int64_t kLookPairs = 2048;

hipError_t launch_preference_loss(hipStream_t st, const dlr_preference &p, float *loss, float *chosen,
                                  float *rejected, float *grad) {
    const int64_t blocks = p.pairs ? p.pairs : 1;
    const PairOut o{loss, chosen, rejected, grad};
    const bool look = p.pairs <= kLookPairs;
    // A large workgroup for long sequences, where there are CUs for it (us by
    // 256 / 512 / 1,024 threads: 16 pairs of 1,000 tokens 5.7 / 4.7 / 5.3, 1,024
    // of 1,465 11 / 12 / 19, 64 of 23,400 - / 30 / 23).
    const int64_t each = p.tokens / blocks;
    hipError_t e;
    if (each > 8192)
        e = launch(k_preference_loss<1024>, blocks, 1024, st, p, o, look);
    else if (each > 512 && blocks <= 2 * kCus)
        e = launch(k_preference_loss<512>, blocks, 512, st, p, o, look);
    else
        e = launch(k_preference_loss<256>, blocks, 256, st, p, o, look);
    if (e != hipSuccess || look) return e;
    const int64_t parts = (2 * p.pairs + 8191) / 8192 < 64 ? (2 * p.pairs + 8191) / 8192 : 64;
    return launch(k_preference_order, parts, 1024, st, p, o, (2 * p.pairs + parts - 1) / parts);
}

// Whether the rows can go through the DMA kernels: 16-byte chunks of rows that
// start at 16 bytes.
static bool head_by_dma(const dlr_head &h) {
    return (reinterpret_cast<uintptr_t>(h.head) | reinterpret_cast<uintptr_t>(h.hidden)) % 16 == 0 &&
           h.head_stride % 8 == 0 && h.hidden_stride % 8 == 0 && h.dim % 8 == 0;
}

// The workspace: the targets' logits, the picked rows and their count, the
// tiles' statistics.
struct HeadSpace {
    float *zy;
    int32_t *row;
    int64_t *count;
    float2 *part;
};
static int64_t head_part(int64_t rows) { return (rows * 8 + 8 + 255) / 256 * 256; }  // where the statistics begin

static HeadSpace head_space(void *workspace, int64_t rows) {
    char *w = static_cast<char *>(workspace);
    return {reinterpret_cast<float *>(w + 8), reinterpret_cast<int32_t *>(w + 8 + rows * 4),
            reinterpret_cast<int64_t *>(w), reinterpret_cast<float2 *>(w + head_part(rows))};
}

// Whether the rows that take part are picked first, so that the others cost
// nothing: 3 to 5 us at 277 rows, 7 at 4,096, for what may be half of a long
// call, from about 100 us on.
static bool head_picks(const dlr_head &h) {
    return (double)h.rows * (double)h.vocab * (double)h.dim >= 6.4e10 && h.rows > 64;
}

// Classes [first, end), their statistics from `tiles` on, which moves behind them.
template <typename T, int WV, int WT, int MV, int MT, int S>
static hipError_t launch_head_dma(hipStream_t st, dlr_head h, int64_t first, int64_t end, const HeadPick &pick,
                                  const HeadSpace &w, int64_t &tiles) {
    constexpr int TV = WV * MV * 16, TT = WT * MT * 16;
    const int64_t vtiles = (end - first + TV - 1) / TV, ttiles = (h.rows + TT - 1) / TT;
    h.vocab = end;
    float2 *part = w.part + tiles * h.rows;
    tiles += vtiles;
    return launch(k_head_dma<T, WV, WT, MV, MT, S>, vtiles * ttiles, WV * WT * 64, st, h, first, pick, part, w.zy);
}

template <typename T, int MT, int S>
static hipError_t launch_head_waves(hipStream_t st, dlr_head h, int64_t first, int64_t end, const HeadPick &pick,
                                    const HeadSpace &w, int64_t &tiles) {
    const int64_t vtiles = (end - first + 63) / 64, ttiles = (h.rows + MT * 16 - 1) / (MT * 16);
    h.vocab = end;
    float2 *part = w.part + tiles * h.rows;
    tiles += vtiles;
    return launch(k_head_waves<T, 4, MT, S>, vtiles * ttiles, 256, st, h, first, pick, part, w.zy);
}

// The tiles of more than 16 rows.  What a tile costs: microseconds per stage
// of 64, alone on its CU or two of them on it, measured from 1 x 8 to 32,768
// tiles at dim 512 and 4096; and per round of the CUs a part of its ends (a fit
// for choosing between tiles: a 256 x 256 tile is 1.4 a stage and ends of 9 to 10,
// so that short dimensions cost more than this says, by any tile).
struct HeadTile {
    int64_t tv, tt;
    double alone, two;  // two 0: one workgroup a CU
};
constexpr HeadTile kHeadTiles[] = {
    {256, 256, 1.56, 0}, {256, 192, 1.2, 0}, {256, 128, 0.9, 0}, {128, 64, 0.42, 0.67}, {64, 64, 0.3, 0.55}};
constexpr double kEnds = 3, kLaunch = 3;

static int64_t tiles_of(int64_t classes, int64_t tv) { return (classes + tv - 1) / tv; }

static double head_cost(const HeadTile &t, int64_t rows, int64_t classes, int64_t stages) {
    if (classes <= 0) return 0;
    const int64_t n = tiles_of(classes, t.tv) * tiles_of(rows, t.tt);
    if (t.two == 0 || n <= kCus) return (double)((n + kCus - 1) / kCus) * (t.alone * stages + kEnds);
    return (double)((n + 2 * kCus - 1) / (2 * kCus)) * (t.two * stages + kEnds);
}

// A plan: the first `classes` by tile `first`, the others by tile `rest`.
struct HeadPlan {
    int first, rest;
    int64_t classes;
};

// The cheapest tile for all classes, or a large one for as many classes as
// fill whole rounds of the CUs and the cheapest for the others: 333 x 1536 x
// 50257 is 2.3 rounds of 256 x 128 tiles, paid as 3 (88 us), or one round of
// 256 x 192 tiles and one of 256 x 128 (80).  200 x 4096 x 32000: 72 us by 256
// x 128, 105 by 256 x 256; 2048 x 4096 x 1000: 30 us by 128 x 64, 81.  Over 24
// .. 1,000 tokens, dimensions 264 .. 4096 and 32,000 .. 131,072 classes the plan
// is within 6% of the best of the five tiles for all classes (10% twice), and up
// to 13% better.
static HeadPlan head_plan(int64_t rows, int64_t vocab, int64_t dim) {
    const int64_t stages = (dim + 63) / 64;
    auto best = [&](int64_t classes) {
        int i = 0;
        for (int j = 1; j < 5; ++j)
            if (head_cost(kHeadTiles[j], rows, classes, stages) < head_cost(kHeadTiles[i], rows, classes, stages))
                i = j;
        return i;
    };
    const int whole = best(vocab);
    HeadPlan plan{whole, whole, vocab};
    double cost = head_cost(kHeadTiles[whole], rows, vocab, stages);
    for (int i = 0; i < 3; ++i) {
        const HeadTile &t = kHeadTiles[i];
        const int64_t ttiles = (rows + t.tt - 1) / t.tt, rounds = vocab / t.tv * ttiles / kCus;
        const int64_t classes = rounds * kCus / ttiles * t.tv;
        if (classes <= 0 || classes >= vocab) continue;
        const int rest = best(vocab - classes);
        const double c = head_cost(t, rows, classes, stages) + kLaunch +
                         head_cost(kHeadTiles[rest], rows, vocab - classes, stages);
        if (c < cost) {
            plan = {i, rest, classes};
            cost = c;
        }
    }
    return plan;
}

// Up to this many tiles of 64 classes they go by k_head_waves (1 x 8192 x 1000:
// 18 us against 24, 100 x 8192 x 1500 31 against 42), beyond by k_head_dma, two
// workgroups a CU (300 x 4096 x 3000: 28 against 30).
constexpr int64_t kFewTiles = 128;

// Up to 16 rows the head's bytes are all there is: 256 classes a workgroup once
// that is most of two workgroups a CU, else 64 with a deeper queue (1 row x
// 4096: 131,072 classes 180 us against 190, 65,536 classes 118 against 105).
static int64_t few_rows_tile(int64_t vocab) { return vocab >= 2 * kCus * 192 ? 256 : 64; }

static int64_t head_slice_workspace(int64_t rows, int64_t vocab, int64_t dim) {
    int64_t tiles = tiles_of(vocab, few_rows_tile(vocab));
    if (rows > 16) {
        const HeadPlan plan = head_plan(rows, vocab, dim);
        tiles = tiles_of(plan.classes, kHeadTiles[plan.first].tv) +
                tiles_of(vocab - plan.classes, kHeadTiles[plan.rest].tv);
    }
    const int64_t plain = tiles_of(vocab, kTileV);  // unaligned rows
    return head_part(rows) + rows * (tiles > plain ? tiles : plain) * (int64_t)sizeof(float2);
}

// The rows of one run of launches, whose workgroups of 256 threads for 64 x 64
// logits stay below 2^32 threads; each slice uses the workspace again.
static int64_t head_rows(int64_t vocab) {
    const int64_t most = (INT64_C(1) << 35) / vocab;
    return most < kLaunchRows ? most : kLaunchRows;
}

int64_t head_workspace(int64_t rows, int64_t vocab, int64_t dim) {
    const int64_t slices = (rows + head_rows(vocab) - 1) / head_rows(vocab);
    if (slices <= 1) return head_slice_workspace(rows, vocab, dim);
    const int64_t each = (rows + slices - 1) / slices, last = rows - (rows - 1) / each * each;
    const int64_t a = head_slice_workspace(each, vocab, dim), b = head_slice_workspace(last, vocab, dim);
    return a > b ? a : b;
}

template <typename T>
static hipError_t launch_head_tiles(hipStream_t st, const dlr_head &h, const HeadPick &pick, const HeadSpace &w,
                                    int64_t &tiles) {
    if (!head_by_dma(h)) {
        tiles = (h.vocab + kTileV - 1) / kTileV;
        return launch(k_head_tile<T>, tiles * ((h.rows + kTileT - 1) / kTileT), 256, st, h, w.part, w.zy);
    }
    if (h.rows <= 16 && tiles_of(h.vocab, 64) <= kFewTiles)
        return launch_head_waves<T, 1, 2>(st, h, 0, h.vocab, pick, w, tiles);
    if (h.rows <= 16)
        return few_rows_tile(h.vocab) == 256 ? launch_head_dma<T, 8, 1, 2, 1, 2>(st, h, 0, h.vocab, pick, w, tiles)
                                         : launch_head_dma<T, 4, 1, 1, 1, 4>(st, h, 0, h.vocab, pick, w, tiles);
    auto by = [&](int tile, int64_t first, int64_t end) {
        switch (tile) {
            case 0: return launch_head_dma<T, 2, 4, 8, 4, 2>(st, h, first, end, pick, w, tiles);
            case 1: return launch_head_dma<T, 2, 4, 8, 3, 2>(st, h, first, end, pick, w, tiles);
            case 2: return launch_head_dma<T, 4, 2, 4, 4, 3>(st, h, first, end, pick, w, tiles);
            case 3: return launch_head_dma<T, 4, 1, 2, 4, 3>(st, h, first, end, pick, w, tiles);
            default:
                return tiles_of(end - first, 64) * tiles_of(h.rows, 64) <= kFewTiles
                           ? launch_head_waves<T, 4, 2>(st, h, first, end, pick, w, tiles)
                           : launch_head_dma<T, 4, 1, 1, 4, 4>(st, h, first, end, pick, w, tiles);
        }
    };
    const HeadPlan plan = head_plan(h.rows, h.vocab, h.dim);
    const hipError_t e = by(plan.first, 0, plan.classes);
    return e != hipSuccess || plan.classes == h.vocab ? e : by(plan.rest, plan.classes, h.vocab);
}

static hipError_t launch_head_slice(hipStream_t st, const dlr_head &h, void *workspace, float *logprob, float *lse) {
    const HeadSpace w = head_space(workspace, h.rows);
    const bool picks = head_by_dma(h) && head_picks(h);
    const HeadPick pick{picks ? w.row : nullptr, w.count};
    hipError_t e = hipSuccess;
    if (picks)
        e = launch(k_head_pick, 1, 1024, st, h.target, h.target_bits, h.rows, w.row, w.count, logprob, lse);
    int64_t tiles = 0;
    if (e == hipSuccess)
        e = h.dtype == DLR_DTYPE_BF16 ? launch_head_tiles<__bf16>(st, h, pick, w, tiles)
                                      : launch_head_tiles<_Float16>(st, h, pick, w, tiles);
    if (e != hipSuccess) return e;
    if (h.rows < 16) return launch(k_head_join<1, 256>, h.rows, 256, st, h, pick, tiles, w.part, w.zy, logprob, lse);
    // 256 threads a token while every CU has a workgroup, else 64 (24 tokens of
    // 1,757 tiles 6.5 us, 12.2; 343 of 891 6.5, 9.7; 4,096 of 512 22.6, 7.9; 16
    // threads 42, 27, 11.4).
    if (h.rows <= 4 * kCus)
        return launch(k_head_join<4, 1024>, (h.rows + 3) / 4, 1024, st, h, pick, tiles, w.part, w.zy, logprob, lse);
    return launch(k_head_join<16, 1024>, (h.rows + 15) / 16, 1024, st, h, pick, tiles, w.part, w.zy, logprob, lse);
}

hipError_t launch_head_logprob(hipStream_t st, const dlr_head &all, void *workspace, float *logprob, float *lse) {
    return by_rows(all, head_rows(all.vocab), [&](dlr_head &h, int64_t at) {
        h.hidden = static_cast<const uint16_t *>(h.hidden) + at * h.hidden_stride;
        return launch_head_slice(st, h, workspace, logprob + at, lse + at);
    });
}

}  // namespace dlr

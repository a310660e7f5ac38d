// Log-probabilities of given tokens, the clipped policy loss and the preference
// loss over (rows, vocab) logits, with the losses' gradients in the logits, for
// gfx950.  No reference counterpart: the reference trains on next tokens only
// (lm.hip's cross-entropy); these are the losses of training on rewards and on
// preferences, on the same logits.
//
// Row i, logits z, m = max_j z_j, s = sum_j e^(z_j - m), target t:
//   logp = (z_t - m) - log s
//   policy:      r = e^(logp - old), x = ref - logp, kl = e^x - 1 - x,
//                loss = w (kl_coef kl - min(r A, clip(r, 1 - lo, 1 + hi) A)),
//                d loss / d logp = w (-A r [the unclipped side is the smaller]
//                                     - kl_coef (e^x - 1))
//   preference:  D = sum over a sequence of w (logp - ref), x = beta (D_chosen -
//                D_rejected), loss = (-(1 - eps) log sig(x) - eps log sig(-x)) / pairs
//   d loss / d z_j = (d loss / d logp) ([j = t] - e^(z_j - m) / s)
// A row of weight 0 is not read: its log-probability, loss and gradient are 0
// whatever its logits, target, old, ref and advantage hold.
//
// The logits' type is bf16, fp16 or fp32; rows start at any multiple of the type's
// size (odd vocabularies, padded rows), read and written with 16-byte accesses
// that need no alignment.  Sums, maxima and everything per row are 32 bits or more;
// the gradient is rounded once, to the logits' type.
//
// One workgroup has a row.  Where the gradient needs nothing but the row (the policy
// loss), the row stays in its registers between the statistics and the gradient, so
// each logit moves once in and once out of memory, which is what bounds it: 16384 x 32000
// in bf16 take 342 to 360 us, 5.8 to 6.1 TB/s (a large copy: 5.15).  A row of over 128 KiB
// leaves no room for a second one on its compute unit, so its loads wait for its
// stores (2048 x 128003 in fp16 192 to 209 us, 4.5 to 4.9 TB/s).  A few rows are bound by
// their own latency, 8 us for 64 x 32000, and the host's 12 to 13.
#include <hip/hip_runtime.h>
#include <math.h>

#include "../../include/efla_hip.h"
#include "common.hpp"
#include "internal.hpp"

namespace efla {
namespace tl {

constexpr float kLog2e = 1.44269502f;
constexpr float kLog2eLow = 1.92596299e-8f;  // log2 e - kLog2e
constexpr double kLn2 = 0.69314718055994530942;
constexpr int kMaxThreads = 1024, kMaxWaves = kMaxThreads / kWave;

// 16 bytes of logits, at any multiple of the element's size
template <typename T>
struct Vec {
    static constexpr int N = 16 / sizeof(T);
    typedef __attribute__((__vector_size__(16))) T Full;
    typedef Full Any __attribute__((aligned(sizeof(T))));
    // ONCE: nothing reads it again soon
    template <bool ONCE>
    static __device__ __forceinline__ Full load(const T* p) {
        if constexpr (ONCE) return __builtin_nontemporal_load(reinterpret_cast<const Any*>(p));
        return *reinterpret_cast<const Any*>(p);
    }
    template <bool PAST>
    static __device__ __forceinline__ void store(T* p, Full v) {
        if constexpr (PAST)
            __builtin_nontemporal_store(v, reinterpret_cast<Any*>(p));
        else
            *reinterpret_cast<Any*>(p) = v;
    }
};

// e^d for d <= 0: d log2 e to its nearest float (the constant alone, rounded, would
// shift every term of a sum the same way), then one v_exp_f32
__device__ __forceinline__ float exp_neg(float d) {
    return __builtin_amdgcn_exp2f(fmaf(d, kLog2e, d * kLog2eLow));
}
// the same for a gradient of type T: in 16 bits its own rounding hides the constant's
template <typename T>
__device__ __forceinline__ float exp_grad(float d) {
    if constexpr (sizeof(T) == 4) return exp_neg(d);
    return __builtin_amdgcn_exp2f(d * kLog2e);
}

// log s for s > 0, in 64 bits from one v_log_f32 of the mantissa: its error is that
// of a number in [-1, 0), not that of log2 s
__device__ __forceinline__ double log_of(float s) {
    if (!(s > 0.f && s < INFINITY)) return (double)logf(s);
    int k;
    const float f = frexpf(s, &k);
    return ((double)k + (double)__builtin_amdgcn_logf(f)) * kLn2;
}

// A row's maximum and sum of e^(z - max).  A -inf logit adds nothing, also where it
// is the maximum (the reference point is then 0 and the sum 0); NaN and +inf make
// the sum NaN.
struct Stat {
    float m, s;
};
__device__ __forceinline__ float ref_of(float m) { return m == -INFINITY ? 0.f : m; }
__device__ __forceinline__ void join(Stat& a, float m2, float s2) {
    const float m = fmaxf(a.m, m2), r = ref_of(m);
    // an empty side has m = -inf and contributes its sum times 0 (NaN stays NaN)
    a.s = a.s * exp_neg(a.m - r) + s2 * exp_neg(m2 - r);
    a.m = m;
}

// The waves' statistics (each wave's in all its lanes) as the workgroup's.
__device__ __forceinline__ Stat join_waves(Stat a, Stat* sm) {
    const int waves = blockDim.x / kWave;
    if (waves == 1) return a;
    if (lane_id() == 0) sm[wave_id()] = a;
    __syncthreads();
    const int k = threadIdx.x & (kMaxWaves - 1);
    a = k < waves ? sm[k] : Stat{-INFINITY, 0.f};
#pragma unroll
    for (int off = kMaxWaves / 2; off > 0; off >>= 1)
        join(a, __shfl_xor(a.m, off), __shfl_xor(a.s, off));
    return a;
}

// A row as its whole vectors from a boundary on and the elements before the first and
// behind the last of them, one to a thread.  The boundary is a cache line's, so that no
// line is two waves' (policy loss of 4096 x 50257 in fp32 305 us, 329 from 16-byte
// boundaries), in short rows 16 bytes: loads that are not aligned to these cost a fifth
// (log-probabilities of 4096 x 50257 in bf16: 100 us against 80).  The boundaries are those
// of the logits, also where the gradient has others, whose stores cost less (151 us where
// they agree, 164 where not).
constexpr int kLineVocab = 4096, kLineThreads = 128;  // its edges: up to 70 elements

template <typename T>
struct Span {
    static constexpr int N = Vec<T>::N;
    int head, nv, edges;

    __device__ __forceinline__ Span(const T* z, int V) {
        const int h = (int)(-(uintptr_t)z % (V >= kLineVocab ? 128 : 16) / sizeof(T));
        head = h < V ? h : V;
        nv = (V - head) / N;
        edges = V - nv * N;
    }
    __device__ __forceinline__ int vec(int c) const { return head + c * N; }
    __device__ __forceinline__ int edge(int k) const { return k < head ? k : k + nv * N; }
    // the thread that has element t
    __device__ __forceinline__ int owner(int t) const {
        if (t < head) return t;
        const int c = (t - head) / N;
        return c < nv ? c % (int)blockDim.x : t - nv * N;
    }
};

// Rows of at most blockDim.x * NV vectors stay in registers: thread i holds vectors i,
// i + blockDim.x, ... and one of the edges.
template <typename T, int NV, bool ONCE>
struct Row {
    static constexpr int N = Vec<T>::N;
    Span<T> p;
    typename Vec<T>::Full x[NV];
    T edge;

    // The elements are converted again in each pass: kept as floats a 16-bit row
    // would take twice the registers.
    static __device__ __forceinline__ typename Vec<T>::Full packed(typename Vec<T>::Full v) {
        typedef __attribute__((__vector_size__(16))) uint32_t U4;
        U4 u = __builtin_bit_cast(U4, v);
        if constexpr (sizeof(T) == 2) asm("" : "+v"(u));
        return __builtin_bit_cast(typename Vec<T>::Full, u);
    }

    __device__ __forceinline__ Row(const T* z, const Span<T>& p_) : p(p_) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = threadIdx.x + i * blockDim.x;
#pragma unroll
            for (int j = 0; j < N; ++j) x[i][j] = (T)-INFINITY;
            if (c < p.nv) x[i] = Vec<T>::template load<ONCE>(z + p.vec(c));
        }
        edge = (T)-INFINITY;
        if (threadIdx.x < p.edges) edge = z[p.edge(threadIdx.x)];
    }

    __device__ __forceinline__ Stat stat(Stat* sm) const {
        float m4[4] = {(float)edge, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j) m4[j & 3] = fmaxf(m4[j & 3], (float)x[i][j]);
        float m = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
        const float r = ref_of(m);
        float s4[4] = {exp_neg((float)edge - r), 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const typename Vec<T>::Full v = packed(x[i]);
#pragma unroll
            for (int j = 0; j < N; ++j) s4[j & 3] += exp_neg((float)v[j] - r);
        }
        float s = (s4[0] + s4[1]) + (s4[2] + s4[3]);
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
        return join_waves(Stat{m, s}, sm);
    }

    // coef ([j = t] - e^(z_j - m) / s) but for the target's own part
    template <bool PAST>
    __device__ __forceinline__ void grad(T* g, const Stat& a, float coef) const {
        const float k = -coef / a.s, r = ref_of(a.m);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = threadIdx.x + i * blockDim.x;
            if (c >= p.nv) continue;
            typename Vec<T>::Full y = packed(x[i]);
#pragma unroll
            for (int j = 0; j < N; ++j) y[j] = (T)(k * exp_grad<T>((float)y[j] - r));
            Vec<T>::template store<PAST>(g + p.vec(c), y);
        }
        if (threadIdx.x < p.edges)
            g[p.edge(threadIdx.x)] = (T)(k * exp_grad<T>((float)edge - r));
    }
};

// Longer rows stream: read once for the statistics and again for the gradient (ONCE: if
// for the former alone).
template <typename T, bool ONCE>
struct Row<T, 0, ONCE> {
    static constexpr int N = Vec<T>::N, U = 4;
    const T* z;
    Span<T> p;

    __device__ __forceinline__ Row(const T* z_, const Span<T>& p_) : z(z_), p(p_) {}

    __device__ __forceinline__ Stat stat(Stat* sm) const {
        Stat a{-INFINITY, 0.f};
        for (int c0 = threadIdx.x; c0 < p.nv; c0 += U * blockDim.x) {
            typename Vec<T>::Full x[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = c0 + u * blockDim.x;
#pragma unroll
                for (int j = 0; j < N; ++j) x[u][j] = (T)-INFINITY;
                if (c < p.nv) x[u] = Vec<T>::template load<ONCE>(z + p.vec(c));
            }
            float m = a.m;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < N; ++j) m = fmaxf(m, (float)x[u][j]);
            const float r = ref_of(m);
            float s4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int j = 0; j < N; ++j) s4[j & 3] += exp_neg((float)x[u][j] - r);
            a.s = a.s * exp_neg(a.m - r) + ((s4[0] + s4[1]) + (s4[2] + s4[3]));
            a.m = m;
        }
        if (threadIdx.x < p.edges) {
            const float v = (float)z[p.edge(threadIdx.x)];
            join(a, v, v == -INFINITY ? 0.f : 1.f);
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) join(a, __shfl_xor(a.m, off), __shfl_xor(a.s, off));
        return join_waves(a, sm);
    }

    template <bool PAST>
    __device__ __forceinline__ void grad(T* g, const Stat& a, float coef) const {
        const float k = -coef / a.s, r = ref_of(a.m);
        for (int c0 = threadIdx.x; c0 < p.nv; c0 += U * blockDim.x) {
            typename Vec<T>::Full y[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = c0 + u * blockDim.x;
                if (c < p.nv) y[u] = Vec<T>::template load<PAST>(z + p.vec(c));
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = c0 + u * blockDim.x;
                if (c >= p.nv) continue;
#pragma unroll
                for (int j = 0; j < N; ++j) y[u][j] = (T)(k * exp_grad<T>((float)y[u][j] - r));
                Vec<T>::template store<PAST>(g + p.vec(c), y[u]);
            }
        }
        if (threadIdx.x < p.edges) {
            const int c = p.edge(threadIdx.x);
            g[c] = (T)(k * exp_grad<T>((float)z[c] - r));
        }
    }
};

__device__ __forceinline__ double logp_of(const Stat& a, float zt) {
    return ((double)zt - (double)a.m) - log_of(a.s);
}

// The target's own place, by the thread that wrote it with the rest of the row.
template <typename T>
__device__ __forceinline__ void target_grad(T* g, const Span<T>& p, int t, float zt,
                                            const Stat& a, float coef) {
    if ((int)threadIdx.x == p.owner(t))
        g[t] = (T)(coef - coef / a.s * exp_neg(zt - ref_of(a.m)));
}

template <bool PAST, typename T>
__device__ __forceinline__ void row_zero(T* g, int V) {
    const typename Vec<T>::Full zero = {};
    const Span<T> p(g, V);
    for (int c = threadIdx.x; c < p.nv; c += blockDim.x)
        Vec<T>::template store<PAST>(g + p.vec(c), zero);
    if ((int)threadIdx.x < p.edges) g[p.edge(threadIdx.x)] = (T)0.f;
}

// Rows of a grid that has a second dimension where one would not hold them.
__device__ __forceinline__ long block_row() {
    return blockIdx.x + (long)blockIdx.y * gridDim.x;
}

template <typename T, int NV, bool ONCE>
__global__ void __launch_bounds__(kMaxThreads, NV > 8 ? 4 : 8)
logprob_kernel(const T* __restrict__ logits, const int32_t* __restrict__ targets,
               const float* __restrict__ weights, float* __restrict__ logp, float2* stat,
               float* coef, long rows, int V, long ld) {
    __shared__ Stat sm[kMaxWaves];
    const long row = block_row();
    if (row >= rows) return;
    // rows outside of every sequence keep this coefficient
    if (coef && threadIdx.x == 0) coef[row] = 0.f;
    if (weights && weights[row] == 0.f) {
        if (threadIdx.x == 0) logp[row] = 0.f;
        return;
    }
    const T* z = logits + row * ld;
    const int t = targets[row];
    const Row<T, NV, ONCE> x(z, Span<T>(z, V));
    const float zt = t >= 0 && t < V ? (float)z[t] : NAN;
    const Stat a = x.stat(sm);
    if (threadIdx.x == 0) {
        logp[row] = (float)logp_of(a, zt);
        if (stat) stat[row] = float2{a.m, a.s};
    }
}

// e^y - 1 - y with em = e^y - 1.  Near 0, where it is about y^2 / 2, the difference loses its
// digits (at |y| = 1e-4 a thousandth of it, at 1e-7 all): there a series,
// y^2 (1/2! + y/3! + ... + y^7/9!), within 3 roundings of 2^-24 (the first term left out is
// 2.5e-9 of it at y = -1/2).
__device__ __forceinline__ float kl_of(float y, float em) {
    if (fabsf(y) < 0.5f) {
        float q = 1.f / 362880.f;
        q = fmaf(q, y, 1.f / 40320.f);
        q = fmaf(q, y, 1.f / 5040.f);
        q = fmaf(q, y, 1.f / 720.f);
        q = fmaf(q, y, 1.f / 120.f);
        q = fmaf(q, y, 1.f / 24.f);
        q = fmaf(q, y, 1.f / 6.f);
        q = fmaf(q, y, 0.5f);
        return y * y * q;
    }
    return em == INFINITY ? INFINITY : em - y;  // also where y is infinite
}

struct PolicyArgs {
    const int32_t* targets;
    const float *adv, *old, *ref, *weights;
    float *loss, *logp, *kl;
    long rows, ld, ldg;
    int V;
    float low, high, kl_coef, even;  // even: the weight of a row where there are none
};

template <typename T, int NV, bool PAST>
__global__ void __launch_bounds__(kMaxThreads, NV > 8 ? 4 : 8)
policy_kernel(const T* logits, T* grad, PolicyArgs a) {
    __shared__ Stat sm[kMaxWaves];
    __shared__ float sm_coef;
    const long row = block_row();
    if (row >= a.rows) return;
    const float w = a.weights ? a.weights[row] : a.even;
    T* g = grad ? grad + row * a.ldg : nullptr;
    if (w == 0.f) {
        if (threadIdx.x == 0) {
            a.loss[row] = 0.f;
            a.logp[row] = 0.f;
            if (a.kl) a.kl[row] = 0.f;
        }
        if (g) row_zero<PAST>(g, a.V);
        return;
    }
    const T* z = logits + row * a.ld;
    const int t = a.targets[row];
    const bool tok = t >= 0 && t < a.V;
    const Row<T, NV, (PAST && NV > 0)> x(z, Span<T>(z, a.V));
    const float zt = tok ? (float)z[t] : 0.f;  // read before the gradient may overwrite it
    const float adv = a.adv[row];
    const float old = a.old ? a.old[row] : 0.f, ref = a.ref ? a.ref[row] : 0.f;
    const Stat st = x.stat(sm);
    // the first wave turns the statistics into the row's outputs and its coefficient
    if (wave_id() == 0) {
        const double lp = logp_of(st, zt);
        // fminf and fmaxf drop a NaN, which has to reach the loss and the coefficient
        const float r = a.old ? expf((float)(lp - (double)old)) : lp == lp ? 1.f : NAN;
        const float u = r * adv, c = fminf(fmaxf(r, a.low), a.high) * adv;
        float l = -(c < u ? c : u);
        // an advantage that is NaN is on neither side
        float d = (adv >= 0.f && r > a.high) || (adv < 0.f && r < a.low) ? 0.f : -adv * r;
        float kl = 0.f;
        if (a.ref) {
            const float y = (float)((double)ref - lp);
            const float em = expm1f(y);
            kl = kl_of(y, em);
            if (a.kl_coef != 0.f) {
                l += a.kl_coef * kl;
                d -= a.kl_coef * em;
            }
        }
        if (threadIdx.x == 0) {
            a.loss[row] = tok ? w * l : NAN;
            a.logp[row] = tok ? (float)lp : NAN;
            if (a.kl) a.kl[row] = tok ? kl : NAN;
            sm_coef = w * d;
        }
    }
    if (!g) return;
    __syncthreads();
    if (tok) {
        x.template grad<PAST>(g, st, sm_coef);
        target_grad(g, x.p, t, zt, st, sm_coef);
    } else {
        row_zero<PAST>(g, a.V);
    }
}

// What one workgroup of a launch hands to another is itself the message: a word written
// and read with device-wide atomics, all ones until it is there.
constexpr uint32_t kAbsent = 0xFFFFFFFFu;
constexpr uint64_t kAbsent2 = ~0ull;

template <typename U>
__device__ __forceinline__ void tell(U* p, U v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename U>
__device__ __forceinline__ U hear(U* p, U absent) {
    U v;
    while ((v = __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) == absent)
        __builtin_amdgcn_s_sleep(8);
    return v;
}
// a float as a message: a NaN is never the one that stands for nothing
__device__ __forceinline__ uint32_t word_of(float v) {
    return v != v ? 0x7FC00000u : __builtin_bit_cast(uint32_t, v);
}

constexpr int NT = 256;

// The sums of w (logp - ref) over a pair's two sequences, rows [a0, a1) and [a1, a2): the
// workgroup's first 256 threads add in a fixed order, all get them.  told: logp are
// messages.
struct PairSum {
    double sum[2];

    __device__ __forceinline__ PairSum(float* logp, const float* ref, const float* weights,
                                       int a0, int a1, int a2, bool told) {
        __shared__ double sm[2][NT / kWave];
        if (threadIdx.x < NT) {
            sum[0] = sum[1] = 0.0;
            constexpr int U = 4;  // rows whose loads are on their way together
            for (int i0 = a0 + (int)threadIdx.x; i0 < a2; i0 += U * NT) {
                float w[U], lp[U], rf[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int i = i0 + u * NT;
                    w[u] = lp[u] = rf[u] = 0.f;
                    if (i >= a2) continue;
                    w[u] = weights ? weights[i] : 1.f;
                    if (ref) rf[u] = ref[i];
                    lp[u] = told ? __builtin_bit_cast(
                                       float, hear(reinterpret_cast<uint32_t*>(logp) + i, kAbsent))
                                 : logp[i];
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const double d =
                        w[u] != 0.f ? (double)w[u] * ((double)lp[u] - (double)rf[u]) : 0.0;
                    if (i0 + u * NT < a1)
                        sum[0] += d;
                    else
                        sum[1] += d;
                }
            }
#pragma unroll
            for (int q = 0; q < 2; ++q) {
#pragma unroll
                for (int off = 32; off > 0; off >>= 1) sum[q] += __shfl_xor(sum[q], off);
                if (lane_id() == 0) sm[q][wave_id()] = sum[q];
            }
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            sum[q] = sm[q][0];
#pragma unroll
            for (int k = 1; k < NT / kWave; ++k) sum[q] += sm[q][k];
        }
    }

    // by one wave, a row at most to each lane: the same sums as the workgroup's
    __device__ __forceinline__ PairSum(const float* logp, const float* ref, const float* weights,
                                       int a0, int a1, int a2) {
        const int i = a0 + lane_id();
        const float w = i >= a2 ? 0.f : weights ? weights[i] : 1.f;
        const float lp = i < a2 ? logp[i] : 0.f, rf = ref && i < a2 ? ref[i] : 0.f;
        const double d = w != 0.f ? (double)w * ((double)lp - (double)rf) : 0.0;
        sum[0] = 0.0 + (i < a1 ? d : 0.0);
        sum[1] = 0.0 + (i < a1 ? 0.0 : d);
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) sum[q] += __shfl_xor(sum[q], off);
    }
};

// loss and d loss / dx of a pair whose rewards differ by x
struct PairLoss {
    double loss, dx;

    __device__ __forceinline__ PairLoss(double x, double eps, double inv_pairs) {
        const double u = exp(-fabs(x));          // e^-|x|
        const double lg = log1p(u);              // log sig(-|x|) = -|x| - lg
        const double plus = lg + fmax(-x, 0.0);  // -log sig(x)
        const double minus = lg + fmax(x, 0.0);  // -log sig(-x)
        const double sig = x >= 0 ? 1.0 / (1.0 + u) : u / (1.0 + u);
        const double gis = x >= 0 ? u / (1.0 + u) : 1.0 / (1.0 + u);  // sig(-x)
        // without smoothing the other side's term is not there, also where it is infinite
        loss = ((1.0 - eps) * plus + (eps != 0.0 ? eps * minus : 0.0)) * inv_pairs;
        dx = (eps * sig - (1.0 - eps) * gis) * inv_pairs;
    }
};

// The pairs' sums and losses, and each row's coefficient.  A pair to a workgroup, or, of MANY
// pairs, `each` of them, as many at a time as it has waves: each wave one of up to 64 rows,
// the workgroup the longer ones.  An offset is taken as at least all before it, which the
// workgroup looks through for its first pair, and at most the rows.
template <bool MANY>
__global__ void __launch_bounds__(NT)
pair_kernel(const int32_t* __restrict__ cu, float* logp,
            const float* __restrict__ ref, const float* __restrict__ weights, int rows,
            int pairs, int each, float beta, float eps, float inv_pairs,
            float* __restrict__ loss, float* __restrict__ rewards, float* __restrict__ coef) {
    constexpr int kWaves = NT / kWave;
    __shared__ int sm_low[kWaves];
    const long begin = (long)blockIdx.x * each;
    const long end = begin + each < pairs ? begin + each : pairs;
    int low = 0;
    constexpr int U = 16;  // loads on their way together
    for (long i0 = threadIdx.x; i0 < 2 * begin; i0 += U * NT) {
        int v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = i0 + u * NT < 2 * begin ? cu[i0 + u * NT] : 0;
#pragma unroll
        for (int u = 0; u < U; ++u) low = max(low, v[u]);
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) low = max(low, __shfl_xor(low, off));
    if (lane_id() == 0) sm_low[wave_id()] = low;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kWaves; ++k) low = max(low, sm_low[k]);
    const auto finish = [&](long pair, const int* at, const PairSum& d, int tid, int threads) {
        const PairLoss l((double)beta * (d.sum[0] - d.sum[1]), eps, inv_pairs);
        if (tid == 0) {
            loss[pair] = (float)l.loss;
            rewards[2 * pair] = (float)((double)beta * d.sum[0]);
            rewards[2 * pair + 1] = (float)((double)beta * d.sum[1]);
        }
        if (!coef) return;
        const float c = (float)((double)beta * l.dx);
        for (int i = at[0] + tid; i < at[2]; i += threads) {
            const float w = weights ? weights[i] : 1.f;
            coef[i] = w != 0.f ? (i < at[1] ? c : -c) * w : 0.f;  // 0 also of a NaN
        }
    };
    if constexpr (!MANY) {
        int at[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) at[i] = low = min(max(low, cu[2 * begin + i]), rows);
        finish(begin, at, PairSum(logp, ref, weights, at[0], at[1], at[2], false), threadIdx.x,
               NT);
        return;
    }
    for (long p0 = begin; p0 < end; p0 += kWaves) {
        int at[kWaves][3], own[3] = {0, 0, 0};
#pragma unroll
        for (int q = 0; q < kWaves; ++q)
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                if (p0 + q < end) low = min(max(low, cu[2 * (p0 + q) + i]), rows);
                at[q][i] = low;
                if (q == wave_id()) own[i] = low;
            }
        if (p0 + wave_id() < end && own[2] - own[0] <= kWave)
            finish(p0 + wave_id(), own, PairSum(logp, ref, weights, own[0], own[1], own[2]),
                   lane_id(), kWave);
#pragma unroll
        for (int q = 0; q < kWaves; ++q) {
            if (at[q][2] - at[q][0] <= kWave) continue;
            __syncthreads();  // the last such pair's sums have been read
            finish(p0 + q, at[q],
                   PairSum(logp, ref, weights, at[q][0], at[q][1], at[q][2], false), threadIdx.x,
                   NT);
        }
    }
}

template <typename T, bool PAST>
__global__ void __launch_bounds__(kMaxThreads)
grad_kernel(const T* logits, T* grad, const int32_t* __restrict__ targets,
            const float2* __restrict__ stat, const float* __restrict__ coef, long rows, int V,
            long ld, long ldg) {
    // the last rows first: of more logits than the 256 MB cache holds it has those that the
    // statistics read last (8191 x 32000 in bf16 200 us in all, 230 from the first on)
    const long row = backwards(block_row(), rows);
    if (row < 0 || row >= rows) return;
    T* g = grad + row * ldg;
    const int t = targets[row];
    const float c = coef[row];
    // 0: a row without weight or outside of every sequence, whose logits may be anything (one
    // that counts has NaN here where its statistics are), or a pair without a gradient
    if (c == 0.f || t < 0 || t >= V) {
        row_zero<PAST>(g, V);
        return;
    }
    const T* z = logits + row * ld;
    const Stat a{stat[row].x, stat[row].y};
    const float zt = (float)z[t];  // in place its own thread overwrites it, later
    const Row<T, 0, false> x(z, Span<T>(z, V));
    x.template grad<PAST>(g, a, c);
    target_grad(g, x.p, t, zt, a, c);
}

// The preference loss of more logits than the 256 MB cache holds, in one launch.  Each
// logit is read twice, the second time once its pair's sums are known; launches for
// either pass read them from memory twice.  Here a workgroup takes one row's
// statistics and an earlier row's gradient, which follows its own statistics by no more
// than the longest pair and what is in flight: between them the row stays in the cache.
// The rows are drawn from a counter, so that a workgroup waits only for what has been
// drawn before (a gradient for its pair's sums, a pair's last row for the pair's other
// rows), by workgroups that run already and do their statistics first: every wait ends
// whatever else the GPU does.  32 pairs of 4100 x 50257 in all: fp32 323 us against 384
// in three launches, bf16 178 against 195; 8 pairs of 2048 x 128000 in bf16 187 against 204.
// Drawing takes 13 ns, one workgroup after another, so that shorter rows are faster in
// three launches: 8 pairs of 8191 x 32000 in bf16 195 us against 207.
struct PairInfo {
    int pair, mid, end;  // of the pair that starts at this row
    uint32_t coef;       // d loss / d (sum of the chosen rows' w logp): a message
};
struct Plan {
    uint32_t next;  // the row to be drawn, alone in its cache line
    int pad[63];
    int lag;  // rows by which gradients follow statistics
    int pad2[63];
    // then: uint64_t stat[rows] (+ 1 where odd), PairInfo info[rows], int first[rows]
};
constexpr int kPlanThreads = 1024;

struct PrefArgs {
    const int32_t *targets, *cu;
    const float *ref, *weights;
    float *loss, *rewards, *logp;
    Plan* plan;
    uint64_t* stat;
    PairInfo* info;
    int* first;
    long ld, ldg;
    int rows, pairs, V;
    int slack;  // rows in flight
    float beta, eps, inv_pairs;
};

// The first workgroup reads the offsets (each at least all before it and at most the
// rows), writes every row's pair and the lag, and finishes pairs without rows; the others
// take the messages back.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(PrefArgs a) {
    const int tid = threadIdx.x;
    if (blockIdx.x > 0) {
        const long step = (long)(gridDim.x - 1) * kPlanThreads;
        for (long i = (long)(blockIdx.x - 1) * kPlanThreads + tid; i < a.rows; i += step) {
            a.stat[i] = kAbsent2;
            reinterpret_cast<uint32_t*>(a.logp)[i] = kAbsent;
        }
        return;
    }
    __shared__ int top[kMaxWaves];
    __shared__ int at[2][kPlanThreads];
    int before = 0, begin = a.rows, longest = 0;
    for (int base = 0; base < a.pairs; base += kPlanThreads) {
        const int p = base + tid;
        int c[3] = {0, 0, 0};
        if (p < a.pairs)
#pragma unroll
            for (int i = 0; i < 3; ++i) c[i] = min(max(a.cu[2 * (long)p + i], 0), a.rows);
        // the largest offset before this pair's: among lanes, waves, blocks of pairs
        int up = max(max(c[0], c[1]), c[2]);
#pragma unroll
        for (int off = 1; off < kWave; off *= 2) {
            const int o = __shfl_up(up, off);
            if (lane_id() >= off) up = max(up, o);
        }
        if (lane_id() == kWave - 1) top[wave_id()] = up;
        int low = __shfl_up(up, 1);
        if (lane_id() == 0) low = 0;
        __syncthreads();
        low = max(low, before);
        for (int k = 0; k < kMaxWaves; ++k) {
            if (k < wave_id()) low = max(low, top[k]);
            before = max(before, top[k]);
        }
        const int a0 = max(low, c[0]), a1 = max(a0, c[1]), a2 = max(a1, c[2]);
        at[0][tid] = a0;
        at[1][tid] = p < a.pairs ? a2 : a0;
        if (p < a.pairs && a0 == a2) {
            a.loss[p] = (float)PairLoss(0.0, a.eps, a.inv_pairs).loss;
            a.rewards[2 * (long)p] = a.rewards[2 * (long)p + 1] = 0.f;
        }
        if (p < a.pairs && a0 < a2) {
            a.info[a0] = PairInfo{p, a1, a2, kAbsent};
            longest = max(longest, a2 - a0);
        }
        if (p == 0) begin = a0;
        __syncthreads();
        for (int q = wave_id(); q < kPlanThreads && base + q < a.pairs; q += kMaxWaves)
            for (int i = at[0][q] + lane_id(); i < at[1][q]; i += kWave) a.first[i] = at[0][q];
        __syncthreads();
    }
    // rows of no sequence: before the first offset and behind the last
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) longest = max(longest, __shfl_xor(longest, off));
    if (lane_id() == 0) top[wave_id()] = longest;
    if (tid == 0) at[0][0] = begin;
    __syncthreads();
    begin = at[0][0];
    for (int k = 0; k < kMaxWaves; ++k) longest = max(longest, top[k]);
    for (long i = tid; i < begin; i += kPlanThreads) a.first[i] = -1;
    for (long i = max(begin, before) + tid; i < a.rows; i += kPlanThreads) a.first[i] = -1;
    if (tid == 0) {
        a.plan->next = 0;
        a.plan->lag = (int)min((long)longest + a.slack, (long)a.rows);
    }
}

template <typename T, bool PAST>
__global__ void __launch_bounds__(kMaxThreads, 8)
preference_kernel(const T* logits, T* grad, PrefArgs a) {
    __shared__ Stat sm[kMaxWaves];
    __shared__ uint32_t sm_draw;
    __shared__ Stat sm_stat;
    __shared__ float sm_coef;
    const int lag = a.plan->lag;
    if (block_row() >= (long)a.rows + lag) return;  // not needed: the grid is for any lag
    if (threadIdx.x == 0) sm_draw = atomicAdd(&a.plan->next, 1u);
    __syncthreads();
    const uint32_t drawn = sm_draw;
    if (drawn < (uint32_t)a.rows) {
        const int row = drawn;
        float lp = 0.f;
        if (!a.weights || a.weights[row] != 0.f) {
            const T* z = logits + row * a.ld;
            const int t = a.targets[row];
            const Row<T, 0, false> x(z, Span<T>(z, a.V));
            const float zt = t >= 0 && t < a.V ? (float)z[t] : NAN;
            const Stat st = x.stat(sm);
            lp = (float)logp_of(st, zt);
            if (threadIdx.x == 0)
                tell(a.stat + row, __builtin_bit_cast(uint64_t, float2{st.m, st.s}));
        }
        if (threadIdx.x == 0) tell(reinterpret_cast<uint32_t*>(a.logp) + row, word_of(lp));
        const int first = a.first[row];
        if (first >= 0 && row + 1 == a.info[first].end) {
            const PairInfo p = a.info[first];
            const PairSum d(a.logp, a.ref, a.weights, first, p.mid, p.end, true);
            if (threadIdx.x == 0) {
                const PairLoss l((double)a.beta * (d.sum[0] - d.sum[1]), a.eps, a.inv_pairs);
                tell(&a.info[first].coef, word_of((float)((double)a.beta * l.dx)));
                a.loss[p.pair] = (float)l.loss;
                a.rewards[2 * (long)p.pair] = (float)((double)a.beta * d.sum[0]);
                a.rewards[2 * (long)p.pair + 1] = (float)((double)a.beta * d.sum[1]);
            }
        }
    }
    if (drawn < (uint32_t)lag) return;
    // where all statistics come first the last rows' gradients follow at once: the cache
    // has these
    const int row = lag == a.rows ? a.rows - 1 - (int)(drawn - lag) : (int)(drawn - lag);
    T* g = grad + row * a.ldg;
    const int t = a.targets[row], first = a.first[row];
    const float w = a.weights ? a.weights[row] : 1.f;
    if (w == 0.f) {
        row_zero<PAST>(g, a.V);
        return;
    }
    const T* z = logits + row * a.ld;
    const bool tok = t >= 0 && t < a.V;
    const float zt = tok ? (float)z[t] : 0.f;  // in place its own thread overwrites it, later
    if (threadIdx.x == 0) {
        // in place also a row of zeros waits for its statistics to have been read
        const float2 st = __builtin_bit_cast(float2, hear(a.stat + row, kAbsent2));
        sm_stat = Stat{st.x, st.y};
        if (tok && first >= 0) {
            const float c = __builtin_bit_cast(float, hear(&a.info[first].coef, kAbsent));
            sm_coef = (row < a.info[first].mid ? c : -c) * w;
        }
    }
    __syncthreads();
    if (!tok || first < 0) {
        row_zero<PAST>(g, a.V);
        return;
    }
    const Row<T, 0, false> x(z, Span<T>(z, a.V));
    const Stat st = sm_stat;
    const float coef = sm_coef;
    x.template grad<PAST>(g, st, coef);
    target_grad(g, x.p, t, zt, st, coef);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
static size_t dtype_size(int dtype) {
    return dtype == kDtypeF32 ? 4 : dtype == kDtypeF16 || dtype == kDtypeBF16 ? 2 : 0;
}

// What the three entries ask of the logits and, where there is one, the gradient.
static int check(const void* logits, const int32_t* targets, const void* grad, size_t rows,
                 size_t vocab, size_t ld, size_t ldg, int dtype) {
    const size_t size = dtype_size(dtype);
    if (size == 0 || vocab == 0 || ld < vocab || (grad && ldg < vocab)) return kInvalidValue;
    if (!logits || !targets) return kInvalidValue;
    if ((uintptr_t)logits % size || (uintptr_t)grad % size) return kInvalidValue;
    // in place the gradient overwrites the row that its own workgroup has read
    if (grad == logits && ldg != ld) return kInvalidValue;
    if (rows > 0x7FFFFFFFull || vocab > 0x7FFFFFFFull) return kInvalidConfiguration;
    size_t n;
    if (!mul_ok(rows, ld, size, &n) || !mul_ok(rows, ldg, size, &n) || n > (size_t)1 << 62)
        return kInvalidConfiguration;
    return kSuccess;
}

#define TL_TYPED(dtype, T, ...)          \
    do {                                 \
        if ((dtype) == kDtypeBF16) {     \
            typedef bf16 T;              \
            __VA_ARGS__                  \
        } else if ((dtype) == kDtypeF16) { \
            typedef f16 T;               \
            __VA_ARGS__                  \
        } else {                         \
            typedef float T;             \
            __VA_ARGS__                  \
        }                                \
    } while (0)

// The form for rows of this length: vectors per thread (0: streamed) and threads.
struct Form {
    int nv;
    unsigned threads;
};
static Form form_with(size_t vocab, size_t nv, int k) {
    const size_t least = vocab >= kLineVocab ? kLineThreads : kWave;
    const size_t need = (nv + k - 1) / k;
    return Form{k, need < least ? (unsigned)least : (unsigned)((need + kWave - 1) / kWave * kWave)};
}
// The policy loss: waves that fill whole rounds of a compute unit's four SIMDs, so the number
// of vectors, 4 to 8 (to 16 where 8 do not hold the row), that leaves the fewest places of
// such rounds empty, the smaller where two do.  In bf16, us with 4 to 8 vectors: 16384 x
// 32000 354, 385, 357, 359, 359; x 28000 341, 310, 314, 309, 308; x 17000 197, 187, 186,
// 187, 188; x 1000 18.7, 20.6, 21.8, 23.3, 23.7; 8192 x 36000 211 with 5, 201 with 6, 204,
// 206; 4096 x 50257 147 with 7, 151 with 8; 2048 x 100000 161 with 13, 176 with 16.
static Form policy_form(size_t vocab, int dtype) {
    const size_t nv = vocab / (16 / dtype_size(dtype));
    if (nv > 16 * kMaxThreads) return Form{0, kMaxThreads};
    int best = 0;
    size_t places = 0;
    for (int k = 4; k <= (nv <= 8 * kMaxThreads ? 8 : 16); ++k) {
        const size_t need = (nv + k - 1) / k, round = (need + 4 * kWave - 1) / (4 * kWave);
        if (need > kMaxThreads || (best && k * round >= places)) continue;
        best = k;
        places = k * round;
    }
    return form_with(vocab, nv, best);
}
// Log-probabilities, which write nothing, take workgroups as small as 8 vectors make them
// (bf16, us with 4 to 8: 16384 x 28000 168, 161, 168, 142, 138; x 9000 56, 51, 47, 50, 54),
// in rows of a few waves the number that leaves the fewest places empty (x 5000 32, 30, 31,
// 33, 35; x 1000 11.0, 12.2, 13.4, 15.1, 16.6).  Where that would be over 640 threads the row
// is streamed by 512 (4096 x 50257 67, 81 in registers; x 40000 58 and 57), and by 1024
// where the policy loss streams too (2048 x 128003 82 with either): both then sum a row in
// the same order.
static Form logprob_form(size_t vocab, int dtype) {
    const size_t nv = vocab / (16 / dtype_size(dtype));
    if (nv > 8 * 640) return Form{0, nv > 16 * kMaxThreads ? unsigned(kMaxThreads) : 512u};
    Form best = form_with(vocab, nv, 8);
    if (nv > 8 * 256) return best;
    for (int k = 7; k >= 4; --k) {
        const Form f = form_with(vocab, nv, k);
        if (f.nv * f.threads < best.nv * best.threads) best = f;
    }
    return best;
}

#define TL_IF(cond, NAME, ...)          \
    do {                                \
        if (cond) {                     \
            constexpr bool NAME = true; \
            __VA_ARGS__                 \
        } else {                        \
            constexpr bool NAME = false; \
            __VA_ARGS__                 \
        }                               \
    } while (0)

#define TL_CASE(k, NV, ...)      \
    case k: {                    \
        constexpr int NV = k;    \
        __VA_ARGS__              \
        break;                   \
    }
#define TL_POLICY_FORM(form, NV, ...)     \
    switch ((form).nv) {                  \
        TL_CASE(4, NV, __VA_ARGS__)       \
        TL_CASE(5, NV, __VA_ARGS__)       \
        TL_CASE(6, NV, __VA_ARGS__)       \
        TL_CASE(7, NV, __VA_ARGS__)       \
        TL_CASE(8, NV, __VA_ARGS__)       \
        TL_CASE(9, NV, __VA_ARGS__)       \
        TL_CASE(10, NV, __VA_ARGS__)      \
        TL_CASE(11, NV, __VA_ARGS__)      \
        TL_CASE(12, NV, __VA_ARGS__)      \
        TL_CASE(13, NV, __VA_ARGS__)      \
        TL_CASE(14, NV, __VA_ARGS__)      \
        TL_CASE(15, NV, __VA_ARGS__)      \
        TL_CASE(16, NV, __VA_ARGS__)      \
        TL_CASE(0, NV, __VA_ARGS__)       \
    }
#define TL_LOGPROB_FORM(form, NV, ...)    \
    switch ((form).nv) {                  \
        TL_CASE(4, NV, __VA_ARGS__)       \
        TL_CASE(5, NV, __VA_ARGS__)       \
        TL_CASE(6, NV, __VA_ARGS__)       \
        TL_CASE(7, NV, __VA_ARGS__)       \
        TL_CASE(8, NV, __VA_ARGS__)       \
        TL_CASE(0, NV, __VA_ARGS__)       \
    }

// A workgroup each; a grid's dimension times its threads stays below 2^32.
static dim3 row_grid(size_t rows) {
    const size_t x = (size_t)1 << 20;
    return rows <= x ? dim3((unsigned)rows) : dim3((unsigned)x, (unsigned)((rows + x - 1) / x));
}

// Whether logits and gradient are more than the 256 MB cache: then the gradient is stored
// past it (policy loss of 16384 x 32000 in bf16 360 us, 369 through it; preference loss of
// 8191 x 32000, whose second read the cache serves, 202 and 249), and what is read for the
// last time read past it (log-probabilities of 16384 x 32000 98 us against 105, of 4096 x
// 50257 in fp32 120 against 130; preference losses 1 to 4 %); else what comes next finds
// them there.  The gradient is counted beside the logits also where it overwrites them or
// there is none; between 128 and 256 MiB of logits those calls have not been measured.
static bool past_cache(size_t rows, size_t vocab, int dtype) {
    return 2 * rows * vocab * dtype_size(dtype) > ((size_t)256 << 20);
}

static int logprob(const void* logits, const int32_t* targets, const float* weights, float* logp,
                   float2* stat, float* coef, size_t rows, size_t vocab, size_t ld, int dtype,
                   Form f, bool once, hipStream_t st) {
    TL_TYPED(dtype, T, {
        TL_LOGPROB_FORM(f, NV, {
            TL_IF(once, ONCE, {
                EFLA_LAUNCH("token_logprob", (logprob_kernel<T, NV, ONCE>), row_grid(rows),
                            dim3(f.threads), st, (const T*)logits, targets, weights, logp, stat,
                            coef, (long)rows, (int)vocab, (long)ld);
            });
        });
    });
    return (int)hipPeekAtLastError();
}

// Logits that the cache does not hold, in rows whose work hides the drawing: their
// preference loss streams them.  420 MB in 16 pairs, us drawn and in three launches: rows of
// 55 KiB (28000 in bf16) 232 and 201, 78 KiB 209 and 203, 94 KiB 199 and 205, 98 KiB 198 and
// 206, 125 KiB 190 and 205; in fp32, of half as many logits, 62 KiB 195 and 198, 94 KiB 188
// and 203, 109 KiB 185 and 205.
static bool streams(size_t rows, size_t vocab, int dtype) {
    const size_t row = vocab * dtype_size(dtype);
    return row >= (size_t)96 << 10 && rows * row > (size_t)256 << 20;
}
// Whether the preference loss takes the launch that draws rows (see there): for such logits
// of pairs that the cache holds (8000 x 50257 in bf16, 30 % of the rows without weight: 4
// pairs 302 us against 340, 3 pairs 320 against 341, 2 pairs 344 against 345, one 382 against
// 352; all with weight: 409 against 425, 411 and 425, 420 and 428), and for a few short rows,
// where two launches instead of three count (45 x 32000 in bf16 18.0 us against 21.4; 256
// rows 22.7 against 21.3, 45 x 128000 in fp32 33 against 31).
static bool draws(size_t rows, size_t pairs, size_t vocab, int dtype) {
    const size_t all = rows * vocab * dtype_size(dtype);
    return streams(rows, vocab, dtype) ? pairs != 0 && all / pairs <= (size_t)256 << 20
                                       : rows <= 128 && all <= (size_t)16 << 20;
}
// LDS that nobody uses: over half of a compute unit's, so that it has one workgroup, where the
// rows in flight would else be as much as the cache (32 pairs of 2048 x 128000 in fp32 411 us,
// 432 with two; in bf16 187 with either, of 4100 x 50257 219 with one and 179 with two).
static unsigned draw_lds(size_t vocab, int dtype) {
    return vocab * dtype_size(dtype) > (size_t)256 << 10 ? 84 << 10 : 0;
}
constexpr size_t kInFlight = (size_t)64 << 20;  // logits between a workgroup's two rows

// Workgroups of the pairs' launch: as many at most as run at once with room to spare, since
// each looks through the offsets before its own (131072 rows of 200 in bf16, 65536 pairs: 243
// us with 1024 workgroups, 264 with 512, 252 with 2048, 1140 with one to a pair; 16384 x 1000,
// 8192 pairs: 40.8, 43.0, 43.2, 61.8).
constexpr size_t kPairGroups = 1024;

// The preference loss's scratch, of either kind.
static size_t preference_scratch(size_t rows) {
    return sizeof(Plan) + (rows + 1) * sizeof(uint64_t) + rows * (sizeof(PairInfo) + sizeof(int));
}
constexpr size_t kMaxPrefRows = (size_t)1 << 30;  // they are drawn in 32 bits

// Threads for a row that is streamed: four vectors each, and enough for a pair's sums.
static unsigned stream_threads(size_t vocab, int dtype) {
    const size_t t = (vocab / (64 / dtype_size(dtype)) + kWave - 1) / kWave * kWave;
    return (unsigned)(t < NT ? NT : t > kMaxThreads ? kMaxThreads : t);
}

}  // namespace tl
}  // namespace efla

using namespace efla;

extern "C" int token_logprob_forward_hip(const void* logits, const int32_t* targets,
                                         const float* weights, float* logp, size_t rows,
                                         size_t vocab_size, size_t ld, int dtype,
                                         hipStream_t stream) {
    if (rows == 0) return kSuccess;
    const int rc = tl::check(logits, targets, nullptr, rows, vocab_size, ld, 0, dtype);
    if (rc != kSuccess) return rc;
    if (!logp) return kInvalidValue;
    return tl::logprob(logits, targets, weights, logp, nullptr, nullptr, rows, vocab_size, ld,
                       dtype, tl::logprob_form(vocab_size, dtype),
                       tl::past_cache(rows, vocab_size, dtype), stream);
}

extern "C" int policy_loss_forward_backward_hip(
    const void* logits, const int32_t* targets, const float* advantages, const float* old_logp,
    const float* ref_logp, const float* weights, float* loss, float* logp, float* kl,
    void* grad_logits, size_t rows, size_t vocab_size, size_t ld, size_t ld_grad, float clip_low,
    float clip_high, float kl_coef, int dtype, hipStream_t stream) {
    if (rows == 0) return kSuccess;
    const int rc =
        tl::check(logits, targets, grad_logits, rows, vocab_size, ld, ld_grad, dtype);
    if (rc != kSuccess) return rc;
    if (!advantages || !loss || !logp) return kInvalidValue;
    if (!(clip_low >= 0.f && clip_low <= 1.f) || !(clip_high >= 0.f)) return kInvalidValue;
    if (!(kl_coef >= 0.f && kl_coef < INFINITY)) return kInvalidValue;
    if (!ref_logp && (kl_coef != 0.f || kl)) return kInvalidValue;
    tl::PolicyArgs a;
    a.targets = targets;
    a.adv = advantages, a.old = old_logp, a.ref = ref_logp, a.weights = weights;
    a.loss = loss, a.logp = logp, a.kl = kl;
    a.rows = (long)rows, a.V = (int)vocab_size, a.ld = (long)ld, a.ldg = (long)ld_grad;
    a.low = 1.f - clip_low, a.high = 1.f + clip_high, a.kl_coef = kl_coef;
    a.even = 1.f / (float)rows;
    const tl::Form f = tl::policy_form(vocab_size, dtype);
    TL_TYPED(dtype, T, {
        TL_POLICY_FORM(f, NV, {
            TL_IF(tl::past_cache(rows, vocab_size, dtype), PAST, {
                EFLA_LAUNCH("policy_loss", (tl::policy_kernel<T, NV, PAST>), tl::row_grid(rows),
                            dim3(f.threads), stream, (const T*)logits, (T*)grad_logits, a);
            });
        });
    });
    return (int)hipPeekAtLastError();
}

extern "C" size_t preference_loss_workspace_size(size_t rows) {
    return rows > tl::kMaxPrefRows ? 0 : tl::preference_scratch(rows);
}

extern "C" int preference_loss_forward_backward_hip(
    const void* logits, const int32_t* targets, const float* ref_logp, const float* weights,
    const int32_t* cu_seqlens, float* loss, float* rewards, float* logp, void* grad_logits,
    size_t pairs, size_t rows, size_t vocab_size, size_t ld, size_t ld_grad, float beta,
    float label_smoothing, int dtype, void* workspace, size_t workspace_bytes,
    hipStream_t stream) {
    if (pairs == 0 && rows == 0) return kSuccess;
    if (rows != 0) {
        const int rc =
            tl::check(logits, targets, grad_logits, rows, vocab_size, ld, ld_grad, dtype);
        if (rc != kSuccess) return rc;
        if (!logp) return kInvalidValue;
    } else if (tl::dtype_size(dtype) == 0) {
        return kInvalidValue;
    }
    if (!(beta > 0.f && beta < INFINITY) || !(label_smoothing >= 0.f && label_smoothing < 1.f))
        return kInvalidValue;
    if (pairs != 0 && (!cu_seqlens || !loss || !rewards)) return kInvalidValue;
    if (pairs > 0x3FFFFFFFull || rows > tl::kMaxPrefRows) return kInvalidConfiguration;
    const size_t need = tl::preference_scratch(rows);
    void* ws = workspace;
    WsLease lease;
    if (!grad_logits) {
        ws = nullptr;
    } else if (!workspace) {
        const int rc = workspace_acquire(need, stream, &ws, lease);
        if (rc != kSuccess) return rc;
    } else if (workspace_bytes < need || (uintptr_t)workspace % 16) {
        return kInvalidValue;
    }
    const float inv_pairs = pairs ? 1.f / (float)pairs : 0.f;
    const unsigned threads = tl::stream_threads(vocab_size, dtype);
    const bool draws = rows != 0 && tl::draws(rows, pairs, vocab_size, dtype);
    if (draws && grad_logits) {
        tl::PrefArgs a;
        a.targets = targets, a.cu = cu_seqlens, a.ref = ref_logp, a.weights = weights;
        a.loss = loss, a.rewards = rewards, a.logp = logp;
        a.plan = (tl::Plan*)ws;
        a.stat = (uint64_t*)(a.plan + 1);
        a.info = (tl::PairInfo*)(a.stat + rows + (rows & 1));
        a.first = (int*)(a.info + rows);
        a.ld = (long)ld, a.ldg = (long)ld_grad;
        a.rows = (int)rows, a.pairs = (int)pairs, a.V = (int)vocab_size;
        a.slack = (int)(tl::kInFlight / (vocab_size * tl::dtype_size(dtype)));
        a.beta = beta, a.eps = label_smoothing, a.inv_pairs = inv_pairs;
        const size_t fill = (rows + 4 * tl::kPlanThreads - 1) / (4 * tl::kPlanThreads);
        EFLA_LAUNCH("preference_plan", tl::plan_kernel, dim3((unsigned)(1 + (fill < 64 ? fill : 64))),
                    dim3(tl::kPlanThreads), stream, a);
        const int rc = (int)hipPeekAtLastError();
        if (rc != kSuccess) return rc;
        // the lag is known on the device: as many as it may take
        TL_TYPED(dtype, T, {
            TL_IF(tl::past_cache(rows, vocab_size, dtype), PAST, {
                EFLA_LAUNCH_LDS("preference_loss", (tl::preference_kernel<T, PAST>),
                                tl::row_grid(2 * rows), dim3(threads),
                                tl::draw_lds(vocab_size, dtype), stream, (const T*)logits,
                                (T*)grad_logits, a);
            });
        });
        return (int)hipPeekAtLastError();
    }
    float2* stat = (float2*)ws;
    float* coef = stat ? (float*)(stat + rows) : nullptr;
    if (rows != 0) {
        // the same sums as where rows are drawn, so that these do not depend on the gradient
        const tl::Form f = draws || tl::streams(rows, vocab_size, dtype)
                               ? tl::Form{0, threads}
                               : tl::logprob_form(vocab_size, dtype);
        const int rc = tl::logprob(logits, targets, weights, logp, stat, coef, rows, vocab_size,
                                   ld, dtype, f, false, stream);
        if (rc != kSuccess) return rc;
    }
    if (pairs != 0) {
        const size_t each = (pairs + tl::kPairGroups - 1) / tl::kPairGroups;
        TL_IF(each > 1, MANY, {
            EFLA_LAUNCH("preference_pairs", tl::pair_kernel<MANY>,
                        dim3((unsigned)((pairs + each - 1) / each)), dim3(tl::NT), stream,
                        cu_seqlens, logp, ref_logp, weights, (int)rows, (int)pairs, (int)each,
                        beta, label_smoothing, inv_pairs, loss, rewards, coef);
        });
        const int rc = (int)hipPeekAtLastError();
        if (rc != kSuccess) return rc;
    }
    if (grad_logits && rows != 0) {
        TL_TYPED(dtype, T, {
            TL_IF(tl::past_cache(rows, vocab_size, dtype), PAST, {
                EFLA_LAUNCH("preference_grad", (tl::grad_kernel<T, PAST>), tl::row_grid((rows + 7) & ~(size_t)7),
                            dim3(threads), stream, (const T*)logits, (T*)grad_logits, targets,
                            stat, coef, (long)rows, (int)vocab_size, (long)ld, (long)ld_grad);
            });
        });
    }
    return (int)hipPeekAtLastError();
}

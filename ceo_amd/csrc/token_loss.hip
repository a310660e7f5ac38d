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
#include <hip/hip_runtime.h>
#include <math.h>

#include "../../include/efla_hip.h"
#include "common.hpp"
#include "internal.hpp"

namespace efla {
namespace tl {

constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.69314718055994530942;

// 16 bytes of logits, at any multiple of the element's size
template <typename T>
struct Vec {
    static constexpr int N = 16 / sizeof(T);
    typedef __attribute__((__vector_size__(16))) T Full;
    typedef Full Any __attribute__((aligned(sizeof(T))));
    static __device__ __forceinline__ Full load(const T* p) {
        return *reinterpret_cast<const Any*>(p);
    }
    static __device__ __forceinline__ void store(T* p, Full v) { *reinterpret_cast<Any*>(p) = v; }
};

// e^d for d <= 0 (one rounding of d log2 e, one v_exp_f32)
__device__ __forceinline__ float exp_neg(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

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

template <int NT>
__device__ __forceinline__ Stat join_all(Stat a, Stat* sm) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) join(a, __shfl_xor(a.m, off), __shfl_xor(a.s, off));
    if constexpr (NT > kWave) {
        if (lane_id() == 0) sm[wave_id()] = a;
        __syncthreads();
        a = sm[0];
#pragma unroll
        for (int k = 1; k < NT / kWave; ++k) join(a, sm[k].m, sm[k].s);
    }
    return a;
}

// One pass over a row's logits: each thread its part, block by block.
template <typename T, int NT>
__device__ __forceinline__ Stat row_stat(const T* z, long V, Stat* sm) {
    constexpr int N = Vec<T>::N;
    Stat a{-INFINITY, 0.f};
    const long nv = V / N;
    for (long c = threadIdx.x; c < nv; c += NT) {
        const typename Vec<T>::Full x = Vec<T>::load(z + c * N);
        float m = a.m;
#pragma unroll
        for (int i = 0; i < N; ++i) m = fmaxf(m, (float)x[i]);
        const float r = ref_of(m);
        float s = a.s * exp_neg(a.m - r);
#pragma unroll
        for (int i = 0; i < N; ++i) s += exp_neg((float)x[i] - r);
        a = Stat{m, s};
    }
    const long c = nv * N + threadIdx.x;
    if (c < V) join(a, (float)z[c], (float)z[c] == -INFINITY ? 0.f : 1.f);
    return join_all<NT>(a, sm);
}

__device__ __forceinline__ double logp_of(const Stat& a, float zt) {
    return (double)(zt - a.m) - log_of(a.s);
}

// d loss / d z over one row: coef ([j = t] - e^(z_j - m) / s)
template <typename T, int NT>
__device__ __forceinline__ void row_grad(const T* z, T* g, long V, long t, const Stat& a,
                                         float coef, long first, long step) {
    constexpr int N = Vec<T>::N;
    const float k = -coef / a.s, r = ref_of(a.m);
    const long nv = V / N;
    for (long c = first; c < nv; c += step) {
        const typename Vec<T>::Full x = Vec<T>::load(z + c * N);
        typename Vec<T>::Full y;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float d = k * exp_neg((float)x[i] - r);
            if (c * N + i == t) d += coef;
            y[i] = (T)d;
        }
        Vec<T>::store(g + c * N, y);
    }
    const long c = nv * N + first;
    if (c < V) {
        float d = k * exp_neg((float)z[c] - r);
        if (c == t) d += coef;
        g[c] = (T)d;
    }
}

template <typename T>
__device__ __forceinline__ void row_zero(T* g, long V, long first, long step) {
    constexpr int N = Vec<T>::N;
    const typename Vec<T>::Full zero = {};
    const long nv = V / N;
    for (long c = first; c < nv; c += step) Vec<T>::store(g + c * N, zero);
    const long c = nv * N + first;
    if (c < V) g[c] = (T)0.f;
}

constexpr int NT = 256;

template <typename T>
__global__ void __launch_bounds__(NT)
logprob_kernel(const T* __restrict__ logits, const int32_t* __restrict__ targets,
               const float* __restrict__ weights, float* __restrict__ logp, float2* stat,
               float* coef, long V, long ld) {
    __shared__ Stat sm[NT / kWave];
    const long row = blockIdx.x;
    // rows outside of every sequence keep this coefficient
    if (coef && threadIdx.x == 0) coef[row] = 0.f;
    if (weights && weights[row] == 0.f) {
        if (threadIdx.x == 0) logp[row] = 0.f;
        return;
    }
    const T* z = logits + row * ld;
    const long t = targets[row];
    const Stat a = row_stat<T, NT>(z, V, sm);
    if (threadIdx.x == 0) {
        logp[row] = t >= 0 && t < V ? (float)logp_of(a, (float)z[t]) : NAN;
        if (stat) stat[row] = float2{a.m, a.s};
    }
}

struct PolicyArgs {
    const int32_t* targets;
    const float *adv, *old, *ref, *weights;
    float *loss, *logp, *kl;
    long rows, V, ld, ldg;
    float low, high, kl_coef, even;  // even: the weight of a row where there are none
};

template <typename T>
__global__ void __launch_bounds__(NT) policy_kernel(const T* logits, T* grad, PolicyArgs a) {
    __shared__ Stat sm[NT / kWave];
    const long row = blockIdx.x;
    const float w = a.weights ? a.weights[row] : a.even;
    T* g = grad ? grad + row * a.ldg : nullptr;
    if (w == 0.f) {
        if (threadIdx.x == 0) {
            a.loss[row] = 0.f;
            a.logp[row] = 0.f;
            if (a.kl) a.kl[row] = 0.f;
        }
        if (g) row_zero(g, a.V, threadIdx.x, NT);
        return;
    }
    const T* z = logits + row * a.ld;
    const long t = a.targets[row];
    const bool tok = t >= 0 && t < a.V;
    const float zt = tok ? (float)z[t] : 0.f;  // read before the gradient may overwrite it
    const Stat st = row_stat<T, NT>(z, a.V, sm);
    const double lp = logp_of(st, zt);
    const float adv = a.adv[row];
    const float r = a.old ? expf((float)(lp - (double)a.old[row])) : 1.f;
    const float rc = fminf(fmaxf(r, a.low), a.high);
    float l = -fminf(r * adv, rc * adv);
    float d = (adv >= 0.f ? r <= a.high : r >= a.low) ? -adv * r : 0.f;
    float kl = 0.f;
    if (a.ref) {
        const float x = (float)((double)a.ref[row] - lp);
        const float em = expm1f(x);
        kl = em - x;
        if (a.kl_coef != 0.f) {
            l += a.kl_coef * kl;
            d -= a.kl_coef * em;
        }
    }
    if (threadIdx.x == 0) {
        a.loss[row] = tok ? w * l : NAN;
        a.logp[row] = tok ? (float)lp : NAN;
        if (a.kl) a.kl[row] = tok ? kl : NAN;
    }
    if (g) {
        if (tok)
            row_grad<T, NT>(z, g, a.V, t, st, w * d, threadIdx.x, NT);
        else
            row_zero(g, a.V, threadIdx.x, NT);
    }
}

// One pair of sequences: their sums, the pair's loss, and each row's coefficient.
__global__ void __launch_bounds__(NT)
pair_kernel(const int32_t* __restrict__ cu, const float* __restrict__ logp,
            const float* __restrict__ ref, const float* __restrict__ weights, long rows,
            float beta, float eps, float inv_pairs, float* __restrict__ loss,
            float* __restrict__ rewards, float* __restrict__ coef) {
    __shared__ double sm[2][NT / kWave];
    const long pair = blockIdx.x;
    long at[3];
    long low = 0;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const long c = cu[2 * pair + i];
        low = c < low ? low : c > rows ? rows : c;
        at[i] = low;
    }
    double sum[2] = {0.0, 0.0};
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        for (long i = at[q] + threadIdx.x; i < at[q + 1]; i += NT) {
            const float w = weights ? weights[i] : 1.f;
            if (w != 0.f) sum[q] += (double)w * ((double)logp[i] - (ref ? (double)ref[i] : 0.0));
        }
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) sum[q] += __shfl_xor(sum[q], off);
        if (lane_id() == 0) sm[q][wave_id()] = sum[q];
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        sum[q] = sm[q][0];
#pragma unroll
        for (int k = 1; k < NT / kWave; ++k) sum[q] += sm[q][k];
    }
    const double x = (double)beta * (sum[0] - sum[1]);
    const double u = exp(-fabs(x));            // e^-|x|
    const double lg = log1p(u);                // log sig(-|x|) = -|x| - lg
    const double plus = lg + fmax(-x, 0.0);    // -log sig(x)
    const double minus = lg + fmax(x, 0.0);    // -log sig(-x)
    const double sig = x >= 0 ? 1.0 / (1.0 + u) : u / (1.0 + u);
    const double gis = x >= 0 ? u / (1.0 + u) : 1.0 / (1.0 + u);  // sig(-x)
    const double dx = ((double)eps * sig - (1.0 - (double)eps) * gis) * (double)inv_pairs;
    if (threadIdx.x == 0) {
        loss[pair] = (float)(((1.0 - (double)eps) * plus + (double)eps * minus) * (double)inv_pairs);
        rewards[2 * pair] = (float)((double)beta * sum[0]);
        rewards[2 * pair + 1] = (float)((double)beta * sum[1]);
    }
    if (coef) {
        const float c = (float)((double)beta * dx);
        for (long i = at[0] + threadIdx.x; i < at[2]; i += NT)
            coef[i] = (i < at[1] ? c : -c) * (weights ? weights[i] : 1.f);
    }
}

template <typename T>
__global__ void __launch_bounds__(NT)
grad_kernel(const T* logits, T* grad, const int32_t* __restrict__ targets,
            const float* __restrict__ weights, const float2* __restrict__ stat,
            const float* __restrict__ coef, long V, long ld, long ldg) {
    const long row = blockIdx.x;
    T* g = grad + row * ldg;
    const long t = targets[row];
    if ((weights && weights[row] == 0.f) || t < 0 || t >= V) {
        row_zero(g, V, threadIdx.x, NT);
        return;
    }
    row_grad<T, NT>(logits + row * ld, g, V, t, Stat{stat[row].x, stat[row].y}, coef[row],
                    threadIdx.x, NT);
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

static int logprob(const void* logits, const int32_t* targets, const float* weights, float* logp,
                   float2* stat, float* coef, size_t rows, size_t vocab, size_t ld, int dtype,
                   hipStream_t st) {
    TL_TYPED(dtype, T, {
        EFLA_LAUNCH("token_logprob", (logprob_kernel<T>), dim3((unsigned)rows), dim3(NT), st,
                    (const T*)logits, targets, weights, logp, stat, coef, (long)vocab, (long)ld);
    });
    return (int)hipPeekAtLastError();
}

// The preference loss's scratch: the rows' statistics and coefficients.
static size_t preference_scratch(size_t rows) { return rows * (sizeof(float2) + sizeof(float)); }

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
                       dtype, stream);
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
    a.rows = (long)rows, a.V = (long)vocab_size, a.ld = (long)ld, a.ldg = (long)ld_grad;
    a.low = 1.f - clip_low, a.high = 1.f + clip_high, a.kl_coef = kl_coef;
    a.even = 1.f / (float)rows;
    TL_TYPED(dtype, T, {
        EFLA_LAUNCH("policy_loss", (tl::policy_kernel<T>), dim3((unsigned)rows), dim3(tl::NT),
                    stream, (const T*)logits, (T*)grad_logits, a);
    });
    return (int)hipPeekAtLastError();
}

extern "C" size_t preference_loss_workspace_size(size_t rows) {
    return rows > 0x7FFFFFFFull ? 0 : tl::preference_scratch(rows);
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
    }
    if (!(beta > 0.f && beta < INFINITY) || !(label_smoothing >= 0.f && label_smoothing < 1.f))
        return kInvalidValue;
    if (pairs != 0 && (!cu_seqlens || !loss || !rewards)) return kInvalidValue;
    if (pairs > 0x3FFFFFFFull) return kInvalidConfiguration;
    const size_t need = tl::preference_scratch(rows);
    float2* stat = (float2*)workspace;
    WsLease lease;
    if (!grad_logits) {
        stat = nullptr;
    } else if (!workspace) {
        const int rc = workspace_acquire(need, stream, (void**)&stat, lease);
        if (rc != kSuccess) return rc;
    } else if (workspace_bytes < need || (uintptr_t)workspace % 16) {
        return kInvalidValue;
    }
    float* coef = stat ? (float*)(stat + rows) : nullptr;
    if (rows != 0) {
        const int rc = tl::logprob(logits, targets, weights, logp, stat, coef, rows, vocab_size,
                                   ld, dtype, stream);
        if (rc != kSuccess) return rc;
    }
    if (pairs != 0) {
        EFLA_LAUNCH("preference_pairs", tl::pair_kernel, dim3((unsigned)pairs), dim3(tl::NT),
                    stream, cu_seqlens, logp, ref_logp, weights, (long)rows, beta,
                    label_smoothing, 1.f / (float)pairs, loss, rewards, coef);
        const int rc = (int)hipPeekAtLastError();
        if (rc != kSuccess) return rc;
    }
    if (grad_logits && rows != 0) {
        TL_TYPED(dtype, T, {
            EFLA_LAUNCH("preference_grad", (tl::grad_kernel<T>), dim3((unsigned)rows),
                        dim3(tl::NT), stream, (const T*)logits, (T*)grad_logits, targets, weights,
                        stat, coef, (long)vocab_size, (long)ld, (long)ld_grad);
        });
    }
    return (int)hipPeekAtLastError();
}

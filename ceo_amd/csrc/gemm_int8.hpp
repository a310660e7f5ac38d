// Products in 8-bit integers with a scale for each token and channel, for gfx950
// (included by gemm_int8.hip).
//
//   sx_m = max_k |x_mk| / 127, qx_mk = x_mk / sx_m to the nearest whole number (ties to even)
//   sw_n, qw_kn the same over the columns of the weight, once, when it is packed
//   y_mn = act((sum_k qx_mk qw_kn) sx_m sw_n + bias_n) + residual_mn, rounded once
//
// The sums are whole and exact (k <= 131072: below 2^31), so nothing depends on how they
// are split.  A packed weight is one row of whole 128-byte lines per channel, zero
// behind k, after the scales; quantised tokens are rows of the same length.
#pragma once
#include "common.hpp"
#include "gemm_fast.hpp"

namespace efla {
namespace i8 {

typedef __attribute__((__vector_size__(4 * sizeof(int)))) int int4v;
typedef __attribute__((__vector_size__(16 * sizeof(int)))) int int16v;

constexpr long kLine = 128;
inline __host__ __device__ long up_to(long x, long m) { return (x + m - 1) / m * m; }

// --- quantising -----------------------------------------------------------------
// A row's (column's) scale from its largest magnitude.  NaN where that is not finite: the
// row's products are NaN then.
__device__ __forceinline__ float scale_of(float amax) {
    return amax < INFINITY ? amax / 127.f : NAN;
}

// x / scale to the nearest whole number, ties to even, as an exact quotient would round:
// eight of them, a byte each.  A fused multiply and add of 1.5 2^23 rounds x inv to a whole
// number that its low byte holds.  inv is 1 / scale rounded, so x inv is off by 127 * 2^-23 at
// most, and the whole number by one at most, next to a half: what lies within 2^-14 of one
// (one vector in sixty) is looked at again.  There x - r scale, which one fused operation gives
// without rounding (x and scale have 24 bits, r 7, and the difference is below scale),
// says on which side of the half x lies.
// A row of zeros, or one that holds NaN or an infinity, has inv 0: 0 everywhere.
struct Quantizer {
    float scale, inv;
    __device__ __forceinline__ explicit Quantizer(float s)
        : scale(s), inv(s > 0.f ? 1.f / s : 0.f) {}
    template <typename Vec>
    __device__ __forceinline__ uint2 operator()(const Vec& x) const {
        constexpr float kRound = 12582912.f;
        float v[8], t[8], far = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[e] = (float)x[e];
            t[e] = fmaf(v[e], inv, kRound);
            far = fmaxf(far, fabsf(fmaf(v[e], inv, kRound - t[e])));
        }
        if (far > 0.5f - 0x1p-14f) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float d = fmaf(kRound - t[e], scale, v[e]), a = fabsf(d), h = 0.5f * scale;
                const bool odd = __float_as_uint(t[e]) & 1;
                t[e] += a > h || (a == h && odd) ? copysignf(1.f, d) : 0.f;
            }
        }
        auto four = [&](int e) {
            const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(t[e + 1]), __float_as_uint(t[e]),
                                                      0x0C0C0400u);
            return lo | __builtin_amdgcn_perm(__float_as_uint(t[e + 3]), __float_as_uint(t[e + 2]),
                                              0x04000C0Cu);
        };
        return make_uint2(four(0), four(4));
    }
};

// The larger magnitude, NaN if either is: magnitudes are compared as whole numbers, in
// which NaN is above infinity.
__device__ __forceinline__ float amax2(float a, float x) {
    return __uint_as_float(max(__float_as_uint(a), __float_as_uint(x) & 0x7FFFFFFFu));
}
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xF,
                                                               0xF, true));
}
// over N = 16, 32 or 64 neighbouring lanes, in each of them
template <int N>
__device__ __forceinline__ float lanes_amax(float m) {
    m = amax2(m, dpp<0xB1>(m));   // quad_perm [1, 0, 3, 2]
    m = amax2(m, dpp<0x4E>(m));   // quad_perm [2, 3, 0, 1]
    m = amax2(m, dpp<0x141>(m));  // row_half_mirror
    m = amax2(m, dpp<0x140>(m));  // row_mirror
    if constexpr (N > 16) m = amax2(m, __shfl_xor(m, 16));
    if constexpr (N > 32) m = amax2(m, __shfl_xor(m, 32));
    return m;
}
// The largest magnitude of vectors of 8, two 16-bit ones at a time
template <typename T>
struct Amax {
    typedef typename gf::Piece<8, T>::vec Vec;
    typedef __attribute__((__vector_size__(8 * sizeof(uint16_t)))) uint16_t U8;
    U8 m{};
    __device__ __forceinline__ void add(Vec x) {
        const U8 b = __builtin_bit_cast(U8, x) & (uint16_t)0x7FFF;
        m = __builtin_elementwise_max(m, b);
    }
    __device__ __forceinline__ float get() const {
        uint16_t t = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) t = t > m[e] ? t : m[e];
        return (float)__builtin_bit_cast(T, t);
    }
};
template <>
struct Amax<float> {
    typedef gf::Piece<8, float>::vec Vec;
    float m = 0.f;
    __device__ __forceinline__ void add(Vec x) {
#pragma unroll
        for (int e = 0; e < 8; ++e) m = amax2(m, x[e]);
    }
    __device__ __forceinline__ float get() const { return m; }
};

// A row of k elements in LPR threads (lr: this one's place), the first 8 LPR HOLD of them in
// registers.  Whole vectors and the last, partial one are loaded apart: a vector that may be
// put together from elements is taken apart where its two ways meet, and that waits for
// its load (a row of 4096 in one wave: 8 loads one by one, 9.5 us; 4.2 together).
template <typename T, int LPR, int HOLD>
struct Row {
    typedef gf::Piece<8, T> P8;
    typedef typename P8::vec Vec;
    static constexpr long kHeld = 8L * LPR * HOLD;
    Vec v[HOLD], last;
    __device__ __forceinline__ static Vec at(const T* x, long c, long k) {  // whole, or zero
        Vec y{};
        if (c + 8 <= k) y = *reinterpret_cast<const typename P8::uvec*>(x + c);
        return y;
    }
    __device__ __forceinline__ void load(const T* x, long k, int lr) {
#pragma unroll
        for (int i = 0; i < HOLD; ++i) v[i] = at(x, 8 * (lr + LPR * i), k);
        last = Vec{};
        if (k % 8 && lr == k / 8 % LPR) {
#pragma unroll
            for (int e = 0; e < 7; ++e)
                if (e < k % 8) last[e] = x[k / 8 * 8 + e];
        }
    }
    __device__ __forceinline__ float amax(const T* x, long k, int lr) const {  // of this thread's
        Amax<T> m;
#pragma unroll
        for (int i = 0; i < HOLD; ++i) m.add(v[i]);
        m.add(last);
        for (long c = kHeld + 8 * lr; c < k; c += 8 * LPR) m.add(at(x, c, k));
        return m.get();
    }
    // q: kp bytes, zero behind k
    __device__ __forceinline__ void store(const T* x, long k, long kp, int lr, float scale,
                                          uint8_t* q) {
        // Below the normal range's reciprocals (never in fp16) everything is taken 2^64 times as
        // large, which is exact.  A scale with few bits may leave more than 127 steps: cut off.
        if (scale < 0x1p-100f && scale > 0.f) {
            const float s = scale;
            auto up = [&](Vec& y) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    y[e] = (T)(fminf(fmaxf((float)y[e], -127.f * s), 127.f * s) * 0x1p64f);
            };
#pragma unroll
            for (int i = 0; i < HOLD; ++i) up(v[i]);
            up(last);
            const Quantizer qz(s * 0x1p64f);
            for (long c = kHeld + 8 * lr; c < kp; c += 8 * LPR) {
                Vec y = at(x, c, k);
                up(y);
                *reinterpret_cast<uint2*>(q + c) = qz(y);
            }
            scale *= 0x1p64f;
            kp = kp < kHeld ? kp : kHeld;
        }
        const Quantizer qz(scale);
#pragma unroll
        for (int i = 0; i < HOLD; ++i) {
            const long c = 8 * (lr + LPR * i);
            if (c < kp) *reinterpret_cast<uint2*>(q + c) = qz(v[i]);
        }
        for (long c = kHeld + 8 * lr; c < kp; c += 8 * LPR)
            *reinterpret_cast<uint2*>(q + c) = qz(at(x, c, k));
        if (k % 8 && lr == k / 8 % LPR) *reinterpret_cast<uint2*>(q + k / 8 * 8) = qz(last);
    }
};

// LPR threads to a row: a wave, four rows to a workgroup, or (few rows) the whole workgroup,
// where one wave's chain of instructions is what a row takes.  Bound by memory.
template <typename T, int LPR, int HOLD>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* __restrict__ x, long ldx,
                                                            long m, long k, long kp,
                                                            uint8_t* __restrict__ q,
                                                            float* __restrict__ scales) {
    __shared__ float part[4];
    const long row = LPR == 64 ? (long)blockIdx.x * 4 + wave_id() : (long)blockIdx.x;
    const int lr = threadIdx.x & (LPR - 1);
    if (row >= m) return;  // whole waves; never where the workgroup shares a row
    x += row * ldx;
    Row<T, LPR, HOLD> r;
    r.load(x, k, lr);
    float a = lanes_amax<64>(r.amax(x, k, lr));
    if constexpr (LPR == 256) {
        if (lane_id() == 0) part[wave_id()] = a;
        __syncthreads();
        a = amax2(amax2(part[0], part[1]), amax2(part[2], part[3]));
    }
    const float s = scale_of(a);
    r.store(x, k, kp, lr, s, q + row * kp);
    if (lr == 0) scales[row] = s;
}

// Columns' largest magnitudes, as whole numbers, into amax (zero before).
template <typename T>
__global__ void __launch_bounds__(256) column_amax_kernel(const T* __restrict__ w, long ld, long k,
                                                          long n, uint32_t* __restrict__ amax) {
    const long c = (long)blockIdx.x * 256 + threadIdx.x;
    if (c >= n) return;
    float m = 0.f;
    for (long r = blockIdx.y; r < k; r += gridDim.y) m = amax2(m, to_f(w[r * ld + c]));
    atomicMax(amax + c, __float_as_uint(m));
}

// 64 x 64 tiles of the weight, turned through LDS and quantised: a row of q per channel.
template <typename T>
__global__ void __launch_bounds__(256) pack_weight_kernel(const T* __restrict__ w, long ld, long k,
                                                          long n, long kp,
                                                          const uint32_t* __restrict__ amax,
                                                          uint8_t* __restrict__ q) {
    __shared__ float tile[64][65];
    const int c = threadIdx.x & 63, r0 = threadIdx.x >> 6;
    const long n0 = (long)blockIdx.x * 64;
    for (long k0 = (long)blockIdx.y * 64; k0 < kp; k0 += (long)gridDim.y * 64) {
        for (int r = r0; r < 64; r += 4)
            tile[r][c] = n0 + c < n && k0 + r < k ? to_f(w[(k0 + r) * ld + n0 + c]) : 0.f;
        __syncthreads();
        // a row of 64 in 8 threads
        for (int i = threadIdx.x; i < 512; i += 256) {
            const long col = n0 + (i >> 3);
            if (col >= n) continue;
            float s = scale_of(__uint_as_float(amax[col]));
            const bool tiny = s < 0x1p-100f;  // as in Row::store
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = tile[8 * (i & 7) + e][i >> 3];
                if (tiny) v[e] = fminf(fmaxf(v[e], -127.f * s), 127.f * s) * 0x1p64f;
            }
            const Quantizer qz(tiny ? s * 0x1p64f : s);
            *reinterpret_cast<uint2*>(q + col * kp + k0 + 8 * (i & 7)) = qz(v);
        }
        __syncthreads();
    }
}

__global__ void __launch_bounds__(256) column_scales_kernel(uint32_t* __restrict__ amax, long n) {
    const long c = (long)blockIdx.x * 256 + threadIdx.x;
    if (c < n) reinterpret_cast<float*>(amax)[c] = scale_of(__uint_as_float(amax[c]));
}

// --- epilogue -----------------------------------------------------------------------
template <typename T>
struct Out {
    T* y;
    long ldy;
    const T* bias;      // [n] or NULL
    const T* residual;  // or NULL
    long ldr;
    const float* sw;
    int gelu;
};

// acc sx sw + bias.  A token of values near the type's largest: acc sx may pass fp32's range
// where the weights are small, so it is taken 2^-64 times as large (acc is below 2^31).
template <typename T, typename Acc, typename Sw, typename Bias, int N>
__device__ __forceinline__ void scaled(float (&v)[N], const Acc& acc, float sx, const Sw& sw,
                                       const Bias& bias) {
    if (!__is_same(T, f16) && __builtin_expect(sx > 0x1p96f, 0)) {
#pragma unroll
        for (int e = 0; e < N; ++e)
            v[e] = fmaf((float)acc[e] * (sx * 0x1p-64f) * sw[e], 0x1p64f, (float)bias[e]);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] = fmaf((float)acc[e] * sx, sw[e], (float)bias[e]);
    }
}

// --- few rows -------------------------------------------------------------------------
// M <= 16 MT rows.  Bound by the weight, which is read once.  A wave takes 16 channels and
// a range of k; the weights are the MFMA's A operand (16 x 16 x 64), read straight from
// memory, 16 bytes a lane.  kw waves of a workgroup share their channels and split k; their
// sums meet in LDS.  HOLD > 0: the workgroup quantises the tokens into LDS itself, all rows at
// once, LPR lanes to a row (8 HOLD elements of each lane in registers).  Loads return in
// the order in which they are issued, so the tokens are asked for before the weights and
// quantised while those are on their way, and what the epilogue needs right behind.  HOLD 0:
// the tokens are read quantised (32 channels a wave, so that they are read half as often: 48 x 4096
// x 1024 16.1 us, 11.9 with 16).
constexpr int kAhead = 8;  // 64-byte steps of k whose weights a wave has in flight
// waves of a workgroup: enough that 32 lanes have a row
template <int MT, int LPR, int HOLD>
constexpr int kFewWaves = HOLD > 0 && LPR == 32 ? 8 * MT : 8;

template <typename T, int MT, int LPR, int HOLD>
__global__ void __launch_bounds__((64 * kFewWaves<MT, LPR, HOLD>),
                                  sizeof(T) == 2 && HOLD <= 4 ? 4 : 2)
few_kernel(const T* __restrict__ x, long ldx, const uint8_t* __restrict__ xq,
           const float* __restrict__ xs, const uint8_t* __restrict__ wq, int M, int N, long k,
           long kp, int kw, Out<T> o) {
    constexpr bool FUSED = HOLD > 0;
    constexpr int NW = kFewWaves<MT, LPR, HOLD>;
    typedef gf::Piece<4, T> P;
    typedef gf::Piece<4, float> F;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int w = wave_id(), l = lane_id(), r = l & 15, g = l >> 4;
    const int cw = NW / kw, wk = w % kw;
    const long n0 = ((long)blockIdx.x * cw + w / kw) * 16;
    const int steps = (int)(kp / 64), s0 = steps * wk / kw, s1 = steps * (wk + 1) / kw;
    const uint8_t* wp = wq + (n0 + r < N ? n0 + r : N - 1) * kp + 16 * g;
    const int own = threadIdx.x / LPR, lr = threadIdx.x % LPR;
    Row<T, LPR, FUSED ? HOLD : 1> row;
    if constexpr (FUSED) row.load(x + own * ldx, own < M ? k : 0, lr);
    int4v a[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
        const int s = s0 + i < s1 ? s0 + i : s0;
        a[i] = *reinterpret_cast<const int4v*>(wp + 64L * s);
    }
    // lane l ends up with rows 16 t + r, channels n .. n + 3
    const long n = n0 + 4 * g;
    const bool mine = wk == 0 && n < N;
    typename F::vec sw{};
    typename P::vec bias{}, res[MT];
    if (mine) {
        sw = F::load(o.sw + n, N - n);
        if (o.bias) bias = P::load(o.bias + n, N - n);
#pragma unroll
        for (int t = 0; t < MT; ++t)
            if (o.residual && 16 * t + r < M)
                res[t] = P::load(o.residual + (16 * t + r) * o.ldr + n, N - n);
    }
    const long ldq = FUSED ? kp + 16 : kp;
    float* sc = reinterpret_cast<float*>(lds);  // 16 MT scales
    uint8_t* rows = lds + 64 * MT;
    if constexpr (FUSED) {
        const float s = scale_of(lanes_amax<LPR>(row.amax(x, 0, lr)));
        row.store(x, own < M ? k : 0, kp, lr, s, rows + own * ldq);
        if (lr == 0) sc[own] = s;
        __syncthreads();
    }
    int4v acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = int4v{};
    // (64 lanes a row: LDS has 8 rows, whose products rows 8 to 15 repeat)
    const uint8_t* bp[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int m = 16 * t + r;
        bp[t] = (FUSED ? rows + (LPR == 64 ? r & 7 : m) * ldq : xq + (m < M ? m : M - 1) * ldq) +
                16 * g;
    }
    for (int s = s0; s < s1; s += kAhead) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (s + i >= s1) break;
            const int4v wa = a[i];
            if (s + i + kAhead < s1)
                a[i] = *reinterpret_cast<const int4v*>(wp + 64L * (s + i + kAhead));
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const int4v b = *reinterpret_cast<const int4v*>(bp[t] + 64L * (s + i));
                acc[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wa, b, acc[t], 0, 0, 0);
            }
        }
    }
    if (kw > 1) {
        if constexpr (FUSED) __syncthreads();  // the tokens have been read
        int4v* part = reinterpret_cast<int4v*>(rows);
#pragma unroll
        for (int t = 0; t < MT; ++t) part[(w * MT + t) * 64 + l] = acc[t];
        __syncthreads();
        if (wk != 0) return;
        for (int j = 1; j < kw; ++j)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[t] += part[((w + j) * MT + t) * 64 + l];
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int m = 16 * t + r;
        if (m >= M || !mine) continue;
        const float sx = FUSED ? sc[m] : xs[m];
        float v[4];
        scaled<T>(v, acc[t], sx, sw, bias);
        typename P::vec y;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (o.gelu) v[e] = gelu::gelu_f<true>(v[e]);
            if (o.residual) v[e] += (float)res[t][e];
            y[e] = (T)v[e];
        }
        P::store(o.y + m * o.ldy + n, y, N - n);
    }
}

// What the output's pieces are: whole and aligned, of any alignment and length, or whole and
// stored past the L2s (an output that they do not hold takes the operands' place in them).
enum Form { kWhole, kRagged, kPast };

// The epilogue of a lane of tile_kernel, whose 8 columns stay the same over its rows: their
// scales and bias are read once, and four rows' scales and residuals ahead of their use
// (read where they are used, each waited behind its branch).
template <typename T, int FORM>
struct Columns {
    static constexpr bool RAGGED = FORM == kRagged;
    typedef gf::Piece<8, T, RAGGED> P;
    typedef gf::Piece<8, float, RAGGED> F;
    long n, cnt;
    float sw[8], bias[8];
    __device__ __forceinline__ Columns(const Out<T>& o, long n, long N) : n(n), cnt(N - n) {
#pragma unroll
        for (int e = 0; e < 8; ++e) sw[e] = bias[e] = 0.f;
        if (cnt <= 0) return;
        const typename F::vec s = F::load(o.sw + n, cnt);
#pragma unroll
        for (int e = 0; e < 8; ++e) sw[e] = s[e];
        if (!o.bias) return;
        const typename P::vec b = P::load(o.bias + n, cnt);
#pragma unroll
        for (int e = 0; e < 8; ++e) bias[e] = (float)b[e];
    }
    struct Rows {  // rows m0, m0 + 8, + 16, + 24
        float sx[4];
        typename P::vec res[4];
        __device__ __forceinline__ void load(const Out<T>& o, const Columns& c,
                                             const float* __restrict__ xs, long m0, long M) {
#pragma unroll
            for (int s = 0; s < 4; ++s) sx[s] = xs[min(m0 + 8 * s, M - 1)];
            if (!o.residual || c.cnt <= 0) return;
#pragma unroll
            for (int s = 0; s < 4; ++s)
                res[s] = P::load(o.residual + min(m0 + 8 * s, M - 1) * o.ldr + c.n, c.cnt);
        }
    };
    __device__ __forceinline__ void finish(const Out<T>& o, long m, const int (&acc)[8],
                                           const Rows& r, int s) const {
        float v[8];
        scaled<T>(v, acc, r.sx[s], sw, bias);
        if (o.gelu) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = gelu::gelu_f<true>(v[e]);
        }
        if (o.residual) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += (float)r.res[s][e];
        }
        typename P::vec y;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = (T)v[e];
        T* to = o.y + m * o.ldy + n;
        if constexpr (FORM == kPast)
            __builtin_nontemporal_store(y, reinterpret_cast<typename P::vec*>(to));
        else
            P::store(to, y, cnt);
    }
};

// --- many rows ------------------------------------------------------------------------
// The tiles of gemm_fast.hpp with both operands k-contiguous and two 8-bit integers in the
// place of each 16-bit element: 256 x 256 x 128 (eight waves of 128 x 64) or 128 x 128 x 128
// (four of 64 x 64, two workgroups to a CU), copied straight into LDS one block ahead,
// MFMA 32 x 32 x 32.  Rows are padded to whole blocks, so there is no tail in k.

// A wave's part of the output, rows mw .., columns nw ..: lane l holds for tile (i, j) row
// mw + 32 j + (l & 31) and columns nw + 32 i + 8 q + 4 (l >> 5) + e in acc[i][j][4 q + e].  They go
// through the wave's 8 KB of free LDS at wp, 32 rows at a time, into 8-column pieces.
template <typename T, int FORM, int TMJ>
__device__ __forceinline__ void tile_epilogue(const Out<T>& o, const int16v (&acc)[2][TMJ],
                                              const float* __restrict__ xs, long mw, long nw,
                                              long M, long N, int l, char* wp) {
    const Columns<T, FORM> col(o, nw + 8 * (l & 7), N);
    // (fp32 residuals and ragged ones leave no registers to read a pass ahead in)
    constexpr bool AHEAD = sizeof(T) == 2 && FORM != kRagged;
    typename Columns<T, FORM>::Rows rows[2];
    if (AHEAD && mw < M) rows[0].load(o, col, xs, mw + (l >> 3), M);
#pragma unroll
    for (int j = 0; j < TMJ; ++j) {
        const long r0 = mw + 32 * j;
        if (r0 >= M) break;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                *reinterpret_cast<int4v*>(wp + gf::ep_off<2>(l & 31, 32 * i + 8 * q + 4 * (l >> 5))) =
                    int4v{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2],
                          acc[i][j][4 * q + 3]};
        // the next pass's scales and residual are on their way while this one is
        // finished: its accumulators have left their registers
        if (AHEAD && j + 1 < TMJ && r0 + 32 < M)
            rows[(j + 1) & 1].load(o, col, xs, r0 + 32 + (l >> 3), M);
        if (!AHEAD) rows[j & 1].load(o, col, xs, r0 + (l >> 3), M);
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int row = 8 * s + (l >> 3), c = 8 * (l & 7);
            const int4v v0 = *reinterpret_cast<const int4v*>(wp + gf::ep_off<2>(row, c));
            const int4v v1 = *reinterpret_cast<const int4v*>(wp + gf::ep_off<2>(row, c + 4));
            const int v[8] = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
            if (r0 + row < M && col.cnt > 0) col.finish(o, r0 + row, v, rows[j & 1], s);
        }
    }
}

// Fragments and products of one 32-deep step of a tile's block, reads of the next between them
template <int TS, int TMJ>
struct Steps {
    int4v fb[2][2], fa[2][TMJ];
    __device__ __forceinline__ void read(int c, const char* as, const char* bs, int wm, int wn,
                                         int ks, int l) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            fb[c][i] = __builtin_bit_cast(int4v, gf::frag<true, TS>(bs, wn + 32 * i, ks, l));
#pragma unroll
        for (int j = 0; j < TMJ; ++j)
            fa[c][j] = __builtin_bit_cast(int4v, gf::frag<true, TS>(as, wm + 32 * j, ks, l));
    }
    __device__ __forceinline__ void mma(int c, int16v (&acc)[2][TMJ]) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < TMJ; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[c][i], fa[c][j], acc[i][j], 0,
                                                                  0, 0);
        // one LDS read between consecutive MFMAs
        constexpr int NR = 2 + TMJ, NM = TMJ * 2, R = NR < NM ? NR : NM;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // DS read
        }
        if constexpr (NM > R) __builtin_amdgcn_sched_group_barrier(0x008, NM - R, 0);
    }
};

template <typename T, int TS, int FORM>
__global__ void __launch_bounds__(64 * gf::tile_waves<TS>(), TS == 128 ? 2 : 1)
tile_kernel(gf::Opnd A, gf::Opnd B, long M, long N, int niter, const float* __restrict__ xs,
            Out<T> o) {
    constexpr int TILE = gf::tile_bytes<TS>(), TNI = 2, TMJ = TS / 64, KS = 4;
    __shared__ __attribute__((aligned(1024))) char smem[4 * TILE];
    const long tm_n = (M + TS - 1) / TS, tn_n = (N + TS - 1) / TS, nitems = tm_n * tn_n;
    // XCD bands, then groups of 8 tile rows
    auto decode = [&](long it, int& m0, int& n0) {
        long id = it;
        if (nitems % 8 == 0) id = (id % 8) * (nitems / 8) + id / 8;
        const long span = 8 * tn_n, gi = id / span, first = gi * 8;
        const long gsize = (tm_n - first) < 8 ? (tm_n - first) : 8;
        m0 = __builtin_amdgcn_readfirstlane((int)((first + (id % span) % gsize) * TS));
        n0 = __builtin_amdgcn_readfirstlane((int)(((id % span) / gsize) * TS));
    };
    const int w = mf::wave();
    const int wm = (w & 1) * (TS / 2), wn = (w >> 1) * (32 * TNI);
    auto As = [&](int b) { return smem + 2 * b * TILE; };
    auto Bs = [&](int b) { return smem + (2 * b + 1) * TILE; };
    long it = blockIdx.x;
    if (it >= nitems) return;
    long fit = it;
    int fkt = 0, fm0, fn0;
    bool fmore = true;
    decode(fit, fm0, fn0);
    auto fetch = [&](int b, int l) {
        if (!fmore) return;
        gf::copy_tile<true, TS>(A, fm0, (long)fkt * gf::BK, As(b), w, l);
        gf::copy_tile<true, TS>(B, fn0, (long)fkt * gf::BK, Bs(b), w, l);
        if (++fkt == niter) {
            fkt = 0;
            fit += gridDim.x;
            fmore = fit < nitems;
            if (fmore) decode(fit, fm0, fn0);
        }
    };
    int m0 = fm0, n0 = fn0;
    fetch(0, mf::lane());
    mf::dma_wait();
    __syncthreads();
    int buf = 0;
    for (;;) {
        const int l = mf::tid_in((int)it) & 63;
        fetch(buf ^ 1, l);
        int16v acc[TNI][TMJ];
#pragma unroll
        for (int i = 0; i < TNI; ++i)
#pragma unroll
            for (int j = 0; j < TMJ; ++j) acc[i][j] = int16v{};
        const bool act = m0 + wm < M && n0 + wn < N;
        Steps<TS, TMJ> st;
        auto read = [&](int c, int b, int ks) { st.read(c, As(b), Bs(b), wm, wn, ks, l); };
        auto mma_step = [&](int c) { st.mma(c, acc); };
        if (act) read(0, buf, 0);
        for (int kt = 0; kt < niter; ++kt) {
            __builtin_amdgcn_s_setprio(1);
            if (act) {
#pragma unroll
                for (int ks = 0; ks + 1 < KS; ++ks) {
                    read((ks + 1) & 1, buf, ks + 1);
                    mma_step(ks & 1);
                }
            }
            __builtin_amdgcn_s_setprio(0);
            mf::dma_wait();
            __syncthreads();
            __builtin_amdgcn_s_setprio(1);
            if (kt + 1 < niter) fetch(buf, l);
            if (act) {
                read(KS & 1, buf ^ 1, 0);  // after the last iteration: not used
                mma_step((KS - 1) & 1);
            }
            buf ^= 1;
        }
        __builtin_amdgcn_s_setprio(0);
        {
            const int le = mf::tid_in(~(int)it) & 63;
            char* wp = smem + 2 * (buf ^ 1) * TILE + (4096 * TNI) * w;
            tile_epilogue<T, FORM>(o, acc, xs, (long)m0 + wm, (long)n0 + wn, M, N, le, wp);
        }
        it += gridDim.x;
        if (it >= nitems) break;
        __syncthreads();
        decode(it, m0, n0);
    }
}

// The same for outputs of no more 128 x 128 tiles than there are compute units, each of which has
// one alone: eight waves in two groups of four that take the blocks of k in turn, two
// buffers each, and add up in LDS.  A lone tile waits for its one wave a SIMD, not for its
// loads: four waves with two buffers, with three blocks under way, and this, us:
//   65 x 1024 x 1024 10.2 / 9.3 / 7.9   65 x 4096 x 1024 24.2 / 22.4 / 18.3
//   65 x 1024 x 32000 11.9 / 11.1 / 10.8   517 x 1001 x 3088 fp16 11.4 / 10.6 / 9.4
template <typename T, int FORM>
__global__ void __launch_bounds__(512, 2)
lone_tile_kernel(gf::Opnd A, gf::Opnd B, long M, long N, int niter, const float* __restrict__ xs,
                 Out<T> o) {
    constexpr int TS = 128, TMJ = 2, KS = 4, TILE = gf::tile_bytes<TS>();
    __shared__ __attribute__((aligned(1024))) char smem[4 * 2 * TILE];
    const int tm_n = (int)((M + TS - 1) / TS);
    const int m0 = (int)(blockIdx.x % tm_n) * TS, n0 = (int)(blockIdx.x / tm_n) * TS;
    const int wave = mf::wave(), w = wave & 3, group = wave >> 2, l = mf::lane();
    const int wm = (w & 1) * (TS / 2), wn = (w >> 1) * 64;
    // the group's block i is block 2 i + group
    const int mine = (niter + 1 - group) / 2, most = (niter + 1) / 2;
    char* base = smem + group * 4 * TILE;
    auto fetch = [&](int i) {
        if (i >= mine) return;
        const long k0 = (2L * i + group) * gf::BK;
        char* to = base + (i & 1) * 2 * TILE;
        gf::copy_tile<true, TS>(A, m0, k0, to, w, l);
        gf::copy_tile<true, TS>(B, n0, k0, to + TILE, w, l);
    };
    fetch(0);
    int16v acc[2][TMJ];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < TMJ; ++j) acc[i][j] = int16v{};
    Steps<TS, TMJ> st;
    for (int i = 0; i < most; ++i) {
        mf::dma_wait();
        __syncthreads();
        // every wave has read the block before: its buffer takes the next
        fetch(i + 1);
        if (i < mine) {
            const char *as = base + (i & 1) * 2 * TILE, *bs = as + TILE;
            st.read(0, as, bs, wm, wn, 0, l);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                if (ks + 1 < KS) st.read((ks + 1) & 1, as, bs, wm, wn, ks + 1, l);
                st.mma(ks & 1, acc);
            }
        }
    }
    // the second group's sums through LDS, 16 KB a wave; each group then finishes half of the rows
    __syncthreads();
    int4v* part = reinterpret_cast<int4v*>(smem) + 1024 * w;
    auto pass = [&](int j, bool put) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                int4v& at = part[((j * 2 + i) * 4 + q) * 64 + l];
                int4v v{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2],
                        acc[i][j][4 * q + 3]};
                if (put) {
                    at = v;
                } else {
                    v += at;
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] = v[e];
                }
            }
    };
    // rows 32 j of a wave's 64 are group j's
    if (group == 0) pass(1, true);
    else pass(0, true);
    __syncthreads();
    int16v half[2][1];
    if (group == 0) {
        pass(0, false);
        half[0][0] = acc[0][0], half[1][0] = acc[1][0];
    } else {
        pass(1, false);
        half[0][0] = acc[0][1], half[1][0] = acc[1][1];
    }
    __syncthreads();
    tile_epilogue<T, FORM, 1>(o, half, xs, (long)m0 + wm + 32 * group, (long)n0 + wn, M, N, l,
                              smem + 8192 * wave);
}

}  // namespace i8
}  // namespace efla

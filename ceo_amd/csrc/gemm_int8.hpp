// Products in 8-bit integers with a scale for each token and channel, for gfx950
// (included by gemm_int8.hip).
//
//   sx_m = max_k |x_mk| (1 / 127), qx_mk = x_mk / sx_m to the nearest whole number (ties to even)
//   sw_n, qw_kn the same over the columns of the weight, once, when it is packed
//   y_mn = act((sum_k qx_mk qw_kn) sx_m sw_n + bias_n) + residual_mn, rounded once
//
// The sums are whole and exact (k <= 131072: below 2^31), so nothing depends on how they
// are split.  k is filled up with zeros to whole blocks of 128.  A packed weight lies, after
// the scales, in the order in which a wave's lanes load it: pieces of 16 channels by 64 k, of
// which lane l = 16 g + r has channel r, k 16 g .. + 15, one behind the other.  (In rows a load takes
// 16 lines of 16 lanes, at a quarter of the rate: mid_kernel for 128 x 4096 x 1024 19 us, 8.6 so.)
// Quantised tokens are the same or rows, whichever the product's kernel reads.
#pragma once
#include "common.hpp"
#include "gemm_fast.hpp"

namespace efla {
namespace i8 {

typedef __attribute__((__vector_size__(4 * sizeof(int)))) int int4v;
typedef __attribute__((__vector_size__(16 * sizeof(int)))) int int16v;

constexpr long kLine = 128;
inline __host__ __device__ long up_to(long x, long m) { return (x + m - 1) / m * m; }
constexpr int kPiece = 1024;  // bytes of 16 rows by 64 k
// where in 16 rows' pieces row r's 8 values from k = c on lie (c % 8 == 0)
__device__ __forceinline__ long piece_at(int r, long c) {
    return (c >> 6) * kPiece + ((c >> 4) & 3) * 256 + 16 * r + (c & 8);
}

// --- quantising -----------------------------------------------------------------
// A row's (column's) scale from its largest magnitude, times 1 / 127 rounded to fp32.  NaN where that is not finite: the
// row's products are NaN then.
__device__ __forceinline__ float scale_of(float amax) {
    return amax < INFINITY ? amax * (1.f / 127.f) : NAN;
}

// x / scale to the nearest whole number, ties to even, as an exact quotient would round:
// eight of them, a byte each.  A fused multiply and add of 1.5 2^23 rounds x inv to a whole
// number that its low byte holds.  inv is 1 / scale rounded, so x inv is off by 127 * 2^-23 at
// most, and the whole number by one at most, next to a half: what lies within 2^-14 of one
// (one vector in a thousand) is looked at again.  There x - r scale, which one fused operation gives
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
    // kp bytes, zero behind k; q(c) is where the eight from c on go
    template <typename At>
    __device__ __forceinline__ void store(const T* x, long k, long kp, int lr, float scale,
                                          At q) {
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
                *reinterpret_cast<uint2*>(q(c)) = qz(y);
            }
            scale *= 0x1p64f;
            kp = kp < kHeld ? kp : kHeld;
        }
        const Quantizer qz(scale);
#pragma unroll
        for (int i = 0; i < HOLD; ++i) {
            const long c = 8 * (lr + LPR * i);
            if (c < kp) *reinterpret_cast<uint2*>(q(c)) = qz(v[i]);
        }
        for (long c = kHeld + 8 * lr; c < kp; c += 8 * LPR)
            *reinterpret_cast<uint2*>(q(c)) = qz(at(x, c, k));
        if (k % 8 && lr == k / 8 % LPR) *reinterpret_cast<uint2*>(q(k / 8 * 8)) = qz(last);
    }
};

// LPR threads to a row: a wave, four rows to a workgroup, or (few rows) the whole workgroup,
// where one wave's chain of instructions is what a row takes.  Bound by memory.  Rows of kp
// bytes, or pieces.
template <typename T, int LPR, int HOLD>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* __restrict__ x, long ldx,
                                                            long m, long k, long kp, int pieces,
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
    q += pieces ? row / 16 * 16 * kp : row * kp;
    const int r16 = (int)(row & 15);
    r.store(x, k, kp, lr, s, [&](long c) { return q + (pieces ? piece_at(r16, c) : c); });
    if (lr == 0) scales[row] = s;
}

// Packing: the weight is read twice, for its columns' scales and for its values, once in its life (a call, bf16:
// 1024 x 1024 16 us, 4096 x 1024 20, 1024 x 32000 65).
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

// 64 x 64 tiles of the weight, turned through LDS and quantised into pieces.
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
            *reinterpret_cast<uint2*>(q + col / 16 * 16 * kp +
                                      piece_at((int)(col & 15), k0 + 8 * (i & 7))) = qz(v);
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
// quantised while those are on their way, and what the epilogue needs right behind.  Up to 8
// tokens have a wave a row (4 x 1024 x 4096 5.4 us, with 32 lanes 6.2, with two waves 5.9), long
// ones two (4 x 4096 x 1024 7.7, with one 8.8).  HOLD 0: the tokens are read quantised, in pieces.
constexpr int kAhead = 8;  // 64-byte steps of k whose weights a wave has in flight
// waves of a workgroup: enough that LPR lanes have a row, 8 rows where that is a wave or two
template <int MT, int LPR, int HOLD>
constexpr int kFewWaves = HOLD == 0 ? 8 : LPR == 32 ? 8 * MT : LPR / 8;
// LDS in front of the rows: their scales, and two waves' halves of a largest magnitude
template <int MT, int LPR>
constexpr int kFewFront = LPR > 64 ? 128 : 64 * MT;

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
    const uint8_t* wp = wq + (n0 < N ? n0 : 0) * kp + 16 * l;
    const int own = threadIdx.x / LPR, lr = threadIdx.x % LPR;
    Row<T, LPR, FUSED ? HOLD : 1> row;
    if constexpr (FUSED) row.load(x + own * ldx, own < M ? k : 0, lr);
    int4v a[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
        const int s = s0 + i < s1 ? s0 + i : s0;
        a[i] = *reinterpret_cast<const int4v*>(wp + (long)kPiece * s);
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
    const long ldq = kp + 16;
    float* sc = reinterpret_cast<float*>(lds);  // 16 MT scales
    uint8_t* rows = lds + kFewFront<MT, LPR>;
    if constexpr (FUSED) {
        float m = lanes_amax<LPR < 64 ? LPR : 64>(row.amax(x, 0, lr));
        if constexpr (LPR > 64) {
            float* part = sc + 16;
            if (l == 0) part[w] = m;
            __syncthreads();
            m = amax2(m, part[w ^ 1]);
        }
        const float s = scale_of(m);
        row.store(x, own < M ? k : 0, kp, lr, s, [&](long c) { return rows + own * ldq + c; });
        if (lr == 0) sc[own] = s;
        __syncthreads();
    }
    int4v acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = int4v{};
    // (64 or more lanes a row: LDS has 8 rows, whose products rows 8 to 15 repeat)
    const uint8_t* bp[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
        bp[t] = FUSED ? rows + (LPR >= 64 ? r & 7 : 16 * t + r) * ldq + 16 * g
                      : xq + (16 * t < M ? 16 * t : 0) * kp + 16 * l;
    constexpr long kStep = FUSED ? 64 : kPiece;
    for (int s = s0; s < s1; s += kAhead) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (s + i >= s1) break;
            const int4v wa = a[i];
            if (s + i + kAhead < s1)
                a[i] = *reinterpret_cast<const int4v*>(wp + (long)kPiece * (s + i + kAhead));
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const int4v b = *reinterpret_cast<const int4v*>(bp[t] + kStep * (s + i));
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
    struct Read {  // as loaded: converting would wait for it
        typename F::vec sw{};
        typename P::vec bias{};
        __device__ __forceinline__ Read(const Out<T>& o, long n, long N) {
            if (n < N) sw = F::load(o.sw + n, N - n);
            if (n < N && o.bias) bias = P::load(o.bias + n, N - n);
        }
    };
    __device__ __forceinline__ Columns(const Read& r, long n, long N) : n(n), cnt(N - n) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            sw[e] = r.sw[e];
            bias[e] = (float)r.bias[e];
        }
    }
    template <int S>
    struct Rows {  // rows m0, m0 + 8, + 16, ..
        float sx[S];
        typename P::vec res[S];
        __device__ __forceinline__ void load(const Out<T>& o, long n, long N,
                                             const float* __restrict__ xs, long m0, long M) {
#pragma unroll
            for (int s = 0; s < S; ++s) sx[s] = xs[min(m0 + 8 * s, M - 1)];
            if (!o.residual || n >= N) return;
#pragma unroll
            for (int s = 0; s < S; ++s)
                res[s] = P::load(o.residual + min(m0 + 8 * s, M - 1) * o.ldr + n, N - n);
        }
    };
    template <int S>
    __device__ __forceinline__ void finish(const Out<T>& o, long m, const int (&acc)[8],
                                           const Rows<S>& r, int s) const {
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

// --- some rows ------------------------------------------------------------------------
// 64 x 64 tiles, eight waves that split k, for outputs of few tiles: nothing waits for another
// wave until the sums meet in LDS, 16 KB a wave, and each wave finishes eight rows.  A wave reads
// its blocks of 128 straight from memory, one ahead, the weights as A operand like few_kernel.
// Bound by its start, one block's latency and the joining for short k (128 x 1024 x 1024 5.0 us) and
// by what a compute unit loads, 64 bytes a clock, for long (8192 more of k 11 us).
constexpr int kMid = 64;

template <typename T, int FORM>
__global__ void __launch_bounds__(512, 2)
mid_kernel(const uint8_t* __restrict__ xq, const float* __restrict__ xs,
           const uint8_t* __restrict__ wq, long M, long N, long kp, Out<T> o) {
    constexpr int W = 8, G = kMid / 16;
    __shared__ __attribute__((aligned(16))) int4v part[W][G * G * 64];
    const int w = mf::wave(), l = lane_id();
    // bands of tiles for the XCDs, tokens first
    const long items = gridDim.x, tm = (M + kMid - 1) / kMid;
    long id = blockIdx.x;
    if (items % 8 == 0) id = (id % 8) * (items / 8) + id / 8;
    const long m0 = id % tm * kMid, n0 = id / tm * kMid;
    const int blocks = (int)(kp / kLine), b0 = blocks * w / W, b1 = blocks * (w + 1) / W;
    const uint8_t *wp[G], *xp[G];
#pragma unroll
    for (int i = 0; i < G; ++i) {
        wp[i] = wq + (n0 + 16 * i < N ? n0 + 16 * i : n0) * kp;
        xp[i] = xq + (m0 + 16 * i < M ? m0 + 16 * i : m0) * kp;
    }
    const unsigned lo = 16 * l;
    int4v a[2][2][G], b[2][2][G];
    auto load = [&](int c, int blk) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < G; ++i) {
                const long at = (long)kPiece * (2 * blk + s);
                a[c][s][i] = *reinterpret_cast<const int4v*>(wp[i] + at + lo);
                b[c][s][i] = *reinterpret_cast<const int4v*>(xp[i] + at + lo);
            }
    };
    int4v acc[G][G];
#pragma unroll
    for (int i = 0; i < G; ++i)
#pragma unroll
        for (int t = 0; t < G; ++t) acc[i][t] = int4v{};
    auto mma = [&](int c) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < G; ++i)
#pragma unroll
                for (int t = 0; t < G; ++t)
                    acc[i][t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[c][s][i], b[c][s][t],
                                                                      acc[i][t], 0, 0, 0);
    };
    if (b0 < b1) load(0, b0);
    // what the epilogue needs: row 8 w + (l & 7) of the tile, columns 8 (l >> 3) ..
    const long row = m0 + 8 * w + (l & 7);
    typedef Columns<T, FORM> Col;
    const long n = n0 + 8 * (l >> 3);
    const typename Col::Read read(o, n, N);
    typename Col::template Rows<1> rows;
    rows.load(o, n, N, xs, row, M);
    int blk = b0;
    for (; blk + 2 <= b1; blk += 2) {
        load(1, blk + 1);
        __builtin_amdgcn_sched_barrier(0);  // (the loads would be put behind the products)
        mma(0);
        if (blk + 2 < b1) load(0, blk + 2);
        __builtin_amdgcn_sched_barrier(0);
        mma(1);
    }
    if (blk < b1) mma(0);
#pragma unroll
    for (int i = 0; i < G; ++i)
#pragma unroll
        for (int t = 0; t < G; ++t) part[w][(i * G + t) * 64 + l] = acc[i][t];
    __syncthreads();
    // tokens 16 t + r are lane 16 g + r's, channels 16 i + 4 g ..
    const int at = (((l >> 3) / 2) * G + w / 2) * 64 + ((l >> 3) % 2) * 32 + 8 * (w % 2) + (l & 7);
    int4v v0{}, v1{};
#pragma unroll
    for (int j = 0; j < W; ++j) {
        v0 += part[j][at];
        v1 += part[j][at + 16];
    }
    const int v[8] = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
    if (row < M && n < N) Col(read, n, N).finish(o, row, v, rows, 0);
}

// --- many rows ------------------------------------------------------------------------
// The tiles of gemm_fast.hpp, the tokens k-contiguous with two 8-bit integers in the
// place of each 16-bit element, the weights in pieces: 256 x 256 x 128 (eight waves of 128 x 64) or 128 x 128 x 128
// (four of 64 x 64, two workgroups to a CU), copied straight into LDS one block ahead,
// MFMA 32 x 32 x 32.  Rows are padded to whole blocks, so there is no tail in k.

// A wave's part of the output, rows mw .., columns nw ..: lane l holds for tile (i, j) row
// mw + 32 j + (l & 31) and columns nw + 32 i + 8 q + 4 (l >> 5) + e in acc[i][j][4 q + e].  They go
// through the wave's 8 KB of free LDS at wp, 32 rows at a time, into 8-column pieces.
template <typename T, int FORM, int TMJ>
__device__ __forceinline__ void tile_epilogue(const Out<T>& o, const int16v (&acc)[2][TMJ],
                                              const float* __restrict__ xs, long mw, long nw,
                                              long M, long N, int l, char* wp) {
    typedef Columns<T, FORM> Col;
    const long n = nw + 8 * (l & 7);
    const Col col(typename Col::Read(o, n, N), n, N);
    // (fp32 residuals and ragged ones leave no registers to read a pass ahead in)
    constexpr bool AHEAD = sizeof(T) == 2 && FORM != kRagged;
    typename Col::template Rows<4> rows[2];
    if (AHEAD && mw < M) rows[0].load(o, n, N, xs, mw + (l >> 3), M);
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
            rows[(j + 1) & 1].load(o, n, N, xs, r0 + 32 + (l >> 3), M);
        if (!AHEAD) rows[j & 1].load(o, n, N, xs, r0 + (l >> 3), M);
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

// TS channels of a block of k, in the order in which they lie, by the waves of a tile
struct Weight {
    const char* base;
    long kp;
    int groups;  // of 16 channels
};
template <int TS>
__device__ __forceinline__ void copy_weight(const Weight& B, int n0, int blk, char* tile, int w,
                                            int l) {
    constexpr int NW = gf::tile_waves<TS>();
    const int g0 = n0 >> 4;
    const char* base = B.base + (long)g0 * 16 * B.kp + 2L * kPiece * blk;
#pragma unroll
    for (int i = 0; i < TS / 8 / NW; ++i) {
        const int q = NW * i + w, group = min(q >> 1, B.groups - 1 - g0);
        mf::dma16(base, (unsigned)(group * (int)(16 * B.kp) + (q & 1) * kPiece + 16 * l),
                  tile + kPiece * q);
    }
}
// channels n .. n + 31 of it, k step ks
__device__ __forceinline__ int4v weight_frag(const char* tile, int n, int ks, int l) {
    const int group = (n >> 4) + ((l >> 4) & 1), lane = 16 * (2 * (ks & 1) + (l >> 5)) + (l & 15);
    return *reinterpret_cast<const int4v*>(tile + kPiece * (2 * group + (ks >> 1)) + 16 * lane);
}

// Fragments and products of one 32-deep step of a tile's block, reads of the next between them
template <int TS, int TMJ>
struct Steps {
    int4v fb[2][2], fa[2][TMJ];
    __device__ __forceinline__ void read(int c, const char* as, const char* bs, int wm, int wn,
                                         int ks, int l) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            fb[c][i] = weight_frag(bs, wn + 32 * i, ks, l);
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
tile_kernel(gf::Opnd A, Weight B, long M, long N, int niter, const float* __restrict__ xs,
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
        copy_weight<TS>(B, fn0, fkt, Bs(b), w, l);
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

// The same for outputs of no more 128 x 128 tiles than there are compute units and too many for
// mid_kernel: each has one alone, eight waves in two groups of four that take the blocks of k in turn, two
// buffers each, and add up in LDS.  A lone tile waits for its one wave a SIMD, not for its
// loads: four waves with two buffers, with three blocks under way, and this, us:
//   65 x 1024 x 32000 11.9 / 11.1 / 10.8   517 x 1001 x 3088 fp16 11.4 / 10.6 / 9.4
template <typename T, int FORM>
__global__ void __launch_bounds__(512, 2)
lone_tile_kernel(gf::Opnd A, Weight B, long M, long N, int niter, const float* __restrict__ xs,
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
        copy_weight<TS>(B, n0, 2 * i + group, to + TILE, w, l);
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

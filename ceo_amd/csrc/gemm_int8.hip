// Entry points of the 8-bit integer products (kernels: gemm_int8.hpp).
#include <hip/hip_runtime.h>
#include <math.h>

#include <algorithm>

#include "../../include/efla_hip.h"
#include "gemm_int8.hpp"
#include "internal.hpp"

namespace efla {
namespace i8 {

constexpr size_t kMaxK = 131072;  // 127^2 of them stay below 2^31
// a row's 256 threads, and 4 a channel, are fewer than 2^32 in a launch
constexpr size_t kMaxM = (1 << 24) - 1, kMaxN = (1 << 29) - 1;

static size_t dtype_size(int d) {
    return d == kDtypeF32 ? 4 : d == kDtypeF16 || d == kDtypeBF16 ? 2 : 0;
}
static size_t scales_bytes(size_t n) { return (size_t)up_to((long)(n * sizeof(float)), kLine); }

static long tiles(long m, long n, long ts) { return ((m + ts - 1) / ts) * ((n + ts - 1) / ts); }

// Up to here the weights are streamed past the tokens (few_kernel).  Measured, few_kernel / mid_kernel,
// us: 32 x 4096 x 1024 6.6 / 8.0, 64 x 4096 x 1024 10.0 / 8.3, 64 x 1024 x 4096 6.6 / 4.9.
constexpr long kFewRows = 32;

// Whether mid_kernel has the tiles: one to a compute unit, or two where k is long, since lone_tile_kernel
// has longer rounds (mid_kernel / lone_tile_kernel, us: 128 x 1024 x 1024 5.0 / 8.4, 512 x 4096 x 1024
// 9.1 / 18.7, 512 x 4096 x 4096 17.6 / 22.4; two rounds of short ones 512 x 1024 x 4096 9.1 / 9.0;
// four 1024 x 4096 x 4096 34 / 27).
static bool mid(long m, long n, long kp) {
    const long cus = device_cu_count() > 0 ? device_cu_count() : 256;
    return m > kFewRows && tiles(m, n, kMid) <= (kp > 1024 ? 2 : 1) * cus;
}

// Fewer rows than this are quantised by a workgroup each, more by a wave, unless a wave's registers
// do not hold the row.
constexpr long kWaveRows = 2048;

// Whether few_kernel quantises the tokens itself: a second launch is longer than what it takes
// every workgroup, while rows are short, or the tokens 8 and the weights small (4 x 4096 x 1024
// 7.9 us, apart 6.2 + 3.4 and the second launch).  What a wave's registers and 64 KiB of
// LDS hold: 16-bit tokens, 32 of 1024 or 8 of 4096 values.
static bool fused(size_t m, size_t n, size_t kp, size_t size) {
    if (m > (size_t)kFewRows) return false;  // the other kernels read quantised tokens
    if (kp <= 1024) return m <= (size == 2 ? 32 : 16);
    return size == 2 && m <= 8 && kp <= 4096 && n <= 16384;
}

template <typename T, int MT, int LPR, int HOLD>
static void few_launch(const T* x, long ldx, const uint8_t* xq, const float* xs, const uint8_t* wq,
                       long m, long n, long k, long kp, const Out<T>& o, hipStream_t st) {
    constexpr long NW = kFewWaves<MT, LPR, HOLD>;
    const long cus = device_cu_count() > 0 ? device_cu_count() : 256;
    const long cols = (n + 15) / 16;
    // waves that split k: until three quarters of the compute units have a workgroup
    long kw = 1;
    while (kw < NW && cols * kw < NW * cus * 3 / 4 && kp / 64 / (2 * kw) >= 2) kw *= 2;
    const long cw = NW / kw;
    const dim3 grid((unsigned)((cols + cw - 1) / cw)), block(64 * NW);
    const size_t parts = kw > 1 ? (size_t)NW * MT * 64 * 16 : 0;
    const size_t rows = HOLD ? (size_t)(64 * NW / LPR) * (size_t)(kp + 16) : 0;
    const size_t lds = kFewFront<MT, LPR> + std::max(parts, rows);
    EFLA_LAUNCH_LDS("linear_int8", (few_kernel<T, MT, LPR, HOLD>), grid, block, lds, st, x, ldx,
                    xq, xs, wq, (int)m, (int)n, k, kp, (int)kw, o);
}

// Whether 256-tiles, one to a compute unit, are the faster ones, 128-tiles two: rounds of what the
// chip holds, of 1.67 / 1.0 us a block of k and 7.3 / 4.4 us for the epilogue and the
// first block.  (Measured with either, us: 16384 x 1024 x 1024 24.5 / 27.7, 16384 x 2048 x 1024 38 / 44,
// 16384 x 1024 x 4096 88 / 95, 1463 x 80 x 12070 21.7 / 20.1.)
static bool large_tiles(long m, long n, long kp) {
    const long cus = device_cu_count() > 0 ? device_cu_count() : 256;
    const double it = (double)(kp / kLine);
    const long big = (tiles(m, n, 256) + cus - 1) / cus;
    const long small = (tiles(m, n, 128) + 2 * cus - 1) / (2 * cus);
    return (double)big * (1.67 * it + 7.3) < (double)small * (1.0 * it + 4.4);
}

template <typename T, int TS, int FORM>
static void tile_launch(const uint8_t* xq, const float* xs, const uint8_t* wq, long m, long n,
                        long kp, const Out<T>& o, hipStream_t st) {
    const long cus = device_cu_count() > 0 ? device_cu_count() : 256;
    const long items = tiles(m, n, TS);
    const dim3 grid((unsigned)std::min(items, TS == 256 ? cus : 2 * cus));
    const gf::Opnd A{(const char*)xq, kp / 2, (int)m};
    const Weight B{(const char*)wq, kp, (int)((n + 15) / 16)};
    EFLA_LAUNCH("linear_int8", (tile_kernel<T, TS, FORM>), grid, dim3(64 * gf::tile_waves<TS>()),
                st, A, B, m, n, (int)(kp / kLine), xs, o);
}

template <typename T, int FORM>
static void lone_launch(const uint8_t* xq, const float* xs, const uint8_t* wq, long m, long n,
                        long kp, const Out<T>& o, hipStream_t st) {
    const gf::Opnd A{(const char*)xq, kp / 2, (int)m};
    const Weight B{(const char*)wq, kp, (int)((n + 15) / 16)};
    EFLA_LAUNCH("linear_int8", (lone_tile_kernel<T, FORM>), dim3((unsigned)tiles(m, n, 128)),
                dim3(512), st, A, B, m, n, (int)(kp / kLine), xs, o);
}

template <typename T, int FORM>
static void mid_launch(const uint8_t* xq, const float* xs, const uint8_t* wq, long m, long n,
                       long kp, const Out<T>& o, hipStream_t st) {
    EFLA_LAUNCH("linear_int8", (mid_kernel<T, FORM>), dim3((unsigned)tiles(m, n, kMid)), dim3(512),
                st, xq, xs, wq, m, n, kp, o);
}

static size_t scratch(size_t m, size_t k, size_t n, size_t size) {
    const size_t kp = (size_t)up_to((long)k, kLine);
    return fused(m, n, kp, size) ? 0 : scales_bytes(m) + (m + 15) / 16 * 16 * kp;
}

template <typename T>
static int linear(const T* x, long ldx, const uint8_t* packed, const T* bias, const T* residual,
                  long ldr, T* y, long ldy, long m, long k, long n, int gelu, uint8_t* ws,
                  hipStream_t st) {
    const long kp = up_to(k, kLine);
    const float* sw = (const float*)packed;
    const uint8_t* wq = packed + scales_bytes((size_t)n);
    const Out<T> o{y, ldy, bias, residual, ldr, sw, gelu};
    float* xs = nullptr;
    uint8_t* xq = nullptr;
    const bool pieces = m <= kFewRows || mid(m, n, kp);
    if (!fused((size_t)m, (size_t)n, (size_t)kp, sizeof(T))) {
        xs = (float*)ws;
        xq = ws + scales_bytes((size_t)m);
#define I8_QUANT(LPR, HOLD)                                                                      \
    EFLA_LAUNCH("quantize_rows", (quantize_rows_kernel<T, LPR, HOLD>),                            \
                dim3((unsigned)(LPR == 64 ? (m + 3) / 4 : m)), dim3(256), st, x, ldx, m, k, kp, pieces, \
                xq, xs)
        if (kp > 4096) I8_QUANT(256, 8);
        else if (m < kWaveRows && kp > 512) I8_QUANT(256, 2);
        else if (kp <= 1024) I8_QUANT(64, 2);
        else I8_QUANT(64, 8);
#undef I8_QUANT
        EFLA_CHECK(hipPeekAtLastError());
    }
    const size_t a = 8 * sizeof(T);
    const bool whole = n % 8 == 0 && (uintptr_t)y % a == 0 && ldy % 8 == 0 &&
                       (!bias || (uintptr_t)bias % a == 0) &&
                       (!residual || ((uintptr_t)residual % a == 0 && ldr % 8 == 0));
    if (m <= kFewRows) {
#define I8_FEW(MT, LPR, HOLD) \
    few_launch<T, MT, LPR, HOLD>(x, ldx, xq, xs, wq, m, n, k, kp, o, st)
        if (!xq && kp > 1024) {
            if constexpr (sizeof(T) == 2) I8_FEW(1, 128, 4);
        } else if (!xq && m <= 8) {
            I8_FEW(1, 64, 2);
        } else if (!xq && m <= 16) {
            I8_FEW(1, 32, 4);
        } else if (!xq) {
            if constexpr (sizeof(T) == 2) I8_FEW(2, 32, 4);
        } else if (m <= 16) {
            I8_FEW(1, 32, 0);
        } else {
            I8_FEW(2, 32, 0);
        }
#undef I8_FEW
        return (int)hipPeekAtLastError();
    }
    if (!xq) return kInvalidConfiguration;  // what follows reads quantised tokens
    if (mid(m, n, kp)) {
        if (whole) mid_launch<T, kWhole>(xq, xs, wq, m, n, kp, o, st);
        else mid_launch<T, kRagged>(xq, xs, wq, m, n, kp, o, st);
        return (int)hipPeekAtLastError();
    }
    const long cus = device_cu_count() > 0 ? device_cu_count() : 256;
    const bool lone = tiles(m, n, 128) <= cus, large = !lone && large_tiles(m, n, kp);
    // past the L2s from their 32 MB on (16384 x 1024 x 4096 with a residual 113 -> 104 us, without
    // any 88 to 92 either way)
    const bool past = (size_t)m * (size_t)n * sizeof(T) >= (size_t)32 << 20;
#define I8_TILE(TS, FORM) tile_launch<T, TS, FORM>(xq, xs, wq, m, n, kp, o, st)
    if (large && whole && past) I8_TILE(256, kPast);
    else if (large && whole) I8_TILE(256, kWhole);
    else if (large) I8_TILE(256, kRagged);
    else if (lone && whole) lone_launch<T, kWhole>(xq, xs, wq, m, n, kp, o, st);
    else if (lone) lone_launch<T, kRagged>(xq, xs, wq, m, n, kp, o, st);
    else if (whole) I8_TILE(128, kWhole);
    else I8_TILE(128, kRagged);
#undef I8_TILE
    return (int)hipPeekAtLastError();
}

template <typename T>
static int pack(const T* w, long ld, uint8_t* packed, long k, long n, hipStream_t st) {
    const long kp = up_to(k, kLine);
    uint32_t* amax = (uint32_t*)packed;
    uint8_t* q = packed + scales_bytes((size_t)n);
    const int rc = fill_zero(amax, (size_t)n * sizeof(float), st);
    if (rc != kSuccess) return rc;
    const dim3 cols((unsigned)((n + 255) / 256), (unsigned)std::min(64L, (k + 31) / 32));
    EFLA_LAUNCH("int8_weight_amax", column_amax_kernel<T>, cols, dim3(256), st, w, ld, k, n, amax);
    const dim3 tiles((unsigned)((n + 63) / 64), (unsigned)std::min(1024L, (kp + 63) / 64));
    EFLA_LAUNCH("int8_weight_pack", pack_weight_kernel<T>, tiles, dim3(256), st, w, ld, k, n, kp,
                amax, q);
    EFLA_LAUNCH("int8_weight_scales", column_scales_kernel, dim3((unsigned)((n + 255) / 256)),
                dim3(256), st, amax, n);
    return (int)hipPeekAtLastError();
}

}  // namespace i8
}  // namespace efla

using namespace efla;

extern "C" size_t int8_weight_size(size_t k, size_t n) {
    if (k == 0 || k > i8::kMaxK || n == 0 || n > i8::kMaxN) return 0;
    return i8::scales_bytes(n) + (n + 15) / 16 * 16 * (size_t)i8::up_to((long)k, i8::kLine);
}

extern "C" int int8_weight_pack_hip(const void* weight, size_t ld, void* packed, size_t k,
                                    size_t n, int dtype, hipStream_t stream) {
    const size_t size = i8::dtype_size(dtype);
    if (size == 0 || k == 0 || n == 0 || ld < n || !weight || !packed) return kInvalidValue;
    if ((uintptr_t)weight % size || (uintptr_t)packed % i8::kLine) return kInvalidValue;
    if (k > i8::kMaxK || n > i8::kMaxN || ld > (1ull << 40)) return kInvalidConfiguration;
    if (dtype == kDtypeBF16)
        return i8::pack((const bf16*)weight, (long)ld, (uint8_t*)packed, (long)k, (long)n, stream);
    if (dtype == kDtypeF16)
        return i8::pack((const f16*)weight, (long)ld, (uint8_t*)packed, (long)k, (long)n, stream);
    return i8::pack((const float*)weight, (long)ld, (uint8_t*)packed, (long)k, (long)n, stream);
}

extern "C" size_t linear_int8_workspace_size(size_t m, size_t k, size_t n, int dtype) {
    const size_t size = i8::dtype_size(dtype);
    if (size == 0 || k == 0 || k > i8::kMaxK || n == 0 || n > i8::kMaxN || m > i8::kMaxM)
        return 0;
    return i8::scratch(m, k, n, size);
}

extern "C" int linear_int8_hip(const void* x, size_t ldx, const void* packed, const void* bias,
                               const void* residual, size_t ld_residual, void* output,
                               size_t ld_output, size_t m, size_t k, size_t n, int gelu,
                               int dtype, void* workspace, size_t workspace_bytes,
                               hipStream_t stream) {
    const size_t size = i8::dtype_size(dtype);
    if (size == 0 || k == 0 || n == 0) return kInvalidValue;
    if (k > i8::kMaxK || n > i8::kMaxN || m > i8::kMaxM || ldx > (1ull << 40) ||
        ld_output > (1ull << 40) || ld_residual > (1ull << 40))
        return kInvalidConfiguration;
    if (m == 0) return kSuccess;
    if (!x || !packed || !output || ldx < k || ld_output < n || (residual && ld_residual < n))
        return kInvalidValue;
    if (((uintptr_t)x | (uintptr_t)output | (uintptr_t)bias | (uintptr_t)residual) % size ||
        (uintptr_t)packed % i8::kLine)
        return kInvalidValue;
    const size_t need = i8::scratch(m, k, n, size);
    void* ws = workspace;
    WsLease lease;
    if (need != 0 && !ws) {
        const int rc = workspace_acquire(need, stream, &ws, lease);
        if (rc != kSuccess) return rc;
    } else if (need != 0 && (workspace_bytes < need || (uintptr_t)ws % 16)) {
        return kInvalidValue;
    }
#define I8_LINEAR(T)                                                                             \
    i8::linear<T>((const T*)x, (long)ldx, (const uint8_t*)packed, (const T*)bias,                \
                  (const T*)residual, (long)ld_residual, (T*)output, (long)ld_output, (long)m,   \
                  (long)k, (long)n, gelu, (uint8_t*)ws, stream)
    if (dtype == kDtypeBF16) return I8_LINEAR(bf16);
    if (dtype == kDtypeF16) return I8_LINEAR(f16);
    return I8_LINEAR(float);
#undef I8_LINEAR
}

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

static size_t dtype_size(int d) {
    return d == kDtypeF32 ? 4 : d == kDtypeF16 || d == kDtypeBF16 ? 2 : 0;
}
static size_t scales_bytes(size_t n) { return (size_t)up_to((long)(n * sizeof(float)), kLine); }

// Rows up to which the weights are streamed (few_kernel).
constexpr size_t kFewRows = 64;
// Tokens that a workgroup quantises into LDS itself (64 KiB with their scales).
constexpr size_t kFusedBytes = 63 << 10;

template <typename T, int MT>
static void few_launch(const T* x, long ldx, const uint8_t* xq, const float* xs, const uint8_t* wq,
                       long m, long n, long k, long kp, const Out<T>& o, hipStream_t st) {
    const long cus = device_cu_count() > 0 ? device_cu_count() : 256;
    const long tiles = (n + 15) / 16;
    // waves that split k: until each SIMD has two
    int kw = 1;
    while (kw < kFewWaves && tiles * kw < 8 * cus && kp / 64 / (2 * kw) >= 2) kw *= 2;
    const long cw = kFewWaves / kw;
    const dim3 grid((unsigned)((tiles + cw - 1) / cw)), block(64 * kFewWaves);
    const size_t parts = kw > 1 ? (size_t)kFewWaves * MT * 64 * 16 : 0;
    const size_t rows = (size_t)16 * MT * (size_t)(kp + 16);
    const size_t head = 64 * MT;
    if (!xq) {
        const size_t lds = head + std::max(parts, rows);
        EFLA_LAUNCH_LDS("linear_int8", (few_kernel<T, MT, true>), grid, block, lds, st, x, ldx, xq,
                        xs, wq, (int)m, (int)n, k, kp, kw, o);
    } else {
        EFLA_LAUNCH_LDS("linear_int8", (few_kernel<T, MT, false>), grid, block, head + parts, st, x,
                        ldx, xq, xs, wq, (int)m, (int)n, k, kp, kw, o);
    }
}

template <typename T, int TS, bool RAGGED>
static void tile_launch(const uint8_t* xq, const float* xs, const uint8_t* wq, long m, long n,
                        long kp, const Out<T>& o, hipStream_t st) {
    const long cus = device_cu_count() > 0 ? device_cu_count() : 256;
    const long items = ((m + TS - 1) / TS) * ((n + TS - 1) / TS);
    const dim3 grid((unsigned)std::min(items, TS == 256 ? cus : 2 * cus));
    const gf::Opnd A{(const char*)xq, kp / 2, (int)m}, B{(const char*)wq, kp / 2, (int)n};
    EFLA_LAUNCH("linear_int8", (tile_kernel<T, TS, RAGGED>), grid, dim3(64 * gf::tile_waves<TS>()),
                st, A, B, m, n, (int)(kp / kLine), xs, o);
}

// rows that the kernel quantises itself
static bool fused(size_t m, size_t kp) {
    return m <= kFewRows && up_to((long)m, 16) * (long)(kp + 16) <= (long)kFusedBytes;
}

static size_t scratch(size_t m, size_t k) {
    const size_t kp = (size_t)up_to((long)k, kLine);
    return fused(m, kp) ? 0 : scales_bytes(m) + m * kp;
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
    if (!fused((size_t)m, (size_t)kp)) {
        xs = (float*)ws;
        xq = ws + scales_bytes((size_t)m);
        const dim3 grid((unsigned)((m + 3) / 4)), block(256);
        if (kp <= 1024)
            EFLA_LAUNCH("quantize_rows", (quantize_rows_kernel<T, 2>), grid, block, st, x, ldx, m, k,
                        kp, xq, xs);
        else
            EFLA_LAUNCH("quantize_rows", (quantize_rows_kernel<T, 8>), grid, block, st, x, ldx, m, k,
                        kp, xq, xs);
        EFLA_CHECK(hipPeekAtLastError());
    }
    if (m <= (long)kFewRows) {
        if (m <= 16) few_launch<T, 1>(x, ldx, xq, xs, wq, m, n, k, kp, o, st);
        else if (m <= 32) few_launch<T, 2>(x, ldx, xq, xs, wq, m, n, k, kp, o, st);
        else few_launch<T, 4>(x, ldx, xq, xs, wq, m, n, k, kp, o, st);
        return (int)hipPeekAtLastError();
    }
    const size_t a = 8 * sizeof(T);
    const bool whole = n % 8 == 0 && (uintptr_t)y % a == 0 && ldy % 8 == 0 &&
                       (!bias || (uintptr_t)bias % a == 0) &&
                       (!residual || ((uintptr_t)residual % a == 0 && ldr % 8 == 0));
    const long cus = device_cu_count() > 0 ? device_cu_count() : 256;
    const bool large = ((m + 255) / 256) * ((n + 255) / 256) >= cus;
    if (large && whole) tile_launch<T, 256, false>(xq, xs, wq, m, n, kp, o, st);
    else if (large) tile_launch<T, 256, true>(xq, xs, wq, m, n, kp, o, st);
    else if (whole) tile_launch<T, 128, false>(xq, xs, wq, m, n, kp, o, st);
    else tile_launch<T, 128, true>(xq, xs, wq, m, n, kp, o, st);
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
    if (k == 0 || k > i8::kMaxK || n == 0 || n > 0x3FFFFFFFull) return 0;
    return i8::scales_bytes(n) + n * (size_t)i8::up_to((long)k, i8::kLine);
}

extern "C" int int8_weight_pack_hip(const void* weight, size_t ld, void* packed, size_t k,
                                    size_t n, int dtype, hipStream_t stream) {
    const size_t size = i8::dtype_size(dtype);
    if (size == 0 || k == 0 || n == 0 || ld < n || !weight || !packed) return kInvalidValue;
    if ((uintptr_t)weight % size || (uintptr_t)packed % i8::kLine) return kInvalidValue;
    if (k > i8::kMaxK || n > 0x3FFFFFFFull || ld > (1ull << 40)) return kInvalidConfiguration;
    if (dtype == kDtypeBF16)
        return i8::pack((const bf16*)weight, (long)ld, (uint8_t*)packed, (long)k, (long)n, stream);
    if (dtype == kDtypeF16)
        return i8::pack((const f16*)weight, (long)ld, (uint8_t*)packed, (long)k, (long)n, stream);
    return i8::pack((const float*)weight, (long)ld, (uint8_t*)packed, (long)k, (long)n, stream);
}

extern "C" size_t linear_int8_workspace_size(size_t m, size_t k) {
    if (k == 0 || k > i8::kMaxK || m > 0x3FFFFFFFull) return 0;
    return i8::scratch(m, k);
}

extern "C" int linear_int8_hip(const void* x, size_t ldx, const void* packed, const void* bias,
                               const void* residual, size_t ld_residual, void* output,
                               size_t ld_output, size_t m, size_t k, size_t n, int gelu,
                               int dtype, void* workspace, size_t workspace_bytes,
                               hipStream_t stream) {
    const size_t size = i8::dtype_size(dtype);
    if (size == 0 || k == 0 || n == 0) return kInvalidValue;
    if (k > i8::kMaxK || n > 0x3FFFFFFFull || m > 0x3FFFFFFFull || ldx > (1ull << 40) ||
        ld_output > (1ull << 40) || ld_residual > (1ull << 40))
        return kInvalidConfiguration;
    if (m == 0) return kSuccess;
    if (!x || !packed || !output || ldx < k || ld_output < n || (residual && ld_residual < n))
        return kInvalidValue;
    if (((uintptr_t)x | (uintptr_t)output | (uintptr_t)bias | (uintptr_t)residual) % size ||
        (uintptr_t)packed % i8::kLine)
        return kInvalidValue;
    const size_t need = i8::scratch(m, k);
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

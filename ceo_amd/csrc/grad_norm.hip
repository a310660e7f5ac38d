// The norm of many gradients and their clipping for gfx950 (the reference clips
// with a host round trip between its reduction and its scaling, optim.cu:221-232,
// 765-775; here nothing leaves the device).
//
//   norm = sqrt(sum over all elements of g^2),  coef = min(1, max_norm / (norm + 1e-6))
//   g <- coef g   (in fp32, rounded once to g's type)
//
// The tensors' addresses, sizes and types are put into a device table once, when
// the list is created; a call is then two launches whatever their number.  The
// elements are dealt out in units of kUnit; a map gives each unit's tensor.  The
// first kernel leaves one sum per workgroup, the second adds them, in the same order
// in every workgroup, so the norm does not depend on scheduling.  Squares and sums are
// 64 bits: the norm of any finite gradients is right, also where a square leaves
// fp32's range.  A NaN or an infinity anywhere gives norm NaN or inf, and the
// gradients what the formula says (coef NaN or 0).
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdlib.h>
#include <string.h>

#include "../../include/efla_hip.h"
#include "common.hpp"
#include "internal.hpp"

namespace efla {
namespace gn {

constexpr int NT = 256;
constexpr size_t kUnit = 16384;     // elements
constexpr unsigned kMaxGrid = 2048;  // workgroups, and sums they leave

struct Entry {
    const void* in;
    void* out;
    uint64_t numel;
    uint32_t first;  // its first unit
    int32_t dtype;
};

// A list's device memory: entries, then the units' map, then the workgroups' sums.
struct List {
    int device;
    size_t count, units;
    Entry* entries;
    uint32_t* map;
    double* part;
};

template <typename T>
struct Vec {
    static constexpr int N = 16 / sizeof(T);
    typedef __attribute__((__vector_size__(16))) T Full;
    typedef Full Any __attribute__((aligned(sizeof(T))));
};

template <typename T>
__device__ __forceinline__ double square_sum(const T* p, long n) {
    constexpr int N = Vec<T>::N;
    double s = 0.0;
    const long nv = n / N;
    for (long c = threadIdx.x; c < nv; c += NT) {
        const typename Vec<T>::Full x = *reinterpret_cast<const typename Vec<T>::Any*>(p + c * N);
#pragma unroll
        for (int i = 0; i < N; ++i) s = fma((double)(float)x[i], (double)(float)x[i], s);
    }
    const long c = nv * N + threadIdx.x;
    if (c < n) s = fma((double)(float)p[c], (double)(float)p[c], s);
    return s;
}

template <typename T>
__device__ __forceinline__ void scale(const T* p, T* q, long n, float f) {
    constexpr int N = Vec<T>::N;
    const long nv = n / N;
    for (long c = threadIdx.x; c < nv; c += NT) {
        typename Vec<T>::Full x = *reinterpret_cast<const typename Vec<T>::Any*>(p + c * N);
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = (T)((float)x[i] * f);
        *reinterpret_cast<typename Vec<T>::Any*>(q + c * N) = x;
    }
    const long c = nv * N + threadIdx.x;
    if (c < n) q[c] = (T)((float)p[c] * f);
}

// Every thread gets the workgroup's sum, added in a fixed order.
__device__ __forceinline__ double block_sum(double s, double* sm) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off);
    if (lane_id() == 0) sm[wave_id()] = s;
    __syncthreads();
    s = sm[0];
#pragma unroll
    for (int k = 1; k < NT / kWave; ++k) s += sm[k];
    return s;
}

__global__ void __launch_bounds__(NT) norm_kernel(const Entry* __restrict__ entries,
                                                  const uint32_t* __restrict__ map,
                                                  uint32_t units, double* __restrict__ part) {
    __shared__ double sm[NT / kWave];
    double s = 0.0;
    for (uint32_t u = blockIdx.x; u < units; u += gridDim.x) {
        const Entry e = entries[map[u]];
        const size_t at = (size_t)(u - e.first) * kUnit;
        const long n = (long)(e.numel - at < kUnit ? e.numel - at : kUnit);
        if (e.dtype == kDtypeBF16)
            s += square_sum((const bf16*)e.in + at, n);
        else if (e.dtype == kDtypeF16)
            s += square_sum((const f16*)e.in + at, n);
        else
            s += square_sum((const float*)e.in + at, n);
    }
    s = block_sum(s, sm);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__device__ __forceinline__ double all_parts(const double* __restrict__ part, int parts,
                                            double* sm) {
    double s = 0.0;
    for (int i = threadIdx.x; i < parts; i += NT) s += part[i];
    return sqrt(block_sum(s, sm));
}

__device__ __forceinline__ float coef_of(double norm, float max_norm) {
    const double c = (double)max_norm / (norm + 1e-6);
    return c > 1.0 ? 1.f : (float)c;  // NaN stays NaN
}

__global__ void __launch_bounds__(NT) final_kernel(const double* __restrict__ part, int parts,
                                                   float max_norm, float* __restrict__ norm,
                                                   float* __restrict__ coef) {
    __shared__ double sm[NT / kWave];
    const double v = all_parts(part, parts, sm);
    if (threadIdx.x == 0) {
        norm[0] = (float)v;
        if (coef) coef[0] = coef_of(v, max_norm);
    }
}

__global__ void __launch_bounds__(NT)
clip_kernel(const Entry* __restrict__ entries, const uint32_t* __restrict__ map, uint32_t units,
            const double* __restrict__ part, int parts, float max_norm,
            float* __restrict__ norm) {
    __shared__ double sm[NT / kWave];
    const double v = all_parts(part, parts, sm);
    const float f = coef_of(v, max_norm);
    if (blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)v;
    for (uint32_t u = blockIdx.x; u < units; u += gridDim.x) {
        const Entry e = entries[map[u]];
        if (f == 1.f && e.in == e.out) continue;  // nothing changes
        const size_t at = (size_t)(u - e.first) * kUnit;
        const long n = (long)(e.numel - at < kUnit ? e.numel - at : kUnit);
        if (e.dtype == kDtypeBF16)
            scale((const bf16*)e.in + at, (bf16*)e.out + at, n, f);
        else if (e.dtype == kDtypeF16)
            scale((const f16*)e.in + at, (f16*)e.out + at, n, f);
        else
            scale((const float*)e.in + at, (float*)e.out + at, n, f);
    }
}

static unsigned grid_of(size_t units) {
    return units < kMaxGrid ? (unsigned)units : kMaxGrid;
}

// The current device has to be the list's.
static int check(const List* l, float max_norm, const float* norm) {
    if (!l || !norm || !(max_norm >= 0.f)) return kInvalidValue;
    int dev = 0;
    EFLA_CHECK(hipGetDevice(&dev));
    return dev == l->device ? kSuccess : (int)hipErrorInvalidDevice;
}

static int sums(const List* l, unsigned* parts, hipStream_t st) {
    *parts = grid_of(l->units);
    if (l->units == 0) return kSuccess;
    EFLA_LAUNCH("grad_norm", norm_kernel, dim3(*parts), dim3(NT), st, l->entries, l->map,
                (uint32_t)l->units, l->part);
    return (int)hipPeekAtLastError();
}

}  // namespace gn
}  // namespace efla

using namespace efla;

extern "C" int grad_list_create_hip(void** list, const void* const* grads, void* const* outs,
                                    const size_t* numels, const int* dtypes, size_t count) {
    if (!list) return kInvalidValue;
    *list = nullptr;
    if (count != 0 && (!grads || !numels || !dtypes)) return kInvalidValue;
    if (count > 0x7FFFFFFFull) return kInvalidConfiguration;
    size_t units = 0;
    for (size_t i = 0; i < count; ++i) {
        const int d = dtypes[i];
        const size_t size = d == kDtypeF32 ? 4 : d == kDtypeF16 || d == kDtypeBF16 ? 2 : 0;
        if (size == 0) return kInvalidValue;
        if (numels[i] == 0) continue;
        const void* out = outs ? outs[i] : grads[i];
        if (!grads[i] || !out || ((uintptr_t)grads[i] | (uintptr_t)out) % size)
            return kInvalidValue;
        if (numels[i] > (size_t)1 << 46) return kInvalidConfiguration;
        units += (numels[i] + gn::kUnit - 1) / gn::kUnit;
        if (units > 0x7FFFFFFFull) return kInvalidConfiguration;
    }
    int dev = 0;
    EFLA_CHECK(hipGetDevice(&dev));
    const size_t parts = (size_t)gn::kMaxGrid * sizeof(double);
    const size_t bytes = parts + count * sizeof(gn::Entry) + units * sizeof(uint32_t);
    gn::List* l = (gn::List*)malloc(sizeof(gn::List));
    uint8_t* host = (uint8_t*)malloc(bytes);
    void* mem = nullptr;
    int rc = l && host ? (int)hipMalloc(&mem, bytes) : kOutOfMemory;
    if (rc == kSuccess) {
        memset(host, 0, parts);
        gn::Entry* e = (gn::Entry*)(host + parts);
        uint32_t* map = (uint32_t*)(e + count);
        uint32_t u = 0;
        for (size_t i = 0; i < count; ++i) {
            e[i].in = grads[i];
            e[i].out = outs ? outs[i] : (void*)grads[i];
            e[i].numel = numels[i];
            e[i].first = u;
            e[i].dtype = dtypes[i];
            for (size_t k = 0; k < numels[i]; k += gn::kUnit) map[u++] = (uint32_t)i;
        }
        rc = (int)hipMemcpy(mem, host, bytes, hipMemcpyHostToDevice);
    }
    free(host);
    if (rc != kSuccess) {
        (void)hipFree(mem);
        free(l);
        return rc;
    }
    l->device = dev;
    l->count = count;
    l->units = units;
    l->part = (double*)mem;
    l->entries = (gn::Entry*)((uint8_t*)mem + parts);
    l->map = (uint32_t*)(l->entries + count);
    *list = l;
    return kSuccess;
}

extern "C" int grad_list_destroy_hip(void* list) {
    if (!list) return kSuccess;
    gn::List* l = (gn::List*)list;
    const int rc = (int)hipFree(l->part);  // waits for the device
    free(l);
    return rc;
}

extern "C" int grad_norm_hip(const void* list, float max_norm, float* norm, float* coef,
                             hipStream_t stream) {
    const gn::List* l = (const gn::List*)list;
    int rc = gn::check(l, max_norm, norm);
    if (rc != kSuccess) return rc;
    unsigned parts;
    rc = gn::sums(l, &parts, stream);
    if (rc != kSuccess) return rc;
    EFLA_LAUNCH("grad_norm_final", gn::final_kernel, dim3(1), dim3(gn::NT), stream, l->part,
                (int)parts, max_norm, norm, coef);
    return (int)hipPeekAtLastError();
}

extern "C" int grad_clip_hip(const void* list, float max_norm, float* norm, hipStream_t stream) {
    const gn::List* l = (const gn::List*)list;
    int rc = gn::check(l, max_norm, norm);
    if (rc != kSuccess) return rc;
    unsigned parts;
    rc = gn::sums(l, &parts, stream);
    if (rc != kSuccess) return rc;
    EFLA_LAUNCH("grad_clip", gn::clip_kernel, dim3(parts ? parts : 1), dim3(gn::NT), stream,
                l->entries, l->map, (uint32_t)l->units, l->part, (int)parts, max_norm, norm);
    return (int)hipPeekAtLastError();
}

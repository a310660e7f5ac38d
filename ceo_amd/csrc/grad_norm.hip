// The norm of many gradients and their clipping for gfx950 (the reference clips
// with a host round trip between its reduction and its scaling, optim.cu:221-232,
// 765-775; here nothing leaves the device).
//
//   norm = sqrt(sum over all elements of g^2),  coef = min(1, max_norm / (norm + 1e-6))
//   g <- coef g   (in fp32, rounded once to g's type)
//
// The tensors' addresses, sizes and types are put into a device table once, when
// the list is created; a call is then two launches whatever their number.  The
// elements are dealt out in units of 16 KiB; a map gives each unit's tensor.  The
// first kernel leaves one sum per workgroup, the second adds them, in the same order
// in every workgroup, so the norm does not depend on scheduling.  Squares and sums are
// 64 bits: the norm of any finite gradients is right, also where a square leaves
// fp32's range.  A NaN or an infinity anywhere gives norm NaN or inf, and the
// gradients what the formula says (coef NaN or 0).
//
// Two reads and one write bound it: 368 million bf16 gradients take 351 us, 2.2 GB at
// 6.3 TB/s (a large copy: 5.15; what the 256 MB cache keeps from the first read to the
// second does not come from memory again).  14.5 million take 17 us, a small model's 23
// gradients 7, and the host's two launches 9.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdlib.h>
#include <string.h>

#include "../../include/efla_hip.h"
#include "common.hpp"
#include "internal.hpp"

namespace efla {
namespace gn {

constexpr int NT = 256, kVecs = 4;
constexpr size_t kUnit = NT * kVecs * 16;  // bytes
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
    size_t count, units, bytes;
    Entry* entries;
    uint32_t* map;
    double* part;
};

// A unit, n elements from p on, in a workgroup's registers: 16-byte vectors from a cache
// line's start on, kVecs to a thread, and the elements before and behind them (70 at
// most), one to a thread.  ONCE: nothing reads them again soon.
template <typename T, bool ONCE>
struct Unit {
    static constexpr int N = 16 / sizeof(T);
    typedef __attribute__((__vector_size__(16))) T Full;
    typedef Full Any __attribute__((aligned(sizeof(T))));
    int head, nv, edges, edge;
    Full x[kVecs];
    T one;

    __device__ __forceinline__ Unit(const T* p, int n) {
        const int h = (int)(-(uintptr_t)p % 128 / sizeof(T));
        head = h < n ? h : n;
        nv = (n - head) / N;
        edges = n - nv * N;
        edge = (int)threadIdx.x < head ? threadIdx.x : threadIdx.x + nv * N;
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            const int c = threadIdx.x + i * NT;
            x[i] = Full{};
            if (c >= nv) continue;
            const Any* from = reinterpret_cast<const Any*>(p + head + c * N);
            if constexpr (ONCE)
                x[i] = __builtin_nontemporal_load(from);
            else
                x[i] = *from;
        }
        one = (T)0.f;
        if ((int)threadIdx.x < edges) one = p[edge];
    }
    __device__ __forceinline__ double square_sum() const {
        double s = (double)(float)one * (double)(float)one;
#pragma unroll
        for (int i = 0; i < kVecs; ++i)
#pragma unroll
            for (int j = 0; j < N; ++j) s = fma((double)(float)x[i][j], (double)(float)x[i][j], s);
        return s;
    }
    template <bool PAST>
    __device__ __forceinline__ void scale(T* q, float f) const {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) {
            const int c = threadIdx.x + i * NT;
            if (c >= nv) continue;
            Full y;
#pragma unroll
            for (int j = 0; j < N; ++j) y[j] = (T)((float)x[i][j] * f);
            Any* to = reinterpret_cast<Any*>(q + head + c * N);
            if constexpr (PAST)
                __builtin_nontemporal_store(y, to);
            else
                *to = y;
        }
        if ((int)threadIdx.x < edges) q[edge] = (T)((float)one * f);
    }
};

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

// Where unit u starts in its tensor, and its elements.
template <typename T>
__device__ __forceinline__ void unit_of(const Entry& e, uint32_t u, size_t* at, int* n) {
    constexpr size_t kElems = kUnit / sizeof(T);
    *at = (size_t)(u - e.first) * kElems;
    *n = (int)(e.numel - *at < kElems ? e.numel - *at : kElems);
}

__global__ void __launch_bounds__(NT) norm_kernel(const Entry* __restrict__ entries,
                                                  const uint32_t* __restrict__ map,
                                                  uint32_t units, double* __restrict__ part) {
    __shared__ double sm[NT / kWave];
    double s = 0.0;
    for (uint32_t u = blockIdx.x; u < units; u += gridDim.x) {
        const Entry e = entries[map[u]];
        size_t at;
        int n;
        if (e.dtype == kDtypeBF16) {
            unit_of<bf16>(e, u, &at, &n);
            s += Unit<bf16, false>((const bf16*)e.in + at, n).square_sum();
        } else if (e.dtype == kDtypeF16) {
            unit_of<f16>(e, u, &at, &n);
            s += Unit<f16, false>((const f16*)e.in + at, n).square_sum();
        } else {
            unit_of<float>(e, u, &at, &n);
            s += Unit<float, false>((const float*)e.in + at, n).square_sum();
        }
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

// The clipping factor; the first workgroup writes the norm.
__device__ __forceinline__ float factor(const double* __restrict__ part, int parts,
                                        float max_norm, float* norm, double* sm) {
    const double v = all_parts(part, parts, sm);
    if (blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)v;
    return coef_of(v, max_norm);
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

// One unit: its loads are on their way while the first one's factor is added up.
template <bool PAST, typename T>
__device__ __forceinline__ void clip_unit(const Entry& e, uint32_t u, bool* known, float* f,
                                          const double* part, int parts, float max_norm,
                                          float* norm, double* sm) {
    size_t at;
    int n;
    unit_of<T>(e, u, &at, &n);
    const Unit<T, PAST> x((const T*)e.in + at, n);
    if (!*known) *f = factor(part, parts, max_norm, norm, sm);
    *known = true;
    if (*f == 1.f && e.in == e.out) return;  // nothing changes
    x.template scale<PAST>((T*)e.out + at, *f);
}

template <bool PAST>
__global__ void __launch_bounds__(NT)
clip_kernel(const Entry* __restrict__ entries, const uint32_t* __restrict__ map, uint32_t units,
            const double* __restrict__ part, int parts, float max_norm,
            float* __restrict__ norm) {
    __shared__ double sm[NT / kWave];
    bool known = false;
    float f = 1.f;
    if (units == 0) factor(part, parts, max_norm, norm, sm);
    // the last units first: of more gradients than the 256 MB cache holds it has those that
    // the norm read last (368 million in bf16 380 us, 393 from the first on, all through the cache)
    for (uint32_t k = blockIdx.x; k < ((units + 7) & ~7u); k += gridDim.x) {
        const uint32_t u = (uint32_t)backwards(k, units);
        if (u >= units) continue;
        const Entry e = entries[map[u]];
        if (known && f == 1.f && e.in == e.out) continue;
        if (e.dtype == kDtypeBF16)
            clip_unit<PAST, bf16>(e, u, &known, &f, part, parts, max_norm, norm, sm);
        else if (e.dtype == kDtypeF16)
            clip_unit<PAST, f16>(e, u, &known, &f, part, parts, max_norm, norm, sm);
        else
            clip_unit<PAST, float>(e, u, &known, &f, part, parts, max_norm, norm, sm);
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
    size_t units = 0, total = 0;
    for (size_t i = 0; i < count; ++i) {
        const int d = dtypes[i];
        const size_t size = d == kDtypeF32 ? 4 : d == kDtypeF16 || d == kDtypeBF16 ? 2 : 0;
        if (size == 0) return kInvalidValue;
        if (numels[i] == 0) continue;
        const void* out = outs ? outs[i] : grads[i];
        if (!grads[i] || !out || ((uintptr_t)grads[i] | (uintptr_t)out) % size)
            return kInvalidValue;
        if (numels[i] > (size_t)1 << 46) return kInvalidConfiguration;
        total += numels[i] * size;
        units += (numels[i] * size + gn::kUnit - 1) / gn::kUnit;
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
            const size_t size = dtypes[i] == kDtypeF32 ? 4 : 2;
            for (size_t k = 0; k < numels[i] * size; k += gn::kUnit) map[u++] = (uint32_t)i;
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
    l->bytes = total;
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
    const dim3 grid(parts ? (parts + 7) / 8 * 8 : 1), block(gn::NT);
    // Where gradients and outputs are over half of the 256 MB cache, this pass leaves the cache
    // to the gradients that the norm has read: it reads and writes past it (368 million in
    // bf16 351 us, 412 through it; 23 million 43.6 and 53.6).  In place they are counted twice
    // too; lists of 64 to 128 MiB clipped in place have not been measured.
    if (2 * l->bytes > (size_t)128 << 20)
        EFLA_LAUNCH("grad_clip", (gn::clip_kernel<true>), grid, block, stream, l->entries, l->map,
                    (uint32_t)l->units, l->part, (int)parts, max_norm, norm);
    else
        EFLA_LAUNCH("grad_clip", (gn::clip_kernel<false>), grid, block, stream, l->entries, l->map,
                    (uint32_t)l->units, l->part, (int)parts, max_norm, norm);
    return (int)hipPeekAtLastError();
}

// The states that a beam search carries, put in the order of its survivors, for gfx950:
//
//   new[b, j] = old[b, parents[b, j]]      for texts b, beams j, in every tensor of a list
//
// (the reference carries an EFLA state between calls, src/model/efla.zig:13-86, and has no
// search).  Rows are bytes: recurrent states, the texts so far and whatever else a beam has
// move in one launch.  The tensors' addresses and sizes go into a device table when the
// list is created.
//
// In place: a thread owns one vector of a row's bytes in all beams of a text, and has
// loaded every beam that moves before it stores the first, so any assignment works, cycles
// among them, and no second set of states is needed.  A beam that stays is neither read
// nor written.  A parent outside of 0 .. beams - 1 leaves its row as it was (to outs: the
// beam's own row).  Bound by memory: every row that changes is written once and its source
// read once (a source's second reader finds it in the caches).
#include <hip/hip_runtime.h>
#include <stdlib.h>
#include <string.h>

#include "../../include/efla_hip.h"
#include "common.hpp"
#include "internal.hpp"

namespace efla {
namespace sr {

constexpr int NT = 256;
constexpr int kMaxBeams = 64;
// 16-byte vectors for up to this many beams (64 registers); more go in 4-byte ones.  24 layers of 16 x 64 x 64, all
// rows moving: 4 texts of 16 beams 160 us, 5.0 TB/s, 4 of 32 302, 5.3, 2 of 64 320, 5.0.
constexpr size_t kWideBeams = 16;
constexpr size_t kMaxUnits = (1 << 24) - 1;  // 256 threads each, fewer than 2^32 in a launch

struct Entry {
    const uint8_t* in;
    uint8_t* out;
    uint64_t row;    // bytes
    uint32_t first;  // its first unit
    uint32_t cols;   // units across a row
    uint32_t width;  // bytes of a vector: 16, 4 or 1
    uint32_t pad;
};

struct List {
    int device;
    size_t batch, beams, units;
    Entry* entries;
    uint32_t* map;  // a unit's entry
};

template <int MB, typename V>
__device__ __forceinline__ void move_unit(const Entry& e, long text, uint32_t col,
                                          const int* __restrict__ parents, int beams) {
    const size_t at = ((size_t)col * NT + threadIdx.x) * sizeof(V);
    const bool in = e.in == e.out;
    const uint8_t* src = e.in + (size_t)text * beams * e.row + at;
    uint8_t* dst = e.out + (size_t)text * beams * e.row + at;
    if (at >= e.row) return;
    V x[MB];
    uint64_t moves = 0;
#pragma unroll
    for (int j = 0; j < MB; ++j) {
        if (j < beams) {
            int p = parents[text * beams + j];
            if (p < 0 || p >= beams) p = j;
            if (!in || p != j) {
                moves |= 1ull << j;
                x[j] = *reinterpret_cast<const V*>(src + (size_t)p * e.row);
            }
        }
    }
#pragma unroll
    for (int j = 0; j < MB; ++j)
        if (moves >> j & 1) *reinterpret_cast<V*>(dst + (size_t)j * e.row) = x[j];
}

template <int MB>
__global__ void __launch_bounds__(NT) reorder_kernel(const Entry* __restrict__ entries,
                                                     const uint32_t* __restrict__ map,
                                                     const int* __restrict__ parents, int beams) {
    typedef __attribute__((__vector_size__(16))) uint32_t V16;
    const Entry e = entries[map[blockIdx.x]];
    const uint32_t u = blockIdx.x - e.first;
    const long text = u / e.cols;
    const uint32_t col = u - (uint32_t)text * e.cols;
    if (e.width == 16) {
        if constexpr (MB <= (int)kWideBeams) move_unit<MB, V16>(e, text, col, parents, beams);
    } else if (e.width == 4) {
        move_unit<MB, uint32_t>(e, text, col, parents, beams);
    } else {
        move_unit<MB, uint8_t>(e, text, col, parents, beams);
    }
}

struct Span {
    uintptr_t from, to;
};
static int by_start(const void* a, const void* b) {
    const uintptr_t x = ((const Span*)a)->from, y = ((const Span*)b)->from;
    return x < y ? -1 : x > y;
}

}  // namespace sr
}  // namespace efla

using namespace efla;

extern "C" int state_list_create_hip(void** list, void* const* states, void* const* outs,
                                     const size_t* row_bytes, size_t count, size_t batch,
                                     size_t beams) {
    if (!list) return kInvalidValue;
    *list = nullptr;
    if (count != 0 && (!states || !row_bytes)) return kInvalidValue;
    if (beams == 0 || beams > sr::kMaxBeams) return kInvalidValue;
    if (count > 0xFFFFFFull || batch > 0x7FFFFFFFull) return kInvalidConfiguration;
    for (size_t i = 0; i < count; ++i) {
        size_t all;
        if (!mul_ok(batch, beams, row_bytes[i], &all) || all > (1ull << 46))
            return kInvalidConfiguration;
        if (all != 0 && (!states[i] || (outs && !outs[i]))) return kInvalidValue;
    }
    const size_t sides = outs ? 2 : 1;
    sr::Entry* entries = (sr::Entry*)calloc(count + 1, sizeof(sr::Entry));
    sr::Span* spans = (sr::Span*)malloc((count * sides + 1) * sizeof(sr::Span));
    sr::List* l = (sr::List*)malloc(sizeof(sr::List));
    uint8_t* host = nullptr;
    void* mem = nullptr;
    size_t units = 0, n = 0, bytes = 0;
    int rc = entries && spans && l ? kSuccess : kOutOfMemory;
    for (size_t i = 0; i < count && rc == kSuccess; ++i) {
        sr::Entry& e = entries[i];
        e.in = (const uint8_t*)states[i];
        e.out = (uint8_t*)(outs ? outs[i] : states[i]);
        e.row = row_bytes[i];
        e.first = (uint32_t)units;
        const uintptr_t any = (uintptr_t)e.in | (uintptr_t)e.out | e.row;
        e.width = any % 16 == 0 && beams <= sr::kWideBeams ? 16 : any % 4 == 0 ? 4 : 1;
        const size_t cols = (e.row + sr::NT * e.width - 1) / (sr::NT * e.width);
        units += cols * batch;
        e.cols = (uint32_t)cols;
        if (units > sr::kMaxUnits) rc = kInvalidConfiguration;
        const size_t all = batch * beams * e.row;
        if (all == 0) continue;
        spans[n++] = sr::Span{(uintptr_t)e.in, (uintptr_t)e.in + all};
        if (outs) spans[n++] = sr::Span{(uintptr_t)e.out, (uintptr_t)e.out + all};
    }
    if (rc == kSuccess) {
        // memory that is written belongs to one tensor
        qsort(spans, n, sizeof(sr::Span), sr::by_start);
        for (size_t i = 1; i < n; ++i)
            if (spans[i].from < spans[i - 1].to) rc = kInvalidValue;
    }
    if (rc == kSuccess) {
        bytes = count * sizeof(sr::Entry) + units * sizeof(uint32_t);
        host = (uint8_t*)malloc(bytes + 1);
        if (!host) rc = kOutOfMemory;
    }
    if (rc == kSuccess) {
        memcpy(host, entries, count * sizeof(sr::Entry));
        uint32_t* map = (uint32_t*)(host + count * sizeof(sr::Entry));
        for (size_t i = 0; i < count; ++i)
            for (size_t k = 0; k < entries[i].cols * batch; ++k) *map++ = (uint32_t)i;
        rc = (int)hipGetDevice(&l->device);
    }
    if (rc == kSuccess && bytes != 0) {
        rc = (int)hipMalloc(&mem, bytes);
        if (rc == kSuccess) rc = (int)hipMemcpy(mem, host, bytes, hipMemcpyHostToDevice);
    }
    free(host);
    free(spans);
    free(entries);
    if (rc != kSuccess) {
        if (mem) (void)hipFree(mem);
        free(l);
        return rc;
    }
    l->batch = batch;
    l->beams = beams;
    l->units = units;
    l->entries = (sr::Entry*)mem;
    l->map = mem ? (uint32_t*)((uint8_t*)mem + count * sizeof(sr::Entry)) : nullptr;
    *list = l;
    return kSuccess;
}

extern "C" int state_list_destroy_hip(void* list) {
    if (!list) return kSuccess;
    sr::List* l = (sr::List*)list;
    const int rc = l->entries ? (int)hipFree(l->entries) : kSuccess;  // waits for the device
    free(l);
    return rc;
}

extern "C" int state_reorder_hip(const void* list, const int32_t* parents, hipStream_t stream) {
    const sr::List* l = (const sr::List*)list;
    if (!l || (l->units != 0 && !parents)) return kInvalidValue;
    int dev = 0;
    EFLA_CHECK(hipGetDevice(&dev));
    if (dev != l->device) return (int)hipErrorInvalidDevice;
    if (l->units == 0) return kSuccess;
    const dim3 grid((unsigned)l->units), block(sr::NT);
    const int beams = (int)l->beams;
#define SR_MOVE(MB)                                                                              \
    EFLA_LAUNCH("state_reorder", sr::reorder_kernel<MB>, grid, block, stream, l->entries, l->map, \
                parents, beams)
    if (beams <= 4) SR_MOVE(4);
    else if (beams <= 8) SR_MOVE(8);
    else if (beams <= 16) SR_MOVE(16);
    else SR_MOVE(64);
#undef SR_MOVE
    return (int)hipPeekAtLastError();
}

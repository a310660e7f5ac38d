// Beam search's selection for gfx950: of all continuations of a text's beams, the best.
//
//   value(k, v) = score_k + z_kv - log sum_v exp z_kv      (beam k, token v, logits z)
//               = (z_kv - max_v z_kv) + (score_k - log sum_v exp (z_kv - max_v z_kv))
//
// (the second form keeps the score and the logarithm beside logits of any size)
// and of a text's beams * vocabulary values the `select` largest, ties to the lowest
// k * vocabulary + v.  Two beams' values are compared in 64 bits, one beam's by their logits.
// A finished beam offers the end token at its own score and nothing else.  A beam whose score is
// not finite, or whose logits have no finite sum of exponentials (a NaN, +inf, -inf everywhere),
// offers nothing: its values are -inf.
//
// The logits are read once and nothing of their size is written.  Two launches (or one where a
// text is small, text_kernel):
//
// slice_kernel: a workgroup takes a slice of one row, 1 to 8 16-byte vectors a thread, in
// registers.  Maximum and sum of exponentials are each thread's own first (no barrier
// stands between load and exponentials), then joined.  For the best n of the slice each
// wave finds the n-th largest of its 64 lanes' maxima, bit by bit with one ballot a
// bit: n logits of the slice are no less, so that is a bound, and the largest of the waves'
// bounds leaves a few tens of a slice's thousands.  Those go to LDS and are ranked by
// counting how many are better (logit, then token: no two are equal, so the order in
// which they arrive does not matter).  Where more pass the bound than LDS has places
// (many equal logits) the best are taken out one by one, each from the memory again: right, and slow
// where that is most of a row (64 x 8 x 128003 fp16, 16 selected, nine tenths masked with the lowest value
// 980 us; with -inf, which is never a candidate, 37).
//
// join_kernel: a workgroup per text joins the slices' sums (64 bits), and does the same
// with the slices' best, whose values it forms in 64 bits.  The bound comes from the slices'
// lists' first entries alone: hardly more than n entries reach their n-th largest.  -inf is never a candidate:
// where fewer than `select` finite values exist, the rest are the lowest pairs (k, v)
// that are not among them, which is what the order above gives.
#include <hip/hip_runtime.h>
#include <math.h>

#include <algorithm>

#include "../../include/efla_hip.h"
#include "common.hpp"
#include "internal.hpp"

namespace efla {
namespace bs {

constexpr int NT = 256, NWV = NT / kWave;
constexpr int kMaxSelect = 64, kMaxBeams = 64;
constexpr size_t kMaxBatch = (1 << 22) - 1;  // 1024 threads each, fewer than 2^32 in a launch
constexpr int kPlaces = 512;   // candidates that LDS holds, a slice's
constexpr int kJoinPlaces = 2048;  // and a text's
constexpr int kVectors = 512;  // and 16-byte vectors that have some

// What is left of a slice: one of its best logits; none: token -1.
struct Cand {
    float z;
    int token;
};

// Whole numbers in the order of the floats that they stand for.
__device__ __forceinline__ uint32_t ordered(float f) {
    const uint32_t b = __float_as_uint(f);
    return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ uint64_t ordered(double f) {
    const uint64_t b = (uint64_t)__double_as_longlong(f);
    return b ^ ((b >> 63) ? ~0ull : 1ull << 63);
}
__device__ __forceinline__ float unordered(uint32_t k) {
    return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}

// A bound that at least n of the wave's 64 keys reach: their n-th largest with its bits
// below LOW cleared.  n <= 64.
template <int LOW>
__device__ __forceinline__ uint32_t wave_bound(uint32_t key, int n) {
    uint32_t got = 0;
#pragma unroll
    for (int b = 31; b >= LOW; --b) {
        const uint32_t t = got | (1u << b);
        if (__popcll(__ballot(key >= t)) >= n) got = t;
    }
    return got;
}

// The same from 256 keys in LDS, one a thread, for larger n, of which 64 groups say little (the
// least of 64 groups' largest lets 300 of 2000 logits through, the 64th of 256 groups' 75;
// up to 32 that costs more than it saves).  The keys have the thread in their low byte,
// so that no two are equal.  A barrier is behind the keys and one in front of *got, which
// holds 0 before.
__device__ __forceinline__ uint32_t with_thread(uint32_t key) {
    return (key & ~255u) | (threadIdx.x & 255u);
}
__device__ __forceinline__ void block_bound(const uint32_t (&keys)[256], int n, uint32_t* got) {
    const uint32_t mine = keys[threadIdx.x];
    int rank = 0;
#pragma unroll 2
    for (int k = 0; k < 256; k += 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(&keys[k]);
        rank += (x.x > mine) + (x.y > mine) + (x.z > mine) + (x.w > mine);
    }
    if (rank == n - 1) *got = mine & ~255u;
}
constexpr int kFewSelect = 32;  // up to here wave_bound does

// Over the wave, in every lane: within rows of 16 by lane permutations, then across them.
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xF,
                                                               0xF, true));
}
template <typename Op>
__device__ __forceinline__ float wave_join(float x, Op op) {
    x = op(x, dpp<0xB1>(x));   // quad_perm [1, 0, 3, 2]
    x = op(x, dpp<0x4E>(x));   // quad_perm [2, 3, 0, 1]
    x = op(x, dpp<0x141>(x));  // row_half_mirror
    x = op(x, dpp<0x140>(x));  // row_mirror
    x = op(x, __shfl_xor(x, 16));
    return op(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float wave_max(float x) {
    return wave_join(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float wave_sum(float x) {
    return wave_join(x, [](float a, float b) { return a + b; });
}

// The largest of a vector's floats, -inf where it has none (NaN is passed over).
template <typename T, typename Vec>
__device__ __forceinline__ float vec_max(Vec x) {
    if constexpr (__is_same(T, f16)) {  // two at a time
        typedef __attribute__((__vector_size__(4))) f16 Pair;
        struct Pairs {
            Pair p[4];
        };
        const Pairs q = __builtin_bit_cast(Pairs, x);
        Pair m = __builtin_elementwise_max(__builtin_elementwise_max(q.p[0], q.p[1]),
                                           __builtin_elementwise_max(q.p[2], q.p[3]));
        return fmaxf((float)m[0], (float)m[1]);
    }
    constexpr int N = 16 / sizeof(T);
    float m = to_f(x[0]);
#pragma unroll
    for (int j = 1; j < N; ++j) m = fmaxf(m, to_f(x[j]));
    return m;
}
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float exp_diff(float d) {  // e^d
    return __builtin_amdgcn_exp2f(d * kLog2e);
}

// c = m log2 e up to here is rounded by 2^20 1.45 / 2^24 at most.
constexpr float kNear = 0x1p20f;

// A row's vectors start at cache lines: element i of the row is at i + shift, shift its
// first element's place in its line, and slice s holds [s L, (s + 1) L) of that.
template <typename T, int VPT>
__global__ void __launch_bounds__(NT)
slice_kernel(const T* __restrict__ logits, long ld, int V, int n,
             const float* __restrict__ scores, const uint8_t* __restrict__ finished,
             float2* __restrict__ stats, Cand* __restrict__ cands) {
    constexpr int N = 16 / sizeof(T), L = NT * VPT * N;
    typedef __attribute__((__vector_size__(16))) T Vec;
    __shared__ Vec piece[kVectors];
    __shared__ int piece_at[kVectors];  // its first token
    __shared__ uint64_t place[kPlaces];
    __shared__ float wm[NWV], ws[NWV];
    __shared__ __attribute__((aligned(16))) uint32_t lanes[NT];
    __shared__ uint32_t exact;
    __shared__ uint64_t best[NWV];
    __shared__ int pieces, count;
    const long row = blockIdx.y;
    // a beam that offers no continuation is not read
    if ((finished && finished[row]) || !(fabsf(scores[row]) < INFINITY)) return;
    const T* p = logits + row * ld;
    const int shift = (int)((uintptr_t)p % 128 / sizeof(T));
    const long v0 = (long)blockIdx.x * L - shift;  // the slice's first token
    if (threadIdx.x == 0) pieces = count = 0, exact = 0;

    Vec x[VPT];
    if (v0 >= 0 && v0 + L <= V) {  // the whole slice lies in the row
        const Vec* q = reinterpret_cast<const Vec*>(p + v0);
#pragma unroll
        for (int i = 0; i < VPT; ++i) x[i] = q[threadIdx.x + i * NT];
    } else {
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const long v = v0 + (long)(threadIdx.x + i * NT) * N;
            if (v >= 0 && v + N <= V) {
                x[i] = *reinterpret_cast<const Vec*>(p + v);
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j)
                    x[i][j] = v + j >= 0 && v + j < V ? p[v + j] : (T)-INFINITY;
            }
        }
    }
    float vm[VPT], m = -INFINITY;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        vm[i] = vec_max<T>(x[i]);
        vm[i] = fmaxf(vm[i], -INFINITY) + 0.f;  // no NaN, and -0 is 0
        m = fmaxf(m, vm[i]);
    }
    // Up to kNear the sum of 2^(z log2 e - c), c = m log2 e rounded: one fused operation and one
    // exponential an element; what the rounding of c left out, an exponent of 0.1 at most, is
    // taken back at the end, so that only z - m meets the constant's own error.  Further from zero it
    // would be hundreds, and z - m comes first.  A thread without a logit above -inf: 0, or NaN from a NaN.
    const float m0 = m == -INFINITY ? 0.f : m;
    float s = 0.f;
    auto sum = [&](auto term) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            asm volatile("" : "+v"(x[i]));  // converted again: the fp32 values take four times the registers
#pragma unroll
            for (int j = 0; j < N; ++j) s += term(to_f(x[i][j]));
        }
    };
    if (__is_same(T, f16) || fabsf(m0) <= kNear) {  // (fp16's largest value is nearer)
        float f = kLog2e;
        asm("" : "+v"(f));  // a vector register: 64 x 8 x 128003 fp16 27.7 us, 28.2 from a scalar one
        const float c0 = m0 * f;
        sum([&](float z) { return __builtin_amdgcn_exp2f(fmaf(z, f, -c0)); });
        s *= __builtin_amdgcn_exp2f(-fmaf(m0, f, -c0));
    } else {
        sum([&](float z) { return exp_diff(z - m0); });
    }
    const float M = wave_max(m), M0 = M == -INFINITY ? 0.f : M;
    s = wave_sum(s * exp_diff(fminf(m0 - M0, 0.f)));
    if (lane_id() == 0) {
        wm[wave_id()] = M;
        ws[wave_id()] = s;
    }
    lanes[threadIdx.x] = n <= kFewSelect ? ordered(m) : with_thread(ordered(m));
    __syncthreads();
    uint32_t least;
    if (n <= kFewSelect) {
        uint32_t group = lanes[lane_id()];
#pragma unroll
        for (int k = 1; k < NWV; ++k) group = max(group, lanes[lane_id() + k * kWave]);
        least = wave_bound<sizeof(T) == 2 && !__is_same(T, f16) ? 16 : 12>(group, n);
    } else {
        block_bound(lanes, n, &exact);
        __syncthreads();
        least = exact;
    }
    // vectors that reach the bound
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        if (vm[i] == -INFINITY || ordered(vm[i]) < least) continue;
        const int at = atomicAdd(&pieces, 1);
        if (at < kVectors) {
            piece[at] = x[i];
            piece_at[at] = (int)(v0 + (long)(threadIdx.x + i * NT) * N);
        }
    }
    const long slot = row * gridDim.x + blockIdx.x;
    if (threadIdx.x == 0) {
        float W = wm[0];
#pragma unroll
        for (int k = 1; k < NWV; ++k) W = fmaxf(W, wm[k]);
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < NWV; ++k)
            sum += wm[k] == -INFINITY ? ws[k] : ws[k] * exp_diff(wm[k] - W);
        stats[slot] = make_float2(W, sum);
    }
    __syncthreads();
    // key: the logit, then the lower token; 0: none
    auto key_of = [](T logit, uint32_t v) {
        const float z = to_f(logit) + 0.f;
        return z > -INFINITY ? (uint64_t)ordered(z) << 32 | (uint32_t)~v : 0ull;
    };
    Cand* out = cands + slot * n;
    auto write = [&](int rank, uint64_t key) {
        out[rank] = Cand{unordered((uint32_t)(key >> 32)), (int)~(uint32_t)key};
    };
    // their elements that do
    const int np = pieces;
    if (np <= kVectors) {
        for (int i = threadIdx.x; i < np * N; i += NT) {
            const T* e = reinterpret_cast<const T*>(&piece[i / N]);
            const uint64_t key = key_of(e[i % N], (uint32_t)(piece_at[i / N] + i % N));
            if (key != 0 && (uint32_t)(key >> 32) >= least) {
                const int at = atomicAdd(&count, 1);
                if (at < kPlaces) place[at] = key;
            }
        }
    }
    __syncthreads();
    const int c = count;
    if (np <= kVectors && c <= kPlaces) {
        for (int i = threadIdx.x; i < c; i += NT) {
            const uint64_t mine = place[i];
            int rank = 0;
#pragma unroll 4
            for (int k = 0; k < c; ++k) rank += place[k] > mine;
            if (rank < n) write(rank, mine);
        }
        for (int i = c + threadIdx.x; i < n; i += NT) out[i] = Cand{0.f, -1};
        return;
    }
    // too many (equal logits): the best, then the best below it, n times; read again, since
    // the loop would keep every key in registers
    uint64_t last = ~0ull;
    for (int r = 0; r < n; ++r) {
        uint64_t top = 0;
        for (int i = threadIdx.x; i < L; i += NT) {
            const long v = v0 + i;
            if (v < 0 || v >= V) continue;
            const uint64_t key = key_of(p[v], (uint32_t)v);
            if (key < last && key > top) top = key;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const uint64_t other = __shfl_xor(top, o);
            if (other > top) top = other;
        }
        __syncthreads();  // `best` has been read
        if (lane_id() == 0) best[wave_id()] = top;
        __syncthreads();
        last = best[0];
#pragma unroll
        for (int k = 1; k < NWV; ++k)
            if (best[k] > last) last = best[k];
        if (threadIdx.x == 0) out[r] = Cand{0.f, -1};
        if (threadIdx.x == 0 && last != 0) write(r, last);
    }
}

// A candidate of the join: its value and its place in the order of ties.
struct Best {
    double value;
    int beam, token;
};
// With its logit, as `ordered`.  A beam's own order is that of its logits, which 64 bits do not always
// leave in the values (a score of -1e30 for a beam that does not count, a logit of 1e30).
struct Candidate : Best {
    uint32_t z;
};
__device__ __forceinline__ bool better(const Candidate& a, const Candidate& b) {
    if (a.value != b.value) return a.value > b.value;
    if (a.beam != b.beam) return a.beam < b.beam;
    if (a.z != b.z) return a.z > b.z;
    return a.token < b.token;
}
// Whether value = (z - top) + offset may be that of another logit of the beam too.  Logits differ by
// 2^-24 of the larger at least, and the value's two roundings are 2^-52 of |z| + |top| + |offset|
// together: two of those are less, unless z is this small.  (0 is as far from the others as they from it.)
__device__ __forceinline__ bool merges(float z, float top, double offset) {
    return z != 0.f && fabs((double)z) * 0x1p26 < fabs((double)top) + fabs(offset);
}

// Whole numbers in the values' order, 0: not a candidate.
__device__ __forceinline__ uint32_t key_of(double v) {
    return v > -(double)INFINITY ? (uint32_t)(ordered(v + 0.0) >> 32) : 0u;
}

// What a text's selection is written to.
struct Selected {
    float* scores;
    int* parents;
    int* tokens;
    uint8_t* finished;
};

// Candidates that reach the bound, in the order in which they arrive.
struct Places {
    Best at[kJoinPlaces];
    uint32_t z[kJoinPlaces];
    int count, merged;  // whether logits have to be compared
    __device__ __forceinline__ void clear() { count = merged = 0; }
    __device__ __forceinline__ void take(const Candidate& c, float top, double offset) {
        const int i = atomicAdd(&count, 1);
        if (i < kJoinPlaces) {
            at[i] = c;
            z[i] = c.z;
        }
        if (merges(unordered(c.z), top, offset)) merged = 1;
    }
};

// The n best of the candidates in `place`, or, where it has not held them all (equal values), of
// those that `each` hands to a function, a thread its own, into `res` in order; all threads.
template <int NTJ, typename Each>
__device__ __forceinline__ void rank(int n, int beams, const Places& place, Best* res,
                                     Candidate* wbest, Each each) {
    const int found = place.count;
    if (found <= kJoinPlaces) {
        const bool merged = place.merged;
        for (int i = threadIdx.x; i < found; i += NTJ) {
            const Best b = place.at[i];
            int rank = 0;
            if (merged) {
                const Candidate c{b, place.z[i]};
                for (int k = 0; k < found; ++k)
                    rank += better(Candidate{place.at[k], place.z[k]}, c);
            } else {
                // without branches, so that the reads need not wait for each other
#pragma unroll 4
                for (int k = 0; k < found; ++k) {
                    const Best x = place.at[k];
                    const bool before =
                        (x.beam < b.beam) | ((x.beam == b.beam) & (x.token < b.token));
                    rank += (x.value > b.value) | ((x.value == b.value) & before);
                }
            }
            if (rank < n) res[rank] = b;
        }
    } else {
        // the best, then the best behind it, n times
        Candidate last{{(double)INFINITY, -1, -1}, 0};
        for (int r = 0; r < n; ++r) {
            Candidate b{{-(double)INFINITY, beams, 0}, 0};
            each([&](const Candidate& x) {
                if (x.value > -(double)INFINITY && better(last, x) && better(x, b)) b = x;
            });
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) {
                const Candidate x{{__shfl_xor(b.value, o), __shfl_xor(b.beam, o),
                                   __shfl_xor(b.token, o)}, __shfl_xor(b.z, o)};
                if (better(x, b)) b = x;
            }
            __syncthreads();  // `wbest` has been read
            if (lane_id() == 0) wbest[wave_id()] = b;
            __syncthreads();
            last = wbest[0];
#pragma unroll
            for (int k = 1; k < NTJ / kWave; ++k)
                if (better(wbest[k], last)) last = wbest[k];
            if (threadIdx.x == 0) res[r] = last;
        }
    }
    __syncthreads();
}

// The selected, the first wave's.  (Others have read the text's marks in front of a barrier.)
__device__ __forceinline__ void write(Best* res, int found, int n, int V, long text, long row0,
                                      const uint8_t* finished, int end_token, int keep_slots,
                                      const Selected& out) {
    if (wave_id() != 0) return;
    const int r = lane_id();
    // fewer finite values than asked for: the lowest pairs that are not among them
    if (found < n) {
        if (r == 0) {
            int beam = 0, token = 0;
            for (int to = found; to < n;) {
                bool taken = false;
                for (int k = 0; k < found; ++k)
                    taken |= res[k].beam == beam && res[k].token == token;
                if (!taken) res[to++] = Best{-(double)INFINITY, beam, token};
                if (++token == V) token = 0, ++beam;
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    const Best b = res[r < n ? r : n - 1];
    int to = r;
    if (keep_slots) {
        // the first child of a beam takes that beam's slot, the others the free ones in order
        uint64_t used = 0;
        bool first = true;
        for (int k = 0; k < n; ++k) {
            const int other = __builtin_amdgcn_readlane(b.beam, k);
            used |= 1ull << other;
            if (k < r && other == b.beam) first = false;
        }
        const uint64_t late = __ballot(!first && r < n);
        to = b.beam;
        if (!first) {
            uint64_t open = ~used;
            for (int k = __popcll(late & ((1ull << r) - 1)); k > 0; --k) open &= open - 1;
            to = __ffsll((unsigned long long)open) - 1;
        }
    }
    // the marks may be written over those that they come from: all are read before
    bool ended = b.token == end_token;
    if (finished) ended |= finished[row0 + b.beam] != 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (r >= n) return;
    const long at = text * n + to;
    out.scores[at] = (float)b.value;
    out.parents[at] = b.beam;
    out.tokens[at] = b.token;
    if (out.finished) out.finished[at] = ended;
}

constexpr int kHeads = 2;

// An entry a thread is held, NTJ of them; more are read twice.  (Eight entries a thread: 17 KB
// of code that a workgroup runs through once, 8.5 us for 800 entries of each of 16 texts; 1024
// threads 6.7.)
template <int NTJ>
__global__ void __launch_bounds__(NTJ)
join_kernel(const float2* __restrict__ stats, const Cand* __restrict__ cands, int slices,
            const float* __restrict__ scores, const uint8_t* finished, int V,
            int beams, int n, int end_token, int keep_slots, Selected out) {
    __shared__ double offset[kMaxBeams];  // score - log sum exp (z - top)
    __shared__ float tops[kMaxBeams];     // the largest logit
    __shared__ int state[kMaxBeams];      // 0: live, 1: finished, 2: offers nothing
    __shared__ Places place;
    __shared__ Best res[kMaxSelect];
    __shared__ Candidate wbest[NTJ / kWave];
    __shared__ __attribute__((aligned(16))) uint32_t groups[256];
    __shared__ uint32_t exact;
    const long text = blockIdx.x, row0 = text * beams;
    const int per = slices * n, total = beams * per;
    const Cand* mine = cands + row0 * per;
    // On their way while the sums are joined: an entry a thread, and the lists' heads, a few to
    // each lane or (many to select) one to each of 256 threads.  Where there are fewer lists,
    // their second entries are among them, and so on.  (What beams that were not read
    // left there is not looked at.)
    const int e0 = (int)threadIdx.x;
    const Cand held = e0 < total ? mine[e0] : Cand{0.f, -1};
    const int lists = beams * slices;
    const bool few = n <= kFewSelect;
    int from[kHeads];
    Cand head[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
        const int j = few ? lane_id() + i * kWave : e0 + i * 256, depth = j / lists;
        from[i] = depth < n ? (j - depth * lists) * n + depth : total;
        head[i] = depth < n ? mine[from[i]] : Cand{0.f, -1};
    }
    if (threadIdx.x == 0) place.clear(), exact = 0;
    // 16 lanes to a beam
    for (int k = threadIdx.x / 16; k < beams; k += NTJ / 16) {
        const int l = threadIdx.x % 16;
        const float2* st = stats + (row0 + k) * slices;
        float2 a = l < slices ? st[l] : make_float2(-INFINITY, 0.f);
        const float score = scores[row0 + k];
        const bool fin = finished && finished[row0 + k], ok = fabsf(score) < INFINITY;
        float M = a.x;
        for (int i = l + 16; i < slices; i += 16) M = fmaxf(M, st[i].x);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 16));
        double s = 0.0;
        for (int i = l; i < slices; i += 16) {
            if (i != l) a = st[i];
            // a slice without a logit above -inf: 0, or NaN from a NaN
            s += a.x < M ? (double)a.y * (double)exp_diff(a.x - M) : (double)a.y;
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) s += __shfl_xor(s, o, 16);
        const double ls = fin ? 0.0 : log(s);
        if (l == 0) {
            const bool live = ok && fabs(ls) < (double)INFINITY && (fin || M > -INFINITY);
            state[k] = !live ? 2 : fin ? 1 : 0;
            offset[k] = (double)score - ls;
            tops[k] = M;
        }
    }
    __syncthreads();
    // entry e from what the slice left; a finished beam has one entry
    auto best_of = [&](int e, const Cand& x) {
        Candidate b{{-(double)INFINITY, 0, 0}, 0};
        if (e >= total) return b;
        b.beam = (int)((unsigned)e / (unsigned)per);
        if (state[b.beam] == 0) {
            if (x.token >= 0) b.value = ((double)x.z - (double)tops[b.beam]) + offset[b.beam];
            b.token = x.token;
            b.z = ordered(x.z);
        } else if (state[b.beam] == 1 && e == b.beam * per) {
            b.value = offset[b.beam];
            b.token = end_token;
        }
        return b;
    };
    const Candidate first = best_of(e0, held);
    // The bound from the largest of some lists: 64 lanes', in every wave by itself, or 256 threads'.
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kHeads; ++i)
        top = max(top, key_of(best_of(from[i], head[i]).value));
    for (int j = (few ? lane_id() + kHeads * kWave : e0 + kHeads * 256); j < lists;
         j += few ? kWave : 256)
        top = max(top, key_of(best_of(j * n, mine[j * n]).value));
    uint32_t least;
    if (few) {
        least = wave_bound<4>(top, n);
    } else {
        if (e0 < 256) groups[e0] = with_thread(top);
        __syncthreads();
        if (e0 < 256) block_bound(groups, n, &exact);
        __syncthreads();
        least = exact;
    }
    least = max(least, 1u);
    auto take = [&](const Candidate& b) {
        if (key_of(b.value) >= least) place.take(b, tops[b.beam], offset[b.beam]);
    };
    take(first);
    for (int e = e0 + NTJ; e < total; e += NTJ) take(best_of(e, mine[e]));
    __syncthreads();
    rank<NTJ>(n, beams, place, res, wbest, [&](auto f) {
        for (int e = e0; e < total; e += NTJ) f(best_of(e, mine[e]));
    });
    write(res, place.count, n, V, text, row0, finished, end_token, keep_slots, out);
}

// A whole text in a workgroup, for texts of few logits (kTextLogits), where a second launch is
// longer than the work: each beam is some waves', and what slice_kernel and join_kernel
// do follows in one place.  The logits that the bound leaves are few threads', which
// read theirs again.  A call through Python, this and both launches, us (bf16 unless said):
//   1 x 2 x 798 11.0 / 15.5   1 x 4 x 8000 11.2 / 15.3   256 x 4 x 8000 11.2 / 15.3
//   85 x 5 x 7936 fp32 11.2 / 15.9   1000 x 4 x 2000 22 / 30   1 x 4 x 32000 20.3 / 15.3
constexpr int kTextThreads = 1024, kTextBeams = kTextThreads / kWave;
constexpr size_t kTextLogits = 49152;

template <typename T>
__global__ void __launch_bounds__(kTextThreads)
text_kernel(const T* __restrict__ logits, long ld, int V, int beams, int n,
            const float* __restrict__ scores, const uint8_t* finished, int end_token,
            int keep_slots, Selected out) {
    constexpr int N = 16 / sizeof(T), NTJ = kTextThreads, W = NTJ / kWave, U = 4;
    typedef __attribute__((__vector_size__(16))) T Vec;
    __shared__ double offset[kTextBeams];  // score - log sum exp (z - top); -inf: offers nothing
    __shared__ float tops[kTextBeams];     // the largest logit
    __shared__ Places place;
    __shared__ Best res[kMaxSelect];
    __shared__ Candidate wbest[W];
    __shared__ float wm[W], ws[W];
    __shared__ uint32_t groups[NTJ];
    const long text = blockIdx.x, row0 = text * beams;
    if (threadIdx.x == 0) place.clear();
    const int waves = W / beams, P = waves * kWave;  // a beam's
    const int k = wave_id() / waves, t = (int)threadIdx.x - k * P;
    const bool has = k < beams;
    const float score = has ? scores[row0 + k] : -INFINITY;
    const bool ok = fabsf(score) < INFINITY, fin = has && finished && finished[row0 + k];
    const bool live = ok && !fin;  // a beam that offers no continuation is not read
    // the row's vectors from 16-byte boundaries on, and the elements before and behind them
    const T* p = logits + (row0 + (has ? k : 0)) * ld;
    const int to16 = (int)(-(uintptr_t)p % 16 / sizeof(T)), head = to16 < V ? to16 : V;
    const int nv = live ? (V - head) / N : 0, edges = live ? V - nv * N : 0;
    const Vec* q = reinterpret_cast<const Vec*>(p + head);
    const int edge = t < head ? t : t + nv * N;
    float m = -INFINITY, s = 0.f;
    auto add = [&](float top, auto sum_of) {  // logits whose largest is `top`
        const float now = fmaxf(m, top) + 0.f, m0 = now == -INFINITY ? 0.f : now;
        s = s * exp_diff(fminf(m - m0, 0.f)) + sum_of(m0);
        m = now;
    };
    for (int v0 = t; v0 < nv; v0 += U * P) {
        Vec x[U];
#pragma unroll
        for (int i = 0; i < U; ++i) {
#pragma unroll
            for (int j = 0; j < N; ++j) x[i][j] = (T)-INFINITY;
            if (v0 + i * P < nv) x[i] = q[v0 + i * P];
        }
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < U; ++i) top = fmaxf(top, vec_max<T>(x[i]));
        add(top, [&](float m0) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < U; ++i)
#pragma unroll
                for (int j = 0; j < N; ++j) sum += exp_diff(to_f(x[i][j]) - m0);
            return sum;
        });
    }
    if (t < edges) {
        const float z = to_f(p[edge]);
        add(z, [&](float m0) { return exp_diff(z - m0); });
    }
    const float M = wave_max(m), M0 = M == -INFINITY ? 0.f : M;
    const float sum = wave_sum(s * exp_diff(fminf(m == -INFINITY ? 0.f : m - M0, 0.f)));
    if (lane_id() == 0) {
        wm[wave_id()] = M;
        ws[wave_id()] = sum;
    }
    __syncthreads();
    if (has && t == 0) {
        float Mb = -INFINITY;
        for (int i = 0; i < waves; ++i) Mb = fmaxf(Mb, wm[k * waves + i]);
        double S = 0.0;
        for (int i = 0; i < waves; ++i) {
            const float a = wm[k * waves + i], b = ws[k * waves + i];
            S += a < Mb ? (double)b * (double)exp_diff(a - Mb) : (double)b;
        }
        const double ls = fin ? 0.0 : log(S);
        const bool offers = ok && fabs(ls) < (double)INFINITY && (fin || Mb > -INFINITY);
        offset[k] = offers ? (double)score - ls : -(double)INFINITY;
        tops[k] = Mb;
    }
    __syncthreads();
    const double off = has ? offset[k] : -(double)INFINITY;
    const float beam_top = has ? tops[k] : 0.f;
    auto value_of = [&](float z) { return ((double)z - (double)beam_top) + off; };
    auto best_of = [&](T logit, int token) {
        const float z = to_f(logit) + 0.f;  // -0 is 0
        return Candidate{{value_of(z), k, token}, ordered(z)};
    };
    // a thread's candidates whose keys are no less than `from`, and some that are; a finished
    // beam has one
    auto each = [&](uint32_t from, auto f) {
        if (!(off > -(double)INFINITY)) return;
        if (fin) {
            if (t == 0) f(Candidate{{off, k, end_token}, ordered(0.f)});
            return;
        }
        for (int v = t; v < nv; v += P) {
            const Vec x = q[v];
            if (key_of(value_of(vec_max<T>(x))) < from) continue;
#pragma unroll
            for (int j = 0; j < N; ++j) f(best_of(x[j], head + v * N + j));
        }
        if (t < edges) f(best_of(p[edge], edge));
    };
    const uint32_t mine = fin ? (t == 0 ? key_of(off) : 0u) : key_of(value_of(m));
    groups[threadIdx.x] = mine;
    __syncthreads();
    uint32_t group = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) group = max(group, groups[lane_id() + i * kWave]);
    const uint32_t least = max(wave_bound<4>(group, n), 1u);
    if (mine >= least)
        each(least, [&](const Candidate& b) {
            if (key_of(b.value) >= least) place.take(b, beam_top, off);
        });
    __syncthreads();
    rank<NTJ>(n, beams, place, res, wbest, [&](auto f) { each(1, f); });
    write(res, place.count, n, V, text, row0, finished, end_token, keep_slots, out);
}

static size_t dtype_size(int d) {
    return d == kDtypeF32 ? 4 : d == kDtypeF16 || d == kDtypeBF16 ? 2 : 0;
}

// Vectors a thread: as many as leave the chip four workgroups for each of its compute units.
static int vectors(size_t rows, size_t vocab, size_t size) {
    const size_t cus = device_cu_count() > 0 ? device_cu_count() : 256;
    for (int v = 8; v > 1; v /= 2)
        if (rows * ((vocab * size + NT * 16 * v - 1) / (NT * 16 * v)) >= 4 * cus) return v;
    return 1;
}
// Slices of a row of whatever alignment.
static size_t slices_of(size_t vocab, size_t size, int vpt, bool lines) {
    const size_t l = (size_t)NT * vpt * 16 / size, shift = lines ? 0 : 128 / size - 1;
    return (vocab + shift + l - 1) / l;
}

// Whether a text is one workgroup's.
static bool one_workgroup(size_t beams, size_t vocab, size_t n) {
    return beams <= kTextBeams && n <= kFewSelect && beams * vocab <= kTextLogits;
}

static size_t slice_bytes(size_t n) { return sizeof(float2) + n * sizeof(Cand); }

// Room for the slices of either element size at any alignment, growing with every argument.  vectors()
// takes fewer than 8 only where twice as many would leave fewer than 4 cus slices in all, so that there are no
// more than 8 cus and one a row; with 8 the 4-byte logits have the most, and one vector of those is the
// finest cut.
static size_t scratch(size_t batch, size_t beams, size_t vocab, size_t n) {
    if (one_workgroup(beams, vocab, n)) return 0;
    const size_t cus = device_cu_count() > 0 ? device_cu_count() : 256, rows = batch * beams;
    const size_t finest = rows * slices_of(vocab, 4, 1, false);
    const size_t few = 8 * cus + rows, many = rows * slices_of(vocab, 4, 8, false);
    return std::max(many, std::min(few, finest)) * slice_bytes(n);
}

template <typename T>
static void launch(const void* logits, const float* scores, const uint8_t* finished,
                   const uint8_t* ws, size_t rows, size_t vocab, size_t ld, size_t n,
                   int vpt, size_t slices, hipStream_t st) {
    float2* stats = (float2*)ws;
    Cand* cands = (Cand*)(stats + rows * slices);
    const T* z = (const T*)logits;
    for (size_t r0 = 0; r0 < rows; r0 += 32768) {
        const dim3 grid((unsigned)slices, (unsigned)(rows - r0 < 32768 ? rows - r0 : 32768));
        const size_t s0 = r0 * slices;
#define BS_SLICE(VPT)                                                                          \
    EFLA_LAUNCH("beam_slice", (slice_kernel<T, VPT>), grid, dim3(NT), st, z + r0 * ld, (long)ld, \
                (int)vocab, (int)n, scores + r0, finished ? finished + r0 : nullptr, \
                stats + s0, cands + s0 * n)
        if (vpt == 1) BS_SLICE(1);
        else if (vpt == 2) BS_SLICE(2);
        else if (vpt == 4) BS_SLICE(4);
        else BS_SLICE(8);
#undef BS_SLICE
    }
}

}  // namespace bs
}  // namespace efla

using namespace efla;

extern "C" size_t beam_select_workspace_size(size_t batch, size_t beams, size_t vocab_size,
                                             size_t select) {
    if (beams > bs::kMaxBeams || select > bs::kMaxSelect || vocab_size > 0x3FFFFFFFull ||
        batch > bs::kMaxBatch)
        return 0;
    return bs::scratch(batch, beams, vocab_size, select);
}

extern "C" int beam_select_hip(const void* logits, const float* scores, const uint8_t* finished,
                               float* out_scores, int32_t* out_parents, int32_t* out_tokens,
                               uint8_t* out_finished, size_t batch, size_t beams,
                               size_t vocab_size, size_t ld, size_t select, int32_t end_token,
                               int keep_slots, int dtype, void* workspace, size_t workspace_bytes,
                               hipStream_t stream) {
    const size_t size = bs::dtype_size(dtype);
    if (size == 0 || beams == 0 || beams > bs::kMaxBeams || select == 0 ||
        select > bs::kMaxSelect || vocab_size == 0 || ld < vocab_size)
        return kInvalidValue;
    if ((keep_slots && select != beams) || beams * vocab_size < select) return kInvalidValue;
    if ((finished || out_finished) && (end_token < 0 || (size_t)end_token >= vocab_size))
        return kInvalidValue;
    if (batch == 0) return kSuccess;
    if (!logits || !scores || !out_scores || !out_parents || !out_tokens) return kInvalidValue;
    if ((uintptr_t)logits % size) return kInvalidValue;
    size_t rows, elems;
    if (vocab_size > 0x3FFFFFFFull || batch > bs::kMaxBatch || !mul_ok(batch, beams, &rows) ||
        !mul_ok(rows, ld, size, &elems) || elems > (1ull << 62))
        return kInvalidConfiguration;
    const bs::Selected out{out_scores, out_parents, out_tokens, out_finished};
    if (bs::one_workgroup(beams, vocab_size, select)) {
#define BS_TEXT(T)                                                                                \
    EFLA_LAUNCH("beam_text", bs::text_kernel<T>, dim3((unsigned)batch), dim3(bs::kTextThreads),  \
                stream, (const T*)logits, (long)ld, (int)vocab_size, (int)beams, (int)select,    \
                scores, finished, (int)end_token, keep_slots, out)
        if (dtype == kDtypeBF16) BS_TEXT(bf16);
        else if (dtype == kDtypeF16) BS_TEXT(f16);
        else BS_TEXT(float);
#undef BS_TEXT
        return (int)hipPeekAtLastError();
    }
    const size_t need = bs::scratch(batch, beams, vocab_size, select);
    void* ws = workspace;
    WsLease lease;
    if (!ws) {
        const int rc = workspace_acquire(need, stream, &ws, lease);
        if (rc != kSuccess) return rc;
    } else if (workspace_bytes < need || (uintptr_t)ws % 8) {
        return kInvalidValue;
    }
    const int vpt = bs::vectors(rows, vocab_size, size);
    const bool lines = (uintptr_t)logits % 128 == 0 && ld * size % 128 == 0;
    const size_t slices = bs::slices_of(vocab_size, size, vpt, lines);
    if (rows * slices * bs::slice_bytes(select) > need) return kInvalidConfiguration;
    if (dtype == kDtypeBF16)
        bs::launch<bf16>(logits, scores, finished, (const uint8_t*)ws, rows, vocab_size, ld,
                         select, vpt, slices, stream);
    else if (dtype == kDtypeF16)
        bs::launch<f16>(logits, scores, finished, (const uint8_t*)ws, rows, vocab_size, ld,
                        select, vpt, slices, stream);
    else
        bs::launch<float>(logits, scores, finished, (const uint8_t*)ws, rows, vocab_size, ld,
                          select, vpt, slices, stream);
    EFLA_CHECK(hipPeekAtLastError());
    const float2* stats = (const float2*)ws;
#define BS_JOIN(NTJ)                                                                             \
    EFLA_LAUNCH("beam_join", bs::join_kernel<NTJ>, dim3((unsigned)batch), dim3(NTJ), stream, stats, \
                (const bs::Cand*)(stats + rows * slices), (int)slices, scores, finished,          \
                (int)vocab_size, (int)beams, (int)select, (int)end_token, keep_slots, out)
    if (beams * slices * select <= 256) BS_JOIN(256);
    else BS_JOIN(1024);
#undef BS_JOIN
    return (int)hipPeekAtLastError();
}

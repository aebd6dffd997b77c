// Global gradient norm over many tensors, clipping in place, and the Adam step
// that applies the clipping coefficient without rewriting the gradients.
//
//   norm = (sum |g|^p)^(1/p) over all elements of all tensors, p = 1 or 2, or max |g|
//   c    = min(1, max_norm / (norm + 1e-6)),   g <- g * c
//
// Nothing here has a counterpart in the reference, which never bounds its
// gradients.  A launch takes a table of tensors by value (no copy to the
// device, so it can be captured into a graph); the tensors are cut into
// chunks, each of n <= 2048 workgroups sums every n-th chunk, and the
// workgroups' sums are added in a fixed order: the norm is the same bits in
// every run.
// Sums are held in 64 bits: squares of float32 values neither overflow nor
// vanish there.
#include "kernels.h"

#include <type_traits>

namespace gs {

constexpr int NORM_THREADS = 256;
constexpr int NORM_TABLE = 240;     // tensors per launch of the norm and scale kernels (kernel arguments: 3.9 KB)
constexpr int NORM_GROUPS = 2048;   // workgroups of the norm kernel at most: eight per CU
constexpr int ADAM_TABLE = 40;      // tensors per launch of the Adam kernel
constexpr int CHUNK_BYTES = 16384;  // a chunk of a tensor, from its start rounded down to 16 bytes: four vectors a thread
constexpr int ADAM_CHUNK = 2048;    // elements of a workgroup of the dense Adam kernel: two vectors a thread
constexpr int SPARSE_CHUNK = 8192;  // elements of the rows of a workgroup of the sparse one, about

// 16 bytes per tensor.
struct NormTable {
    const void* ptr[NORM_TABLE];
    uint32_t first[NORM_TABLE];       // first chunk of each tensor
    uint32_t shape[NORM_TABLE];       // type | (bytes of the last chunk) << 2
    uint32_t chunks;                  // of the launch
    int n;
};

typedef float f32x4 __attribute__((ext_vector_type(4)));

struct AdamEntry {
    float *param, *exp_avg, *exp_avg_sq;
    const float* grad;
    int64_t count;                    // elements, or rows for the sparse kernel
    uint32_t width;                   // elements per row
    AdamConst c;
};
struct AdamTable {
    AdamEntry e[ADAM_TABLE];
    uint32_t first[ADAM_TABLE];       // first workgroup of each tensor
    int n;
};

// What the norm leaves for its consumers at the start of the temp area.
struct NormResult {
    double norm;
    float coefficient;
};

template <typename Table>
__device__ __forceinline__ int find_tensor(const Table& t, uint32_t chunk) {
    int lo = 0, hi = t.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= chunk) lo = mid; else hi = mid - 1;
    }
    return lo;
}

__device__ __forceinline__ float bf16_to_float(uint16_t v) { return __builtin_bit_cast(float, (uint32_t)v << 16); }
// Round to nearest, ties to even; a NaN keeps its upper bits and stays a NaN.
__device__ __forceinline__ uint16_t float_to_bf16(float f) {
    const uint32_t u = __builtin_bit_cast(uint32_t, f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);
    return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}

__device__ __forceinline__ float f16_to_float(uint16_t v) { return (float)__builtin_bit_cast(_Float16, v); }
__device__ __forceinline__ uint16_t float_to_f16(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }

__device__ __forceinline__ int type_bytes(int type) { return type == GSO_F32 ? 4 : 2; }

// What a workgroup does with one chunk: vectors of 16 bytes that lie wholly in the tensor, and the elements before the
// first and after the last of those one by one.
struct Chunk {
    char* base;          // 16-byte aligned
    int begin, end;      // bytes of the chunk that belong to the tensor
    int type;
};
__device__ __forceinline__ Chunk chunk_of(const NormTable& t, int k, uint32_t chunk) {
    Chunk c;
    const uintptr_t p = (uintptr_t)t.ptr[k];
    const uint32_t within = chunk - t.first[k], last = (k + 1 < t.n ? t.first[k + 1] : t.chunks) - 1;
    c.type = (int)(t.shape[k] & 3u);
    c.base = (char*)(p & ~(uintptr_t)15) + (size_t)within * CHUNK_BYTES;
    c.begin = within == 0 ? (int)(p & 15) : 0;
    c.end = chunk == last ? (int)(t.shape[k] >> 2) : CHUNK_BYTES;
    return c;
}
template <typename V, typename E>
__device__ __forceinline__ void for_chunk(const Chunk& c, int tid, V vectors, E element) {   // tid: 0 .. NORM_THREADS - 1
    const int lo = (c.begin + 15) >> 4, hi = c.end >> 4;
    vectors(lo, hi);
    const int es = type_bytes(c.type);
    if (c.begin != 0 || (c.end & 15) != 0) {   // at most seven elements at either end
        const int head_end = lo << 4 < c.end ? lo << 4 : c.end, tail = hi >= lo ? hi << 4 : c.end;
        const int x = tid < 64 ? c.begin + tid * es : tail + (tid - 64) * es;
        if (tid < 8 ? x < head_end : tid >= 64 && tid < 72 && x < c.end) element(x);
    }
}

// One value's share of the sum.  For the largest absolute value the sum is replaced by the maximum of the absolute
// values' bits: they order as the values do, and a NaN lies above infinity, so that it wins.
template <int KIND>
struct Share;
template <>
struct Share<2> {
    typedef double T;
    static __device__ __forceinline__ T zero() { return 0.0; }
    static __device__ __forceinline__ void add(T& a, float v) { a = __builtin_fma((double)v, (double)v, a); }
    static __device__ __forceinline__ T join(T a, T b) { return a + b; }
    static __device__ __forceinline__ uint64_t bits(T a) { return __builtin_bit_cast(uint64_t, a); }
    static __device__ __forceinline__ T of(uint64_t b) { return __builtin_bit_cast(double, b); }
    static __device__ __forceinline__ double norm(T a) { return sqrt(a); }
};
template <>
struct Share<1> : Share<2> {
    static __device__ __forceinline__ void add(T& a, float v) { a += (double)fabsf(v); }
    static __device__ __forceinline__ double norm(T a) { return a; }
};
template <>
struct Share<0> {
    typedef uint32_t T;
    static __device__ __forceinline__ T zero() { return 0u; }
    static __device__ __forceinline__ void add(T& a, float v) {
        const uint32_t u = __builtin_bit_cast(uint32_t, v) & 0x7fffffffu;
        a = a > u ? a : u;
    }
    static __device__ __forceinline__ T join(T a, T b) { return a > b ? a : b; }
    static __device__ __forceinline__ uint64_t bits(T a) { return a; }
    static __device__ __forceinline__ T of(uint64_t b) { return (uint32_t)b; }
    static __device__ __forceinline__ double norm(T a) { return (double)__builtin_bit_cast(float, a); }
};

template <typename S>
__device__ __forceinline__ typename S::T wave_join(typename S::T v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const uint64_t b = S::bits(v);
        const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)b, d, WAVE), hi = (uint32_t)__shfl_xor((int)(uint32_t)(b >> 32), d, WAVE);
        v = S::join(v, S::of((uint64_t)hi << 32 | lo));
    }
    return v;
}

// The workgroup's threads joined in a fixed order; the result is valid in every thread.
template <typename S, int THREADS>
__device__ __forceinline__ typename S::T block_join(typename S::T v) {
    __shared__ uint64_t s_w[THREADS / WAVE];
    v = wave_join<S>(v);
    if ((threadIdx.x & (WAVE - 1)) == 0) s_w[threadIdx.x / WAVE] = S::bits(v);
    __syncthreads();
    v = S::of(s_w[0]);
#pragma unroll
    for (int w = 1; w < THREADS / WAVE; ++w) v = S::join(v, S::of(s_w[w]));
    return v;
}

// Calls f with the type as a constant: one copy of the loop for each, where a test per value would cost more than the sum.
template <typename F>
__device__ __forceinline__ void with_type(int type, F f) {
    if (type == GSO_F32) f(std::integral_constant<int, GSO_F32>());
    else if (type == GSO_BF16) f(std::integral_constant<int, GSO_BF16>());
    else f(std::integral_constant<int, GSO_F16>());
}

template <typename S, int TYPE>
__device__ __forceinline__ void add_vector(typename S::T& a, const uint4& v) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (TYPE == GSO_F32) {
            S::add(a, __builtin_bit_cast(float, w[j]));
        } else if (TYPE == GSO_BF16) {
            S::add(a, __builtin_bit_cast(float, w[j] << 16));
            S::add(a, __builtin_bit_cast(float, w[j] & 0xffff0000u));
        } else {
            S::add(a, f16_to_float((uint16_t)w[j]));
            S::add(a, f16_to_float((uint16_t)(w[j] >> 16)));
        }
    }
}

template <int TYPE>
__device__ __forceinline__ uint4 scale_vector(const uint4& v, float s) {
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (TYPE == GSO_F32) w[j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, w[j]) * s);
        else if (TYPE == GSO_BF16)
            w[j] = (uint32_t)float_to_bf16(__builtin_bit_cast(float, w[j] << 16) * s) |
                   (uint32_t)float_to_bf16(__builtin_bit_cast(float, w[j] & 0xffff0000u) * s) << 16;
        else
            w[j] = (uint32_t)float_to_f16(f16_to_float((uint16_t)w[j]) * s) |
                   (uint32_t)float_to_f16(f16_to_float((uint16_t)(w[j] >> 16)) * s) << 16;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

template <bool ONCE>
__device__ __forceinline__ uint4 load_vector(const char* p) {
    const f32x4* q = reinterpret_cast<const f32x4*>(p);
    return __builtin_bit_cast(uint4, ONCE ? __builtin_nontemporal_load(q) : *q);
}

template <typename S, bool ONCE>
__device__ __forceinline__ void add_chunk(typename S::T& a, const Chunk& c, int tid) {
    for_chunk(c, tid, [&](int lo, int hi) {
        uint4 v[4];
        if (hi - lo == CHUNK_BYTES / 16) {
#pragma unroll
            for (int u = 0; u < 4; ++u) v[u] = load_vector<ONCE>(c.base + 16 * (u * NORM_THREADS + tid));
        } else {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int i = u * NORM_THREADS + tid;
                v[u] = i >= lo && i < hi ? load_vector<ONCE>(c.base + 16 * i) : make_uint4(0, 0, 0, 0);   // zeros add nothing
            }
        }
        with_type(c.type, [&](auto type) {
#pragma unroll
            for (int u = 0; u < 4; ++u) add_vector<S, decltype(type)::value>(a, v[u]);
        });
    }, [&](int x) {
        if (c.type == GSO_F32) S::add(a, *(const float*)(c.base + x));
        else if (c.type == GSO_BF16) S::add(a, bf16_to_float(*(const uint16_t*)(c.base + x)));
        else S::add(a, f16_to_float(*(const uint16_t*)(c.base + x)));
    });
}

// Non-temporal both ways: the scaled gradients are next read by an optimizer that streams six times as much, and keeping
// them out of the caches leaves there what the norm has put in (1.5 GB: 475 us, 6.4 TB/s; 554 us with ordinary accesses).
__device__ __forceinline__ void scale_chunk(const Chunk& c, int tid, float s) {
    for_chunk(c, tid, [&](int lo, int hi) {
        uint4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = u * NORM_THREADS + tid;
            if (i >= lo && i < hi) v[u] = load_vector<true>(c.base + 16 * i);
        }
        with_type(c.type, [&](auto type) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int i = u * NORM_THREADS + tid;
                if (i >= lo && i < hi)
                    __builtin_nontemporal_store(__builtin_bit_cast(f32x4, scale_vector<decltype(type)::value>(v[u], s)),
                                                reinterpret_cast<f32x4*>(c.base + 16 * i));
            }
        });
    }, [&](int x) {
        char* p = c.base + x;
        if (c.type == GSO_F32) *(float*)p = *(const float*)p * s;
        else if (c.type == GSO_BF16) *(uint16_t*)p = float_to_bf16(bf16_to_float(*(const uint16_t*)p) * s);
        else *(uint16_t*)p = float_to_f16(f16_to_float(*(const uint16_t*)p) * s);
    });
}

// ONCE: non-temporal loads, for a norm alone and before an Adam step: 7.0 TB/s on 1.5 GB where ordinary ones reach 6.2.
// A clip reads the gradients again at once; ordinary loads leave up to 256 MB in the last-level cache for it.  Before a
// step, with / without (us): sparse, a tenth visible, 1 M Gaussians (252 MB) 174 / 182, 6 M (1.5 GB) 950 / 990, 0.3 M 57
// either way; dense, 0.1 M (25 MB) 41.5 / 39.4, 0.3 M 110 / 100, 1 M 343 / 308, 2.5 M 870 / 832, 6 M 2118 / 2104: a dense
// step finds part of its gradients in the cache after ordinary loads, which this rule does not use.
template <int KIND, bool ONCE>
__global__ void __launch_bounds__(NORM_THREADS) norm_kernel(const NormTable t, uint64_t* __restrict__ partial) {
    typedef Share<KIND> S;
    typename S::T a = S::zero();
    // The first chunks of all tensors, one a lane: a chunk's tensor is then found with a few ballots, where a walk through
    // the kernel's arguments in memory costs a round of loads for every chunk.
    constexpr int HELD = (NORM_TABLE + WAVE - 1) / WAVE;
    uint32_t first[HELD];
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
        const int i = j * WAVE + (int)(threadIdx.x & (WAVE - 1));
        first[j] = i < t.n ? t.first[i] : 0xffffffffu;
    }
    for (uint32_t chunk = blockIdx.x; chunk < t.chunks; chunk += gridDim.x) {
        int k = -1;
#pragma unroll
        for (int j = 0; j < HELD; ++j) k += __popcll(__ballot(first[j] <= chunk));
        add_chunk<S, ONCE>(a, chunk_of(t, k, chunk), (int)threadIdx.x);
    }
    a = block_join<S, NORM_THREADS>(a);
    if (threadIdx.x == 0) partial[blockIdx.x] = S::bits(a);
}

// The coefficient is formed in 64 bits from the unrounded norm and rounded once; a NaN norm gives a NaN.
__device__ __forceinline__ float clip_coefficient(double norm, double max_norm) {
    const double c = max_norm / (norm + 1e-6);
    return c > 1.0 ? 1.0f : (float)c;
}

constexpr int FINISH_THREADS = 1024;
template <int KIND>
__global__ void __launch_bounds__(FINISH_THREADS) norm_finish_kernel(const uint64_t* __restrict__ partial, int count,
                                                                     double max_norm, NormResult* __restrict__ result,
                                                                     float* __restrict__ norm_out) {
    typedef Share<KIND> S;
    typename S::T a = S::zero();
    for (int i = threadIdx.x; i < count; i += 4 * FINISH_THREADS) {
        typename S::T v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = i + u * FINISH_THREADS < count ? S::of(partial[i + u * FINISH_THREADS]) : S::zero();
#pragma unroll
        for (int u = 0; u < 4; ++u) a = S::join(a, v[u]);
    }
    a = block_join<S, FINISH_THREADS>(a);
    if (threadIdx.x == 0) {
        const double norm = S::norm(a);
        result->norm = norm;
        result->coefficient = clip_coefficient(norm, max_norm);
        *norm_out = (float)norm;
    }
}

// A norm that gso_grad_norm has left in `temp` becomes a coefficient.
__global__ void coefficient_kernel(NormResult* __restrict__ result, double max_norm, float* __restrict__ norm_out) {
    result->coefficient = clip_coefficient(result->norm, max_norm);
    *norm_out = (float)result->norm;
}

// A few chunks are one workgroup's work, four of them at a time, and one launch's: the norm, and where it is a clip the
// scaling behind it (up to 16 chunks, 256 KB: 4.7 us a call; three launches 9.6.  30 chunks take 6.3 and 17.5 us alone,
// the other way 7.0 and 16.9).
constexpr int SMALL_THREADS = 4 * NORM_THREADS;
template <int KIND, bool SCALE>
__global__ void __launch_bounds__(SMALL_THREADS) norm_small_kernel(const NormTable t, double max_norm,
                                                                   NormResult* __restrict__ result, float* __restrict__ norm_out) {
    typedef Share<KIND> S;
    const int tid = (int)threadIdx.x & (NORM_THREADS - 1);
    const uint32_t group = (uint32_t)__builtin_amdgcn_readfirstlane((int)threadIdx.x / NORM_THREADS);
    typename S::T a = S::zero();
    for (uint32_t chunk = group; chunk < t.chunks; chunk += SMALL_THREADS / NORM_THREADS)
        add_chunk<S, false>(a, chunk_of(t, find_tensor(t, chunk), chunk), tid);
    const double norm = S::norm(block_join<S, SMALL_THREADS>(a));
    const float s = clip_coefficient(norm, max_norm);
    if (threadIdx.x == 0) {
        result->norm = norm;
        result->coefficient = s;
        *norm_out = (float)norm;
    }
    if (!SCALE || s == 1.0f) return;
    for (uint32_t chunk = group; chunk < t.chunks; chunk += SMALL_THREADS / NORM_THREADS)
        scale_chunk(chunk_of(t, find_tensor(t, chunk), chunk), tid, s);
}

// Where the consumers of a norm find the coefficient: finished (count = 0), or in at most NORM_GROUPS sums, which every
// workgroup joins for itself in the order of norm_finish_kernel; that saves a launch where the consumer has few
// workgroups.
struct Coefficient {
    const NormResult* result;
    const uint64_t* partial;
    float* norm;
    double max_norm;
    int count, kind;
};
static_assert(NORM_GROUPS <= 2 * FINISH_THREADS, "two sums a thread of norm_finish_kernel");
template <int KIND>
__device__ __forceinline__ float join_coefficient(const Coefficient& c) {
    typedef Share<KIND> S;
    constexpr int PARTS = FINISH_THREADS / NORM_THREADS;   // threads of the other kernel that a thread stands for
    __shared__ uint64_t s_w[FINISH_THREADS / WAVE];
    typename S::T v[PARTS];
#pragma unroll
    for (int j = 0; j < PARTS; ++j) {
        const int i = (int)threadIdx.x + j * NORM_THREADS;
        v[j] = S::join(i < c.count ? S::of(c.partial[i]) : S::zero(),
                       i + FINISH_THREADS < c.count ? S::of(c.partial[i + FINISH_THREADS]) : S::zero());
    }
#pragma unroll
    for (int j = 0; j < PARTS; ++j) {
        if (j * NORM_THREADS >= c.count) {   // nothing from here on
            if ((threadIdx.x & (WAVE - 1)) == 0) s_w[threadIdx.x / WAVE + j * (NORM_THREADS / WAVE)] = S::bits(S::zero());
            continue;
        }
        const typename S::T w = wave_join<S>(v[j]);
        if ((threadIdx.x & (WAVE - 1)) == 0) s_w[threadIdx.x / WAVE + j * (NORM_THREADS / WAVE)] = S::bits(w);
    }
    __syncthreads();
    typename S::T a = S::of(s_w[0]);
#pragma unroll
    for (int w = 1; w < FINISH_THREADS / WAVE; ++w) a = S::join(a, S::of(s_w[w]));
    const double norm = S::norm(a);
    if (blockIdx.x == 0 && threadIdx.x == 0) *c.norm = (float)norm;
    return clip_coefficient(norm, c.max_norm);
}
__device__ __forceinline__ float coefficient_of(const Coefficient& c) {
    if (c.count == 0) return c.result->coefficient;
    return c.kind == 2 ? join_coefficient<2>(c) : c.kind == 1 ? join_coefficient<1>(c) : join_coefficient<0>(c);
}

__global__ void __launch_bounds__(NORM_THREADS) scale_kernel(const NormTable t, const Coefficient coefficient) {
    const float s = coefficient_of(coefficient);
    if (s == 1.0f) return;   // under the ceiling nothing changes, and nothing is read
    scale_chunk(chunk_of(t, find_tensor(t, blockIdx.x), blockIdx.x), (int)threadIdx.x, s);
}

// Bound by its seven streams, 28 bytes an element.  Two vectors of each a thread, all loads first, non-temporal: every
// value is used once in a step (158 M elements: 785 us, 5.6 TB/s; one vector a thread 819).
__global__ void __launch_bounds__(NORM_THREADS) adam_clipped_kernel(const AdamTable t, const Coefficient coefficient) {
    const float s = coefficient_of(coefficient);
    const int k = find_tensor(t, blockIdx.x);
    const AdamEntry& e = t.e[k];
    const int64_t base = (int64_t)(blockIdx.x - t.first[k]) * ADAM_CHUNK;
    const int count = e.count - base < ADAM_CHUNK ? (int)(e.count - base) : ADAM_CHUNK;
    float *p = e.param + base, *m = e.exp_avg + base, *v = e.exp_avg_sq + base;
    const float* g = e.grad + base;
    int done = 0;
    if ((((uintptr_t)p | (uintptr_t)m | (uintptr_t)v | (uintptr_t)g) & 15) == 0) {
        done = count & ~3;
        f32x4 P[2], G[2], M[2], V[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int i = 4 * (u * NORM_THREADS + (int)threadIdx.x);
            if (i < done) {
                P[u] = __builtin_nontemporal_load((const f32x4*)(p + i));
                G[u] = __builtin_nontemporal_load((const f32x4*)(g + i));
                M[u] = __builtin_nontemporal_load((const f32x4*)(m + i));
                V[u] = __builtin_nontemporal_load((const f32x4*)(v + i));
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int i = 4 * (u * NORM_THREADS + (int)threadIdx.x);
            if (i < done) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float mm = M[u][j], vv = V[u][j];
                    P[u][j] = adam_update(P[u][j], G[u][j] * s, &mm, &vv, e.c);
                    M[u][j] = mm;
                    V[u][j] = vv;
                }
                __builtin_nontemporal_store(P[u], (f32x4*)(p + i));
                __builtin_nontemporal_store(M[u], (f32x4*)(m + i));
                __builtin_nontemporal_store(V[u], (f32x4*)(v + i));
            }
        }
    }
    for (int i = done + (int)threadIdx.x; i < count; i += NORM_THREADS) {
        float mm = m[i], vv = v[i];
        p[i] = adam_update(p[i], g[i] * s, &mm, &vv, e.c);
        m[i] = mm;
        v[i] = vv;
    }
}

// The sparse step touches few rows (a view sees about a tenth of a large scene), so a thread per element of all rows
// would leave most lanes without a load: the workgroup first lists its visible rows, then its threads walk the elements
// of the listed rows only, four each in flight (2.5 M rows, a tenth visible at random: 300 us, 355 with a thread per
// vector of all rows; rows of 12 or 16 bytes at random use a sixth of the lines that they touch, which is what bounds it).
// The list's order is that of arrival; every element is updated on its own, so nothing depends on it.
__global__ void __launch_bounds__(NORM_THREADS) adam_clipped_sparse_kernel(const AdamTable t, const uint8_t* __restrict__ visible,
                                                                           const Coefficient coefficient) {
    __shared__ uint16_t s_row[SPARSE_CHUNK];
    __shared__ uint32_t s_count;
    const float s = coefficient_of(coefficient);
    const int k = find_tensor(t, blockIdx.x);
    const AdamEntry& e = t.e[k];
    const uint32_t W = e.width, R = W < SPARSE_CHUNK ? SPARSE_CHUNK / W : 1;
    const int64_t row0 = (int64_t)(blockIdx.x - t.first[k]) * R;
    const uint32_t nrows = e.count - row0 < (int64_t)R ? (uint32_t)(e.count - row0) : R;
    if (threadIdx.x == 0) s_count = 0;
    __syncthreads();
    const int lane = threadIdx.x & (WAVE - 1);
    for (uint32_t r0 = 0; r0 < nrows; r0 += 4 * NORM_THREADS) {
        bool on[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint32_t r = r0 + u * NORM_THREADS + threadIdx.x;
            on[u] = r < nrows && visible[row0 + r] != 0;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint64_t mask = __ballot(on[u]);
            if (mask == 0) continue;
            uint32_t at = 0;
            if (lane == 0) at = atomicAdd(&s_count, (uint32_t)__popcll(mask));
            at = (uint32_t)__builtin_amdgcn_readlane((int)at, 0) + (uint32_t)__popcll(mask & ((1ull << lane) - 1));
            if (on[u]) s_row[at] = (uint16_t)(r0 + u * NORM_THREADS + threadIdx.x);
        }
    }
    __syncthreads();
    const uint32_t total = s_count * W;   // at most SPARSE_CHUNK, or one row
    // x / W by one multiplication: x and W stay below 2^13 unless the row is the only one
    const uint32_t magic = W > 1 && W < SPARSE_CHUNK ? 0xffffffffu / W + 1 : 0;
    float *p = e.param + row0 * W, *m = e.exp_avg + row0 * W, *v = e.exp_avg_sq + row0 * W;
    const float* g = e.grad + row0 * W;
    for (uint32_t x0 = threadIdx.x; x0 < total; x0 += 4 * NORM_THREADS) {
        uint32_t i[4];
        float P[4], G[4], M[4], V[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint32_t x = x0 + u * NORM_THREADS < total ? x0 + u * NORM_THREADS : x0;
            const uint32_t n = W == 1 ? x : (uint32_t)(((uint64_t)x * magic) >> 32);
            i[u] = (uint32_t)s_row[n] * W + (x - n * W);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            P[u] = p[i[u]];
            G[u] = g[i[u]];
            M[u] = m[i[u]];
            V[u] = v[i[u]];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (x0 + u * NORM_THREADS >= total) break;
            p[i[u]] = adam_update(P[u], G[u] * s, &M[u], &V[u], e.c);
            m[i[u]] = M[u];
            v[i[u]] = V[u];
        }
    }
}

// ------------------------------------------------------------------ host
// Chunks of a tensor, counted from its start rounded down to 16 bytes.
static int64_t chunks_of(const void* p, int64_t numel, int type) {
    return ((int64_t)((uintptr_t)p & 15) + numel * (type == GSO_F32 ? 4 : 2) + CHUNK_BYTES - 1) / CHUNK_BYTES;
}

// Chunks are counted in 32 bits.
bool norm_fits(int n, const int64_t* numels) {
    int64_t c = 0;
    for (int i = 0; i < n; ++i) {
        if (numels[i] >= (1ll << 43)) return false;
        c += numels[i] / (CHUNK_BYTES / 4) + 2;
        if (c >= (1ll << 31)) return false;
    }
    return true;
}

size_t norm_temp_bytes(int n) {
    const size_t launches = ((size_t)(n > 0 ? n : 1) + NORM_TABLE - 1) / NORM_TABLE;
    return 256 + launches * NORM_GROUPS * sizeof(uint64_t);
}

static uint64_t* norm_partials(void* temp) { return (uint64_t*)((char*)temp + 256); }

// Calls launch(table, whether it is the only one) for every group of tensors that fits a table.
template <typename F>
static hipError_t for_each_table(int n, const void* const* ptrs, const int64_t* numels, const int* types, F launch) {
    bool first = true;
    for (int i = 0; i < n;) {
        NormTable t;
        t.n = 0;
        t.chunks = 0;
        for (; i < n && t.n < NORM_TABLE; ++i) {
            if (numels[i] <= 0) continue;
            const int64_t bytes = (int64_t)((uintptr_t)ptrs[i] & 15) + numels[i] * (types[i] == GSO_F32 ? 4 : 2);
            t.ptr[t.n] = ptrs[i];
            t.first[t.n] = t.chunks;
            t.shape[t.n] = (uint32_t)types[i] | (uint32_t)((bytes - 1) % CHUNK_BYTES + 1) << 2;
            t.chunks += (uint32_t)chunks_of(ptrs[i], numels[i], types[i]);
            ++t.n;
        }
        if (t.n == 0) break;
        launch(t, first && i == n);
        first = false;
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <int KIND>
static void launch_norm(const NormTable& t, bool read_again, unsigned groups, uint64_t* p, hipStream_t st) {
    if (read_again) hipLaunchKernelGGL((norm_kernel<KIND, false>), dim3(groups), dim3(NORM_THREADS), 0, st, t, p);
    else hipLaunchKernelGGL((norm_kernel<KIND, true>), dim3(groups), dim3(NORM_THREADS), 0, st, t, p);
}

template <int KIND>
static void launch_small(const NormTable& t, bool scale, double max_norm, NormResult* r, float* norm, hipStream_t st) {
    if (scale) hipLaunchKernelGGL((norm_small_kernel<KIND, true>), dim3(1), dim3(SMALL_THREADS), 0, st, t, max_norm, r, norm);
    else hipLaunchKernelGGL((norm_small_kernel<KIND, false>), dim3(1), dim3(SMALL_THREADS), 0, st, t, max_norm, r, norm);
}

template <int KIND>
static void launch_finish(const uint64_t* p, int count, double max_norm, NormResult* r, float* norm, hipStream_t st) {
    hipLaunchKernelGGL(norm_finish_kernel<KIND>, dim3(1), dim3(FINISH_THREADS), 0, st, p, count, max_norm, r, norm);
}

// The norm of the gradients for whoever reads it next: *c says where the coefficient is found; for a norm alone the
// result is in the temp area and in *norm.  A clip of a few chunks is done at once (*scaled).  `consumers`: workgroups
// of what reads the coefficient.
constexpr uint32_t SMALL_CHUNKS = 16;
constexpr int64_t JOIN_CONSUMERS = 1024;   // clip of 10 MB: 9.5 us with, 11.2 without; of 25 MB (1539): 16.9 and 15.5
enum NormUse { NORM_ONLY, NORM_CLIP, NORM_STEP };
static hipError_t launch_norm_for(NormUse use, int n, const void* const* grads, const int64_t* numels, const int* types,
                                  int kind, double max_norm, int64_t consumers, void* temp, float* norm, hipStream_t st,
                                  Coefficient* c, bool* scaled) {
    NormResult* r = (NormResult*)temp;
    int count = 0, small = 0;
    hipError_t e = for_each_table(n, grads, numels, types, [&](const NormTable& t, bool alone) {
        if (alone && t.chunks <= SMALL_CHUNKS) {
            small = 1;
            if (kind == 2) launch_small<2>(t, use == NORM_CLIP, max_norm, r, norm, st);
            else if (kind == 1) launch_small<1>(t, use == NORM_CLIP, max_norm, r, norm, st);
            else launch_small<0>(t, use == NORM_CLIP, max_norm, r, norm, st);
            return;
        }
        const uint32_t rounds = (t.chunks + NORM_GROUPS - 1) / NORM_GROUPS;   // of every workgroup; some take one chunk less
        const unsigned groups = (t.chunks + rounds - 1) / rounds;
        uint64_t* p = norm_partials(temp) + count;
        if (kind == 2) launch_norm<2>(t, use == NORM_CLIP, groups, p, st);
        else if (kind == 1) launch_norm<1>(t, use == NORM_CLIP, groups, p, st);
        else launch_norm<0>(t, use == NORM_CLIP, groups, p, st);
        count += (int)groups;
    });
    if (e != hipSuccess) return e;
    *scaled = small && use == NORM_CLIP;
    // without a consumer (a sparse step that no group takes) nobody would join
    const bool join_later = use != NORM_ONLY && count > 0 && count <= NORM_GROUPS && consumers > 0 && consumers <= JOIN_CONSUMERS;
    if (!small && !join_later) {
        if (kind == 2) launch_finish<2>(norm_partials(temp), count, max_norm, r, norm, st);
        else if (kind == 1) launch_finish<1>(norm_partials(temp), count, max_norm, r, norm, st);
        else launch_finish<0>(norm_partials(temp), count, max_norm, r, norm, st);
        e = hipGetLastError();
    }
    *c = {r, norm_partials(temp), norm, max_norm, join_later ? count : 0, kind};
    return e;
}

// The same where gso_grad_norm has been called for these gradients and this temp area.
static hipError_t launch_coefficient(int kind, double max_norm, void* temp, float* norm, hipStream_t st, Coefficient* c) {
    hipLaunchKernelGGL(coefficient_kernel, dim3(1), dim3(1), 0, st, (NormResult*)temp, max_norm, norm);
    *c = {(NormResult*)temp, norm_partials(temp), norm, max_norm, 0, kind};
    return hipGetLastError();
}

hipError_t launch_grad_norm(int n, const void* const* grads, const int64_t* numels, const int* types, int kind, void* temp,
                            float* norm, hipStream_t st) {
    Coefficient c;
    bool scaled;
    return launch_norm_for(NORM_ONLY, n, grads, numels, types, kind, 0.0, 0, temp, norm, st, &c, &scaled);
}

hipError_t launch_clip_grads(int n, void* const* grads, const int64_t* numels, const int* types, int kind, double max_norm,
                             bool norm_known, void* temp, float* norm, hipStream_t st) {
    Coefficient c;
    bool scaled = false;
    const void* const* g = (const void* const*)grads;
    int64_t chunks = 0;
    for (int i = 0; i < n; ++i) chunks += chunks_of(g[i], numels[i], types[i]);
    const hipError_t e = norm_known ? launch_coefficient(kind, max_norm, temp, norm, st, &c)
                                    : launch_norm_for(NORM_CLIP, n, g, numels, types, kind, max_norm, chunks, temp, norm, st, &c,
                                                      &scaled);
    if (e != hipSuccess || scaled) return e;
    return for_each_table(n, g, numels, types, [&](const NormTable& t, bool) {
        hipLaunchKernelGGL(scale_kernel, dim3(t.chunks), dim3(NORM_THREADS), 0, st, t, c);
    });
}

// Workgroups of a tensor's update.
static int64_t adam_groups(const GsoAdamTensor& a, bool sparse) {
    const int64_t R = a.width < SPARSE_CHUNK ? SPARSE_CHUNK / a.width : 1;
    return sparse ? (a.rows + R - 1) / R : (a.rows * a.width + ADAM_CHUNK - 1) / ADAM_CHUNK;
}

hipError_t launch_adam_clipped(int ngrads, const void* const* grads, const int64_t* numels, const int* types, int n,
                               const GsoAdamTensor* tensors, const uint8_t* visible, int kind, double max_norm,
                               bool norm_known, void* temp, float* norm, hipStream_t st) {
    Coefficient c;
    bool scaled;
    int64_t all = 0;
    for (int i = 0; i < n; ++i) all += adam_groups(tensors[i], visible != nullptr);
    hipError_t e = norm_known ? launch_coefficient(kind, max_norm, temp, norm, st, &c)
                              : launch_norm_for(NORM_STEP, ngrads, grads, numels, types, kind, max_norm, all, temp, norm, st, &c,
                                                &scaled);
    for (int i = 0; i < n && e == hipSuccess;) {
        AdamTable t;
        t.n = 0;
        int64_t groups = 0;
        for (; i < n && t.n < ADAM_TABLE; ++i) {
            const GsoAdamTensor& a = tensors[i];
            const int64_t numel = a.rows * a.width;
            if (numel <= 0) continue;
            const int64_t more = adam_groups(a, visible != nullptr);
            if (t.n > 0 && groups + more > 0x7fffffff) break;
            t.e[t.n] = {a.param, a.exp_avg, a.exp_avg_sq, a.grad, visible ? a.rows : numel, (uint32_t)a.width,
                        adam_const(a.lr, a.beta1, a.beta2, a.eps, a.bias_correction1, a.bias_correction2_sqrt)};
            t.first[t.n] = (uint32_t)groups;
            groups += more;
            ++t.n;
        }
        if (t.n == 0) break;
        const dim3 grid((unsigned)groups), block(NORM_THREADS);
        if (visible) hipLaunchKernelGGL(adam_clipped_sparse_kernel, grid, block, 0, st, t, visible, c);
        else hipLaunchKernelGGL(adam_clipped_kernel, grid, block, 0, st, t, c);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace gs

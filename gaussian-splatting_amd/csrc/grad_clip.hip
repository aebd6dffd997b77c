// Global gradient norm over many tensors, clipping in place, and the Adam step
// that applies the clipping coefficient without rewriting the gradients.
//
//   norm = (sum |g|^p)^(1/p) over all elements of all tensors, p = 1 or 2, or max |g|
//   c    = min(1, max_norm / (norm + 1e-6)),   g <- g * c
//
// Nothing here has a counterpart in the reference, which never bounds its
// gradients.  A launch takes a table of tensors by value (no copy to the
// device, so it can be captured into a graph); the elements are cut into
// chunks, one workgroup sums one chunk, and the chunks' sums are added in a
// fixed order: the norm is the same bits in every run and on every replica.
// Sums are held in 64 bits: squares of float32 values neither overflow nor
// vanish there.
#include "kernels.h"

namespace gs {

constexpr int NORM_THREADS = 256;
constexpr int NORM_TABLE = 128;     // tensors per launch of the norm and scale kernels (kernel arguments: 2.7 KB)
constexpr int ADAM_TABLE = 40;      // tensors per launch of the Adam kernel
constexpr int64_t CHUNK = 4096;     // elements of one workgroup

struct NormTable {
    const void* ptr[NORM_TABLE];
    int64_t numel[NORM_TABLE];
    uint32_t first[NORM_TABLE + 1];   // first chunk of each tensor; first[n] = chunks of the launch
    uint8_t type[NORM_TABLE];
    int n;
};

struct AdamEntry {
    float *param, *exp_avg, *exp_avg_sq;
    const float* grad;
    int64_t numel;
    uint32_t width;                   // elements per row, for the visibility flags
    AdamConst c;
};
struct AdamTable {
    AdamEntry e[ADAM_TABLE];
    uint32_t first[ADAM_TABLE + 1];
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

__device__ __forceinline__ float load_element(const void* p, int type, int64_t i) {
    if (type == GSO_F32) return ((const float*)p)[i];
    if (type == GSO_BF16) return bf16_to_float(((const uint16_t*)p)[i]);
    return (float)((const _Float16*)p)[i];
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

// The workgroup's threads joined in a fixed order; the result is valid in every thread.
template <typename S, int THREADS>
__device__ __forceinline__ typename S::T block_join(typename S::T v) {
    __shared__ uint64_t s_w[THREADS / WAVE];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const uint64_t b = S::bits(v);
        const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)b, d, WAVE), hi = (uint32_t)__shfl_xor((int)(uint32_t)(b >> 32), d, WAVE);
        v = S::join(v, S::of((uint64_t)hi << 32 | lo));
    }
    if ((threadIdx.x & (WAVE - 1)) == 0) s_w[threadIdx.x / WAVE] = S::bits(v);
    __syncthreads();
    v = S::of(s_w[0]);
#pragma unroll
    for (int w = 1; w < THREADS / WAVE; ++w) v = S::join(v, S::of(s_w[w]));
    return v;
}

template <int KIND>
__global__ void __launch_bounds__(NORM_THREADS) norm_kernel(const NormTable t, uint64_t* __restrict__ partial) {
    typedef Share<KIND> S;
    const int k = find_tensor(t, blockIdx.x);
    const int64_t begin = (int64_t)(blockIdx.x - t.first[k]) * CHUNK;
    const int64_t end = begin + CHUNK < t.numel[k] ? begin + CHUNK : t.numel[k];
    typename S::T a = S::zero();
    for (int64_t i = begin + threadIdx.x; i < end; i += NORM_THREADS) S::add(a, load_element(t.ptr[k], t.type[k], i));
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
    for (int i = threadIdx.x; i < count; i += FINISH_THREADS) a = S::join(a, S::of(partial[i]));
    a = block_join<S, FINISH_THREADS>(a);
    if (threadIdx.x == 0) {
        const double norm = S::norm(a);
        result->norm = norm;
        result->coefficient = clip_coefficient(norm, max_norm);
        *norm_out = (float)norm;
    }
}

__global__ void __launch_bounds__(NORM_THREADS) scale_kernel(const NormTable t, const NormResult* __restrict__ result) {
    const float c = result->coefficient;
    if (c == 1.0f) return;   // under the ceiling nothing changes, and nothing is read
    const int k = find_tensor(t, blockIdx.x);
    const int64_t begin = (int64_t)(blockIdx.x - t.first[k]) * CHUNK;
    const int64_t end = begin + CHUNK < t.numel[k] ? begin + CHUNK : t.numel[k];
    void* p = const_cast<void*>(t.ptr[k]);
    for (int64_t i = begin + threadIdx.x; i < end; i += NORM_THREADS) {
        const float v = load_element(p, t.type[k], i) * c;
        if (t.type[k] == GSO_F32) ((float*)p)[i] = v;
        else if (t.type[k] == GSO_BF16) ((uint16_t*)p)[i] = float_to_bf16(v);
        else ((_Float16*)p)[i] = (_Float16)v;
    }
}

__global__ void __launch_bounds__(NORM_THREADS) adam_clipped_kernel(const AdamTable t, const uint8_t* __restrict__ visible,
                                                                    const NormResult* __restrict__ result) {
    const float c = result->coefficient;
    const int k = find_tensor(t, blockIdx.x);
    const AdamEntry& e = t.e[k];
    const int64_t begin = (int64_t)(blockIdx.x - t.first[k]) * CHUNK;
    const int64_t end = begin + CHUNK < e.numel ? begin + CHUNK : e.numel;
    for (int64_t i = begin + threadIdx.x; i < end; i += NORM_THREADS) {
        if (visible && !visible[i / e.width]) continue;
        float m = e.exp_avg[i], v = e.exp_avg_sq[i];
        e.param[i] = adam_update(e.param[i], e.grad[i] * c, &m, &v, e.c);
        e.exp_avg[i] = m;
        e.exp_avg_sq[i] = v;
    }
}

// ------------------------------------------------------------------ host
static int64_t chunks_of(int64_t numel) { return (numel + CHUNK - 1) / CHUNK; }

// Chunks are counted in 32 bits.
bool norm_fits(int n, const int64_t* numels) {
    int64_t c = 0;
    for (int i = 0; i < n; ++i) c += chunks_of(numels[i]);
    return c < (1ll << 31);
}

size_t norm_temp_bytes(int n, const int64_t* numels) {
    int64_t c = 0;
    for (int i = 0; i < n; ++i) c += chunks_of(numels[i]);
    return 256 + (size_t)(c > 0 ? c : 1) * sizeof(uint64_t);
}

static uint64_t* norm_partials(void* temp) { return (uint64_t*)((char*)temp + 256); }

// Calls launch(table, first partial) for every group of tensors that fits a table.
template <typename F>
static hipError_t for_each_table(int n, const void* const* ptrs, const int64_t* numels, const int* types, F launch) {
    int64_t done = 0;
    for (int i = 0; i < n;) {
        NormTable t;
        t.n = 0;
        t.first[0] = 0;
        for (; i < n && t.n < NORM_TABLE; ++i) {
            if (numels[i] <= 0) continue;
            t.ptr[t.n] = ptrs[i];
            t.numel[t.n] = numels[i];
            t.type[t.n] = (uint8_t)types[i];
            t.first[t.n + 1] = t.first[t.n] + (uint32_t)chunks_of(numels[i]);
            ++t.n;
        }
        if (t.n == 0) break;
        launch(t, done);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        done += t.first[t.n];
    }
    return hipSuccess;
}

hipError_t launch_grad_norm(int n, const void* const* grads, const int64_t* numels, const int* types, int kind, void* temp,
                            int* partials, hipStream_t st) {
    int64_t count = 0;
    const hipError_t e = for_each_table(n, grads, numels, types, [&](const NormTable& t, int64_t done) {
        uint64_t* p = norm_partials(temp) + done;
        const dim3 grid(t.first[t.n]), block(NORM_THREADS);
        if (kind == 2) hipLaunchKernelGGL(norm_kernel<2>, grid, block, 0, st, t, p);
        else if (kind == 1) hipLaunchKernelGGL(norm_kernel<1>, grid, block, 0, st, t, p);
        else hipLaunchKernelGGL(norm_kernel<0>, grid, block, 0, st, t, p);
        count = done + t.first[t.n];
    });
    *partials = (int)count;
    return e;
}

hipError_t launch_norm_finish(void* temp, int partials, int kind, double max_norm, float* norm, hipStream_t st) {
    NormResult* r = (NormResult*)temp;
    const uint64_t* p = norm_partials(temp);
    const dim3 grid(1), block(FINISH_THREADS);
    if (kind == 2) hipLaunchKernelGGL(norm_finish_kernel<2>, grid, block, 0, st, p, partials, max_norm, r, norm);
    else if (kind == 1) hipLaunchKernelGGL(norm_finish_kernel<1>, grid, block, 0, st, p, partials, max_norm, r, norm);
    else hipLaunchKernelGGL(norm_finish_kernel<0>, grid, block, 0, st, p, partials, max_norm, r, norm);
    return hipGetLastError();
}

hipError_t launch_clip_grads(int n, void* const* grads, const int64_t* numels, const int* types, int kind, double max_norm,
                             void* temp, int partials, float* norm, hipStream_t st) {
    const hipError_t e = launch_norm_finish(temp, partials, kind, max_norm, norm, st);
    if (e != hipSuccess) return e;
    return for_each_table(n, (const void* const*)grads, numels, types, [&](const NormTable& t, int64_t) {
        hipLaunchKernelGGL(scale_kernel, dim3(t.first[t.n]), dim3(NORM_THREADS), 0, st, t, (const NormResult*)temp);
    });
}

hipError_t launch_adam_clipped(int n, const GsoAdamTensor* tensors, const uint8_t* visible, int kind, double max_norm,
                               void* temp, int partials, float* norm, hipStream_t st) {
    hipError_t e = launch_norm_finish(temp, partials, kind, max_norm, norm, st);
    for (int i = 0; i < n && e == hipSuccess;) {
        AdamTable t;
        t.n = 0;
        t.first[0] = 0;
        for (; i < n && t.n < ADAM_TABLE; ++i) {
            const GsoAdamTensor& a = tensors[i];
            const int64_t numel = a.rows * a.width;
            if (numel <= 0) continue;
            t.e[t.n] = {a.param, a.exp_avg, a.exp_avg_sq, a.grad, numel, (uint32_t)a.width,
                        adam_const(a.lr, a.beta1, a.beta2, a.eps, a.bias_correction1, a.bias_correction2_sqrt)};
            t.first[t.n + 1] = t.first[t.n] + (uint32_t)chunks_of(numel);
            ++t.n;
        }
        if (t.n == 0) break;
        hipLaunchKernelGGL(adam_clipped_kernel, dim3(t.first[t.n]), dim3(NORM_THREADS), 0, st, t, visible,
                           (const NormResult*)temp);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace gs

// Keeping a model within a row budget.  Alpha compositing is attention: along a
// ray the Gaussians' weights are non-negative and sum to at most one, and a
// view's forward returns their sums per Gaussian.  The rows of the parameters
// and of the optimizer state are the cache that these weights read, new rows
// are appended at its end, and eviction keeps the newest rows and the heaviest
// of the others:
//
//   w_i <- decay * w_i + sigmoid(o_i) * sum over views of contribution_v[i]
//   keep = { i >= N - recent }  and the (budget - recent) first of the others
//          in the order (larger weight, then lower index), a NaN last
//
// The number of kept rows is known before any row is looked at, so nothing here
// makes the host wait.  The k-th largest weight is found by a radix select on
// the weights' bits (three histograms of 11, 11 and 10 bits), then one pass
// counts and one writes the kept rows in ascending order.  All counts are
// integers: the result is the same in every run.
#include "kernels.h"

namespace gs {

// ------------------------------------------------------------------ accumulated weights
constexpr int WEIGHT_VIEWS = 32;   // views per launch
struct WeightArgs {
    const float* contribution[WEIGHT_VIEWS];
    const float* opacity;
    float* weights;
    int64_t N;
    float decay;
    int views;
};

__global__ void __launch_bounds__(256) accumulate_weights_kernel(const WeightArgs a) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= a.N) return;
    float s = 0.0f;
    for (int v = 0; v < a.views; ++v) s += a.contribution[v][i];
    if (a.opacity) s /= 1.0f + expf(-a.opacity[i]);
    a.weights[i] = a.weights[i] * a.decay + s;
}

// ------------------------------------------------------------------ selection
constexpr int HIST_BINS = 2048;
constexpr int SELECT_THREADS = 256;
constexpr int SELECT_ROWS = 4096;   // rows of one workgroup

struct SelectState {
    uint32_t hist[3][HIST_BINS];
    uint32_t key;     // the bits of the threshold found so far
    uint32_t need;    // how many rows that equal them are still to be kept
};

// Unsigned integers that order as the weights do: NaN lowest, then -inf .. +inf, and -0 equal to +0.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__global__ void __launch_bounds__(256) select_clear_kernel(SelectState* __restrict__ s, uint32_t need) {
    for (int i = blockIdx.x * 256 + threadIdx.x; i < 3 * HIST_BINS; i += gridDim.x * 256) (&s->hist[0][0])[i] = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        s->key = 0;
        s->need = need;
    }
}

__device__ __forceinline__ int pass_shift(int pass) { return pass == 0 ? 21 : pass == 1 ? 10 : 0; }
__device__ __forceinline__ int pass_bits(int pass) { return pass == 2 ? 10 : 11; }

__global__ void __launch_bounds__(SELECT_THREADS) select_hist_kernel(int64_t old, const float* __restrict__ weights,
                                                                     SelectState* __restrict__ s, int pass) {
    __shared__ uint32_t h[HIST_BINS];
    for (int b = threadIdx.x; b < HIST_BINS; b += SELECT_THREADS) h[b] = 0;
    __syncthreads();
    const uint32_t prefix = s->key;
    const int shift = pass_shift(pass), bits = pass_bits(pass);
    const int64_t begin = (int64_t)blockIdx.x * SELECT_ROWS;
    const int64_t end = begin + SELECT_ROWS < old ? begin + SELECT_ROWS : old;
    for (int64_t i = begin + threadIdx.x; i < end; i += SELECT_THREADS) {
        const uint32_t k = weight_key(weights[i]);
        if (pass == 0 || (k >> (shift + bits)) == prefix) atomicAdd(&h[(k >> shift) & ((1u << bits) - 1)], 1u);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < HIST_BINS; b += SELECT_THREADS)
        if (h[b]) atomicAdd(&s->hist[pass][b], h[b]);
}

// The bin that holds the need-th largest key, and how many of it are needed.
__global__ void __launch_bounds__(256) select_bin_kernel(SelectState* __restrict__ s, int pass) {
    __shared__ uint32_t sums[256];
    const uint32_t need = s->need;
    uint32_t c[8], own = 0;
    for (int j = 0; j < 8; ++j) {   // thread 0 has the highest bins
        c[j] = s->hist[pass][HIST_BINS - 1 - (threadIdx.x * 8 + j)];
        own += c[j];
    }
    sums[threadIdx.x] = own;
    __syncthreads();
    uint32_t above = 0;
    for (int i = 0; i < (int)threadIdx.x; ++i) above += sums[i];
    __syncthreads();
    for (int j = 0; j < 8; ++j) {
        if (above < need && need <= above + c[j]) {
            s->key = (s->key << pass_bits(pass)) | (uint32_t)(HIST_BINS - 1 - (threadIdx.x * 8 + j));
            s->need = need - above;
        }
        above += c[j];
    }
}

__device__ __forceinline__ uint32_t block_sum_u32(uint32_t v, uint32_t* s_w) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += (uint32_t)__shfl_xor((int)v, d, WAVE);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_w[threadIdx.x >> 6] = v;
    __syncthreads();
    return s_w[0] + s_w[1] + s_w[2] + s_w[3];
}

// Per workgroup: rows above the threshold (the recent ones among them) and rows that equal it.
__global__ void __launch_bounds__(SELECT_THREADS) select_count_kernel(int64_t N, int64_t old,
                                                                      const float* __restrict__ weights,
                                                                      const SelectState* __restrict__ s,
                                                                      uint2* __restrict__ counts) {
    __shared__ uint32_t s_w[4];
    const uint32_t key = s->key;
    uint32_t above = 0, level = 0;
    for (int j = 0; j < SELECT_ROWS / SELECT_THREADS; ++j) {
        const int64_t i = (int64_t)blockIdx.x * SELECT_ROWS + j * SELECT_THREADS + threadIdx.x;
        if (i >= N) break;
        const uint32_t k = i < old ? weight_key(weights[i]) : 0u;
        above += (i >= old || k > key) ? 1u : 0u;
        level += (i < old && k == key) ? 1u : 0u;
    }
    above = block_sum_u32(above, s_w);
    level = block_sum_u32(level, s_w);
    if (threadIdx.x == 0) counts[blockIdx.x] = make_uint2(above, level);
}

__global__ void __launch_bounds__(SELECT_THREADS) select_write_kernel(int64_t N, int64_t old,
                                                                      const float* __restrict__ weights,
                                                                      const SelectState* __restrict__ s,
                                                                      const uint2* __restrict__ counts,
                                                                      int32_t* __restrict__ rows) {
    __shared__ uint32_t s_w[4];
    __shared__ uint32_t s_a[4], s_l[4];
    const uint32_t key = s->key, need = s->need;
    uint32_t above = 0, level = 0;   // rows of the workgroups before this one
    for (uint32_t b = threadIdx.x; b < blockIdx.x; b += SELECT_THREADS) {
        above += counts[b].x;
        level += counts[b].y;
    }
    above = block_sum_u32(above, s_w);
    level = block_sum_u32(level, s_w);
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const uint64_t below = (1ull << lane) - 1;
    for (int j = 0; j < SELECT_ROWS / SELECT_THREADS; ++j) {
        const int64_t i = (int64_t)blockIdx.x * SELECT_ROWS + j * SELECT_THREADS + threadIdx.x;
        const uint32_t k = i < old ? weight_key(weights[i]) : 0u;
        const bool a = i < N && (i >= old || k > key), l = i < old && k == key;
        const uint64_t ma = __ballot(a), ml = __ballot(l);
        __syncthreads();
        if (lane == 0) {
            s_a[w] = (uint32_t)__popcll(ma);
            s_l[w] = (uint32_t)__popcll(ml);
        }
        __syncthreads();
        uint32_t pa = above, pl = level;
        for (int x = 0; x < w; ++x) {
            pa += s_a[x];
            pl += s_l[x];
        }
        pa += (uint32_t)__popcll(ma & below);
        pl += (uint32_t)__popcll(ml & below);
        if (a || (l && pl < need)) rows[pa + (pl < need ? pl : need)] = (int32_t)i;
        above += s_a[0] + s_a[1] + s_a[2] + s_a[3];
        level += s_l[0] + s_l[1] + s_l[2] + s_l[3];
    }
}

__global__ void __launch_bounds__(256) select_tail_kernel(int64_t first, int64_t count, int32_t* __restrict__ rows) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < count) rows[i] = (int32_t)(first + i);
}

// ------------------------------------------------------------------ rows of many tensors
constexpr int ROWS_TABLE = 96;   // tensors per launch
constexpr int64_t ROWS_CHUNK = 4096;   // units of one workgroup
struct RowsTable {
    const void* src[ROWS_TABLE];
    void* dst[ROWS_TABLE];
    int64_t pitch[ROWS_TABLE];           // bytes between source rows
    uint32_t units[ROWS_TABLE];          // units of a row
    uint32_t first[ROWS_TABLE + 1];      // first chunk of each tensor
    uint8_t unit_shift[ROWS_TABLE];      // a unit is 1 << unit_shift bytes: 4, 2 or 1
    int n;
};

__global__ void __launch_bounds__(256) gather_rows_multi_kernel(const RowsTable t, const int32_t* __restrict__ rows,
                                                                int64_t K) {
    int lo = 0, hi = t.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= blockIdx.x) lo = mid; else hi = mid - 1;
    }
    const uint32_t M = t.units[lo];
    const int sh = t.unit_shift[lo];
    const int64_t total = K * M;
    const int64_t begin = (int64_t)(blockIdx.x - t.first[lo]) * ROWS_CHUNK;
    const int64_t end = begin + ROWS_CHUNK < total ? begin + ROWS_CHUNK : total;
    for (int64_t i = begin + threadIdx.x; i < end; i += 256) {
        const int64_t r = i / M;
        const char* s = (const char*)t.src[lo] + (int64_t)rows[r] * t.pitch[lo] + ((i - r * M) << sh);
        if (sh == 2) ((uint32_t*)t.dst[lo])[i] = *(const uint32_t*)s;
        else if (sh == 1) ((uint16_t*)t.dst[lo])[i] = *(const uint16_t*)s;
        else ((uint8_t*)t.dst[lo])[i] = *(const uint8_t*)s;
    }
}

// ------------------------------------------------------------------ host
hipError_t launch_accumulate_weights(int64_t N, float* weights, int views, const float* const* contributions,
                                     const float* opacity, float decay, hipStream_t st) {
    if (N <= 0) return hipSuccess;
    int first = 0;
    do {
        WeightArgs a;
        a.views = views - first < WEIGHT_VIEWS ? views - first : WEIGHT_VIEWS;
        for (int v = 0; v < WEIGHT_VIEWS; ++v) a.contribution[v] = v < a.views ? contributions[first + v] : nullptr;
        a.opacity = opacity;
        a.weights = weights;
        a.N = N;
        a.decay = first == 0 ? decay : 1.0f;
        hipLaunchKernelGGL(accumulate_weights_kernel, dim3((unsigned)((N + 255) / 256)), dim3(256), 0, st, a);
        first += WEIGHT_VIEWS;
    } while (first < views);
    return hipGetLastError();
}

size_t evict_temp_bytes(int64_t N) {
    const size_t nb = (size_t)((N + SELECT_ROWS - 1) / SELECT_ROWS);
    return align_up(sizeof(SelectState), 256) + align_up((nb + 1) * sizeof(uint2), 256);
}

hipError_t launch_evict_select(int64_t N, const float* weights, int64_t budget, int64_t recent, int32_t* rows, void* temp,
                               hipStream_t st) {
    const int64_t keep = budget < N ? budget : N;
    if (keep <= 0) return hipSuccess;
    if (recent > N) recent = N;
    if (keep == N || keep == recent) {   // no row has to be compared: the last `keep` rows
        hipLaunchKernelGGL(select_tail_kernel, dim3((unsigned)((keep + 255) / 256)), dim3(256), 0, st, N - keep, keep, rows);
        return hipGetLastError();
    }
    const int64_t old = N - recent;
    SelectState* s = (SelectState*)temp;
    uint2* counts = (uint2*)((char*)temp + align_up(sizeof(SelectState), 256));
    const unsigned nb_old = (unsigned)((old + SELECT_ROWS - 1) / SELECT_ROWS), nb = (unsigned)((N + SELECT_ROWS - 1) / SELECT_ROWS);
    hipLaunchKernelGGL(select_clear_kernel, dim3(24), dim3(256), 0, st, s, (uint32_t)(keep - recent));
    for (int pass = 0; pass < 3; ++pass) {
        hipLaunchKernelGGL(select_hist_kernel, dim3(nb_old), dim3(SELECT_THREADS), 0, st, old, weights, s, pass);
        hipLaunchKernelGGL(select_bin_kernel, dim3(1), dim3(256), 0, st, s, pass);
    }
    hipLaunchKernelGGL(select_count_kernel, dim3(nb), dim3(SELECT_THREADS), 0, st, N, old, weights, s, counts);
    hipLaunchKernelGGL(select_write_kernel, dim3(nb), dim3(SELECT_THREADS), 0, st, N, old, weights, s, counts, rows);
    return hipGetLastError();
}

hipError_t launch_gather_rows_multi(int n, const GsoRowCopy* copies, const int32_t* rows, int64_t K, hipStream_t st) {
    for (int i = 0; i < n;) {
        RowsTable t;
        t.n = 0;
        t.first[0] = 0;
        int64_t chunks = 0;
        for (; i < n && t.n < ROWS_TABLE; ++i) {
            const GsoRowCopy& c = copies[i];
            if (c.row_bytes <= 0 || K <= 0) continue;
            const uint64_t bits = (uint64_t)c.row_bytes | (uint64_t)c.src_pitch | (uint64_t)(uintptr_t)c.src | (uint64_t)(uintptr_t)c.dst;
            const int sh = (bits & 3) == 0 ? 2 : (bits & 1) == 0 ? 1 : 0;
            const int64_t more = ((K * (c.row_bytes >> sh)) + ROWS_CHUNK - 1) / ROWS_CHUNK;
            if (t.n > 0 && chunks + more > 0x7fffffff) break;
            t.src[t.n] = c.src;
            t.dst[t.n] = c.dst;
            t.pitch[t.n] = c.src_pitch;
            t.units[t.n] = (uint32_t)(c.row_bytes >> sh);
            t.unit_shift[t.n] = (uint8_t)sh;
            chunks += more;
            t.first[++t.n] = (uint32_t)chunks;
        }
        if (t.n == 0) break;
        hipLaunchKernelGGL(gather_rows_multi_kernel, dim3((unsigned)chunks), dim3(256), 0, st, t, rows, K);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace gs

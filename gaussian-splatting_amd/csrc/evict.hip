// Keeping a model within a row budget.  Alpha compositing is attention: a
// pixel's weights alpha * T over the Gaussians of its ray are non-negative and
// sum to at most one; their sums over a view's pixels are the gradient of the
// image with respect to the Gaussians' colours.  The rows of the parameters
// and of the optimizer state are the cache that these weights read, new rows
// are appended at its end, and eviction keeps the newest rows and the heaviest
// of the others:
//
//   w_i <- decay * w_i + s_i * sum over views of contribution_v[i]
//
// with s = 1 for contributions that are weights.  With s = sigmoid(opacity) and
// the forward's gauss_sum (T over the pixels that test the Gaussian, whatever
// its alpha there) the sum is an upper bound of the weight, and no more: it
// overrates splats that are small against a tile.
//
//   keep = { i >= N - recent }  and the (budget - recent) first of the others
//          in the order (larger weight, then lower index), a NaN last
//
// The number of kept rows is known before any row is looked at, so nothing here
// makes the host wait.  The k-th largest weight is found by a radix select on
// the weights' bits (three histograms of 11, 11 and 10 bits).  The third pass
// knows 22 of them and leaves two bits per row: above all weights with these 22
// bits, or one of them.  Counting and writing the kept rows reads those bits, and
// the weights of the rows among the second only.  All counts are integers: the
// result is the same in every run.
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

typedef float f32x4 __attribute__((ext_vector_type(4)));

// Bound by its reads, 4 bytes a view and Gaussian.  Four Gaussians a thread where every pointer allows 16-byte accesses;
// the loads of eight views are issued before the first is added, non-temporal because a view's weights are read once
// (8 views of 6 M Gaussians: 43 us, 6.1 TB/s; 50 us with ordinary loads, 75 with one Gaussian a thread).
template <int VEC>
__global__ void __launch_bounds__(256) accumulate_weights_kernel(const WeightArgs a) {
    typedef float vec __attribute__((ext_vector_type(VEC)));
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * VEC;
    if (i >= a.N) return;
    if (VEC > 1 && i + VEC > a.N) {   // the last one to three
        for (int64_t j = i; j < a.N; ++j) {
            float s = 0.0f;
            for (int v = 0; v < a.views; ++v) s += a.contribution[v][j];
            if (a.opacity) s /= 1.0f + expf(-a.opacity[j]);
            a.weights[j] = a.weights[j] * a.decay + s;
        }
        return;
    }
    vec w = *reinterpret_cast<const vec*>(a.weights + i), o = 0.0f, s = 0.0f;
    if (a.opacity) o = *reinterpret_cast<const vec*>(a.opacity + i);
    for (int v = 0; v < a.views; v += 8) {
        vec c[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            c[u] = v + u < a.views ? __builtin_nontemporal_load(reinterpret_cast<const vec*>(a.contribution[v + u] + i)) : vec(0.0f);
#pragma unroll
        for (int u = 0; u < 8; ++u) s += c[u];
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
        if (a.opacity) s[j] /= 1.0f + expf(-o[j]);
        w[j] = w[j] * a.decay + s[j];
    }
    *reinterpret_cast<vec*>(a.weights + i) = w;
}

// ------------------------------------------------------------------ selection
constexpr int HIST_BINS = 2048;
constexpr int HIST_THREADS = 1024;
constexpr int HIST_GROUPS = 512;        // two workgroups per CU: each adds its whole histogram to the global one once
constexpr int SELECT_THREADS = 256;
constexpr int SELECT_ROWS = 4096;       // rows of a tile: sixteen a thread
constexpr int SELECT_GROUPS = 2048;     // workgroups of the counting and writing kernels, a run of tiles each

struct SelectState {
    uint32_t hist[3][HIST_BINS];
    uint2 at[4];      // before each pass, and after the last: the bits of the threshold found so far, and how many rows
                      // that equal them are still to be kept
};

// Two bits of every row, a segment of 256 rows in eight words: bit l of word j is row 4 l + j of the segment, as a ballot
// over lanes with four rows each gives it.
constexpr int SEGMENT = 256;
struct SegmentBits {
    uint64_t above[4], level[4];
};

// Unsigned integers that order as the weights do: NaN lowest, then -inf .. +inf, and -0 equal to +0.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0u;
    const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__global__ void __launch_bounds__(256) select_clear_kernel(SelectState* __restrict__ s, uint32_t need) {
    for (int i = blockIdx.x * 256 + threadIdx.x; i < 3 * HIST_BINS; i += gridDim.x * 256) (&s->hist[0][0])[i] = 0;
    if (blockIdx.x == 0 && threadIdx.x == 0) s->at[0] = make_uint2(0u, need);
}

constexpr int pass_shift(int pass) { return pass == 0 ? 21 : pass == 1 ? 10 : 0; }
constexpr int pass_bits(int pass) { return pass == 2 ? 10 : 11; }

__device__ __forceinline__ uint32_t wave_scan_u32(uint32_t v) {   // inclusive
#pragma unroll
    for (int d = 1; d < WAVE; d <<= 1) {
        const uint32_t o = (uint32_t)__shfl_up((int)v, d, WAVE);
        if ((int)(threadIdx.x & 63) >= d) v += o;
    }
    return v;
}

// The bin of a finished histogram (of pass PASS) that holds the at.y-th largest key, and how many of it are needed.
template <int PASS, int THREADS>
__device__ __forceinline__ uint2 find_bin(const uint32_t* hist, uint2 at) {
    constexpr int PER = HIST_BINS / THREADS;
    __shared__ uint32_t s_w[THREADS / WAVE];
    __shared__ uint2 s_found;
    uint32_t c[PER], own = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {   // thread 0 has the highest bins
        c[j] = hist[HIST_BINS - 1 - ((int)threadIdx.x * PER + j)];
        own += c[j];
    }
    const uint32_t incl = wave_scan_u32(own);
    if ((threadIdx.x & 63) == 63) s_w[threadIdx.x >> 6] = incl;
    __syncthreads();
    uint32_t above = incl - own;
    for (int w = 0; w < (int)(threadIdx.x >> 6); ++w) above += s_w[w];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        if (above < at.y && at.y <= above + c[j])
            s_found = make_uint2((at.x << pass_bits(PASS)) | (uint32_t)(HIST_BINS - 1 - ((int)threadIdx.x * PER + j)), at.y - above);
        above += c[j];
    }
    __syncthreads();
    return s_found;
}

// Copies of the workgroup's histogram, side by side, a quarter of the lanes each: few bins hold most weights (20 M rows of
// one weight: 117 us for the selection, 267 with a single copy; of random weights 100 us either way).
constexpr int HIST_COPIES = 4;

// One pass of the radix select, bound by reading the weights: 17.8 us for 20 M (4.5 TB/s, 3 us of it the launch, the bin
// search and the merge; the third, which leaves the rows' bits, 20.5).  VECS: 16-byte loads a thread has in flight.  The rows that no view has seen all weigh zero;
// they are counted per wave with a ballot, and only the others go to LDS.
template <int PASS, int VECS>
__global__ void __launch_bounds__(HIST_THREADS) select_hist_kernel(int64_t old, const float* __restrict__ weights,
                                                                   SelectState* __restrict__ s,
                                                                   SegmentBits* __restrict__ segments) {
    __shared__ uint32_t h[HIST_BINS * HIST_COPIES];
    constexpr int shift = pass_shift(PASS), bits = pass_bits(PASS), step = 4 * VECS * HIST_THREADS;
    constexpr uint32_t ZERO = 0x80000000u;   // weight_key(0)
    for (int b = threadIdx.x; b < HIST_BINS * HIST_COPIES; b += HIST_THREADS) h[b] = 0;
    uint32_t prefix = 0;
    if (PASS > 0) {
        // every workgroup finds the bin of the pass before for itself, which saves a launch between the passes
        constexpr int BEFORE = PASS > 0 ? PASS - 1 : 0;
        const uint2 at = find_bin<BEFORE, HIST_THREADS>(s->hist[BEFORE], s->at[BEFORE]);
        prefix = at.x;
        if (blockIdx.x == 0 && threadIdx.x == 0) s->at[PASS] = at;
    } else {
        __syncthreads();
    }
    uint32_t* own = h + (threadIdx.x & (HIST_COPIES - 1));
    const bool count_zeros = PASS == 0 || (uint32_t)((uint64_t)ZERO >> (shift + bits)) == prefix;
    uint32_t zeros = 0;
    const int lane = threadIdx.x & (WAVE - 1);
    // four rows of a lane, `valid` of them
    auto add = [&](const f32x4& w, int64_t i, int valid) {
        uint64_t word[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t k = weight_key(w[j]), top = (uint32_t)((uint64_t)k >> (shift + bits));
            bool in = j < valid && (PASS == 0 || top == prefix);
            if (PASS == 2) {
                word[j] = __ballot(j < valid && top > prefix);
                word[4 + j] = __ballot(in);
            }
            if (count_zeros) {
                zeros += (uint32_t)__popcll(__ballot(j < valid && k == ZERO));
                in = in && k != ZERO;
            }
            if (in) atomicAdd(own + ((k >> shift) & ((1u << bits) - 1)) * HIST_COPIES, 1u);
        }
        if (PASS == 2) {
            uint64_t mine = word[0];   // lane x stores word x
#pragma unroll
            for (int x = 1; x < 8; ++x) mine = lane == x ? word[x] : mine;
            const int64_t first = i - 4 * lane;   // of the wave's segment
            if (lane < 8 && first < old)
                reinterpret_cast<uint64_t*>(segments + first / SEGMENT)[lane] = mine;
        }
    };
    const bool aligned = ((uintptr_t)weights & 15) == 0;
    for (int64_t base = (int64_t)blockIdx.x * step; base < old; base += (int64_t)gridDim.x * step) {
        const int64_t i0 = base + 4 * (int)threadIdx.x;
        if (aligned && base + step <= old) {
            f32x4 w[VECS];
#pragma unroll
            for (int q = 0; q < VECS; ++q) w[q] = *reinterpret_cast<const f32x4*>(weights + i0 + 4 * q * HIST_THREADS);
#pragma unroll
            for (int q = 0; q < VECS; ++q) add(w[q], i0 + 4 * q * HIST_THREADS, 4);
        } else {
            for (int q = 0; q < VECS; ++q) {
                const int64_t i = i0 + 4 * q * HIST_THREADS;
                const int valid = old - i >= 4 ? 4 : old > i ? (int)(old - i) : 0;
                f32x4 w = 0.0f;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (j < valid) w[j] = weights[i + j];
                add(w, i, valid);
            }
        }
    }
    if (zeros && lane == 0) atomicAdd(own + ((ZERO >> shift) & ((1u << bits) - 1)) * HIST_COPIES, zeros);
    __syncthreads();
    for (int b = threadIdx.x; b < HIST_BINS; b += HIST_THREADS) {
        uint32_t n = 0;
#pragma unroll
        for (int c = 0; c < HIST_COPIES; ++c) n += h[b * HIST_COPIES + c];
        if (n) atomicAdd(&s->hist[PASS][b], n);
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

// The threshold of a finished select, and whether all rows that share its upper 22 bits equal it (ties at zero, or one row):
// then the bits alone tell what is kept.
struct Threshold {
    uint32_t key, need;
    bool one;
};
__device__ __forceinline__ Threshold threshold_of(const SelectState* __restrict__ s, uint2 at) {
    return {at.x, at.y, s->hist[2][at.x & 1023u] == s->hist[1][s->at[2].x & 2047u]};
}

// A lane's bit of a word that is the same in all lanes.
__device__ __forceinline__ bool lane_bit(uint64_t word) { return __builtin_amdgcn_inverse_ballot_w64(word); }

// A segment's rows above the threshold (the recent ones among them) and at it, for a wave.
__device__ __forceinline__ SegmentBits load_segment(int64_t segment, int64_t old, const SegmentBits* __restrict__ segments) {
    SegmentBits b = {};
    if (segment * SEGMENT < old) b = segments[segment];
    return b;
}
__device__ __forceinline__ void resolve_segment(SegmentBits& b, int64_t segment, int64_t N, int64_t old,
                                                const float* __restrict__ weights, const Threshold& t) {
    const int64_t first = segment * SEGMENT, i = first + 4 * (int)(threadIdx.x & (WAVE - 1));
    if (!t.one && (b.level[0] | b.level[1] | b.level[2] | b.level[3]) != 0) {
        float w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = lane_bit(b.level[j]) ? weights[i + j] : 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool in = lane_bit(b.level[j]);
            const uint32_t k = weight_key(w[j]);
            b.above[j] |= __ballot(in && k > t.key);
            b.level[j] = __ballot(in && k == t.key);
        }
    }
    if (first + SEGMENT > old) {
#pragma unroll
        for (int j = 0; j < 4; ++j) b.above[j] |= __ballot(i + j >= old && i + j < N);
    }
}
__device__ __forceinline__ uint32_t count_rows(const uint64_t (&word)[4]) {
    return (uint32_t)(__popcll(word[0]) + __popcll(word[1]) + __popcll(word[2]) + __popcll(word[3]));
}

constexpr int SELECT_WAVES = SELECT_THREADS / WAVE;
constexpr int WAVE_SEGMENTS = SELECT_ROWS / SEGMENT / SELECT_WAVES;   // of a tile

// Per workgroup, a run of `tiles` tiles: rows above the threshold and rows that equal it (20 M rows: 9.6 us, 16.8 when it
// read the weights).
__global__ void __launch_bounds__(SELECT_THREADS) select_count_kernel(int64_t N, int64_t old, int tiles,
                                                                      const float* __restrict__ weights,
                                                                      SelectState* __restrict__ s,
                                                                      const SegmentBits* __restrict__ segments,
                                                                      uint2* __restrict__ counts) {
    __shared__ uint2 s_w[SELECT_WAVES];
    const uint2 at = find_bin<2, SELECT_THREADS>(s->hist[2], s->at[2]);
    if (blockIdx.x == 0 && threadIdx.x == 0) s->at[3] = at;
    const Threshold t = threshold_of(s, at);
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / WAVE);
    uint32_t above = 0, level = 0;
    const int64_t first = (int64_t)blockIdx.x * tiles * (SELECT_ROWS / SEGMENT), all = (N + SEGMENT - 1) / SEGMENT;
    const int64_t end = first + tiles * (SELECT_ROWS / SEGMENT) < all ? first + tiles * (SELECT_ROWS / SEGMENT) : all;
    for (int64_t x = first + wave * WAVE_SEGMENTS; x < end; x += SELECT_WAVES * WAVE_SEGMENTS) {
        SegmentBits b[WAVE_SEGMENTS];   // the loads of all of them first
#pragma unroll
        for (int y = 0; y < WAVE_SEGMENTS; ++y) b[y] = load_segment(x + y, old, segments);
#pragma unroll
        for (int y = 0; y < WAVE_SEGMENTS; ++y) {
            resolve_segment(b[y], x + y, N, old, weights, t);
            above += count_rows(b[y].above);
            level += count_rows(b[y].level);
        }
    }
    if ((threadIdx.x & 63) == 0) s_w[wave] = make_uint2(above, level);
    __syncthreads();
    if (threadIdx.x == 0) {
        uint2 c = make_uint2(0u, 0u);
        for (int w = 0; w < SELECT_WAVES; ++w) {
            c.x += s_w[w].x;
            c.y += s_w[w].y;
        }
        counts[blockIdx.x] = c;
    }
}

// The bits of the words below a lane.
__device__ __forceinline__ uint32_t count_below(const uint64_t (&word)[4]) {
    uint32_t n = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        n = __builtin_amdgcn_mbcnt_hi((uint32_t)(word[j] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)word[j], n));
    return n;
}

// The kept rows of a tile are gathered in LDS and leave in one run (16 M of 20 M rows: 23 us, 34 with each lane storing its
// own, 27 when it read the weights); bound by its stores, 64 MB, and the chain of loads in front of them.
__global__ void __launch_bounds__(SELECT_THREADS) select_write_kernel(int64_t N, int64_t old, int tiles,
                                                                      const float* __restrict__ weights,
                                                                      const SelectState* __restrict__ s,
                                                                      const SegmentBits* __restrict__ segments,
                                                                      const uint2* __restrict__ counts,
                                                                      int32_t* __restrict__ rows) {
    __shared__ uint32_t s_w[4];
    __shared__ uint2 s_count[SELECT_WAVES];
    __shared__ __attribute__((aligned(16))) int32_t s_rows[SELECT_ROWS + 4];
    const Threshold t = threshold_of(s, s->at[3]);
    const uint32_t need = t.need;
    uint32_t above = 0, level = 0;   // rows of the workgroups before this one
    {
        constexpr int LOADS = SELECT_GROUPS / SELECT_THREADS;   // all at once
        uint2 c[LOADS];
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            const uint32_t b = u * SELECT_THREADS + threadIdx.x;
            c[u] = b < blockIdx.x ? counts[b] : make_uint2(0u, 0u);
        }
#pragma unroll
        for (int u = 0; u < LOADS; ++u) {
            above += c[u].x;
            level += c[u].y;
        }
    }
    above = block_sum_u32(above, s_w);
    level = block_sum_u32(level, s_w);
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / WAVE);
    for (int k = 0; k < tiles; ++k) {
        const int64_t tile = (int64_t)blockIdx.x * tiles + k;
        if (tile * SELECT_ROWS >= N) break;
        const int64_t segment = tile * (SELECT_ROWS / SEGMENT) + wave * WAVE_SEGMENTS;
        SegmentBits b[WAVE_SEGMENTS];
        uint32_t na = 0, nl = 0;
#pragma unroll
        for (int x = 0; x < WAVE_SEGMENTS; ++x) b[x] = load_segment(segment + x, old, segments);
#pragma unroll
        for (int x = 0; x < WAVE_SEGMENTS; ++x) {
            resolve_segment(b[x], segment + x, N, old, weights, t);
            na += count_rows(b[x].above);
            nl += count_rows(b[x].level);
        }
        if ((threadIdx.x & 63) == 0) s_count[wave] = make_uint2(na, nl);
        __syncthreads();
        uint32_t pa = 0, pl = level, tile_above = 0, tile_level = 0;   // rows before the segment: above, in the tile; at the threshold
        for (int w = 0; w < SELECT_WAVES; ++w) {
            const uint2 c = s_count[w];
            pa += w < wave ? c.x : 0u;
            pl += w < wave ? c.y : 0u;
            tile_above += c.x;
            tile_level += c.y;
        }
        const uint32_t level_at = level < need ? level : need;   // rows at the threshold kept before the tile
        const uint32_t level_end = level + tile_level;
        const bool all_level = level_end <= need;
        const uint32_t kept = tile_above + (all_level ? level_end : need) - level_at;
        // the list starts where its first row falls in sixteen bytes of the output, so that it leaves in whole vectors
        int32_t* to = rows + (above + level_at);
        const uint32_t skip = (uint32_t)((uintptr_t)to >> 2) & 3u;
        if (all_level || level >= need) {   // every tile but one: the rows at the threshold stay all, or go all
            uint32_t out = skip + pa + (all_level ? pl - level : 0u);
#pragma unroll
            for (int x = 0; x < WAVE_SEGMENTS; ++x) {
#pragma unroll
                for (int j = 0; j < 4; ++j) b[x].above[j] |= all_level ? b[x].level[j] : 0ull;
                uint32_t at = out + count_below(b[x].above);
                const uint32_t i = (uint32_t)((segment + x) * SEGMENT) + 4 * (threadIdx.x & (WAVE - 1));
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (lane_bit(b[x].above[j])) s_rows[at++] = (int32_t)(i + j);
                out += count_rows(b[x].above);
            }
        } else {
#pragma unroll
            for (int x = 0; x < WAVE_SEGMENTS; ++x) {
                uint32_t n = pa + count_below(b[x].above), l = pl + count_below(b[x].level);
                const uint32_t i = (uint32_t)((segment + x) * SEGMENT) + 4 * (threadIdx.x & (WAVE - 1));
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const bool is_above = lane_bit(b[x].above[j]), is_level = lane_bit(b[x].level[j]);
                    if (is_above || (is_level && l < need)) s_rows[skip + n + (l < need ? l : need) - level_at] = (int32_t)(i + j);
                    n += is_above ? 1u : 0u;
                    l += is_level ? 1u : 0u;
                }
                pa += count_rows(b[x].above);
                pl += count_rows(b[x].level);
            }
        }
        __syncthreads();
        const uint32_t end = skip + kept, vectors = end >> 2;
        int4* out4 = reinterpret_cast<int4*>(to - skip);
        for (uint32_t v = threadIdx.x + (skip ? 1u : 0u); v < vectors; v += SELECT_THREADS) out4[v] = reinterpret_cast<int4*>(s_rows)[v];
        if (threadIdx.x < 8) {   // what is left of the first vector and of the last
            const uint32_t x = threadIdx.x < 4 ? threadIdx.x : (vectors << 2) + threadIdx.x - 4;
            if (x >= skip && x < end && (threadIdx.x < 4 ? skip != 0 && vectors > 0 : true)) to[x - skip] = s_rows[x];
        }
        above += tile_above;
        level = level_end;
        __syncthreads();
    }
}

// The whole selection in one workgroup, the keys in registers: one launch, which is what a small model's costs (5000 rows:
// 10.7 us a call, six launches 19; with sixteen keys a thread 16384 rows take 22 us, more than the six launches).
constexpr int SMALL_THREADS = 1024;
constexpr int SMALL_PER = 8;
constexpr int SMALL_ROWS = SMALL_PER * SMALL_THREADS;
template <int PASS>
__device__ __forceinline__ uint2 small_pass(uint32_t* h, const uint32_t (&key)[SMALL_PER], uint32_t valid, uint2 at) {
    constexpr int shift = pass_shift(PASS), bits = pass_bits(PASS);
    for (int b = threadIdx.x; b < HIST_BINS; b += SMALL_THREADS) h[b] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < SMALL_PER; ++j) {
        const bool in = (valid >> j & 1u) && (PASS == 0 || (uint32_t)((uint64_t)key[j] >> (shift + bits)) == at.x);
        const uint32_t bin = (key[j] >> shift) & ((1u << bits) - 1);
        // the lanes that share the first active lane's bin are added at once: weights repeat
        const uint64_t act = __ballot(in);
        if (act == 0) continue;
        const int leader = __builtin_ctzll(act);
        const bool same = in && bin == (uint32_t)__builtin_amdgcn_readlane((int)bin, leader);
        const uint64_t m = __ballot(same);
        if ((int)(threadIdx.x & 63) == leader) atomicAdd(&h[bin], (uint32_t)__popcll(m));
        else if (in && !same) atomicAdd(&h[bin], 1u);
    }
    __syncthreads();
    return find_bin<PASS, SMALL_THREADS>(h, at);
}

__global__ void __launch_bounds__(SMALL_THREADS) select_small_kernel(int N, int old, uint32_t need_all,
                                                                     const float* __restrict__ weights,
                                                                     int32_t* __restrict__ rows) {
    __shared__ uint32_t h[HIST_BINS];
    __shared__ uint32_t s_scan[SMALL_THREADS / WAVE];
    const int i = SMALL_PER * (int)threadIdx.x;
    uint32_t key[SMALL_PER], valid = 0;
#pragma unroll
    for (int j = 0; j < SMALL_PER; ++j) {
        key[j] = i + j < old ? weight_key(weights[i + j]) : 0u;
        valid |= (i + j < old ? 1u : 0u) << j;
    }
    uint2 at = make_uint2(0u, need_all);
    at = small_pass<0>(h, key, valid, at);
    at = small_pass<1>(h, key, valid, at);
    at = small_pass<2>(h, key, valid, at);
    uint32_t above = 0, level = 0;
#pragma unroll
    for (int j = 0; j < SMALL_PER; ++j) {
        const bool v = valid >> j & 1u;
        above |= ((v ? key[j] > at.x : i + j < N) ? 1u : 0u) << j;
        level |= (v && key[j] == at.x ? 1u : 0u) << j;
    }
    const uint32_t own = (uint32_t)__popc(above) | (uint32_t)__popc(level) << 16;   // each at most SMALL_ROWS in all: 16 bits hold it
    uint32_t before = wave_scan_u32(own);
    if ((threadIdx.x & 63) == 63) s_scan[threadIdx.x >> 6] = before;
    __syncthreads();
    before -= own;
    for (int w = 0; w < (int)(threadIdx.x >> 6); ++w) before += s_scan[w];
    uint32_t pl = before >> 16, out = (before & 0xffffu) + (pl < at.y ? pl : at.y);
#pragma unroll
    for (int j = 0; j < SMALL_PER; ++j) {
        const bool l = level >> j & 1u;
        if ((above >> j & 1u) || (l && pl < at.y)) rows[out++] = i + j;
        pl += l ? 1u : 0u;
    }
}

__global__ void __launch_bounds__(256) select_tail_kernel(int64_t first, int64_t count, int32_t* __restrict__ rows) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < count) rows[i] = (int32_t)(first + i);
}

// ------------------------------------------------------------------ rows of many tensors
// A row is cut into the widest units that every address is a multiple of: 16, 8, 4, 2 or 1 bytes.  A workgroup copies a
// run of rows; a run starts at a multiple of sixteen bytes of the copy.
constexpr int ROWS_TABLE = 96;              // tensors per launch
constexpr int ROWS_BYTES = 16384;           // bytes of a workgroup, about
struct RowsTable {
    const void* src[ROWS_TABLE];
    void* dst[ROWS_TABLE];
    int64_t pitch[ROWS_TABLE];           // bytes between source rows
    uint32_t units[ROWS_TABLE];          // units of a row
    uint32_t first[ROWS_TABLE];          // first workgroup of each tensor
    uint8_t unit_shift[ROWS_TABLE];      // a unit is 1 << unit_shift bytes
    int n;
};

// Rows of a workgroup: a multiple of sixteen.
__host__ __device__ inline uint32_t rows_per_group(uint32_t units, int unit_shift) {
    const uint64_t row_bytes = (uint64_t)units << unit_shift;
    const uint32_t r = (uint32_t)(ROWS_BYTES / (row_bytes < ROWS_BYTES ? row_bytes : (uint64_t)ROWS_BYTES));
    return r < 16 ? 16u : r & ~15u;
}

// A run of rows: unit x of the copy is unit x mod M of row rows[x / M].
struct RowRun {
    const char* src;
    int64_t pitch;
    const int32_t* rows;
    uint32_t M, magic;
    // x / M for x < 2^32, by one multiplication where x * M < 2^32 (magic = 0: it is not, or M = 1)
    __device__ __forceinline__ uint32_t row(uint32_t x) const { return M == 1 ? x : (uint32_t)(((uint64_t)x * magic) >> 32); }
    __device__ __forceinline__ const char* at(uint32_t r) const { return src + (int64_t)rows[r] * pitch; }
};

// Unit by unit: rows of more than about 32 KB, whose units a multiplication cannot divide, and copies that do not start
// at a multiple of sixteen bytes.
template <typename T>
__device__ __forceinline__ void copy_units(const RowRun& s, T* __restrict__ dst, uint64_t total) {
    for (uint64_t x = threadIdx.x; x < total; x += 256) {
        const uint32_t r = (uint32_t)(x / s.M);
        dst[x] = reinterpret_cast<const T*>(s.at(r))[x - (uint64_t)r * s.M];
    }
}

// Sixteen bytes of the copy at a time.  They lie side by side in the source as well when they are in one row, or in rows
// that follow each other there: then one load fetches them, which needs no alignment of its own.
template <typename T>
using vector_of = f32x4 __attribute__((aligned(sizeof(T))));

// At most two rows in a vector.  Four vectors are in flight per thread, and all row numbers are read before the first of
// them: loads return in order, and a row number behind a vector would wait for it.  Four of five of 2.5 M rows: 45 floats
// 5.5 TB/s of reads and writes, 3 floats 4.8 (3.5 with row numbers between the vectors, 3.5 with four 4-byte loads for
// a vector, 2.6 with a float a thread).
template <typename T>
__device__ __forceinline__ void copy_wide(const RowRun& s, T* __restrict__ dst, uint32_t vectors) {
    constexpr uint32_t N = 16 / sizeof(T);
    for (uint32_t q0 = threadIdx.x; q0 < vectors; q0 += 4 * 256) {
        const T *here[4], *next[4];   // unit j of a vector is here[j], or next[j] behind the row's end
        uint32_t left[4];             // units of the vector's first row
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint32_t x = (q0 + u * 256 < vectors ? q0 + u * 256 : q0) * N, r = s.row(x), c = x - r * s.M;
            here[u] = next[u] = reinterpret_cast<const T*>(s.at(r)) + c;
            left[u] = s.M - c;
            if (left[u] < N) next[u] = reinterpret_cast<const T*>(s.at(r + 1)) - left[u];
        }
        f32x4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (here[u] == next[u]) {
                v[u] = *reinterpret_cast<const vector_of<T>*>(here[u]);
            } else {
                union { f32x4 v; T t[N]; } e;
#pragma unroll
                for (uint32_t j = 0; j < N; ++j) e.t[j] = (j < left[u] ? here[u] : next[u])[j];
                v[u] = e.v;
            }
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (q0 + u * 256 < vectors) __builtin_nontemporal_store(v[u], (f32x4*)dst + q0 + u * 256);
    }
}

// Three rows and more in a vector.
template <typename T>
__device__ __forceinline__ void copy_narrow(const RowRun& s, T* __restrict__ dst, uint32_t vectors) {
    constexpr uint32_t N = 16 / sizeof(T);
    const bool dense = s.pitch == (int64_t)(s.M * sizeof(T));
    for (uint32_t q = threadIdx.x; q < vectors; q += 256) {
        const uint32_t x = q * N, c0 = x - s.row(x) * s.M;
        int32_t at[N];
#pragma unroll
        for (uint32_t j = 0; j < N; ++j) at[j] = s.rows[s.row(x + j)];
        f32x4 v;
        // rows that follow each other, each one: repeated and unordered rows can span as much as a run does
        bool run = dense;
#pragma unroll
        for (uint32_t j = 1; j < N; ++j) run = run && at[j] - at[j - 1] == (int32_t)(s.row(x + j) - s.row(x + j - 1));
        if (run) {
            v = *reinterpret_cast<const vector_of<T>*>(s.src + (int64_t)at[0] * s.pitch + c0 * sizeof(T));
        } else {
            union { f32x4 v; T t[N]; } e;
#pragma unroll
            for (uint32_t j = 0; j < N; ++j)
                e.t[j] = reinterpret_cast<const T*>(s.src + (int64_t)at[j] * s.pitch)[x + j - s.row(x + j) * s.M];
            v = e.v;
        }
        __builtin_nontemporal_store(v, (f32x4*)dst + q);
    }
}

template <typename T>
__device__ __forceinline__ void copy_run(const RowRun& s, T* __restrict__ dst, uint32_t total) {
    constexpr uint32_t N = 16 / sizeof(T);
    const uint32_t vectors = total / N;
    if (s.M + 1 >= N) copy_wide<T>(s, dst, vectors);
    else copy_narrow<T>(s, dst, vectors);
    const uint32_t x = vectors * N + threadIdx.x;
    if (x < total) {
        const uint32_t r = s.row(x);
        dst[x] = reinterpret_cast<const T*>(s.at(r))[x - r * s.M];
    }
}

template <typename T>
__device__ __forceinline__ void copy_rows(const RowRun& s, char* dst, uint64_t total) {
    if ((s.magic || s.M == 1) && ((uintptr_t)dst & 15) == 0) copy_run<T>(s, (T*)dst, (uint32_t)total);
    else copy_units<T>(s, (T*)dst, total);
}

__global__ void __launch_bounds__(256) gather_rows_multi_kernel(const RowsTable t, const int32_t* __restrict__ rows,
                                                                int64_t K) {
    int k = 0, hi = t.n - 1;
    while (k < hi) {
        const int mid = (k + hi + 1) >> 1;
        if (t.first[mid] <= blockIdx.x) k = mid; else hi = mid - 1;
    }
    const uint32_t M = t.units[k];
    const int sh = t.unit_shift[k];
    const uint32_t R = rows_per_group(M, sh);
    const int64_t row0 = (int64_t)(blockIdx.x - t.first[k]) * R;
    const uint64_t total = (uint64_t)(K - row0 < (int64_t)R ? K - row0 : (int64_t)R) * M;
    char* dst = (char*)t.dst[k] + ((row0 * M) << sh);
    const uint32_t magic = M > 1 && (uint64_t)R * M * M < (1ull << 32) ? 0xffffffffu / M + 1 : 0;
    const RowRun s = {(const char*)t.src[k], t.pitch[k], rows + row0, M, magic};
    if (sh == 4) copy_rows<f32x4>(s, dst, total);
    else if (sh == 3) copy_rows<uint2>(s, dst, total);
    else if (sh == 2) copy_rows<uint32_t>(s, dst, total);
    else if (sh == 1) copy_rows<uint16_t>(s, dst, total);
    else copy_rows<uint8_t>(s, dst, total);
}

// ------------------------------------------------------------------ host
hipError_t launch_accumulate_weights(int64_t N, float* weights, int views, const float* const* contributions,
                                     const float* opacity, float decay, hipStream_t st) {
    if (N <= 0) return hipSuccess;
    uintptr_t bits = (uintptr_t)weights | (uintptr_t)opacity;
    for (int v = 0; v < views; ++v) bits |= (uintptr_t)contributions[v];
    int first = 0;
    do {
        WeightArgs a;
        a.views = views - first < WEIGHT_VIEWS ? views - first : WEIGHT_VIEWS;
        for (int v = 0; v < WEIGHT_VIEWS; ++v) a.contribution[v] = v < a.views ? contributions[first + v] : nullptr;
        a.opacity = opacity;
        a.weights = weights;
        a.N = N;
        a.decay = first == 0 ? decay : 1.0f;
        if ((bits & 15) == 0)
            hipLaunchKernelGGL(accumulate_weights_kernel<4>, dim3((unsigned)((N + 1023) / 1024)), dim3(256), 0, st, a);
        else
            hipLaunchKernelGGL(accumulate_weights_kernel<1>, dim3((unsigned)((N + 255) / 256)), dim3(256), 0, st, a);
        first += WEIGHT_VIEWS;
    } while (first < views);
    return hipGetLastError();
}

static size_t select_fixed_bytes() { return align_up(sizeof(SelectState), 256) + align_up(SELECT_GROUPS * sizeof(uint2), 256); }

size_t evict_temp_bytes(int64_t N) {
    return select_fixed_bytes() + (N > SMALL_ROWS ? (size_t)((N + SEGMENT - 1) / SEGMENT) * sizeof(SegmentBits) : 0);
}

// One vector a thread while that gives every workgroup at most one step, four from there on.
template <int PASS>
static void launch_hist(int64_t old, const float* weights, SelectState* s, SegmentBits* segments, hipStream_t st) {
    const int64_t steps = (old + 4 * HIST_THREADS - 1) / (4 * HIST_THREADS);
    if (steps <= HIST_GROUPS) {
        hipLaunchKernelGGL((select_hist_kernel<PASS, 1>), dim3((unsigned)steps), dim3(HIST_THREADS), 0, st, old, weights, s, segments);
    } else {
        constexpr int VECS = 4;
        const int64_t wide = (steps + VECS - 1) / VECS;
        hipLaunchKernelGGL((select_hist_kernel<PASS, VECS>), dim3((unsigned)(wide < HIST_GROUPS ? wide : HIST_GROUPS)),
                           dim3(HIST_THREADS), 0, st, old, weights, s, segments);
    }
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
    if (N <= SMALL_ROWS) {
        hipLaunchKernelGGL(select_small_kernel, dim3(1), dim3(SMALL_THREADS), 0, st, (int)N, (int)old, (uint32_t)(keep - recent),
                           weights, rows);
        return hipGetLastError();
    }
    SelectState* s = (SelectState*)temp;
    uint2* counts = (uint2*)((char*)temp + align_up(sizeof(SelectState), 256));
    SegmentBits* segments = (SegmentBits*)((char*)temp + select_fixed_bytes());
    const int64_t all = (N + SELECT_ROWS - 1) / SELECT_ROWS;
    const int tiles = (int)((all + SELECT_GROUPS - 1) / SELECT_GROUPS);
    const dim3 groups((unsigned)((all + tiles - 1) / tiles));
    hipLaunchKernelGGL(select_clear_kernel, dim3(24), dim3(256), 0, st, s, (uint32_t)(keep - recent));
    launch_hist<0>(old, weights, s, segments, st);
    launch_hist<1>(old, weights, s, segments, st);
    launch_hist<2>(old, weights, s, segments, st);
    hipLaunchKernelGGL(select_count_kernel, groups, dim3(SELECT_THREADS), 0, st, N, old, tiles, weights, s, segments, counts);
    hipLaunchKernelGGL(select_write_kernel, groups, dim3(SELECT_THREADS), 0, st, N, old, tiles, weights, s, segments, counts, rows);
    return hipGetLastError();
}

hipError_t launch_gather_rows_multi(int n, const GsoRowCopy* copies, const int32_t* rows, int64_t K, hipStream_t st) {
    for (int i = 0; i < n;) {
        RowsTable t;
        t.n = 0;
        int64_t chunks = 0;
        for (; i < n && t.n < ROWS_TABLE; ++i) {
            const GsoRowCopy& c = copies[i];
            if (c.row_bytes <= 0 || K <= 0) continue;
            const uint64_t bits = (uint64_t)c.row_bytes | (uint64_t)c.src_pitch | (uint64_t)(uintptr_t)c.src | (uint64_t)(uintptr_t)c.dst;
            const int sh = (bits & 15) == 0 ? 4 : (bits & 7) == 0 ? 3 : (bits & 3) == 0 ? 2 : (bits & 1) == 0 ? 1 : 0;
            const int64_t per = rows_per_group((uint32_t)(c.row_bytes >> sh), sh);
            const int64_t more = (K + per - 1) / per;
            if (t.n > 0 && chunks + more > 0x7fffffff) break;
            t.src[t.n] = c.src;
            t.dst[t.n] = c.dst;
            t.pitch[t.n] = c.src_pitch;
            t.units[t.n] = (uint32_t)(c.row_bytes >> sh);
            t.unit_shift[t.n] = (uint8_t)sh;
            t.first[t.n] = (uint32_t)chunks;
            chunks += more;
            ++t.n;
        }
        if (t.n == 0) break;
        hipLaunchKernelGGL(gather_rows_multi_kernel, dim3((unsigned)chunks), dim3(256), 0, st, t, rows, K);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace gs

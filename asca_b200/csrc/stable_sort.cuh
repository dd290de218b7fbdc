// Stable counting sort of n items by a key below `bins`, and the radix sort made of such passes (least significant digit first).
// Three kernels a pass, integer only:
//   1. a CTA counts the digits of its tile                              -> counts[digit][tile]
//   2. one CTA scans the counts in that order, which gives every tile the first place of each of its digits
//   3. a CTA ranks its tile's items: match_any gives a lane its rank among equal digits of its 32, a counter per warp and digit
//      what came before them in the warp's run, a scan over the warps what came before the warp
// The rank is by construction the order of the items, so the result is the same in every run.
#pragma once
#include "common.cuh"

namespace stable_sort {

constexpr int WARPS = 8, PER_LANE = 8, TILE = WARPS * 32 * PER_LANE;
constexpr int MAX_BINS = 2049;   // 8 warps' counters: 64 KiB of shared memory

// What is sorted and where it goes. Source: `ids` with everything at or past `limit` (as unsigned) taken as key `limit`, or, in a
// later pass, the keys and items that the pass before wrote.
struct Pass {
    const uint32_t* ids = nullptr;      // first pass: item i has key min(ids[i], limit)
    uint32_t limit = 0;
    const uint32_t* keys = nullptr;     // later passes
    const int32_t* items = nullptr;
    int64_t n = 0;
    int shift = 0, bins = 0;            // digit = (key >> shift) & mask, below bins
    uint32_t mask = 0xffffffffu;
    uint32_t* out_keys = nullptr;       // nullable
    int32_t* out_items = nullptr;
    int32_t* place = nullptr;           // nullable: place[item] = where it went, -1 for key `limit`
};

inline int64_t tiles(int64_t n) { return ceil_div64(n, TILE); }
inline size_t counts_bytes(int64_t n, int bins) { return ((size_t)tiles(n) * bins * 4 + 255) & ~(size_t)255; }

#ifdef __CUDACC__
__device__ __forceinline__ uint32_t key_of(const Pass& p, int64_t i) { return p.ids ? min(p.ids[i], p.limit) : p.keys[i]; }
__device__ __forceinline__ int digit_of(const Pass& p, uint32_t key) { return (int)((key >> p.shift) & p.mask); }

static __global__ void __launch_bounds__(WARPS * 32) count_kernel(const Pass p, int32_t* __restrict__ counts) {
    extern __shared__ int32_t sh[];
    for (int b = threadIdx.x; b < p.bins; b += WARPS * 32) sh[b] = 0;
    __syncthreads();
    const int64_t lo = (int64_t)blockIdx.x * TILE;
#pragma unroll
    for (int j = 0; j < PER_LANE; ++j) {
        const int64_t i = lo + j * WARPS * 32 + threadIdx.x;
        if (i < p.n) atomicAdd(&sh[digit_of(p, key_of(p, i))], 1);   // integer: any order gives the same counts
    }
    __syncthreads();
    for (int b = threadIdx.x; b < p.bins; b += WARPS * 32) counts[(int64_t)b * gridDim.x + blockIdx.x] = sh[b];
}

// counts[0, m) -> its exclusive scan, in place; one CTA. With `tiles_per_bin`, offsets[b] (nullable, n_off of them) = the first place
// of bin b.
static __global__ void __launch_bounds__(1024) scan_kernel(int32_t* __restrict__ counts, int64_t m, int64_t tiles_per_bin,
                                                           int32_t* __restrict__ offsets, int n_off) {
    __shared__ int32_t wsum[33];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int32_t base = 0;
    for (int64_t i0 = 0; i0 < m; i0 += 4096) {
        const int64_t i = i0 + threadIdx.x * 4;
        int32_t v[4], s = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = i + j < m ? counts[i + j] : 0;
            s += v[j];
        }
        int32_t inc = s;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int32_t y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        if (lane == 31) wsum[w] = inc;
        __syncthreads();
        if (w == 0) {
            const int32_t x = wsum[lane];
            int32_t y = x;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int32_t z = __shfl_up_sync(0xffffffffu, y, o);
                if (lane >= o) y += z;
            }
            wsum[lane] = y - x;
            if (lane == 31) wsum[32] = y;
        }
        __syncthreads();
        int32_t at = base + wsum[w] + inc - s;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (i + j < m) {
                counts[i + j] = at;
                if (offsets && (i + j) % tiles_per_bin == 0 && (i + j) / tiles_per_bin < n_off) offsets[(i + j) / tiles_per_bin] = at;
            }
            at += v[j];
        }
        base += wsum[32];
        __syncthreads();
    }
}

static __global__ void __launch_bounds__(WARPS * 32) place_kernel(const Pass p, const int32_t* __restrict__ start) {
    extern __shared__ int32_t sh[];   // [warp][bin]: counts, then the first place of the warp's next item
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int32_t* run = sh + w * p.bins;
    for (int b = lane; b < p.bins; b += 32) run[b] = 0;
    __syncwarp();
    const int64_t lo = (int64_t)blockIdx.x * TILE + w * 32 * PER_LANE;
    uint32_t key[PER_LANE];
    int32_t item[PER_LANE], rank[PER_LANE];
#pragma unroll
    for (int j = 0; j < PER_LANE; ++j) {
        const int64_t i = lo + j * 32 + lane;
        const bool live = i < p.n;
        key[j] = live ? key_of(p, i) : 0u;
        item[j] = live ? (p.items ? p.items[i] : (int32_t)i) : -1;
    }
#pragma unroll
    for (int j = 0; j < PER_LANE; ++j) {
        const bool live = item[j] >= 0;
        const unsigned act = __ballot_sync(0xffffffffu, live);
        if (live) {
            const int b = digit_of(p, key[j]);
            const unsigned peers = __match_any_sync(act, b);
            const int before = __popc(peers & ((1u << lane) - 1u));
            rank[j] = run[b] + before;
            __syncwarp(act);
            if (before == 0) run[b] += __popc(peers);   // one leader per distinct digit
        }
        __syncwarp();
    }
    __syncthreads();
    for (int b = threadIdx.x; b < p.bins; b += WARPS * 32) {
        int32_t at = start[(int64_t)b * gridDim.x + blockIdx.x];
#pragma unroll
        for (int i = 0; i < WARPS; ++i) {
            const int32_t c = sh[i * p.bins + b];
            sh[i * p.bins + b] = at;
            at += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < PER_LANE; ++j) {
        if (item[j] < 0) continue;
        const int32_t at = run[digit_of(p, key[j])] + rank[j];
        if (p.out_keys) p.out_keys[at] = key[j];
        if (p.out_items) p.out_items[at] = item[j];
        if (p.place) p.place[item[j]] = key[j] == p.limit ? -1 : at;
    }
}

// One pass; counts: counts_bytes(n, bins) of scratch. offsets (nullable): the first place of each of the first n_off bins.
static inline int run(asca_ctx* ctx, const Pass& p, int32_t* counts, int32_t* offsets, int n_off) {
    const int64_t t = tiles(p.n);
    const size_t smem = (size_t)WARPS * p.bins * 4;
    if (smem > 48 * 1024) ASCA_CUDA(ctx, cudaFuncSetAttribute(place_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    count_kernel<<<(unsigned)t, WARPS * 32, (size_t)p.bins * 4, ctx->stream>>>(p, counts);
    ASCA_CHECK_LAUNCH(ctx);
    scan_kernel<<<1, 1024, 0, ctx->stream>>>(counts, t * p.bins, t, offsets, n_off);
    ASCA_CHECK_LAUNCH(ctx);
    place_kernel<<<(unsigned)t, WARPS * 32, smem, ctx->stream>>>(p, counts);
    ASCA_CHECK_LAUNCH(ctx);
    return ASCA_OK;
}
#endif

}  // namespace stable_sort

// Stable counting sort of n items by a key, in passes over its digits (least significant first; one pass where the keys are few).
//
// Up to 4,096 items: one CTA does all passes in one launch. More: two launches a pass, a CTA to a tile of 2,048 items -- the first
// counts the tile's digits, the second adds up what the tiles in front of its own counted and places its items; where that table has
// more than 65,536 entries, a launch between the two scans it once instead of every CTA for itself.
// In both, a warp owns a run of consecutive items; a ballot for every bit of the digit gives a lane its rank among equal digits of its 32
// (match_any, which goes over the distinct digits one by one, takes longer where they are many), a counter per warp and digit what
// came before them in the run, a scan over the warps what came before the warp. The rank is by construction the order
// of the items, so the result is the same in every run. Bound by launches and the latency of a pass's steps, not by bytes.
#pragma once
#include "common.cuh"
#include "row_io.cuh"

#include <algorithm>

namespace stable_sort {

constexpr int PER = 4;                           // items a lane
constexpr int SMALL = 1024 * PER, TILE = 512 * PER;
constexpr int64_t OWN_SCAN = 65536;              // entries of the table that every CTA may add up for itself
constexpr int MAX_BINS = 2049;

// Item i of the first pass has key min(ids[i], limit): everything at or past `limit`, as unsigned, is one key. Pass p writes keys[p & 1]
// (nullable in a single pass) and items[p & 1].
struct Job {
    const uint32_t* ids;
    uint32_t limit;
    int64_t n;
    int passes, digit, bins;      // digit: bits of a pass (one pass: the whole key); bins: digits that a pass may meet
    uint32_t* keys[2];
    int32_t* items[2];
    int32_t *place, *offsets;     // of a single pass, nullable: where each item went, -1 for key `limit`; the first place of each bin
};

inline int64_t tiles(int64_t n) { return ceil_div64(n, TILE); }
inline size_t scratch_bytes(int64_t n, int bins) { return n <= SMALL ? 0 : ((size_t)tiles(n) * bins * 4 + 255) & ~(size_t)255; }

#ifdef __CUDACC__
__device__ __forceinline__ uint32_t mask_of(const Job& j) { return j.passes > 1 ? (1u << j.digit) - 1 : 0xffffffffu; }
// (no indexing by a variable: the arguments stay where they are)
__device__ __forceinline__ uint32_t* keys_to(const Job& j, int pass) { return pass & 1 ? j.keys[1] : j.keys[0]; }
__device__ __forceinline__ int32_t* items_to(const Job& j, int pass) { return pass & 1 ? j.items[1] : j.items[0]; }
__device__ __forceinline__ uint32_t key_of(const Job& j, int pass, int64_t i) { return pass == 0 ? min(j.ids[i], j.limit) : keys_to(j, pass + 1)[i]; }

// A CTA's scan of one value a thread; `total` in every thread.
template <int THREADS>
__device__ __forceinline__ int exclusive_scan(int v, int32_t* wsum, int& total) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    int inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
    }
    if (lane == 31) wsum[w] = inc;
    __syncthreads();
    int x = lane < THREADS / 32 ? wsum[lane] : 0, y = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int z = __shfl_up_sync(0xffffffffu, y, o);
        if (lane >= o) y += z;
    }
    total = __shfl_sync(0xffffffffu, y, 31);
    const int before = __shfl_sync(0xffffffffu, y - x, w);
    __syncthreads();   // wsum may be written again
    return before + inc - v;
}

// What both kernels do with a CTA's items: load, rank inside the warp's run. counts [warp][bins], 16 bits: at most 128 of a warp.
struct Items {
    uint32_t key[PER];
    int32_t item[PER];
    int rank[PER];
};
__device__ __forceinline__ void load_items(const Job& j, int pass, int64_t lo, int per, Items& t) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int64_t at = lo + i * 32 + lane;
        t.item[i] = -1;
        t.key[i] = 0;
        if (i < per && at < j.n) {
            t.key[i] = key_of(j, pass, at);
            t.item[i] = pass == 0 ? (int32_t)at : items_to(j, pass + 1)[at];
        }
    }
}
__device__ __forceinline__ void rank_items(int bins, int shift, uint32_t mask, uint16_t* run, Items& t) {
    const int lane = threadIdx.x & 31;
    for (int b = lane; b < bins; b += 32) run[b] = 0;
    __syncwarp();
    const int bits = 32 - __clz(bins - 1);   // of a digit (one bin: none)
    unsigned peers[PER];
    int b[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        b[i] = (int)((t.key[i] >> shift) & mask);
        peers[i] = __ballot_sync(0xffffffffu, t.item[i] >= 0);
    }
    for (int k = 0; k < bits; ++k) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const bool set = b[i] >> k & 1;
            const unsigned m = __ballot_sync(0xffffffffu, set);
            peers[i] &= set ? m : ~m;
        }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int before = __popc(peers[i] & ((1u << lane) - 1u));
        int had = 0;
        if (t.item[i] >= 0) had = run[b[i]];
        t.rank[i] = had + before;
        __syncwarp();
        if (t.item[i] >= 0 && before == 0) run[b[i]] = (uint16_t)(had + __popc(peers[i]));   // one leader per distinct digit
        __syncwarp();
    }
}
// Exclusive scan of each bin over the CTA's warps, in place, four lanes a bin; the totals to tot (nullable).
template <int THREADS>
__device__ __forceinline__ void scan_warps(uint16_t* counts, int bins, int32_t* tot) {
    constexpr int Q = THREADS / 32 / 4;   // a lane's warps
    const int part = threadIdx.x & 3;
    for (int b0 = 0; b0 < bins; b0 += THREADS / 4) {
        const int b = b0 + (threadIdx.x >> 2);
        int c[Q], s = 0;
#pragma unroll
        for (int i = 0; i < Q; ++i) {
            c[i] = b < bins ? counts[(part * Q + i) * bins + b] : 0;
            s += c[i];
        }
        int inc = s;
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, inc, o, 4);
            if (part >= o) inc += y;
        }
        int at = inc - s;
        if (b < bins) {
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                counts[(part * Q + i) * bins + b] = (uint16_t)at;
                at += c[i];
            }
            if (tot && part == 3) tot[b] = at;
        }
    }
}
// Ranks the items of one CTA of 1,024 threads: `first` gets the first place of each bin, t.rank and the warps' counters the rest.
__device__ __forceinline__ void rank_cta(int bins, int shift, uint32_t mask, uint16_t* counts, int32_t* first, int32_t* wsum, Items& t) {
    rank_items(bins, shift, mask, counts + (threadIdx.x >> 5) * bins, t);
    __syncthreads();
    scan_warps<1024>(counts, bins, first);
    __syncthreads();
    for (int b0 = 0, carry = 0; b0 < bins; b0 += 1024) {
        const int b = b0 + threadIdx.x, v = b < bins ? first[b] : 0;
        int total;
        const int at = carry + exclusive_scan<1024>(v, wsum, total);
        carry += total;
        if (b < bins) first[b] = at;
    }
    __syncthreads();
}
__device__ __forceinline__ void put_items(const Job& j, int pass, const Items& t, const int32_t* base, const uint16_t* run) {
    const int shift = pass * j.digit;
    const uint32_t mask = mask_of(j);
    uint32_t* keys = keys_to(j, pass);
    int32_t* items = items_to(j, pass);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (t.item[i] < 0) continue;
        const int b = (int)((t.key[i] >> shift) & mask), at = base[b] + run[b] + t.rank[i];
        if (keys) keys[at] = t.key[i];
        items[at] = t.item[i];
        if (j.place) j.place[t.item[i]] = t.key[i] == j.limit ? -1 : at;
    }
}

inline size_t smem_bytes(int threads, int bins) { return (size_t)bins * 4 + (size_t)threads / 32 * bins * 2; }

static __global__ void __launch_bounds__(1024) sort_small_kernel(const Job j) {
    extern __shared__ __align__(16) int32_t sh[];   // a bin's total, then first place; the warps' counters
    __shared__ int32_t wsum[32];
    pdl_launch_dependents();
    uint16_t *counts = reinterpret_cast<uint16_t*>(sh + j.bins), *run = counts + (threadIdx.x >> 5) * j.bins;
    const int n = (int)j.n, per = (n + 1023) / 1024;
    for (int pass = 0; pass < j.passes; ++pass) {
        Items t;
        load_items(j, pass, (threadIdx.x >> 5) * per * 32, per, t);
        rank_cta(j.bins, pass * j.digit, mask_of(j), counts, sh, wsum, t);
        if (j.offsets)
            for (int b = threadIdx.x; b < j.bins; b += 1024) j.offsets[b] = sh[b];
        put_items(j, pass, t, sh, run);
        __syncthreads();   // (what the next pass reads)
    }
}

// counts[tile][bin]
static __global__ void __launch_bounds__(512) count_kernel(const Job j, int pass, int32_t* __restrict__ counts) {
    extern __shared__ __align__(16) int32_t sh[];
    pdl_wait();
    pdl_launch_dependents();
    for (int b = threadIdx.x; b < j.bins; b += 512) sh[b] = 0;
    __syncthreads();
    const int64_t lo = (int64_t)blockIdx.x * TILE;
    const uint32_t mask = mask_of(j);
    const int shift = pass * j.digit;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int64_t at = lo + i * 512 + threadIdx.x;
        if (at < j.n) atomicAdd(&sh[(key_of(j, pass, at) >> shift) & mask], 1);   // integer: any order gives the same counts
    }
    __syncthreads();
    for (int b = threadIdx.x; b < j.bins; b += 512) counts[(int64_t)blockIdx.x * j.bins + b] = sh[b];
}

// counts[tile][bin] -> the first place of the tile's items of the bin; one CTA, a thread a bin.
static __global__ void __launch_bounds__(1024) scan_kernel(const Job j, int32_t* __restrict__ counts, int n_tiles) {
    __shared__ int32_t wsum[32];
    pdl_wait();
    pdl_launch_dependents();
    for (int b0 = 0, carry = 0; b0 < j.bins; b0 += 1024) {
        const int b = b0 + threadIdx.x;
        int all = 0;
        if (b < j.bins) {
#pragma unroll 16
            for (int t = 0; t < n_tiles; ++t) all += counts[(int64_t)t * j.bins + b];
        }
        int total;
        int at = carry + exclusive_scan<1024>(all, wsum, total);
        carry += total;
        if (b < j.bins) {
            if (j.offsets) j.offsets[b] = at;
#pragma unroll 16
            for (int t = 0; t < n_tiles; ++t) {
                const int c = counts[(int64_t)t * j.bins + b];
                counts[(int64_t)t * j.bins + b] = at;
                at += c;
            }
        }
    }
}

// SCANNED: the table holds first places (scan_kernel); otherwise counts, which the CTA adds up: 512 / Q bins at a time, Q threads a bin.
template <bool SCANNED>
static __global__ void __launch_bounds__(512) place_kernel(const Job j, int pass, const int32_t* __restrict__ table, int n_tiles, int q) {
    extern __shared__ __align__(16) int32_t sh[];   // first places [bin]; the warps' counters
    __shared__ int32_t wsum[32];
    uint16_t *counts = reinterpret_cast<uint16_t*>(sh + j.bins), *run = counts + (threadIdx.x >> 5) * j.bins;
    const int mine = blockIdx.x;
    pdl_wait();
    pdl_launch_dependents();
    Items t;
    load_items(j, pass, (int64_t)mine * TILE + (threadIdx.x >> 5) * PER * 32, PER, t);
    if (SCANNED) {
        for (int b = threadIdx.x; b < j.bins; b += 512) sh[b] = table[(int64_t)mine * j.bins + b];
    } else {
        for (int b0 = 0, carry = 0; b0 < j.bins; b0 += 512 / q) {
            const int b = b0 + threadIdx.x / q;
            int before = 0, all = 0;
            if (b < j.bins) {
#pragma unroll 8
                for (int i = threadIdx.x % q; i < n_tiles; i += q) {
                    const int c = table[(int64_t)i * j.bins + b];
                    all += c;
                    if (i < mine) before += c;
                }
            }
            for (int o = 1; o < q; o <<= 1) {
                before += __shfl_xor_sync(0xffffffffu, before, o);
                all += __shfl_xor_sync(0xffffffffu, all, o);
            }
            const bool first_lane = threadIdx.x % q == 0;
            int total;
            const int first = carry + exclusive_scan<512>(first_lane ? all : 0, wsum, total);
            carry += total;
            if (b < j.bins && first_lane) {
                sh[b] = first + before;
                if (j.offsets && mine == 0) j.offsets[b] = first;
            }
        }
    }
    rank_items(j.bins, pass * j.digit, mask_of(j), run, t);   // (while the table's entries come in)
    __syncthreads();
    scan_warps<512>(counts, j.bins, nullptr);
    __syncthreads();
    put_items(j, pass, t, sh, run);
}

// Leaves the result in keys / items [(passes - 1) & 1]; table: scratch_bytes(n, bins) of scratch. Every kernel lets the next one's
// launch begin early.
static inline int sort(asca_ctx* ctx, const Job& j, int32_t* table) {
    const size_t smem = smem_bytes(j.n <= SMALL ? 1024 : 512, j.bins);
    if (j.n <= SMALL) {
        if (smem > 40 * 1024) ASCA_CUDA(ctx, cudaFuncSetAttribute(sort_small_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        sort_small_kernel<<<1, 1024, smem, ctx->stream>>>(j);
        ASCA_CHECK_LAUNCH(ctx);
        return ASCA_OK;
    }
    const int n = (int)tiles(j.n);
    const bool scanned = (int64_t)n * j.bins > OWN_SCAN;
    int q = 1;   // threads a bin
    while (q < 32 && (q * 2) * j.bins <= 512) q *= 2;
    if (smem > 40 * 1024) {
        ASCA_CUDA(ctx, cudaFuncSetAttribute(place_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        ASCA_CUDA(ctx, cudaFuncSetAttribute(place_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    }
    for (int p = 0; p < j.passes; ++p) {
        if (p == 0) count_kernel<<<(unsigned)n, 512, (size_t)j.bins * 4, ctx->stream>>>(j, p, table);
        else ASCA_CUDA(ctx, asca_launch_after(ctx, count_kernel, dim3(n), dim3(512), (size_t)j.bins * 4, j, p, table));
        if (scanned) ASCA_CUDA(ctx, asca_launch_after(ctx, scan_kernel, dim3(1), dim3(1024), 0, j, table, n));
        ASCA_CUDA(ctx, asca_launch_after(ctx, scanned ? place_kernel<true> : place_kernel<false>, dim3(n), dim3(512), smem, j, p, (const int32_t*)table, n, q));
        ctx->launches += scanned ? 3 : 2;
    }
    ASCA_CUDA(ctx, cudaGetLastError());
    return ASCA_OK;
}
#endif

}  // namespace stable_sort

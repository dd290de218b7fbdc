// Stable counting sort of n items by a key, in passes over its digits (least significant first; one pass where the keys are few).
//
// Up to 4,096 items: one CTA does all passes in one launch. More: two launches a pass, a CTA to a tile of 2,048 items -- the first
// counts the tile's digits, the second adds up what the tiles in front of its own counted and places its items; where that table has
// more than 16,384 entries, a launch between the two scans it once instead of every CTA for itself (200,000 ids of 50,000 in two passes
// and their rows' sums: 48.6 us, 59.1 each for itself; where the table has 4,160 entries the launch costs 0.7 us more than it saves).
// In both, a warp owns a run of consecutive items; a ballot for every bit of the digit gives a lane its rank among equal digits of its 32
// (match_any, which goes over the distinct digits one by one, takes longer where they are many), a counter per warp and digit what
// came before them in the run, a scan over the warps what came before the warp. The rank is by construction the order
// of the items, so the result is the same in every run. Bound by launches and the latency of a pass's steps, not by bytes:
// 8,192 items 6.8 us, 131,072 7.4, two million 27.
#pragma once
#include "common.cuh"
#include "row_io.cuh"

#include <algorithm>

namespace stable_sort {

constexpr int PER = 4;                           // items a lane
constexpr int SMALL = 1024 * PER, TILE = 512 * PER;
constexpr int64_t OWN_SCAN = 16384;              // entries of the table that every CTA may add up for itself
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

// Memory that the launches of a sort clear besides: `ctas` more CTAs in each of them, an equal share a launch.
struct Fill {
    float* p = nullptr;
    int64_t n = 0;
    int ctas = 0;
};

inline int64_t tiles(int64_t n) { return n <= SMALL ? 1 : ceil_div64(n, TILE); }   // CTAs of a launch
inline int launches(int64_t n, int passes) { return n <= SMALL ? 1 : 2 * passes; }
// the table, and the totals of scan_kernel
inline size_t scratch_bytes(int64_t n, int bins) { return n <= SMALL ? 0 : ((size_t)(tiles(n) + 1) * bins * 4 + 255) & ~(size_t)255; }

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
// Exclusive scan of each bin over the CTA's warps, in place, PARTS lanes a bin; the totals to tot.
template <int THREADS, int PARTS>
__device__ __forceinline__ void scan_warps(uint16_t* counts, int bins, int32_t* tot) {
    constexpr int Q = THREADS / 32 / PARTS;   // a lane's warps
    const int part = threadIdx.x % PARTS;
    for (int b0 = 0; b0 < bins; b0 += THREADS / PARTS) {
        const int b = b0 + threadIdx.x / PARTS;
        int c[Q], s = 0;
#pragma unroll
        for (int i = 0; i < Q; ++i) c[i] = b < bins ? counts[(part * Q + i) * bins + b] : 0;
#pragma unroll
        for (int i = 0; i < Q; ++i) s += c[i];
        int inc = s;
#pragma unroll
        for (int o = 1; o < PARTS; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, inc, o, PARTS);
            if (part >= o) inc += y;
        }
        int at = inc - s;
        if (b < bins) {
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                counts[(part * Q + i) * bins + b] = (uint16_t)at;
                at += c[i];
            }
            if (part == PARTS - 1) tot[b] = at;
        }
    }
}
template <int THREADS>
__device__ __forceinline__ void scan_warps(uint16_t* counts, int bins, int32_t* tot) {
    if (bins <= THREADS / 4) scan_warps<THREADS, 4>(counts, bins, tot);
    else scan_warps<THREADS, 1>(counts, bins, tot);
}
// In place: totals of the bins -> the first place of each. The caller's barrier is in front, one is behind.
template <int THREADS>
__device__ __forceinline__ void scan_bins(int32_t* v, int bins, int32_t* wsum) {
    for (int b0 = 0, carry = 0; b0 < bins; b0 += THREADS) {
        const int b = b0 + threadIdx.x, x = b < bins ? v[b] : 0;
        int total;
        const int at = carry + exclusive_scan<THREADS>(x, wsum, total);
        carry += total;
        if (b < bins) v[b] = at;
    }
    __syncthreads();
}
// Ranks the items of one CTA: `first` gets the first place of each bin, t.rank and the warps' counters the rest.
template <int THREADS>
__device__ __forceinline__ void rank_cta(int bins, int shift, uint32_t mask, uint16_t* counts, int32_t* first, int32_t* wsum, Items& t) {
    rank_items(bins, shift, mask, counts + (threadIdx.x >> 5) * bins, t);
    __syncthreads();
    scan_warps<THREADS>(counts, bins, first);
    __syncthreads();
    scan_bins<THREADS>(first, bins, wsum);
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

inline size_t smem_bytes(int threads, int bins) { return (size_t)bins * 8 + (size_t)threads / 32 * bins * 2; }

// n floats of zeros, by threads `me` of `step`.
__device__ __forceinline__ void clear_floats(float* p, int64_t n, int64_t me, int64_t step) {
    const int64_t head = min(n, (int64_t)(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / 4)), four = (n - head) / 4, rest = n - four * 4;
    for (int64_t i = me; i < four; i += step) st4(p + head + 4 * i, make_float4(0.0f, 0.0f, 0.0f, 0.0f));
    if (me < rest) p[me < head ? me : me + four * 4] = 0.0f;   // (at most six)
}

// f(std::integral_constant of 256, 512 or 1024): the threads that n items keep busy, four each
template <typename F>
inline void with_threads(int64_t n, F f) {
    if (n <= 256 * PER) f(std::integral_constant<int, 256>());
    else if (n <= 512 * PER) f(std::integral_constant<int, 512>());
    else f(std::integral_constant<int, 1024>());
}

// (nothing in front of it on the stream but this sort's own launches, which do not touch that memory: no wait for them)
__device__ __forceinline__ bool filled(const Fill& fill, int n_tiles) {
    if ((int)blockIdx.x < n_tiles) return false;
    pdl_launch_dependents();
    clear_floats(fill.p, fill.n, (int64_t)(blockIdx.x - n_tiles) * blockDim.x + threadIdx.x, (int64_t)fill.ctas * blockDim.x);
    return true;
}

template <int THREADS>
static __global__ void __launch_bounds__(THREADS) sort_small_kernel(const Job j, const Fill fill) {
    extern __shared__ __align__(16) int32_t sh[];   // a bin's first place; the warps' counters
    __shared__ int32_t wsum[32];
    if (filled(fill, 1)) return;
    pdl_launch_dependents();
    uint16_t *counts = reinterpret_cast<uint16_t*>(sh + j.bins), *run = counts + (threadIdx.x >> 5) * j.bins;
    const int n = (int)j.n, per = (n + THREADS - 1) / THREADS;
    for (int pass = 0; pass < j.passes; ++pass) {
        Items t;
        load_items(j, pass, (threadIdx.x >> 5) * per * 32, per, t);
        rank_cta<THREADS>(j.bins, pass * j.digit, mask_of(j), counts, sh, wsum, t);
        if (j.offsets)
            for (int b = threadIdx.x; b < j.bins; b += THREADS) j.offsets[b] = sh[b];
        put_items(j, pass, t, sh, run);
        __syncthreads();   // (what the next pass reads)
    }
}

// counts[tile][bin]
static __global__ void __launch_bounds__(512) count_kernel(const Job j, int pass, int32_t* __restrict__ counts, int n_tiles, const Fill fill) {
    extern __shared__ __align__(16) int32_t sh[];
    if (filled(fill, n_tiles)) return;
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

// counts[tile][bin] -> how many items of the bin the tiles in front have; totals[bin]. A CTA owns eight bins (a 32-byte sector of every
// tile's row), 128 lanes a bin, four tiles a lane in a round.
constexpr int SCAN_BINS = 8;
static __global__ void __launch_bounds__(1024) scan_kernel(const Job j, int32_t* __restrict__ counts, int n_tiles) {
    __shared__ int32_t sums[32][SCAN_BINS], all[SCAN_BINS];   // of a warp's tiles, then of the warps in front
    pdl_wait();
    pdl_launch_dependents();
    const int b = blockIdx.x * SCAN_BINS + threadIdx.x % SCAN_BINS, lane = threadIdx.x / SCAN_BINS, w = threadIdx.x >> 5, x = threadIdx.x & 31;
    int carry = 0;
    for (int t0 = 0; t0 < n_tiles; t0 += 512) {
        int c[4], s = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int t = t0 + lane * 4 + u;
            c[u] = t < n_tiles && b < j.bins ? counts[(int64_t)t * j.bins + b] : 0;
            s += c[u];
        }
        int inc = s;
#pragma unroll
        for (int o = SCAN_BINS; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, inc, o);
            if (x >= o) inc += y;
        }
        if (x >= 32 - SCAN_BINS) sums[w][x % SCAN_BINS] = inc;
        __syncthreads();
        if (w < SCAN_BINS) {   // a warp a bin
            const int v = sums[x][w];
            int y = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int z = __shfl_up_sync(0xffffffffu, y, o);
                if (x >= o) y += z;
            }
            sums[x][w] = y - v;
            if (x == 31) all[w] = y;
        }
        __syncthreads();
        int at = carry + sums[w][x % SCAN_BINS] + inc - s;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int t = t0 + lane * 4 + u;
            if (t < n_tiles && b < j.bins) counts[(int64_t)t * j.bins + b] = at;
            at += c[u];
        }
        carry += all[x % SCAN_BINS];
        __syncthreads();   // (written again)
    }
    if (lane == 0 && b < j.bins) counts[(int64_t)n_tiles * j.bins + b] = carry;
}

// SCANNED: the table holds what scan_kernel leaves; otherwise counts, which the CTA adds up: 512 / Q bins at a time, Q threads a bin.
// The items are put in order inside the tile first, so that what goes out together goes to neighbouring places.
template <bool SCANNED>
static __global__ void __launch_bounds__(512) place_kernel(const Job j, int pass, const int32_t* __restrict__ table, int n_tiles, int q_log, const Fill fill) {
    extern __shared__ __align__(16) int32_t sh[];   // first places [bin]; places inside the tile [bin]; the warps' counters
    __shared__ int32_t wsum[32];
    __shared__ uint32_t keys[TILE];
    __shared__ int32_t items[TILE];
    int32_t *first = sh, *inside = sh + j.bins;
    uint16_t *counts = reinterpret_cast<uint16_t*>(sh + 2 * j.bins), *run = counts + (threadIdx.x >> 5) * j.bins;
    if (filled(fill, n_tiles)) return;
    const int mine = blockIdx.x, shift = pass * j.digit;
    const uint32_t mask = mask_of(j);
    pdl_wait();
    pdl_launch_dependents();
    Items t;
    load_items(j, pass, (int64_t)mine * TILE + (threadIdx.x >> 5) * PER * 32, PER, t);
    if (SCANNED) {
        for (int b0 = 0, carry = 0; b0 < j.bins; b0 += 512) {
            const int b = b0 + threadIdx.x, all = b < j.bins ? table[(int64_t)n_tiles * j.bins + b] : 0;
            const int before = b < j.bins ? table[(int64_t)mine * j.bins + b] : 0;
            int total;
            const int at = carry + exclusive_scan<512>(all, wsum, total);
            carry += total;
            if (b >= j.bins) continue;
            first[b] = at + before;
            if (j.offsets && mine == 0) j.offsets[b] = at;
        }
    } else {
        const int q = 1 << q_log, lane = threadIdx.x & (q - 1);
        for (int b0 = 0, carry = 0; b0 < j.bins; b0 += 512 >> q_log) {
            const int b = b0 + (threadIdx.x >> q_log);
            int before = 0, all = 0;
            if (b < j.bins) {
                for (int i0 = lane; i0 < n_tiles; i0 += 16 << q_log) {
                    int c[16];
#pragma unroll
                    for (int u = 0; u < 16; ++u) c[u] = i0 + (u << q_log) < n_tiles ? table[(i0 + (u << q_log)) * j.bins + b] : 0;
#pragma unroll
                    for (int u = 0; u < 16; ++u) {
                        all += c[u];
                        if (i0 + (u << q_log) < mine) before += c[u];
                    }
                }
            }
            for (int o = 1; o < q; o <<= 1) {
                before += __shfl_xor_sync(0xffffffffu, before, o);
                all += __shfl_xor_sync(0xffffffffu, all, o);
            }
            int total;
            const int at = carry + exclusive_scan<512>(lane == 0 ? all : 0, wsum, total);
            carry += total;
            if (b < j.bins && lane == 0) {
                first[b] = at + before;
                if (j.offsets && mine == 0) j.offsets[b] = at;
            }
        }
    }
    rank_items(j.bins, shift, mask, run, t);
    __syncthreads();
    scan_warps<512>(counts, j.bins, inside);
    __syncthreads();
    scan_bins<512>(inside, j.bins, wsum);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (t.item[i] < 0) continue;
        const int b = (int)((t.key[i] >> shift) & mask), at = run[b] + t.rank[i];
        keys[inside[b] + at] = t.key[i];
        items[inside[b] + at] = t.item[i];
        if (j.place) j.place[t.item[i]] = t.key[i] == j.limit ? -1 : first[b] + at;
    }
    __syncthreads();
    uint32_t* to_keys = keys_to(j, pass);
    int32_t* to_items = items_to(j, pass);
    const int n = (int)min((int64_t)TILE, j.n - (int64_t)mine * TILE);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int p = i * 512 + threadIdx.x;
        if (p >= n) break;
        const uint32_t key = keys[p];
        const int b = (int)((key >> shift) & mask), at = first[b] + p - inside[b];
        if (to_keys) to_keys[at] = key;
        to_items[at] = items[p];
    }
}

// Leaves the result in keys / items [(passes - 1) & 1]; table: scratch_bytes(n, bins) of scratch. Every kernel lets the next one's
// launch begin early.
static inline int sort(asca_ctx* ctx, const Job& j, int32_t* table, const Fill& fill = Fill()) {
    if (j.n <= SMALL) {
        cudaError_t e = cudaSuccess;
        with_threads(j.n, [&](auto threads) {
            auto kern = sort_small_kernel<threads()>;
            const size_t smem = smem_bytes(threads(), j.bins);
            e = asca_allow_smem(kern, smem, smem_bytes(threads(), MAX_BINS));
            if (e == cudaSuccess) kern<<<(unsigned)(1 + fill.ctas), threads(), smem, ctx->stream>>>(j, fill);
        });
        ASCA_CUDA(ctx, e);
        ASCA_CHECK_LAUNCH(ctx);
        return ASCA_OK;
    }
    const size_t smem = smem_bytes(512, j.bins);
    const int n = (int)tiles(j.n);
    const bool scanned = (int64_t)n * j.bins > OWN_SCAN;
    int q_log = 0;   // threads a bin
    while (q_log < 5 && (j.bins << (q_log + 1)) <= 512) ++q_log;
    ASCA_CUDA(ctx, asca_allow_smem(scanned ? place_kernel<true> : place_kernel<false>, smem, smem_bytes(512, MAX_BINS)));
    auto share = [&](int launch) {
        const int64_t from = fill.n * launch / (2 * j.passes);
        return Fill{fill.p + from, fill.n * (launch + 1) / (2 * j.passes) - from, fill.ctas};
    };
    const dim3 grid((unsigned)(n + fill.ctas));
    for (int p = 0; p < j.passes; ++p) {
        if (p == 0) count_kernel<<<grid, 512, (size_t)j.bins * 4, ctx->stream>>>(j, p, table, n, share(0));
        else ASCA_CUDA(ctx, asca_launch_after(ctx, count_kernel, grid, dim3(512), (size_t)j.bins * 4, j, p, table, n, share(2 * p)));
        if (scanned) ASCA_CUDA(ctx, asca_launch_after(ctx, scan_kernel, dim3((unsigned)ceil_div64(j.bins, SCAN_BINS)), dim3(1024), 0, j, table, n));
        ASCA_CUDA(ctx, asca_launch_after(ctx, scanned ? place_kernel<true> : place_kernel<false>, grid, dim3(512), smem, j, p, (const int32_t*)table, n, q_log, share(2 * p + 1)));
        ctx->launches += scanned ? 3 : 2;
    }
    ASCA_CUDA(ctx, cudaGetLastError());
    return ASCA_OK;
}
#endif

}  // namespace stable_sort

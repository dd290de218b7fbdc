// Embedding rows with a scale for a vocabulary of any size, and the table's gradient by sorted tokens.
//
//   x[t] = scale * W[id_t]                      dW[v] (+)= scale * sum over t with id_t = v of dx[t]
//
// An id at or past the vocabulary (as unsigned: -1 is one) is padding: a row of zeros forward, no part of any sum backward.
//
// Backward. The tokens are sorted by id (stable_sort.cuh), so that the rows of one id lie in one run of the sorted order, in token
// order. The order is cut into pieces; a thread owns a few columns of a piece and walks down it with the running sum in registers,
// and a run that lies inside its piece goes straight into the table. A run over several pieces leaves one partial sum a piece (at
// most two of a piece belong to such runs: the one that comes in from the left and the one that goes on to the right), which a last
// launch adds. Where the table is overwritten, the SMs that the sort leaves idle clear its first rows, and blocks among the
// pieces' write the zeros of those behind that no token has. Nothing depends on the order in which blocks run. Bound by HBM
// where the table is large: dx is read once and the table written once (32,768 ids, 48,000 x 2048, bf16 dx: 527 MB in 110 us =
// 4.8 TB/s, of which the sort takes 17 us at little traffic); by the latency of six launches where it is not. A scan of all ids for
// every row of the table, as asca_embed_bwd does it, reads N * V ids.
#include "row_io.cuh"
#include "stable_sort.cuh"

namespace {

// Up to LANES lanes own TOKENS tokens, all of whose rows they have in flight (32,768 rows of 2048 bf16 from 48,000: 33.6 us with 32 lanes,
// 30.9 with 64, 32.7 with 256; of f32: 66, 63, 61); where that leaves SMs without work, blocks beside each other (blockIdx.y)
// share the columns.
constexpr int TOKENS = 4, LANES = 64;
template <int W, typename TT, typename TX>
__global__ void __launch_bounds__(256) embed_scaled_fwd_kernel(const TT* __restrict__ table, const uint32_t* __restrict__ ids, int64_t N, int d,
                                                               uint32_t vocab, float scale, TX* __restrict__ x) {
    using F = frag<W, TT>;
    const int lanes = blockDim.x;
    const int64_t r0 = ((int64_t)blockIdx.x * blockDim.y + threadIdx.y) * TOKENS;
    uint32_t id[TOKENS];
#pragma unroll
    for (int i = 0; i < TOKENS; ++i) id[i] = r0 + i < N ? ids[r0 + i] : 0xffffffffu;
    for (int c = blockIdx.y * lanes * F::E + frag_first<W>(threadIdx.x); c < d; c += gridDim.y * lanes * F::E) {
        F r[TOKENS];
#pragma unroll
        for (int i = 0; i < TOKENS; ++i)
            if (id[i] < vocab) r[i].load(table + (int64_t)id[i] * d, c, lanes, d);
#pragma unroll
        for (int i = 0; i < TOKENS; ++i) {
            if (r0 + i >= N) break;
            float v[F::E] = {};
            if (id[i] < vocab) {
                r[i].get(v);
#pragma unroll
                for (int j = 0; j < F::E; ++j) v[j] *= scale;
            }
            frag<W, TX>::put(x + (r0 + i) * d, c, lanes, d, v);
        }
    }
}

// p[columns] = scale * v, or += with accumulate
template <int W>
__device__ __forceinline__ void add_row(float* row, int c, int lanes, int d, const float (&v)[frag<W, float>::E], float scale, int accumulate) {
    constexpr int E = frag<W, float>::E;
    float o[E], t[E];
    if (accumulate) {
        frag<W, float> r;
        r.load(row, c, lanes, d);
        r.get(t);
    }
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = accumulate ? t[i] + scale * v[i] : scale * v[i];
    frag<W, float>::put(row, c, lanes, d, o);
}

constexpr int MOST_PIECE = 64, AHEAD = 8, ZERO_ROWS = 32;
// Bytes of the table that a CTA beside a sort's tiles clears in each of its launches: about what it has time for. 32,768 ids, 48,000 x
// 2048: 116 us with none, 112 with 128 KiB, 110 with 256, 114 with 512; 6728 ids, 52,608 x 319: 41, 31, 31, 31.
constexpr int64_t FILL_SHARE = 256 << 10;

struct Sum {
    const void* dx;
    const uint32_t* keys;   // sorted
    const int32_t* items;
    int64_t N;
    int d, piece, accumulate;
    uint32_t vocab;
    float scale;
    float *d_table, *part;
    int64_t sums, zeros;    // blocks of the two kinds; they take turns in the grid
    int64_t cleared;        // rows of the table, from the first on, that the sort's launches clear
    bool narrow;            // rows of the table: a warp clears some of its own, or the block some together
};

// The first place in the sorted keys that is not below v.
__device__ __forceinline__ int64_t lower_bound(const uint32_t* keys, int64_t n, uint32_t v) {
    int64_t lo = 0;
    while (n > 0) {
        const int64_t half = n >> 1;
        if (keys[lo + half] < v) {
            lo += half + 1;
            n -= half + 1;
        } else n = half;
    }
    return lo;
}

// The same from `at` on, by a warp: every round looks at 32 places.
__device__ __forceinline__ int64_t warp_lower_bound(const uint32_t* keys, int64_t at, int64_t N, uint32_t v, int lane) {
    int64_t n = N - at;   // the answer is in [at, at + n]
    while (n > 0) {
        const int64_t step = (n + 31) / 32, mine = lane * step;
        const int below = __popc(__ballot_sync(0xffffffffu, mine < n && keys[at + mine] < v));
        if (below == 0) return at;
        const int64_t from = (below - 1) * step + 1;
        n = min(step - 1, n - from);
        at += from;
    }
    return at;
}

// ZERO_ROWS rows of the table: those without a token are cleared. Narrow rows: every warp of the block has rows of its own.
template <int W>
__device__ __forceinline__ void zero_rows(const Sum& a, int64_t block) {
    const int me = threadIdx.x + threadIdx.y * blockDim.x, threads = blockDim.x * blockDim.y, lane = me & 31;
    const int64_t v0 = a.cleared + (a.narrow ? block * (threads >> 5) + (me >> 5) : block) * ZERO_ROWS;
    if (v0 >= a.vocab) return;
    const uint32_t rows = (uint32_t)min((int64_t)ZERO_ROWS, a.vocab - v0);
    // the rows' tokens lie in [lo, hi) of the sorted order: few are looked at one by one, many are looked for row by row
    const int64_t lo = warp_lower_bound(a.keys, 0, a.N, (uint32_t)v0, lane), hi = warp_lower_bound(a.keys, lo, a.N, (uint32_t)v0 + rows, lane);
    unsigned met = 0;
    if (hi - lo <= 128) {
        for (int64_t at = lo + lane; at < hi; at += 32) met |= 1u << (a.keys[at] - (uint32_t)v0);
        met = __reduce_or_sync(0xffffffffu, met);
    } else {
        const uint32_t v = (uint32_t)v0 + lane;
        const int64_t at = lo + lower_bound(a.keys + lo, hi - lo, v);
        met = __ballot_sync(0xffffffffu, at < hi && a.keys[at] == v);
    }
    using F = frag<W, float>;
    const float zero[F::E] = {};
    const int x = a.narrow ? lane : me, lanes = a.narrow ? 32 : threads;
    for (unsigned left = ~met & (rows < 32 ? (1u << rows) - 1 : 0xffffffffu); left; left &= left - 1) {
        float* p = a.d_table + (v0 + __ffs(left) - 1) * a.d;
        for (int c = frag_first<W>(x); c < a.d; c += lanes * F::E) F::put(p, c, lanes, a.d, zero);
    }
}

// part[piece][0]: the sum of a run that came in from the left; part[piece][1]: of a run that begins here and goes on to the right.
// A thread owns some columns of a piece; AHEAD rows are asked for before the first of them is added.
template <int W, typename T>
__global__ void __launch_bounds__(128) embed_pieces_kernel(const Sum a) {
    extern __shared__ uint32_t sh[];   // [block's pieces][key before, keys of the piece, key behind; items]
    pdl_wait();
    pdl_launch_dependents();
    const int64_t all = a.sums + a.zeros, before = (int64_t)blockIdx.x * a.zeros / all;   // zeroing blocks in front of this one
    if ((int64_t)(blockIdx.x + 1) * a.zeros / all > before) {
        zero_rows<W>(a, before);
        return;
    }
    using F = frag<W, T>;
    constexpr int E = F::E;
    const int d = a.d, piece = a.piece, lanes = blockDim.x, wide = lanes * E, groups = (d + wide - 1) / wide;
    const int64_t at0 = blockIdx.x - before, p = at0 / groups * blockDim.y + threadIdx.y, lo = p * piece;
    const int n = lo < a.N ? (int)min((int64_t)piece, a.N - lo) : 0;
    uint32_t* key = sh + threadIdx.y * (2 * piece + 2) + 1;
    int32_t* item = reinterpret_cast<int32_t*>(key + piece + 1);
    for (int i = threadIdx.x; i < n + 2 && n > 0; i += blockDim.x) {
        const int64_t at = lo + i - 1;
        key[i - 1] = at >= 0 && at < a.N ? a.keys[at] : 0xffffffffu;   // (no key of a token)
        if (i > 0 && i <= n) item[i - 1] = a.items[at];
    }
    __syncthreads();
    const int c = (int)(at0 % groups) * wide + frag_first<W>(threadIdx.x);
    if (c >= d) return;
    const T* dx = static_cast<const T*>(a.dx);
    float acc[E] = {};
    bool from_left = n > 0 && key[-1] == key[0];
    for (int i0 = 0; i0 < n; i0 += AHEAD) {
        F r[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            r[u].load(dx + (int64_t)item[min(i0 + u, n - 1)] * d, c, lanes, d);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int i = i0 + u;
            if (i >= n || key[i] >= a.vocab) return;   // the end of the piece, or padding from here on
            float v[E];
            r[u].get(v);
#pragma unroll
            for (int j = 0; j < E; ++j) acc[j] += v[j];
            const bool goes_on = key[i + 1] == key[i];
            if (goes_on && i + 1 < n) continue;
            if (from_left || goes_on) frag<W, float>::put(a.part + (2 * p + (from_left ? 0 : 1)) * d, c, lanes, d, acc);
            else add_row<W>(a.d_table + (int64_t)key[i] * d, c, lanes, d, acc, a.scale, a.accumulate);
#pragma unroll
            for (int j = 0; j < E; ++j) acc[j] = 0.0f;
            from_left = false;
        }
    }
}

// A block owns `pieces` pieces; it has work where a run begins in one of them and goes on past it. A run that comes into up to AHEAD
// further pieces is added up by one thread a column (a block has blockDim.y of them beside each other, each at its own run); for a
// longer one those beside each other take its pieces in turn, eight of them in flight.
constexpr int MOST_JOINED = 32;
template <int W>
__global__ void __launch_bounds__(256) embed_join_kernel(const Sum a, int pieces) {
    using F = frag<W, float>;
    constexpr int E = F::E;
    extern __shared__ uint32_t sh_raw[];
    float(*sh)[E] = reinterpret_cast<float(*)[E]>(sh_raw);   // [lane beside][column lane]
    __shared__ int comes_into[MOST_JOINED];   // further pieces of the run that begins in a piece; AHEAD + 1: more than AHEAD
    __shared__ uint32_t keys[MOST_JOINED];
    const int piece = a.piece, d = a.d, lanes = blockDim.x, beside = blockDim.y, threads = lanes * beside, me = threadIdx.y * lanes + threadIdx.x;
    pdl_wait();
    const int64_t p0 = (int64_t)blockIdx.x * pieces;
    for (int i = me; i < pieces; i += threads) {
        const int64_t p = p0 + i, end = (p + 1) * piece;
        int more = 0;
        if (end < a.N) {
            const uint32_t key = a.keys[end - 1], left = p > 0 ? a.keys[p * piece - 1] : 0xffffffffu;   // (left the same: it began there)
            uint32_t at[AHEAD + 1];
#pragma unroll
            for (int u = 0; u <= AHEAD; ++u) at[u] = end + (int64_t)u * piece < a.N ? a.keys[end + (int64_t)u * piece] : 0xffffffffu;
            if (key < a.vocab && left != key) {
#pragma unroll
                for (int u = 0; u <= AHEAD; ++u) more += at[u] == key;   // (sorted: they are the first ones)
            }
            keys[i] = key;
        }
        comes_into[i] = more;
    }
    __syncthreads();
    const auto add = [](const F& r, float (&acc)[E]) {
        float v[E];
        r.get(v);
#pragma unroll
        for (int j = 0; j < E; ++j) acc[j] += v[j];
    };
    for (int i = threadIdx.y; i < pieces; i += beside) {
        const int more = comes_into[i];
        if (more == 0 || more > AHEAD) continue;
        const int64_t p = p0 + i;
        for (int c = frag_first<W>(threadIdx.x); c < d; c += lanes * E) {
            F first, r[AHEAD];
            float acc[E] = {};
            first.load(a.part + (2 * p + 1) * d, c, lanes, d);
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
                if (u < more) r[u].load(a.part + 2 * (p + 1 + u) * d, c, lanes, d);
            add(first, acc);
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
                if (u < more) add(r[u], acc);
            add_row<W>(a.d_table + (int64_t)keys[i] * d, c, lanes, d, acc, a.scale, a.accumulate);
        }
    }
    for (int i = 0; i < pieces; ++i) {
        if (comes_into[i] <= AHEAD) continue;
        const int64_t p = p0 + i;
        const uint32_t key = keys[i];
        int64_t more = 0;   // pieces that the run comes into from the left
        for (;; more += threads) {
            const int64_t q = p + 1 + more + me;
            const int in = __syncthreads_count(q * piece < a.N && a.keys[q * piece] == key);
            if (in < threads) {
                more += in;
                break;
            }
        }
        for (int c = frag_first<W>(threadIdx.x); c - frag_first<W>(threadIdx.x) < d; c += lanes * E) {   // (the same turns for all)
            float acc[E] = {};
            if (c < d) {
                F r[AHEAD];
                if (threadIdx.y == 0) {
                    r[0].load(a.part + (2 * p + 1) * d, c, lanes, d);
                    add(r[0], acc);
                }
                for (int64_t q0 = threadIdx.y; q0 < more; q0 += (int64_t)AHEAD * beside) {
#pragma unroll
                    for (int u = 0; u < AHEAD; ++u)
                        if (q0 + u * beside < more) r[u].load(a.part + 2 * (p + 1 + q0 + u * beside) * d, c, lanes, d);
#pragma unroll
                    for (int u = 0; u < AHEAD; ++u)
                        if (q0 + u * beside < more) add(r[u], acc);
                }
            }
            if (beside > 1) {
#pragma unroll
                for (int j = 0; j < E; ++j) sh[me][j] = acc[j];
                __syncthreads();
                if (threadIdx.y == 0) {
#pragma unroll 8
                    for (int y = 1; y < beside; ++y) {
#pragma unroll
                        for (int j = 0; j < E; ++j) acc[j] += sh[y * lanes + threadIdx.x][j];
                    }
                }
                __syncthreads();
            }
            if (threadIdx.y == 0 && c < d) add_row<W>(a.d_table + (int64_t)key * d, c, lanes, d, acc, a.scale, a.accumulate);
        }
    }
}

// Few tokens: everything in one launch. A CTA owns some rows of the table and some columns, which it clears first where the table is
// overwritten; it picks the tokens of its rows from all of them, in their order, and sorts those (2048 x 64: 5.7 us; 9.5 where every
// CTA sorted all tokens). A row of up to SHORT tokens is summed by the lanes that share a row, others of the CTA doing other rows
// meanwhile; a longer one by the whole CTA, each of the lanes beside each other taking tokens in turn. Bound by its launch and the
// latency of these steps. SHORT = 8, 16, 32 with a cold cache: 2048 x 64 of 256 6.1 us, 7.0, 7.2; 300 x 800 of 90 6.6, 7.2, 7.8; 4096 x 64
// of 48,000 21.3, 21.5, 21.1.
constexpr int SHORT = 16;
template <int W, int THREADS, typename T>
__global__ void __launch_bounds__(THREADS) embed_small_kernel(const Sum a, const stable_sort::Job j, int lanes, int rows) {
    using F = frag<W, T>;
    constexpr int E = F::E;
    extern __shared__ uint32_t sh[];   // keys and tokens, twice; places; counters. Behind the sort: the sums of the lanes beside each other
    __shared__ int32_t wsum[32];
    __shared__ int32_t long_runs[stable_sort::SMALL / SHORT], n_long;   // where they begin in the sorted order
    const int n = (int)j.n, per = (n + THREADS - 1) / THREADS, room = (n + 7) & ~7;
    uint32_t* keys[2] = {sh, sh + room};
    int32_t* items[2] = {reinterpret_cast<int32_t*>(sh) + 2 * room, reinterpret_cast<int32_t*>(sh) + 3 * room};
    int32_t* first = reinterpret_cast<int32_t*>(sh) + 4 * room;
    uint16_t *counts = reinterpret_cast<uint16_t*>(first + j.bins), *run = counts + (threadIdx.x >> 5) * j.bins;
    const uint32_t mask = stable_sort::mask_of(j);
    const int d = a.d, beside = THREADS / lanes, x = threadIdx.x % lanes, y = threadIdx.x / lanes;
    const int wide = lanes * E, c = blockIdx.y * wide + frag_first<W>(x);
    const bool in = c < d;
    const int64_t v0 = (int64_t)blockIdx.x * rows, v1 = min(v0 + rows, (int64_t)a.vocab);
    if (!a.accumulate) {
        const float zero[E] = {};
        if (gridDim.y == 1) stable_sort::clear_floats(a.d_table + v0 * d, (v1 - v0) * d, threadIdx.x, THREADS);
        else if (in)
            for (int64_t v = v0 + y; v < v1; v += beside) frag<W, float>::put(a.d_table + v * d, c, lanes, d, zero);
    }
    if (threadIdx.x == 0) n_long = 0;
    int m;   // tokens of the CTA's rows
    {
        uint32_t k[stable_sort::PER];
        unsigned mine[stable_sort::PER];
        const int lo = (threadIdx.x >> 5) * per * 32 + (threadIdx.x & 31);
        int of_warp = 0;
#pragma unroll
        for (int i = 0; i < stable_sort::PER; ++i) k[i] = i < per && lo + i * 32 < n ? j.ids[lo + i * 32] : 0xffffffffu;
#pragma unroll
        for (int i = 0; i < stable_sort::PER; ++i) {
            mine[i] = __ballot_sync(0xffffffffu, k[i] < a.vocab && k[i] - (uint32_t)v0 < (uint32_t)(v1 - v0));
            of_warp += __popc(mine[i]);
        }
        const bool first_lane = (threadIdx.x & 31) == 0;
        int at = __shfl_sync(0xffffffffu, stable_sort::exclusive_scan<THREADS>(first_lane ? of_warp : 0, wsum, m), 0);
#pragma unroll
        for (int i = 0; i < stable_sort::PER; ++i) {
            const unsigned below = (1u << (threadIdx.x & 31)) - 1u;
            if (mine[i] >> (threadIdx.x & 31) & 1) {
                const int p = at + __popc(mine[i] & below);
                keys[0][p] = k[i] - (uint32_t)v0;
                items[0][p] = lo + i * 32;
            }
            at += __popc(mine[i]);
        }
        __syncthreads();
    }
    int now = 0;
    const int per_m = (m + THREADS - 1) / THREADS;
    for (int pass = 0; pass < j.passes; ++pass) {
        stable_sort::Items t;
        const int lo = (threadIdx.x >> 5) * per_m * 32 + (threadIdx.x & 31);
#pragma unroll
        for (int i = 0; i < stable_sort::PER; ++i) {
            const int at = lo + i * 32;
            t.item[i] = -1;
            t.key[i] = 0;
            if (i < per_m && at < m) {
                t.key[i] = keys[now][at];
                t.item[i] = items[now][at];
            }
        }
        const int shift = pass * j.digit;
        stable_sort::rank_cta<THREADS>(j.bins, shift, mask, counts, first, wsum, t);
        now ^= 1;
#pragma unroll
        for (int i = 0; i < stable_sort::PER; ++i) {
            if (t.item[i] < 0) continue;
            const int b = (int)((t.key[i] >> shift) & mask), at = first[b] + run[b] + t.rank[i];
            keys[now][at] = t.key[i];
            items[now][at] = t.item[i];
        }
        __syncthreads();
    }
    const uint32_t* key = keys[now];
    const int32_t* item = items[now];
    const T* dx = static_cast<const T*>(a.dx);
    auto sum = [&](int lo, int step, int end, float (&acc)[E]) {
        for (int i0 = lo; i0 < end; i0 += AHEAD * step) {
            F r[AHEAD];
#pragma unroll
            for (int u = 0; u < AHEAD; ++u)
                if (i0 + u * step < end) r[u].load(dx + (int64_t)item[i0 + u * step] * d, c, lanes, d);
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                if (i0 + u * step >= end) break;
                float v[E];
                r[u].get(v);
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] += v[e];
            }
        }
    };
    for (int p = y; p < m; p += beside) {   // (behind barriers: the zeros are in place)
        if (p > 0 && key[p] == key[p - 1]) continue;   // (not where a row's run begins)
        int end = p + 1;
        while (end < m && key[end] == key[p] && end - p <= SHORT) ++end;
        if (end - p > SHORT) {
            if (x == 0) long_runs[atomicAdd(&n_long, 1)] = p;   // (rows are summed one by one: their order does not matter)
            continue;
        }
        if (!in) continue;
        float acc[E] = {};
        sum(p, 1, end, acc);
        add_row<W>(a.d_table + (v0 + key[p]) * d, c, lanes, d, acc, a.scale, a.accumulate);
    }
    __syncthreads();
    float* part = reinterpret_cast<float*>(first);   // [E][thread]: the places and counters are no longer needed
    for (int l = 0; l < n_long; ++l) {
        const int lo = long_runs[l], end = (int)lower_bound(key, m, key[lo] + 1);
        const int64_t v = v0 + key[lo];
        float acc[E] = {};
        if (in) sum(lo + y, beside, end, acc);
#pragma unroll
        for (int e = 0; e < E; ++e) part[e * THREADS + threadIdx.x] = acc[e];
        __syncthreads();
        for (int s = beside / 2; s > 0; s /= 2) {
            if (y < s) {
#pragma unroll
                for (int e = 0; e < E; ++e) part[e * THREADS + threadIdx.x] += part[e * THREADS + threadIdx.x + s * lanes];
            }
            __syncthreads();
        }
        if (y == 0 && in) {
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = part[e * THREADS + x];
            add_row<W>(a.d_table + v * d, c, lanes, d, acc, a.scale, a.accumulate);
        }
        __syncthreads();
    }
}

// Scratch: sorted keys and items, the pass before's where there are two, the counts, and the partial sums.
struct Plan {
    int passes, digit, bins, piece;
    bool small;   // everything in one launch
    size_t list, counts, part;
    Plan(int64_t N, int64_t d, int64_t vocab) {
        int bits = 1;
        while (((int64_t)1 << bits) <= vocab) ++bits;   // keys 0 .. vocab
        passes = (int)ceil_div64(bits, 11);
        digit = (int)ceil_div64(bits, passes);
        bins = passes == 1 ? (int)vocab + 1 : 1 << digit;
        // Short pieces where the tokens are few: 256 threads on each of the B200's 148 SMs walk down pieces at once, or the walk is what the
        // call waits for (a fixed number, so that the size of the scratch does not depend on a context). With 128, 256, 512 threads:
        // 12,000 x 768 of 256 21.1 us, 19.3, 22.1; 8192 x 512 of 1000 19.5, 20.1, 21.9; 6000 x 64 of 256 15.4, 16.0, 15.4.
        piece = MOST_PIECE;
        while (piece > AHEAD && ceil_div64(N, piece) * std::max<int64_t>(8, ceil_div64(d, 4)) < 148 * 256) piece /= 2;
        // One launch or three (sort, pieces, join): every CTA of the one looks at all tokens and may have to add its columns of all of dx's
        // rows by itself. In one launch and in three, N x d: 12 x 768 4.3 us, 6.6; 100 x 2048 of 48,000 71, 80; 2048 x 64 5.7, 10.8; 4096 x 64
        // 10.3, 15.6; 1000 x 768 8.8, 9.0; 500 x 777 of 30,000 28.3, 25.4; 2048 x 768 bf16 12.6, 11.4; 4096 x 512 of 48,000 45, 34.
        small = N <= stable_sort::SMALL && N * d <= (1 << 18);
        if (small) {
            list = counts = part = 0;
            return;
        }
        list = ((size_t)N * 4 + 255) & ~(size_t)255;
        counts = stable_sort::scratch_bytes(N, bins);
        part = (size_t)ceil_div64(N, piece) * 2 * d * 4;
    }
    size_t bytes() const { return 4 * list + counts + part; }
};

}  // namespace

extern "C" {

int asca_embed_scaled_fwd(asca_ctx* ctx, const void* table, const uint32_t* ids, int64_t N, int64_t d, int64_t vocab, float scale, int table_dtype,
                          int out_dtype, void* x) {
    if (!ctx) return ASCA_ERR_ARG;
    ASCA_REQUIRE(ctx, N >= 0 && d > 0 && d < (1 << 30) && vocab > 0 && vocab < ((int64_t)1 << 31), "embed_scaled_fwd: bad shape");
    ASCA_REQUIRE(ctx, asca_known_dtype(table_dtype) && asca_known_dtype(out_dtype), "embed_scaled_fwd: unknown dtype");
    if (N == 0) return ASCA_OK;
    ASCA_REQUIRE(ctx, table && ids && x, "embed_scaled_fwd: null pointer");
    ASCA_REQUIRE(ctx, N < ((int64_t)1 << 31), "embed_scaled_fwd: at most 2^31 - 1 tokens");
    const asca_span_of out(x, N * d, asca_dtype_size(out_dtype));
    ASCA_REQUIRE(ctx, asca_apart(out, {table, vocab * d, asca_dtype_size(table_dtype)}) && asca_apart(out, {ids, N, 4}), "embed_scaled_fwd: x lies over an input");
    asca_device_scope on(ctx);
    const int v = asca_row_width(d, table, table_dtype, x, out_dtype);
    const int64_t frags = asca_row_frags(d, v);
    asca_with_dtype(table, table_dtype, [&](auto tab) {
        asca_with_dtype(x, out_dtype, [&](auto out) {
            using TT = std::remove_const_t<std::remove_pointer_t<decltype(tab)>>;
            using TX = std::remove_pointer_t<decltype(out)>;
            asca_with_width<TT, TX>(v, [&](auto w) {
                const dim3 block = asca_row_block(std::min<int64_t>(frags, LANES), 256);
                const int64_t blocks = ceil_div64(N, (int64_t)block.y * TOKENS);
                const dim3 grid((unsigned)blocks, asca_column_blocks(ctx, blocks, frags, block.x));
                embed_scaled_fwd_kernel<w(), TT, TX><<<grid, block, 0, ctx->stream>>>(tab, ids, N, (int)d, (uint32_t)vocab, scale, out);
            });
        });
    });
    ASCA_CHECK_LAUNCH(ctx);
    return ASCA_OK;
}

int64_t asca_embed_scaled_bwd_ws(int64_t N, int64_t d, int64_t vocab) {
    if (N < 0 || N >= ((int64_t)1 << 31) || d <= 0 || d >= (1 << 30) || vocab <= 0 || vocab >= ((int64_t)1 << 31)) return ASCA_ERR_ARG;   // (as the call)
    return (int64_t)Plan(N, d, vocab).bytes();
}

int asca_embed_scaled_bwd(asca_ctx* ctx, const void* dx, const uint32_t* ids, int64_t N, int64_t d, int64_t vocab, float scale, int dtype, int accumulate,
                          float* d_table, void* ws, size_t ws_bytes) {
    if (!ctx) return ASCA_ERR_ARG;
    ASCA_REQUIRE(ctx, N >= 0 && d > 0 && d < (1 << 30) && vocab > 0 && vocab < ((int64_t)1 << 31), "embed_scaled_bwd: bad shape");
    ASCA_REQUIRE(ctx, asca_known_dtype(dtype), "embed_scaled_bwd: unknown dtype");
    ASCA_REQUIRE(ctx, N < ((int64_t)1 << 31), "embed_scaled_bwd: at most 2^31 - 1 tokens");
    ASCA_REQUIRE(ctx, d_table, "embed_scaled_bwd: null pointer");
    asca_device_scope on(ctx);
    if (N == 0) {
        if (!accumulate) ASCA_CUDA(ctx, cudaMemsetAsync(d_table, 0, (size_t)vocab * d * 4, ctx->stream));
        return ASCA_OK;
    }
    ASCA_REQUIRE(ctx, dx && ids, "embed_scaled_bwd: null pointer");
    const asca_span_of out(d_table, vocab * d, 4);
    ASCA_REQUIRE(ctx, asca_apart(out, {dx, N * d, asca_dtype_size(dtype)}) && asca_apart(out, {ids, N, 4}), "embed_scaled_bwd: d_table lies over an input");
    const Plan plan(N, d, vocab);
    ASCA_REQUIRE(ctx, asca_aligned(ws, 256) && ws_bytes >= plan.bytes() && (ws || ws_bytes == 0), "embed_scaled_bwd: the workspace has to have asca_embed_scaled_bwd_ws bytes, 256-byte aligned");
    const int v = asca_row_width(d, dx, dtype, d_table, ASCA_F32);
    const int64_t frags = asca_row_frags(d, v);
    dim3 block = asca_row_block(frags, 128);
    const unsigned place = (2 * plan.piece + 2) * 4;   // a piece's keys and items in shared memory
    block.y = std::min(block.y, 4096u / plan.piece);   // 36 KiB at most
    const int64_t pieces = ceil_div64(N, plan.piece), groups = ceil_div64(frags, block.x);
    char* w = (char*)ws;
    stable_sort::Job j{};
    j.ids = ids;
    j.limit = (uint32_t)vocab;
    j.n = N;
    j.passes = plan.passes;
    j.digit = plan.digit;
    j.bins = plan.bins;
    for (int i = 0; i < 2; ++i) j.keys[i] = (uint32_t*)(w + i * plan.list), j.items[i] = (int32_t*)(w + (2 + i) * plan.list);
    Sum a{};
    a.dx = dx; a.N = N; a.d = (int)d; a.piece = plan.piece; a.accumulate = accumulate; a.vocab = (uint32_t)vocab; a.scale = scale; a.d_table = d_table;
    a.keys = j.keys[(plan.passes - 1) & 1];
    a.items = j.items[(plan.passes - 1) & 1];
    a.part = (float*)(w + 4 * plan.list + plan.counts);
    a.sums = ceil_div64(pieces, block.y) * groups;
    // (5000 ids, what the sort does not clear, a warp's own rows and a block's: 3 M x 64 171 us, 381; 1.5 M x 128 145, 212; 700,000 x 256
    // 126, 127; 500,000 x 320 120, 116; 150,000 x 1024 131, 120)
    a.narrow = d <= 256;
    // What SMs the sort leaves idle clear a part of the table meanwhile, rows that have tokens among them (written over afterwards).
    stable_sort::Fill fill;
    if (!accumulate && !plan.small && stable_sort::tiles(N) < ctx->sm_count) {
        fill.ctas = (int)(ctx->sm_count - stable_sort::tiles(N));
        a.cleared = std::min<int64_t>(vocab, fill.ctas * (FILL_SHARE / 4) * stable_sort::launches(N, plan.passes) / d);
        fill.p = d_table;
        fill.n = a.cleared * d;
    }
    a.zeros = accumulate ? 0 : ceil_div64(vocab - a.cleared, a.narrow ? ZERO_ROWS * (int64_t)(block.x * block.y / 32) : ZERO_ROWS);
    if (plan.small) {
        int lanes = 1;
        while (lanes < frags && lanes < 64) lanes *= 2;
        const int64_t across = ceil_div64(frags, lanes), rows = ceil_div64(vocab, std::max<int64_t>(1, 2 * ctx->sm_count / across));   // two CTAs an SM
        const dim3 grid((unsigned)ceil_div64(vocab, rows), (unsigned)across);
        int bits = 0;   // keys 0 .. rows - 1 of a CTA
        while (((int64_t)1 << bits) < rows) ++bits;
        j.passes = (int)ceil_div64(bits, 11);
        j.digit = j.passes > 0 ? (int)ceil_div64(bits, j.passes) : 0;
        j.bins = j.passes == 1 ? (int)rows : 1 << j.digit;
        cudaError_t e = cudaSuccess;
        asca_with_dtype(dx, dtype, [&](auto src) {
            using T = std::remove_const_t<std::remove_pointer_t<decltype(src)>>;
            asca_with_width<T, T>(v, [&](auto wd) {
                stable_sort::with_threads(N, [&](auto threads) {
                    auto kern = embed_small_kernel<wd(), threads(), T>;
                    auto size = [&](size_t n, int bins) {
                        return 16 * ((n + 7) & ~(size_t)7) + std::max((size_t)threads() * 4 * frag<wd(), T>::E, stable_sort::smem_bytes(threads(), bins));
                    };
                    const size_t smem = size((size_t)N, j.bins);
                    e = asca_allow_smem(kern, smem, size(threads() * stable_sort::PER, stable_sort::MAX_BINS));
                    if (e == cudaSuccess) kern<<<grid, threads(), smem, ctx->stream>>>(a, j, lanes, (int)rows);
                });
            });
        });
        ASCA_CUDA(ctx, e);
        ASCA_CHECK_LAUNCH(ctx);
        return ASCA_OK;
    }
    ASCA_REQUIRE(ctx, a.sums + a.zeros < ((int64_t)1 << 31) && ceil_div64(frags, 32) <= 65535, "embed_scaled_bwd: too large");
    ASCA_TRY(stable_sort::sort(ctx, j, (int32_t*)(w + 4 * plan.list), fill));
    cudaError_t e = cudaSuccess;
    asca_with_dtype(dx, dtype, [&](auto src) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(src)>>;
        asca_with_width<T, T>(v, [&](auto wd) {
            // (whole warps: a zeroing block votes)
            e = asca_launch_after(ctx, embed_pieces_kernel<wd(), T>, dim3((unsigned)(a.sums + a.zeros)), block, (size_t)block.y * place, a);
            const dim3 wide = asca_row_block(frags, 256);
            const int64_t each = std::min<int64_t>(MOST_JOINED, ceil_div64(pieces, ctx->sm_count * 8));   // (most pieces have no work)
            if (e == cudaSuccess && pieces > 1)
                e = asca_launch_after(ctx, embed_join_kernel<wd()>, dim3((unsigned)ceil_div64(pieces, each)), wide,
                                      wide.y > 1 ? (size_t)wide.x * wide.y * 4 * frag<wd(), float>::E : 0, a, (int)each);
        });
    });
    ASCA_CUDA(ctx, e);
    ctx->launches += pieces > 1 ? 2 : 1;
    return ASCA_OK;
}

}  // extern "C"

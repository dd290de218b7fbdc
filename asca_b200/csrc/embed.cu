// Embedding rows with a scale for a vocabulary of any size, and the table's gradient by sorted tokens.
//
//   x[t] = scale * W[id_t]                      dW[v] (+)= scale * sum over t with id_t = v of dx[t]
//
// An id at or past the vocabulary (as unsigned: -1 is one) is padding: a row of zeros forward, no part of any sum backward.
//
// Backward. The tokens are sorted by id (stable_sort.cuh), so that the rows of one id lie in one run of the sorted order, in token
// order. The order is cut into pieces of `piece` rows; a thread owns four columns of a piece and walks down it with the running sum
// in registers, and a run that lies inside its piece goes straight into the table. A run over several pieces leaves one partial sum
// a piece (at most two of a piece belong to such runs: the one that comes in from the left and the one that goes on to the right),
// which a second launch adds in order. Nothing depends on the order in which blocks run. Bound by HBM: dx is read once, the table
// written once; a scan of all ids for every row of the table, as asca_embed_bwd does it, reads N * V ids.
#include "row_io.cuh"
#include "stable_sort.cuh"

namespace {

template <int V, typename TT, typename TX>
__global__ void __launch_bounds__(256) embed_scaled_fwd_kernel(const TT* __restrict__ table, const uint32_t* __restrict__ ids, int64_t N, int d,
                                                               uint32_t vocab, float scale, TX* __restrict__ x) {
    const int64_t r = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (r >= N) return;
    const uint32_t id = ids[r];
    const bool live = id < vocab;
    const TT* src = table + (int64_t)(live ? id : 0) * d;
    TX* dst = x + r * (int64_t)d;
    for (int c = threadIdx.x * V; c < d; c += blockDim.x * V) {
        float v[V];
        if (live) ld_row<V>(src + c, v);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = live ? scale * v[i] : 0.0f;
        st_row<V>(dst + c, v);
    }
}

template <int V>
__device__ __forceinline__ void add_row(float* p, const float (&v)[V], float scale, int accumulate) {
    float o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = scale * v[i];
    if (accumulate) {
        float t[V];
        ld_row<V>(p, t);
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] += t[i];
    }
    st_row<V>(p, o);
}

// part[piece][0]: the sum of a run that came in from the left; part[piece][1]: of a run that begins here and goes on to the right
template <int V, typename T>
__global__ void __launch_bounds__(128) embed_pieces_kernel(const T* __restrict__ dx, const uint32_t* __restrict__ keys, const int32_t* __restrict__ items,
                                                           int64_t N, int d, uint32_t vocab, float scale, int accumulate, int piece,
                                                           float* __restrict__ d_table, float* __restrict__ part) {
    const int64_t p = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    const int64_t lo = p * piece;
    const int c = (blockIdx.y * blockDim.x + threadIdx.x) * V;
    if (lo >= N || c >= d) return;
    const int64_t hi = lo + piece < N ? lo + piece : N;
    uint32_t key = keys[lo];
    bool from_left = lo > 0 && keys[lo - 1] == key;
    float acc[V] = {};
    for (int64_t i = lo; i < hi && key < vocab; ) {
        float v[V];
        ld_row<V>(dx + (int64_t)items[i] * d + c, v);
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] += v[j];
        ++i;
        const uint32_t next = i < N ? keys[i] : 0xffffffffu;
        if (next == key && i < hi) continue;
        const bool to_right = next == key;   // (i == hi then)
        if (from_left || to_right) st_row<V>(part + (2 * p + (from_left ? 0 : 1)) * d + c, acc);
        else add_row<V>(d_table + (int64_t)key * d + c, acc, scale, accumulate);
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] = 0.0f;
        key = next;
        from_left = false;
    }
}

// A block owns a piece and some columns; it has work where a run begins in the piece and goes on past it.
template <int V>
__global__ void __launch_bounds__(128) embed_join_kernel(const uint32_t* __restrict__ keys, int64_t N, int d, uint32_t vocab, float scale, int accumulate,
                                                         int piece, const float* __restrict__ part, float* __restrict__ d_table) {
    const int64_t p = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    const int64_t end = (p + 1) * piece;
    const int c = (blockIdx.y * blockDim.x + threadIdx.x) * V;
    if (end >= N || c >= d) return;
    const uint32_t key = keys[end - 1];
    if (key >= vocab || keys[end] != key) return;
    if (p > 0 && keys[p * piece - 1] == key) return;   // (it began further left)
    float acc[V];
    ld_row<V>(part + (2 * p + 1) * d + c, acc);
    for (int64_t q = p + 1; q * piece < N && keys[q * piece] == key; ++q) {
        float v[V];
        ld_row<V>(part + 2 * q * d + c, v);
#pragma unroll
        for (int j = 0; j < V; ++j) acc[j] += v[j];
    }
    add_row<V>(d_table + (int64_t)key * d + c, acc, scale, accumulate);
}

constexpr int PIECE = 64;

// Scratch: sorted keys and items, the pass before's where there are two, the counts, and the partial sums.
struct Plan {
    int bits, passes, digit;
    size_t list, counts, part;
    Plan(int64_t N, int64_t d, int64_t vocab) {
        bits = 1;
        while (((int64_t)1 << bits) <= vocab) ++bits;   // keys 0 .. vocab
        passes = (int)ceil_div64(bits, 11);
        digit = (int)ceil_div64(bits, passes);
        list = ((size_t)N * 4 + 255) & ~(size_t)255;
        counts = stable_sort::counts_bytes(N, 1 << digit);
        part = (size_t)ceil_div64(N, PIECE) * 2 * d * 4;
    }
    size_t bytes() const { return 4 * list + counts + part + 256; }
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
    asca_device_scope on(ctx);
    const bool four = asca_rows_by_four(table, d, table_dtype) && asca_rows_by_four(x, d, out_dtype);
    const int64_t per_row = four ? d / 4 : d;
    const int tx = per_row >= 256 ? 256 : (int)ceil_div64(per_row, 32) * 32, ty = 256 / tx;
    const dim3 grid((unsigned)ceil_div64(N, ty)), block(tx, ty);
    auto go = [&](auto tab, auto out) {
        using TT = std::remove_const_t<std::remove_pointer_t<decltype(tab)>>;
        using TX = std::remove_const_t<std::remove_pointer_t<decltype(out)>>;
        if (four) embed_scaled_fwd_kernel<4, TT, TX><<<grid, block, 0, ctx->stream>>>(tab, ids, N, (int)d, (uint32_t)vocab, scale, out);
        else embed_scaled_fwd_kernel<1, TT, TX><<<grid, block, 0, ctx->stream>>>(tab, ids, N, (int)d, (uint32_t)vocab, scale, out);
    };
    asca_with_dtype(table, table_dtype, [&](auto tab) { asca_with_dtype(x, out_dtype, [&](auto out) { go(tab, out); }); });
    ASCA_CHECK_LAUNCH(ctx);
    return ASCA_OK;
}

int64_t asca_embed_scaled_bwd_ws(int64_t N, int64_t d, int64_t vocab) {
    if (N < 0 || d <= 0 || vocab <= 0) return ASCA_ERR_ARG;
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
    if (!accumulate) ASCA_CUDA(ctx, cudaMemsetAsync(d_table, 0, (size_t)vocab * d * 4, ctx->stream));
    if (N == 0) return ASCA_OK;
    ASCA_REQUIRE(ctx, dx && ids && ws, "embed_scaled_bwd: null pointer");
    const Plan plan(N, d, vocab);
    ASCA_REQUIRE(ctx, asca_aligned(ws, 256) && ws_bytes >= plan.bytes(), "embed_scaled_bwd: the workspace has to have asca_embed_scaled_bwd_ws bytes, 256-byte aligned");
    char* w = (char*)ws;
    uint32_t* keys[2] = {(uint32_t*)w, (uint32_t*)(w + plan.list)};
    int32_t* items[2] = {(int32_t*)(w + 2 * plan.list), (int32_t*)(w + 3 * plan.list)};
    int32_t* counts = (int32_t*)(w + 4 * plan.list);
    float* part = (float*)(w + 4 * plan.list + plan.counts);
    int at = 0;
    for (int i = 0; i < plan.passes; ++i) {
        stable_sort::Pass p;
        p.n = N;
        p.limit = (uint32_t)vocab;
        if (i == 0) p.ids = ids;
        else p.keys = keys[at], p.items = items[at];
        p.shift = i * plan.digit;
        p.bins = 1 << plan.digit;
        p.mask = (uint32_t)p.bins - 1;
        at = i == 0 ? 0 : 1 - at;
        p.out_keys = keys[at];
        p.out_items = items[at];
        ASCA_TRY(stable_sort::run(ctx, p, counts, nullptr, 0));
    }
    const bool four = asca_rows_by_four(dx, d, dtype) && asca_aligned(d_table, 16);
    const int64_t per_row = four ? d / 4 : d;
    const int tx = per_row >= 128 ? 128 : (int)ceil_div64(per_row, 32) * 32, ty = 128 / tx;
    const int64_t pieces = ceil_div64(N, PIECE);
    const dim3 block(tx, ty), grid((unsigned)ceil_div64(pieces, ty), (unsigned)ceil_div64(per_row, tx));
    ASCA_REQUIRE(ctx, grid.y <= 65535, "embed_scaled_bwd: rows too wide");
    asca_with_dtype(dx, dtype, [&](auto src) {
        using T = std::remove_const_t<std::remove_pointer_t<decltype(src)>>;
        if (four) embed_pieces_kernel<4, T><<<grid, block, 0, ctx->stream>>>(src, keys[at], items[at], N, (int)d, (uint32_t)vocab, scale, accumulate, PIECE, d_table, part);
        else embed_pieces_kernel<1, T><<<grid, block, 0, ctx->stream>>>(src, keys[at], items[at], N, (int)d, (uint32_t)vocab, scale, accumulate, PIECE, d_table, part);
    });
    ASCA_CHECK_LAUNCH(ctx);
    if (pieces > 1) {
        if (four) embed_join_kernel<4><<<grid, block, 0, ctx->stream>>>(keys[at], N, (int)d, (uint32_t)vocab, scale, accumulate, PIECE, part, d_table);
        else embed_join_kernel<1><<<grid, block, 0, ctx->stream>>>(keys[at], N, (int)d, (uint32_t)vocab, scale, accumulate, PIECE, part, d_table);
        ASCA_CHECK_LAUNCH(ctx);
    }
    return ASCA_OK;
}

}  // extern "C"

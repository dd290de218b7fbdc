// Tokens sorted by the experts that a router chose for them, their rows moved there and back with the router's weights, and the
// gradients of both moves.
//
// Assignment a = t * K + k gives token t to expert experts[t, k]. perm is the stable order of the assignments by expert, offsets the
// experts' bounds in it, slot its inverse (-1: an expert at or past E as unsigned, -1 among them -- the assignment goes nowhere and
// lies behind offsets[E] in perm).
//
//   sort     xs[slot[a]] = x[t]                          d_x[t] = sum_k d_xs[slot[a]]
//   unsort   out[t] = sum_k w[a] ys[slot[a]]             d_ys[slot[a]] = w[a] d_out[t],  d_w[a] = <d_out[t], ys[slot[a]]>
//
// All four go by token: a token's row is read (or written) once whatever K is, and the sums over k run in the order of k. Rows at and
// behind offsets[E] are neither read nor written. Bound by HBM.
#include "row_io.cuh"
#include "stable_sort.cuh"

namespace {

// a thread owns V columns of a token
template <int V, typename TX, typename TS>
__global__ void __launch_bounds__(256) sort_rows_kernel(const TX* __restrict__ x, const int32_t* __restrict__ slot, int64_t N, int K, int d,
                                                        TS* __restrict__ xs) {
    const int64_t t = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (t >= N) return;
    for (int c = threadIdx.x * V; c < d; c += blockDim.x * V) {
        float v[V];
        ld_row<V>(x + t * d + c, v);
        for (int k = 0; k < K; ++k) {
            const int32_t s = slot[t * K + k];
            if (s >= 0) st_row<V>(xs + (int64_t)s * d + c, v);
        }
    }
}

// weights null: every weight is one
template <int V, typename TS, typename TX>
__global__ void __launch_bounds__(256) unsort_rows_kernel(const TS* __restrict__ ys, const int32_t* __restrict__ slot, const float* __restrict__ weights,
                                                          int64_t N, int K, int d, TX* __restrict__ out) {
    const int64_t t = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
    if (t >= N) return;
    for (int c = threadIdx.x * V; c < d; c += blockDim.x * V) {
        float acc[V] = {};
        for (int k = 0; k < K; ++k) {
            const int32_t s = slot[t * K + k];
            if (s < 0) continue;
            const float w = weights ? weights[t * K + k] : 1.0f;
            float v[V];
            ld_row<V>(ys + (int64_t)s * d + c, v);
#pragma unroll
            for (int i = 0; i < V; ++i) acc[i] = fmaf(w, v[i], acc[i]);
        }
        st_row<V>(out + t * d + c, acc);
    }
}

// A warp owns a token. d_w (nullable); d_ys may be ys; four assignments at a time share one reading of d_out's row.
template <int V, typename TX, typename TS>
__global__ void __launch_bounds__(256) unsort_rows_bwd_kernel(const TX* __restrict__ d_out, const TS* ys, const int32_t* __restrict__ slot,
                                                              const float* __restrict__ weights, int64_t N, int K, int d, TS* d_ys,
                                                              float* __restrict__ d_w) {
    const int lane = threadIdx.x & 31;
    const int64_t t = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (t >= N) return;
    for (int k0 = 0; k0 < K; k0 += 4) {
        int32_t s[4];
        float w[4], dot[4] = {};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            s[j] = k0 + j < K ? slot[t * K + k0 + j] : -1;
            w[j] = s[j] >= 0 && weights ? weights[t * K + k0 + j] : 1.0f;
        }
        for (int c = lane * V; c < d; c += 32 * V) {
            float g[V];
            ld_row<V>(d_out + t * d + c, g);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (s[j] < 0) continue;
                float y[V], o[V];
                if (d_w) ld_row<V>(ys + (int64_t)s[j] * d + c, y);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    if (d_w) dot[j] = fmaf(g[i], y[i], dot[j]);
                    o[i] = w[j] * g[i];
                }
                st_row<V>(d_ys + (int64_t)s[j] * d + c, o);
            }
        }
        if (d_w) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float sum = warp_sum(dot[j]);
                if (lane == 0 && k0 + j < K) d_w[t * K + k0 + j] = s[j] >= 0 ? sum : 0.0f;
            }
        }
    }
}

struct Shape {
    dim3 grid, block;
};
inline Shape by_token(int64_t N, int64_t per_row) {
    const int tx = per_row >= 256 ? 256 : (int)ceil_div64(per_row, 32) * 32, ty = 256 / tx;
    return {dim3((unsigned)ceil_div64(N, ty)), dim3(tx, ty)};
}

int check_rows(asca_ctx* ctx, const char* who, int64_t N, int64_t K, int64_t d, int tok_dtype, int row_dtype) {
    ASCA_REQUIRE(ctx, N >= 0 && K > 0 && d > 0 && d < (1 << 30) && K < (1 << 16) && N < ((int64_t)1 << 31) / K, "%s: bad shape (N * K must fit int32)", who);
    ASCA_REQUIRE(ctx, asca_known_dtype(tok_dtype) && asca_known_dtype(row_dtype), "%s: unknown dtype", who);
    return ASCA_OK;
}

}  // namespace

extern "C" {

int64_t asca_moe_topk_dispatch_ws(int64_t N, int64_t K, int64_t E) {
    if (N < 0 || K <= 0 || E <= 0 || E + 1 > stable_sort::MAX_BINS) return ASCA_ERR_ARG;
    return (int64_t)stable_sort::counts_bytes(N * K, (int)E + 1) + 256;
}

int asca_moe_topk_dispatch(asca_ctx* ctx, const int32_t* experts, int64_t N, int64_t K, int64_t E, int32_t* perm, int32_t* offsets, int32_t* slot,
                           void* ws, size_t ws_bytes) {
    if (!ctx) return ASCA_ERR_ARG;
    ASCA_TRY(check_rows(ctx, "moe_topk_dispatch", N, K, 1, ASCA_F32, ASCA_F32));
    ASCA_REQUIRE(ctx, E >= 1 && E + 1 <= stable_sort::MAX_BINS, "moe_topk_dispatch: 1 to %d experts", stable_sort::MAX_BINS - 1);
    ASCA_REQUIRE(ctx, offsets, "moe_topk_dispatch: null pointer");
    asca_device_scope on(ctx);
    if (N == 0) {
        ASCA_CUDA(ctx, cudaMemsetAsync(offsets, 0, (size_t)(E + 1) * 4, ctx->stream));
        return ASCA_OK;
    }
    ASCA_REQUIRE(ctx, experts && perm && slot && ws, "moe_topk_dispatch: null pointer");
    ASCA_REQUIRE(ctx, asca_aligned(ws, 256) && ws_bytes >= (size_t)asca_moe_topk_dispatch_ws(N, K, E),
                 "moe_topk_dispatch: the workspace has to have asca_moe_topk_dispatch_ws bytes, 256-byte aligned");
    stable_sort::Pass p;
    p.ids = (const uint32_t*)experts;
    p.limit = (uint32_t)E;
    p.n = N * K;
    p.bins = (int)E + 1;
    p.out_items = perm;
    p.place = slot;
    return stable_sort::run(ctx, p, (int32_t*)ws, offsets, (int)E + 1);
}

int asca_moe_sort_rows(asca_ctx* ctx, const void* x, const int32_t* slot, int64_t N, int64_t K, int64_t d, int x_dtype, int xs_dtype, void* xs) {
    if (!ctx) return ASCA_ERR_ARG;
    ASCA_TRY(check_rows(ctx, "moe_sort_rows", N, K, d, x_dtype, xs_dtype));
    if (N == 0) return ASCA_OK;
    ASCA_REQUIRE(ctx, x && slot && xs, "moe_sort_rows: null pointer");
    asca_device_scope on(ctx);
    const bool four = asca_rows_by_four(x, d, x_dtype) && asca_rows_by_four(xs, d, xs_dtype);
    const Shape s = by_token(N, four ? d / 4 : d);
    asca_with_dtype(x, x_dtype, [&](auto a) {
        asca_with_dtype(xs, xs_dtype, [&](auto b) {
            using TX = std::remove_const_t<std::remove_pointer_t<decltype(a)>>;
            using TS = std::remove_pointer_t<decltype(b)>;
            if (four) sort_rows_kernel<4, TX, TS><<<s.grid, s.block, 0, ctx->stream>>>(a, slot, N, (int)K, (int)d, b);
            else sort_rows_kernel<1, TX, TS><<<s.grid, s.block, 0, ctx->stream>>>(a, slot, N, (int)K, (int)d, b);
        });
    });
    ASCA_CHECK_LAUNCH(ctx);
    return ASCA_OK;
}

int asca_moe_unsort_rows(asca_ctx* ctx, const void* ys, const int32_t* slot, const float* weights, int64_t N, int64_t K, int64_t d, int ys_dtype,
                         int out_dtype, void* out) {
    if (!ctx) return ASCA_ERR_ARG;
    ASCA_TRY(check_rows(ctx, "moe_unsort_rows", N, K, d, out_dtype, ys_dtype));
    if (N == 0) return ASCA_OK;
    ASCA_REQUIRE(ctx, ys && slot && out, "moe_unsort_rows: null pointer");
    asca_device_scope on(ctx);
    const bool four = asca_rows_by_four(ys, d, ys_dtype) && asca_rows_by_four(out, d, out_dtype);
    const Shape s = by_token(N, four ? d / 4 : d);
    asca_with_dtype(ys, ys_dtype, [&](auto a) {
        asca_with_dtype(out, out_dtype, [&](auto b) {
            using TS = std::remove_const_t<std::remove_pointer_t<decltype(a)>>;
            using TX = std::remove_pointer_t<decltype(b)>;
            if (four) unsort_rows_kernel<4, TS, TX><<<s.grid, s.block, 0, ctx->stream>>>(a, slot, weights, N, (int)K, (int)d, b);
            else unsort_rows_kernel<1, TS, TX><<<s.grid, s.block, 0, ctx->stream>>>(a, slot, weights, N, (int)K, (int)d, b);
        });
    });
    ASCA_CHECK_LAUNCH(ctx);
    return ASCA_OK;
}

int asca_moe_sort_rows_bwd(asca_ctx* ctx, const void* d_xs, const int32_t* slot, int64_t N, int64_t K, int64_t d, int xs_dtype, int x_dtype, void* d_x) {
    return asca_moe_unsort_rows(ctx, d_xs, slot, nullptr, N, K, d, xs_dtype, x_dtype, d_x);
}

int asca_moe_unsort_rows_bwd(asca_ctx* ctx, const void* d_out, const void* ys, const int32_t* slot, const float* weights, int64_t N, int64_t K, int64_t d,
                             int out_dtype, int ys_dtype, void* d_ys, float* d_w) {
    if (!ctx) return ASCA_ERR_ARG;
    ASCA_TRY(check_rows(ctx, "moe_unsort_rows_bwd", N, K, d, out_dtype, ys_dtype));
    if (N == 0) return ASCA_OK;
    ASCA_REQUIRE(ctx, d_out && slot && d_ys, "moe_unsort_rows_bwd: null pointer");
    ASCA_REQUIRE(ctx, !d_w || ys, "moe_unsort_rows_bwd: the weights' gradient needs ys");
    asca_device_scope on(ctx);
    const bool four = asca_rows_by_four(d_out, d, out_dtype) && asca_rows_by_four(ys, d, ys_dtype) && asca_rows_by_four(d_ys, d, ys_dtype);
    const unsigned grid = (unsigned)ceil_div64(N, 8);
    asca_with_dtype(d_out, out_dtype, [&](auto a) {
        asca_with_dtype(d_ys, ys_dtype, [&](auto b) {
            using TX = std::remove_const_t<std::remove_pointer_t<decltype(a)>>;
            using TS = std::remove_pointer_t<decltype(b)>;
            const TS* y = static_cast<const TS*>(ys);
            if (four) unsort_rows_bwd_kernel<4, TX, TS><<<grid, 256, 0, ctx->stream>>>(a, y, slot, weights, N, (int)K, (int)d, b, d_w);
            else unsort_rows_bwd_kernel<1, TX, TS><<<grid, 256, 0, ctx->stream>>>(a, y, slot, weights, N, (int)K, (int)d, b, d_w);
        });
    });
    ASCA_CHECK_LAUNCH(ctx);
    return ASCA_OK;
}

}  // extern "C"

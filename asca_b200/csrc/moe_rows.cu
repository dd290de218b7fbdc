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
// behind offsets[E] are not written, and no value of theirs is used. Bound by HBM.
#include "row_io.cuh"
#include "stable_sort.cuh"

namespace {

// sort: a thread has its columns of TOKENS tokens in flight (the rows are asked for before the first is used); a block has as many lanes
// a token as a row has groups of columns, 256 at most.
constexpr int TOKENS = 4;

template <int W, typename TX, typename TS>
__global__ void __launch_bounds__(256) sort_rows_kernel(const TX* __restrict__ x, const int32_t* __restrict__ slot, int64_t N, int K, int d,
                                                        TS* __restrict__ xs) {
    using F = frag<W, TX>;
    const int lanes = blockDim.x;
    const uint32_t rows = (uint32_t)N * (uint32_t)K;
    const int64_t t0 = ((int64_t)blockIdx.x * blockDim.y + threadIdx.y) * TOKENS;
    for (int c = frag_first<W>(threadIdx.x); c < d; c += lanes * F::E) {
        F r[TOKENS];
#pragma unroll
        for (int i = 0; i < TOKENS; ++i)
            if (t0 + i < N) r[i].load(x + (t0 + i) * d, c, lanes, d);
#pragma unroll
        for (int i = 0; i < TOKENS; ++i) {
            if (t0 + i >= N) break;
            for (int k = 0; k < K; ++k) {
                const uint32_t s = slot[(t0 + i) * K + k];
                if (s >= rows) continue;   // (nowhere)
                TS* p = xs + (int64_t)s * d;
                if constexpr (std::is_same_v<TX, TS>) r[i].store(p, c, lanes, d);   // bit for bit
                else {
                    float v[F::E];
                    r[i].get(v);
                    frag<W, TS>::put(p, c, lanes, d, v);
                }
            }
        }
    }
}

// unsort and its gradient: some lanes own PAIRS / KS tokens, KS assignments of each at a time: PAIRS rows of the sorted side in flight.
// There is no branch around a load. Forward an assignment that goes nowhere asks for row 0 and does not use it (with another
// assignment's row of the same lanes in its place all loads wait for all slots: 65,536 x 2 x 1024 f32 131 us, 127 here; 16,000 x 4 x 1024
// 58, 56; rows of single columns gain by it, 40,000 x 3 x 777 99, 123 here). In the gradient, where d_ys may be ys and row 0 another
// CTA's to write, it asks for a row of the same lanes (`live`), and where all of them go nowhere nothing is asked for: same times.
constexpr int PAIRS = 4;

// weights null: every weight is one. K = 1: up to 256 lanes a token, so that a block goes over four rows from end to end, which HBM
// likes better than eight warps each at four rows of their own (16,000 x 4096 f32: 88 us, 159 by warps); with several assignments a
// warp's tokens lie close together anyway, and a bf16 row would leave wide blocks lanes (32,768 x 2 x 2048 bf16: 90 us by warps, 99).
// Few tokens: blocks beside each other (blockIdx.y) share the columns.
template <int W, int KS, typename TS, typename TX>
__global__ void __launch_bounds__(256) unsort_rows_kernel(const TS* __restrict__ ys, const int32_t* __restrict__ slot, const float* __restrict__ weights,
                                                          int64_t N, int K, int d, TX* __restrict__ out) {
    using F = frag<W, TS>;
    constexpr int T = PAIRS / KS;
    const int lanes = blockDim.x;
    const uint32_t rows = (uint32_t)N * (uint32_t)K;
    const int64_t t0 = ((int64_t)blockIdx.x * blockDim.y + threadIdx.y) * T;
    for (int c = blockIdx.y * lanes * F::E + frag_first<W>(threadIdx.x); c < d; c += gridDim.y * lanes * F::E) {
        float acc[T][F::E] = {};
        for (int k0 = 0; k0 < K; k0 += KS) {
            F r[T][KS];
            float w[T][KS];
            uint32_t s[T][KS];
#pragma unroll
            for (int i = 0; i < T; ++i) {
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    s[i][j] = t0 + i < N && k0 + j < K ? (uint32_t)slot[(t0 + i) * K + k0 + j] : ~0u;
                    w[i][j] = s[i][j] < rows && weights ? weights[(t0 + i) * K + k0 + j] : 1.0f;
                    r[i][j].load(ys + (int64_t)(s[i][j] < rows ? s[i][j] : 0) * d, c, lanes, d);
                }
            }
#pragma unroll
            for (int i = 0; i < T; ++i) {
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    if (s[i][j] >= rows) continue;   // (adds nothing, whatever its weight)
                    float v[F::E];
                    r[i][j].get(v);
#pragma unroll
                    for (int e = 0; e < F::E; ++e) acc[i][e] = fmaf(w[i][j], v[e], acc[i][e]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < T; ++i)
            if (t0 + i < N) frag<W, TX>::put(out + (t0 + i) * d, c, lanes, d, acc[i]);
    }
}

// The KS assignments of a token share one reading of d_out's row; d_w (nullable) is a sum over it. d_ys may be ys. LANES = 256: a CTA
// a token, or four with K = 1, where tokens are too few to fill the SMs by warps (500 x 2 x 2048: 4.1 us, 10.4 by warps) or a single
// assignment's row is long (16,000 x 4096 f32: 120 us, 141 by warps; 512 groups of eight bf16: 88 and 85).
template <int W, int LANES, int KS, typename TX, typename TS>
__global__ void __launch_bounds__(256) unsort_rows_bwd_kernel(const TX* __restrict__ d_out, const TS* ys, const int32_t* __restrict__ slot,
                                                              const float* __restrict__ weights, int64_t N, int K, int d, TS* d_ys,
                                                              float* __restrict__ d_w) {
    constexpr int T = PAIRS / KS, E = frag<W, TX>::E;
    const int lane = threadIdx.x % LANES;
    const uint32_t rows = (uint32_t)N * (uint32_t)K;
    const int64_t t0 = ((int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES) * T;
    for (int k0 = 0; k0 < K; k0 += KS) {
        uint32_t s[T][KS], live = ~0u;
        float w[T][KS], dot[T][KS] = {};
#pragma unroll
        for (int i = 0; i < T; ++i) {
#pragma unroll
            for (int j = 0; j < KS; ++j) {
                s[i][j] = t0 + i < N && k0 + j < K ? (uint32_t)slot[(t0 + i) * K + k0 + j] : ~0u;
                w[i][j] = s[i][j] < rows && weights ? weights[(t0 + i) * K + k0 + j] : 1.0f;
                live = s[i][j] < rows ? s[i][j] : live;
            }
        }
        for (int c = live < rows ? frag_first<W>(lane) : d; c < d; c += LANES * E) {
            frag<W, TX> rg[T];
            frag<W, TS> ry[T][KS];
#pragma unroll
            for (int i = 0; i < T; ++i) {
                rg[i].load(d_out + min(t0 + i, N - 1) * d, c, LANES, d);
#pragma unroll
                for (int j = 0; j < KS; ++j)
                    if (d_w) ry[i][j].load(ys + (int64_t)(s[i][j] < rows ? s[i][j] : live) * d, c, LANES, d);
            }
#pragma unroll
            for (int i = 0; i < T; ++i) {
                float g[E];
                rg[i].get(g);
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    if (s[i][j] >= rows) continue;
                    float y[E], o[E];
                    if (d_w) ry[i][j].get(y);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        if (d_w && (W > 1 || c + e * LANES < d)) dot[i][j] = fmaf(g[e], y[e], dot[i][j]);
                        o[e] = w[i][j] * g[e];
                    }
                    frag<W, TS>::put(d_ys + (int64_t)s[i][j] * d, c, LANES, d, o);
                }
            }
        }
        if (d_w) {
#pragma unroll
            for (int i = 0; i < T; ++i) {
#pragma unroll
                for (int j = 0; j < KS; ++j) {
#pragma unroll
                    for (int o = (LANES < 32 ? LANES : 32) / 2; o > 0; o >>= 1) dot[i][j] += __shfl_xor_sync(0xffffffffu, dot[i][j], o);
                    if constexpr (LANES == 256) {
                        __shared__ float sums[8];
                        if (lane % 32 == 0) sums[lane / 32] = dot[i][j];
                        __syncthreads();
                        dot[i][j] = 0.0f;
#pragma unroll
                        for (int w = 0; w < 8; ++w) dot[i][j] += sums[w];
                        __syncthreads();
                    }
                    if (t0 + i < N && lane == 0 && k0 + j < K) d_w[(t0 + i) * K + k0 + j] = s[i][j] < rows ? dot[i][j] : 0.0f;
                }
            }
        }
    }
}

// f(assignments of a token that are taken at a time)
template <typename F>
inline void with_assignments(int64_t K, F f) {
    if (K == 1) f(std::integral_constant<int, 1>());
    else if (K == 2) f(std::integral_constant<int, 2>());
    else f(std::integral_constant<int, 4>());
}

int check_rows(asca_ctx* ctx, const char* who, int64_t N, int64_t K, int64_t d, int tok_dtype, int row_dtype) {
    ASCA_REQUIRE(ctx, N >= 0 && K > 0 && d > 0 && d < (1 << 30) && K < (1 << 16) && N < ((int64_t)1 << 31) / K, "%s: bad shape (N * K must fit int32)", who);
    ASCA_REQUIRE(ctx, asca_known_dtype(tok_dtype) && asca_known_dtype(row_dtype), "%s: unknown dtype", who);
    return ASCA_OK;
}

}  // namespace

extern "C" {

int64_t asca_moe_topk_dispatch_ws(int64_t N, int64_t K, int64_t E) {
    if (N < 0 || K <= 0 || K >= (1 << 16) || N >= ((int64_t)1 << 31) / K || E <= 0 || E >= stable_sort::MAX_BINS) return ASCA_ERR_ARG;
    return (int64_t)stable_sort::scratch_bytes(N * K, (int)E + 1);   // (few assignments: none)
}

int asca_moe_topk_dispatch(asca_ctx* ctx, const int32_t* experts, int64_t N, int64_t K, int64_t E, int32_t* perm, int32_t* offsets, int32_t* slot,
                           void* ws, size_t ws_bytes) {
    if (!ctx) return ASCA_ERR_ARG;
    ASCA_TRY(check_rows(ctx, "moe_topk_dispatch", N, K, 1, ASCA_F32, ASCA_F32));
    ASCA_REQUIRE(ctx, E >= 1 && E < stable_sort::MAX_BINS, "moe_topk_dispatch: 1 to %d experts", stable_sort::MAX_BINS - 1);
    ASCA_REQUIRE(ctx, offsets, "moe_topk_dispatch: null pointer");
    asca_device_scope on(ctx);
    if (N == 0) {
        ASCA_CUDA(ctx, cudaMemsetAsync(offsets, 0, (size_t)(E + 1) * 4, ctx->stream));
        return ASCA_OK;
    }
    ASCA_REQUIRE(ctx, experts && perm && slot, "moe_topk_dispatch: null pointer");
    const asca_span_of in(experts, N * K, 4), out[3] = {{perm, N * K, 4}, {offsets, E + 1, 4}, {slot, N * K, 4}};
    for (int i = 0; i < 3; ++i)
        ASCA_REQUIRE(ctx, asca_apart(out[i], in) && asca_apart(out[i], out[(i + 1) % 3]), "moe_topk_dispatch: an output lies over an input or another output");
    ASCA_REQUIRE(ctx, asca_aligned(ws, 256) && ws_bytes >= (size_t)asca_moe_topk_dispatch_ws(N, K, E) && (ws || ws_bytes == 0),
                 "moe_topk_dispatch: the workspace has to have asca_moe_topk_dispatch_ws bytes, 256-byte aligned");
    stable_sort::Job j{};
    j.ids = (const uint32_t*)experts;
    j.limit = (uint32_t)E;
    j.n = N * K;
    j.passes = 1;
    j.bins = (int)E + 1;
    j.items[0] = perm;
    j.place = slot;
    j.offsets = offsets;
    return stable_sort::sort(ctx, j, (int32_t*)ws);
}

int asca_moe_sort_rows(asca_ctx* ctx, const void* x, const int32_t* slot, int64_t N, int64_t K, int64_t d, int x_dtype, int xs_dtype, void* xs) {
    if (!ctx) return ASCA_ERR_ARG;
    ASCA_TRY(check_rows(ctx, "moe_sort_rows", N, K, d, x_dtype, xs_dtype));
    if (N == 0) return ASCA_OK;
    ASCA_REQUIRE(ctx, x && slot && xs, "moe_sort_rows: null pointer");
    const asca_span_of out(xs, N * K * d, asca_dtype_size(xs_dtype));
    ASCA_REQUIRE(ctx, asca_apart(out, {x, N * d, asca_dtype_size(x_dtype)}) && asca_apart(out, {slot, N * K, 4}), "moe_sort_rows: xs lies over an input");
    asca_device_scope on(ctx);
    const int v = asca_row_width(d, x, x_dtype, xs, xs_dtype);
    const dim3 block = asca_row_block(asca_row_frags(d, v), 256), grid((unsigned)ceil_div64(N, (int64_t)block.y * TOKENS));
    asca_with_dtype(x, x_dtype, [&](auto a) {
        asca_with_dtype(xs, xs_dtype, [&](auto b) {
            using TX = std::remove_const_t<std::remove_pointer_t<decltype(a)>>;
            using TS = std::remove_pointer_t<decltype(b)>;
            asca_with_width<TX, TS>(v, [&](auto w) { sort_rows_kernel<w(), TX, TS><<<grid, block, 0, ctx->stream>>>(a, slot, N, (int)K, (int)d, b); });
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
    const asca_span_of to(out, N * d, asca_dtype_size(out_dtype));
    ASCA_REQUIRE(ctx, asca_apart(to, {ys, N * K * d, asca_dtype_size(ys_dtype)}) && asca_apart(to, {slot, N * K, 4}) && asca_apart(to, {weights, N * K, 4}),
                 "moe_unsort_rows: out lies over an input");
    asca_device_scope on(ctx);
    const int v = asca_row_width(d, ys, ys_dtype, out, out_dtype);
    const int64_t frags = asca_row_frags(d, v);
    asca_with_dtype(ys, ys_dtype, [&](auto a) {
        asca_with_dtype(out, out_dtype, [&](auto b) {
            using TS = std::remove_const_t<std::remove_pointer_t<decltype(a)>>;
            using TX = std::remove_pointer_t<decltype(b)>;
            asca_with_width<TX, TS>(v, [&](auto w) {
                with_assignments(K, [&](auto ks) {
                    const dim3 block = asca_row_block(ks() == 1 ? frags : std::min<int64_t>(frags, 32), 256);
                    const int64_t blocks = ceil_div64(N, (int64_t)block.y * (PAIRS / ks()));
                    const dim3 grid((unsigned)blocks, asca_column_blocks(ctx, blocks, frags, block.x));
                    unsort_rows_kernel<w(), ks(), TS, TX><<<grid, block, 0, ctx->stream>>>(a, slot, weights, N, (int)K, (int)d, b);
                });
            });
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
    const asca_span_of g(d_out, N * d, asca_dtype_size(out_dtype)), rows(d_w ? ys : nullptr, N * K * d, asca_dtype_size(ys_dtype)), at(slot, N * K, 4),
        w(weights, N * K, 4), to(d_ys, N * K * d, asca_dtype_size(ys_dtype)), to_w(d_w, N * K, 4);
    ASCA_REQUIRE(ctx, asca_in_place(to, rows) && asca_apart(to, g) && asca_apart(to, at) && asca_apart(to, w) && asca_apart(to, to_w) && asca_apart(to_w, g) &&
                          asca_apart(to_w, rows) && asca_apart(to_w, at) && asca_apart(to_w, w),
                 "moe_unsort_rows_bwd: an output lies over an input (d_ys may be ys) or the other output");
    asca_device_scope on(ctx);
    const int v = std::min(asca_row_width(d, d_out, out_dtype, ys, ys_dtype), asca_row_width(d, d_out, out_dtype, d_ys, ys_dtype));
    const int64_t frags = asca_row_frags(d, v);
    asca_with_dtype(d_out, out_dtype, [&](auto a) {
        asca_with_dtype(d_ys, ys_dtype, [&](auto b) {
            using TX = std::remove_const_t<std::remove_pointer_t<decltype(a)>>;
            using TS = std::remove_pointer_t<decltype(b)>;
            asca_with_width<TX, TS>(v, [&](auto w) {
                with_assignments(K, [&](auto ks) {
                    auto by = [&](auto l) {
                        const unsigned blocks = (unsigned)ceil_div64(N, 256 / l() * (PAIRS / ks()));
                        unsort_rows_bwd_kernel<w(), l(), ks(), TX, TS><<<blocks, 256, 0, ctx->stream>>>(a, static_cast<const TS*>(ys), slot, weights, N,
                                                                                                        (int)K, (int)d, b, d_w);
                    };
                    if ((frags > 32 && N <= 8 * ctx->sm_count) || (ks() == 1 && w() < 8 && frags >= 512)) by(std::integral_constant<int, 256>());
                    else asca_with_lanes(frags, by);
                });
            });
        });
    });
    ASCA_CHECK_LAUNCH(ctx);
    return ASCA_OK;
}

}  // extern "C"

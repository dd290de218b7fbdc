// The L2 norm of the gradients of many tensors, clipping by it in place, and the coefficient that the optimizer step takes.
//
//   norm = sqrt(sum over all elements of all tensors of g^2)          c = min(1, max_norm / (norm + 1e-6))
//
// A CTA owns an equal, contiguous share of all tensors laid end to end, eight 16-byte loads in flight a thread, and adds the squares in
// 64 bits, in which neither the square of a large f32 overflows nor that of a small one vanishes, and a long sum loses nothing. A
// second launch adds the CTAs' sums in a fixed order. (One cluster for small gradients, in one launch, takes longer: 331,000 f32
// 5.5 us by 16 CTAs, 4.0 by two launches.) The tensors' addresses travel with the launch (no copy in front of it, and a captured graph
// keeps them), 128 a launch. Bound by reading the gradients: 1.09 G f32 613 us = 7.1 TB/s, 0.5 G bf16 162 us = 6.2; clipping 0.5 G
// bf16 in place 323 us = 6.2 TB/s.
//
// A norm that is not finite follows the formula: c is 0 for an infinite norm (an infinite gradient then gives NaN), NaN for NaN.
#include "row_io.cuh"

#include <algorithm>
#include <cmath>
#include <memory>
#include <new>
#include <utility>

namespace {

constexpr int MAX_TENSORS = 128, CTAS_PER_SM = 32, LOADS = 8, GRAIN = 256;
constexpr int64_t LEAST = 4 << 10, MOST = 128 << 10, ONE_CTA = 16 << 10, ONE_WARP = 4 << 10;   // bytes of a CTA, a warp
struct Tensors {
    void* p[MAX_TENSORS];
    int64_t n[MAX_TENSORS];
    int64_t off[MAX_TENSORS + 1];   // bytes in front of each tensor, all rounded up to GRAIN
    uint8_t bf16[MAX_TENSORS];
    int count;
};

// f(pointer to the tensor's type, elements, thread, number of threads) for every tensor's part in this CTA's share: all threads for a long
// one; short ones, which a thread would wait for one after the other, go to the warps in turn.
template <typename F>
__device__ __forceinline__ void each_part(const Tensors& t, F f) {
    const int64_t grains = t.off[t.count] / GRAIN, start = grains * blockIdx.x / gridDim.x * GRAIN, end = grains * (blockIdx.x + 1) / gridDim.x * GRAIN;
    int lo = 0, hi = t.count - 1;   // last tensor that begins at or in front of the share
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.off[mid] <= start) lo = mid; else hi = mid - 1;
    }
    for (; lo < t.count && t.off[lo] < end; ++lo) {
        const int size = t.bf16[lo] ? 2 : 4;
        const int64_t a = (start > t.off[lo] ? start - t.off[lo] : 0) / size, b = min((end - t.off[lo]) / size, t.n[lo]);
        if (a >= b) continue;   // (in the padding behind a tensor)
        auto with = [&](int me, auto threads) {
            if (t.bf16[lo]) f(static_cast<__nv_bfloat16*>(t.p[lo]) + a, b - a, me, threads);
            else f(static_cast<float*>(t.p[lo]) + a, b - a, me, threads);
        };
        if ((b - a) * size > ONE_WARP) with(threadIdx.x, std::integral_constant<int, 256>());
        else if ((lo & 7) == (int)threadIdx.x >> 5) with(threadIdx.x & 31, std::integral_constant<int, 32>());
    }
}

// A part of a tensor that may begin anywhere: single elements up to the 16-byte grid, then groups of G (16 bytes), then the rest.
template <typename T>
__device__ __forceinline__ int lead(const T* p, int64_t n) {
    const int off = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
    return (int)min(n, (int64_t)(off ? (int)(16 / sizeof(T)) - off : 0));
}
__device__ __forceinline__ void square_add(double& s, float v) { s = fma((double)v, (double)v, s); }
__device__ __forceinline__ void group_add(double (&s)[4], const raw_row<4, float>& r) {
    square_add(s[0], r.v.x); square_add(s[1], r.v.y); square_add(s[2], r.v.z); square_add(s[3], r.v.w);
}
__device__ __forceinline__ void group_add(double (&s)[4], const raw_row<8, __nv_bfloat16>& r) {
    float v[8];
    unpack(r, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) square_add(s[i & 3], v[i]);
}

__device__ double block_sum_f64(double v, double* red) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) red[w] = v;
    __syncthreads();
    v = lane < (int)(blockDim.x >> 5) ? red[lane] : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The CTA's sum, in every thread.
__device__ __forceinline__ double squares(const Tensors& t, double* red) {
    double s[4] = {};
    each_part(t, [&](auto* p, int64_t n, int me, auto by) {
        using T = std::remove_pointer_t<decltype(p)>;
        constexpr int G = 16 / sizeof(T), threads = decltype(by)::value;
        const int head = lead(p, n);
        const int64_t groups = (n - head) / G;
        int64_t i = me;
        for (; i + (LOADS - 1) * threads < groups; i += LOADS * threads) {
            raw_row<G, T> r[LOADS];
#pragma unroll
            for (int u = 0; u < LOADS; ++u) r[u] = ld_raw<G>(p + head + (i + u * threads) * G);
#pragma unroll
            for (int u = 0; u < LOADS; ++u) group_add(s, r[u]);
        }
        if constexpr (threads == 32) {   // (a short part: all of it in flight)
            for (; i < groups; i += LOADS * threads) {
                raw_row<G, T> r[LOADS];
#pragma unroll
                for (int u = 0; u < LOADS; ++u) r[u] = ld_raw<G>(p + head + min(i + u * threads, groups - 1) * G);
#pragma unroll
                for (int u = 0; u < LOADS; ++u)
                    if (i + u * threads < groups) group_add(s, r[u]);
            }
        }
        for (; i < groups; i += threads) group_add(s, ld_raw<G>(p + head + i * G));
        const int rest = (int)(n - groups * G);   // in front of the groups and behind them
        for (i = me; i < rest; i += threads) square_add(s[0], to_f32(p[i < head ? i : i + groups * G]));
    });
    return block_sum_f64((s[0] + s[1]) + (s[2] + s[3]), red);
}

template <bool ONE>   // the only CTA
__global__ void __launch_bounds__(256) norm_parts_kernel(const __grid_constant__ Tensors t, double* __restrict__ part, float* __restrict__ norm) {
    __shared__ double red[32];
    pdl_launch_dependents();
    const double s = squares(t, red);
    if (threadIdx.x > 0) return;
    if constexpr (ONE) *norm = (float)sqrt(s);
    else part[blockIdx.x] = s;
}

__global__ void __launch_bounds__(256) norm_join_kernel(const double* __restrict__ part, int n, float* __restrict__ norm) {
    __shared__ double red[32];
    pdl_wait();
    pdl_launch_dependents();
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) s += part[i];
    s = block_sum_f64(s, red);
    if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

__global__ void __launch_bounds__(256) clip_kernel(const __grid_constant__ Tensors t, const float* __restrict__ norm, float max_norm) {
    const float c = asca_clip_coefficient(*norm, max_norm);
    if (c == 1.0f) return;   // nothing changes
    each_part(t, [&](auto* p, int64_t n, int me, auto by) {
        using T = std::remove_pointer_t<decltype(p)>;
        constexpr int G = 16 / sizeof(T), threads = decltype(by)::value;
        const int head = lead(p, n);
        const int64_t groups = (n - head) / G;
        auto scale = [&](T* q, const raw_row<G, T>& r) {
            float v[G];
            unpack(r, v);
#pragma unroll
            for (int e = 0; e < G; ++e) v[e] *= c;
            st_row<G>(q, v);
        };
        int64_t i = me;
        for (; i + 3 * threads < groups; i += 4 * threads) {
            raw_row<G, T> r[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) r[u] = ld_raw<G>(p + head + (i + u * threads) * G);
#pragma unroll
            for (int u = 0; u < 4; ++u) scale(p + head + (i + u * threads) * G, r[u]);
        }
        for (; i < groups; i += threads) scale(p + head + i * G, ld_raw<G>(p + head + i * G));
        const int rest = (int)(n - groups * G);
        for (i = me; i < rest; i += threads) {
            T* q = p + (i < head ? i : i + groups * G);
            *q = from_f32<T>(c * to_f32<T>(*q));
        }
    });
}

int check_tensors(asca_ctx* ctx, const char* who, void* const* p, const int64_t* n, const int* dtype, int count) {
    ASCA_REQUIRE(ctx, count >= 0 && (count == 0 || (p && n && dtype)), "%s: bad arguments", who);
    for (int i = 0; i < count; ++i) {
        ASCA_REQUIRE(ctx, n[i] >= 0 && n[i] < ((int64_t)1 << 35) && (n[i] == 0 || p[i]), "%s: tensor %d: bad pointer or size", who, i);
        ASCA_REQUIRE(ctx, asca_known_dtype(dtype[i]), "%s: tensor %d: unknown dtype", who, i);
        ASCA_REQUIRE(ctx, asca_aligned(p[i], asca_dtype_size(dtype[i])), "%s: tensor %d is not aligned to its elements", who, i);
    }
    return ASCA_OK;
}

// The tensors from `at` on that one launch takes (empty ones left out); moves `at` behind them.
Tensors take(void* const* p, const int64_t* n, const int* dtype, int count, int& at) {
    Tensors t;
    int k = 0;
    t.off[0] = 0;
    for (; at < count && k < MAX_TENSORS; ++at) {
        if (n[at] == 0) continue;
        t.p[k] = p[at];
        t.n[k] = n[at];
        t.bf16[k] = dtype[at] == ASCA_BF16;
        t.off[k + 1] = t.off[k] + ceil_div64(n[at] * (int64_t)asca_dtype_size(dtype[at]), GRAIN) * GRAIN;
        ++k;
    }
    t.count = k;
    return t;
}
// Two CTAs an SM where that leaves each of them a share worth a CTA (8 MB: 4.6 us, 7.1 by shares of 128 KiB; 1.3 MB: 4.0 and 6.0); more
// CTAs only in shares of 128 KiB (51 MB: 9.0 us, 10.1 by 64). Few small tensors: one CTA, and no second launch.
int ctas_of(const asca_ctx* ctx, const Tensors& t) {
    const int64_t all = t.off[t.count], share = std::min(MOST, std::max(LEAST, all / (2 * ctx->sm_count)));
    if (all <= ONE_CTA && t.count <= 16) return all > 0;
    return (int)std::min<int64_t>(ceil_div64(all, share), ctx->sm_count * CTAS_PER_SM);
}

}  // namespace

extern "C" {

int64_t asca_grad_norm_ws(asca_ctx* ctx, int count) {
    if (!ctx || count < 0) return ASCA_ERR_ARG;
    return ceil_div64(std::max(count, 1), MAX_TENSORS) * ctx->sm_count * CTAS_PER_SM * (int64_t)sizeof(double);
}

int asca_grad_norm(asca_ctx* ctx, void* const* grads, const int64_t* n, const int* dtype, int count, float* norm, void* ws, size_t ws_bytes) {
    if (!ctx) return ASCA_ERR_ARG;
    ASCA_TRY(check_tensors(ctx, "grad_norm", grads, n, dtype, count));
    ASCA_REQUIRE(ctx, norm && ws && asca_aligned(ws, 8) && ws_bytes >= (size_t)asca_grad_norm_ws(ctx, count),
                 "grad_norm: null pointer, or a workspace of less than asca_grad_norm_ws bytes");
    asca_device_scope on(ctx);
    double* part = (double*)ws;
    int parts = 0;
    for (int at = 0; at < count; ) {
        const Tensors t = take(grads, n, dtype, count, at);
        const int grid = ctas_of(ctx, t);
        if (grid == 0) continue;
        if (grid == 1 && parts == 0 && at == count) {
            norm_parts_kernel<true><<<1, 256, 0, ctx->stream>>>(t, nullptr, norm);
            ASCA_CHECK_LAUNCH(ctx);
            return ASCA_OK;
        }
        norm_parts_kernel<false><<<(unsigned)grid, 256, 0, ctx->stream>>>(t, part + parts, nullptr);
        ASCA_CHECK_LAUNCH(ctx);
        parts += grid;
    }
    if (parts == 0) {   // (no tensors)
        ASCA_CUDA(ctx, cudaMemsetAsync(norm, 0, sizeof(float), ctx->stream));
        return ASCA_OK;
    }
    ASCA_CUDA(ctx, asca_launch_after(ctx, norm_join_kernel, dim3(1), dim3(256), 0, (const double*)part, parts, norm));
    ctx->launches++;
    return ASCA_OK;
}

int asca_clip_grads(asca_ctx* ctx, void* const* grads, const int64_t* n, const int* dtype, int count, const float* norm, float max_norm) {
    if (!ctx) return ASCA_ERR_ARG;
    ASCA_TRY(check_tensors(ctx, "clip_grads", grads, n, dtype, count));
    ASCA_REQUIRE(ctx, norm && max_norm >= 0.0f && std::isfinite(max_norm), "clip_grads: null pointer, or a largest norm that is none");
    for (int i = 0; i < count; ++i)   // (every CTA reads the norm when it begins, some behind others' writes)
        ASCA_REQUIRE(ctx, asca_apart({norm, 1, 4}, {grads[i], n[i], asca_dtype_size(dtype[i])}), "clip_grads: the norm lies in tensor %d", i);
    // an element that two tensors share would be scaled by both
    using Span = std::pair<uintptr_t, uintptr_t>;
    const std::unique_ptr<Span[]> span(new (std::nothrow) Span[(size_t)count + 1]);
    if (!span) return asca_fail(ctx, ASCA_ERR_OOM, "clip_grads: no host memory for the places of %d tensors", count);
    int spans = 0;
    for (int i = 0; i < count; ++i)
        if (n[i] > 0) span[spans++] = {(uintptr_t)grads[i], (uintptr_t)grads[i] + (size_t)n[i] * asca_dtype_size(dtype[i])};
    std::sort(span.get(), span.get() + spans);
    for (int i = 1; i < spans; ++i) ASCA_REQUIRE(ctx, span[i].first >= span[i - 1].second, "clip_grads: two tensors overlap");
    asca_device_scope on(ctx);
    for (int at = 0; at < count; ) {
        const Tensors t = take(grads, n, dtype, count, at);
        const int grid = ctas_of(ctx, t);
        if (grid == 0) continue;
        clip_kernel<<<(unsigned)grid, 256, 0, ctx->stream>>>(t, norm, max_norm);
        ASCA_CHECK_LAUNCH(ctx);
    }
    return ASCA_OK;
}

}  // extern "C"

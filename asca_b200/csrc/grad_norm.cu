// The L2 norm of the gradients of many tensors, clipping by it in place, and the coefficient that the optimizer step takes.
//
//   norm = sqrt(sum over all elements of all tensors of g^2)          c = min(1, max_norm / (norm + 1e-6))
//
// The tensors are cut into pieces of 16,384 elements; a CTA takes every gridDim-th piece and adds the squares in 64 bits, in which
// neither the square of a large f32 overflows nor that of a small one vanishes, and a long sum loses nothing. A second launch adds
// the CTAs' sums in a fixed order. Bound by reading the gradients. The tensors' addresses travel with the launch (no copy in
// front of it, and a captured graph keeps them), 160 a launch.
//
// A norm that is not finite follows the formula: c is 0 for an infinite norm (an infinite gradient then gives NaN), NaN for NaN.
#include "row_io.cuh"

#include <algorithm>
#include <cmath>

namespace {

constexpr int MAX_TENSORS = 160, PIECE = 16384;
struct Tensors {
    void* p[MAX_TENSORS];
    int64_t n[MAX_TENSORS];
    int32_t first[MAX_TENSORS + 1];   // the first piece of each tensor
    uint8_t bf16[MAX_TENSORS];
    int count;
};

// f(pointer to the tensor's type, first element, past the last) for every piece of this CTA
template <typename F>
__device__ __forceinline__ void each_piece(const Tensors& t, F f) {
    const int total = t.first[t.count];
    for (int i = blockIdx.x; i < total; i += gridDim.x) {
        int lo = 0, hi = t.count - 1;   // last tensor whose first piece is at most i
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (t.first[mid] <= i) lo = mid; else hi = mid - 1;
        }
        const int64_t a = (int64_t)(i - t.first[lo]) * PIECE, b = min(a + PIECE, t.n[lo]);
        if (t.bf16[lo]) f(static_cast<__nv_bfloat16*>(t.p[lo]) + a, (int)(b - a));
        else f(static_cast<float*>(t.p[lo]) + a, (int)(b - a));
    }
}

// A piece of a tensor that may begin anywhere: single elements up to the 16-byte grid, then groups of G (16 bytes), then the rest.
template <typename T>
__device__ __forceinline__ int lead(const T* p, int n) {
    const int off = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
    return min(n, off ? (int)(16 / sizeof(T)) - off : 0);
}
__device__ __forceinline__ void square_add(double& s, float v) { s = fma((double)v, (double)v, s); }
__device__ __forceinline__ void group_add(double& s, const float* p) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(p));
    square_add(s, v.x); square_add(s, v.y); square_add(s, v.z); square_add(s, v.w);
}
__device__ __forceinline__ void group_add(double& s, const __nv_bfloat16* p) {
    const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = bf16x2_f32(w[i]);
        square_add(s, v.x); square_add(s, v.y);
    }
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

__global__ void __launch_bounds__(256) norm_parts_kernel(const __grid_constant__ Tensors t, double* __restrict__ part) {
    __shared__ double red[32];
    double s = 0.0;
    each_piece(t, [&](auto* p, int n) {
        constexpr int G = 16 / sizeof(*p);
        const int head = lead(p, n), groups = (n - head) / G;
        for (int i = threadIdx.x; i < groups; i += 256) group_add(s, p + head + i * G);
        const int rest = n - groups * G;   // in front of the groups and behind them
        for (int i = threadIdx.x; i < rest; i += 256) square_add(s, to_f32(p[i < head ? i : i + groups * G]));
    });
    s = block_sum_f64(s, red);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__global__ void __launch_bounds__(256) norm_join_kernel(const double* __restrict__ part, int n, float* __restrict__ norm) {
    __shared__ double red[32];
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) s += part[i];
    s = block_sum_f64(s, red);
    if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

__global__ void __launch_bounds__(256) clip_kernel(const __grid_constant__ Tensors t, const float* __restrict__ norm, float max_norm) {
    const float c = asca_clip_coefficient(*norm, max_norm);
    if (c == 1.0f) return;   // nothing changes
    each_piece(t, [&](auto* p, int n) {
        using T = std::remove_pointer_t<decltype(p)>;
        const int head = min(n, (int)(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T))), groups = (n - head) / 4;
        for (int i = threadIdx.x; i < groups; i += 256) {
            T* q = p + head + i * 4;
            float4 v = ld4(q);
            v.x *= c; v.y *= c; v.z *= c; v.w *= c;
            st4(q, v);
        }
        const int rest = n - groups * 4;
        for (int i = threadIdx.x; i < rest; i += 256) {
            T* q = p + (i < head ? i : i + groups * 4);
            *q = from_f32<T>(c * to_f32<T>(*q));
        }
    });
}

int check_tensors(asca_ctx* ctx, const char* who, void* const* p, const int64_t* n, const int* dtype, int count) {
    ASCA_REQUIRE(ctx, count >= 0 && (count == 0 || (p && n && dtype)), "%s: bad arguments", who);
    for (int i = 0; i < count; ++i) {
        ASCA_REQUIRE(ctx, n[i] >= 0 && n[i] < ((int64_t)1 << 37) && (n[i] == 0 || p[i]), "%s: tensor %d: bad pointer or size", who, i);
        ASCA_REQUIRE(ctx, asca_known_dtype(dtype[i]), "%s: tensor %d: unknown dtype", who, i);
        ASCA_REQUIRE(ctx, asca_aligned(p[i], asca_dtype_size(dtype[i])), "%s: tensor %d is not aligned to its elements", who, i);
    }
    return ASCA_OK;
}

// The tensors from `at` on that one launch takes (empty ones left out); moves `at` behind them.
Tensors take(void* const* p, const int64_t* n, const int* dtype, int count, int& at) {
    Tensors t;
    int k = 0;
    int64_t pieces = 0;
    for (; at < count && k < MAX_TENSORS; ++at) {
        if (n[at] == 0) continue;
        t.p[k] = p[at];
        t.n[k] = n[at];
        t.bf16[k] = dtype[at] == ASCA_BF16;
        t.first[k] = (int32_t)pieces;
        pieces += ceil_div64(n[at], PIECE);
        ++k;
    }
    t.first[k] = (int32_t)pieces;
    t.count = k;
    return t;
}

constexpr int CTAS_PER_SM = 8;

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
        const int grid = std::min(t.first[t.count], ctx->sm_count * CTAS_PER_SM);
        if (grid == 0) continue;
        norm_parts_kernel<<<(unsigned)grid, 256, 0, ctx->stream>>>(t, part + parts);
        ASCA_CHECK_LAUNCH(ctx);
        parts += grid;
    }
    norm_join_kernel<<<1, 256, 0, ctx->stream>>>(part, parts, norm);
    ASCA_CHECK_LAUNCH(ctx);
    return ASCA_OK;
}

int asca_clip_grads(asca_ctx* ctx, void* const* grads, const int64_t* n, const int* dtype, int count, const float* norm, float max_norm) {
    if (!ctx) return ASCA_ERR_ARG;
    ASCA_TRY(check_tensors(ctx, "clip_grads", grads, n, dtype, count));
    ASCA_REQUIRE(ctx, norm && max_norm >= 0.0f && std::isfinite(max_norm), "clip_grads: null pointer, or a largest norm that is none");
    // an element that two tensors share would be scaled by both
    std::vector<std::pair<uintptr_t, uintptr_t>> span;
    for (int i = 0; i < count; ++i)
        if (n[i] > 0) span.push_back({(uintptr_t)grads[i], (uintptr_t)grads[i] + (size_t)n[i] * asca_dtype_size(dtype[i])});
    std::sort(span.begin(), span.end());
    for (size_t i = 1; i < span.size(); ++i) ASCA_REQUIRE(ctx, span[i].first >= span[i - 1].second, "clip_grads: two tensors overlap");
    asca_device_scope on(ctx);
    for (int at = 0; at < count; ) {
        const Tensors t = take(grads, n, dtype, count, at);
        const int grid = std::min(t.first[t.count], ctx->sm_count * CTAS_PER_SM);
        if (grid == 0) continue;
        clip_kernel<<<(unsigned)grid, 256, 0, ctx->stream>>>(t, norm, max_norm);
        ASCA_CHECK_LAUNCH(ctx);
    }
    return ASCA_OK;
}

}  // extern "C"

// The join behind a block in one pass: the norm of the block's output, its gate, the scaled residual and the norm in front of the
// next block; and its gradients.
//
//   n     = y r1 * w_post             r1 = 1 / sqrt(mean y^2 + eps)           (post_norm = 0: n = y)
//   x_out = skip x + branch gate * n
//   xn    = x_out r2 * w_pre          r2 = 1 / sqrt(mean x_out^2 + eps)
//
//   d     = d_out + r2 (t - x_out r2 mean(t x_out r2))       t = d_xn * w_pre           d_w_pre  = sum over rows of d_xn * x_out r2
//   d_x   = skip d                                                                       d_gate   = sum over its rows of branch d * n
//   d_y   = r1 (u - y r1 mean(u y r1))                       u = branch gate d * w_post  d_w_post = sum over rows of branch gate d * y r1
//
// A row belongs to a team: a warp up to 256 columns, else a CTA with eight columns a thread; the row stays in registers between its
// two reductions, so every matrix passes HBM once, which is what bounds both directions. The statistics are taken again in the
// backward pass, whose rows are in registers anyway: nothing is kept for it.
//
// Backward, a team owns a strip of consecutive rows and the same columns in all of them, so that the column sums stay in its
// registers; a strip's sums of the gains go out once, a gate's once for every group of rows in the strip, and a second launch adds
// the strips in a fixed order. A group of rows up to two strips long gets strips that end where groups end: its gate's gradient is
// then written at once.
#include "row_io.cuh"

#include <algorithm>

namespace {

constexpr int MAX_COLS = 8192;

// Columns of thread `tid` of a team of `team`: groups of four, `team` groups apart, or single columns `team` apart.
template <bool FOUR>
__device__ __forceinline__ int col_of(int j, int team, int tid) { return FOUR ? ((j >> 2) * team + tid) * 4 + (j & 3) : j * team + tid; }

template <int EPT, bool FOUR, typename T>
__device__ __forceinline__ void ld_cols(const T* p, int team, int tid, int cols, float (&v)[EPT], float other = 0.0f) {
    if constexpr (FOUR) {
#pragma unroll
        for (int q = 0; q < EPT / 4; ++q) {
            const int c = (q * team + tid) * 4;
            float4 x = make_float4(other, other, other, other);
            if (c < cols) x = ld4(p + c);
            v[4 * q] = x.x; v[4 * q + 1] = x.y; v[4 * q + 2] = x.z; v[4 * q + 3] = x.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < EPT; ++j) v[j] = j * team + tid < cols ? to_f32<T>(p[j * team + tid]) : other;
    }
}
template <int EPT, bool FOUR, typename T>
__device__ __forceinline__ void st_cols(T* p, int team, int tid, int cols, const float (&v)[EPT]) {
    if constexpr (FOUR) {
#pragma unroll
        for (int q = 0; q < EPT / 4; ++q) {
            const int c = (q * team + tid) * 4;
            if (c < cols) st4(p + c, make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]));
        }
    } else {
#pragma unroll
        for (int j = 0; j < EPT; ++j)
            if (j * team + tid < cols) p[j * team + tid] = from_f32<T>(v[j]);
    }
}

// Sums over a team, the same in all its threads. A CTA's teams alternate between two halves of `red` (`turn`), so that one barrier a
// sum is enough: who writes a half again has passed the barrier of the other, behind everybody's reading of this one.
template <bool WARP>
__device__ __forceinline__ float3 team_sum(float3 v, float4 (*red)[32], int& turn) {
    v.x = warp_sum(v.x); v.y = warp_sum(v.y); v.z = warp_sum(v.z);
    if constexpr (!WARP) {
        float4* r = red[turn];
        turn ^= 1;
        const int nw = blockDim.x >> 5;
        if ((threadIdx.x & 31) == 0) r[threadIdx.x >> 5] = make_float4(v.x, v.y, v.z, 0.0f);
        __syncthreads();
        v = make_float3(0.0f, 0.0f, 0.0f);
        for (int i = 0; i < nw; ++i) {
            const float4 a = r[i];
            v.x += a.x; v.y += a.y; v.z += a.z;
        }
    }
    return v;
}

struct Join {
    const void *y, *d_xn;
    const float *x, *w_post, *gate, *w_pre, *d_out;
    float *x_out;
    void *xn, *d_y;
    float *d_x, *d_w_post, *d_gate, *d_w_pre;
    int64_t rows, gate_rows;
    int cols, post, accumulate;
    float skip, branch, eps;
    // backward: rows a strip, strips, the CTAs' sums of the gains [cta][pre, post][cols] and the strips' sums of a gate that reaches past
    // the strip [strip][from the left, to the right][cols]
    int64_t strip, strips;
    float *part_w, *part_g;
};

template <typename T, int EPT, bool FOUR, bool WARP, int MOST>
__global__ void __launch_bounds__(MOST) join_fwd_kernel(const Join a) {
    __shared__ float4 red[2][32];
    const int team = WARP ? 32 : blockDim.x, tid = WARP ? threadIdx.x & 31 : threadIdx.x;
    const int64_t r = WARP ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;
    if (WARP && r >= a.rows) return;
    int turn = 0;
    const int cols = a.cols;
    float y[EPT], x[EPT];
    ld_cols<EPT, FOUR>(static_cast<const T*>(a.y) + r * cols, team, tid, cols, y);
    ld_cols<EPT, FOUR>(a.x + r * cols, team, tid, cols, x);
    if (a.post) {
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < EPT; ++j) s += y[j] * y[j];
        s = team_sum<WARP>(make_float3(s, 0.0f, 0.0f), red, turn).x;
        const float r1 = 1.0f / sqrtf(s / (float)cols + a.eps);
#pragma unroll
        for (int j = 0; j < EPT; ++j) y[j] *= r1;
        if (a.w_post) {
            float w[EPT];
            ld_cols<EPT, FOUR>(a.w_post, team, tid, cols, w);
#pragma unroll
            for (int j = 0; j < EPT; ++j) y[j] *= w[j];
        }
    }
    if (a.gate) {
        float g[EPT];
        ld_cols<EPT, FOUR>(a.gate + r / a.gate_rows * cols, team, tid, cols, g);
#pragma unroll
        for (int j = 0; j < EPT; ++j) y[j] *= g[j];
    }
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < EPT; ++j) {
        x[j] = a.skip * x[j] + a.branch * y[j];
        s += x[j] * x[j];
    }
    st_cols<EPT, FOUR>(a.x_out + r * cols, team, tid, cols, x);
    if (!a.xn) return;
    s = team_sum<WARP>(make_float3(s, 0.0f, 0.0f), red, turn).x;
    const float r2 = 1.0f / sqrtf(s / (float)cols + a.eps);
#pragma unroll
    for (int j = 0; j < EPT; ++j) x[j] *= r2;
    if (a.w_pre) {
        float w[EPT];
        ld_cols<EPT, FOUR>(a.w_pre, team, tid, cols, w);
#pragma unroll
        for (int j = 0; j < EPT; ++j) x[j] *= w[j];
    }
    st_cols<EPT, FOUR>(static_cast<T*>(a.xn) + r * cols, team, tid, cols, x);
}

template <int EPT, bool FOUR>
__device__ __forceinline__ void put_sum(float* p, int team, int tid, int cols, float (&v)[EPT], int accumulate) {
    if (accumulate) {
        float o[EPT];
        ld_cols<EPT, FOUR>(p, team, tid, cols, o);
#pragma unroll
        for (int j = 0; j < EPT; ++j) v[j] += o[j];
    }
    st_cols<EPT, FOUR>(p, team, tid, cols, v);
}

template <typename T, int EPT, bool FOUR, bool WARP, int MOST>
__global__ void __launch_bounds__(MOST) join_bwd_kernel(const Join a) {
    __shared__ float4 red[2][32];
    __shared__ float warp_part[WARP ? 8 * 32 * EPT : 1];
    const int team = WARP ? 32 : blockDim.x, tid = WARP ? threadIdx.x & 31 : threadIdx.x, cols = a.cols;
    const int64_t s = WARP ? (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5) : blockIdx.x;   // the strip
    const int64_t r0 = s * a.strip, r1 = min(r0 + a.strip, a.rows);
    int turn = 0;
    const float over = 1.0f / (float)cols;
    float sw_pre[EPT] = {}, sw_post[EPT] = {}, sg[EPT] = {};
    for (int64_t r = r0; r < r1; ++r) {
        float y[EPT], xo[EPT], dn[EPT], d[EPT], w[EPT], g[EPT];
        ld_cols<EPT, FOUR>(static_cast<const T*>(a.y) + r * cols, team, tid, cols, y);
        ld_cols<EPT, FOUR>(a.x_out + r * cols, team, tid, cols, xo);
        if (a.d_out) ld_cols<EPT, FOUR>(a.d_out + r * cols, team, tid, cols, d);
        float3 sum = make_float3(0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int j = 0; j < EPT; ++j) {
            if (!a.d_out) d[j] = 0.0f;
            g[j] = 1.0f;
            sum.x += y[j] * y[j];
        }
        const int64_t group = r / a.gate_rows;
        if (a.gate) ld_cols<EPT, FOUR>(a.gate + group * cols, team, tid, cols, g);
        if (a.d_xn) {
            ld_cols<EPT, FOUR>(static_cast<const T*>(a.d_xn) + r * cols, team, tid, cols, dn);
            if (a.w_pre) ld_cols<EPT, FOUR>(a.w_pre, team, tid, cols, w);
#pragma unroll
            for (int j = 0; j < EPT; ++j) {
                if (!a.w_pre) w[j] = 1.0f;
                sum.y += xo[j] * xo[j];
                sum.z += dn[j] * w[j] * xo[j];
            }
        }
        sum = team_sum<WARP>(sum, red, turn);
        if (a.d_xn) {
            const float i2 = 1.0f / sqrtf(sum.y * over + a.eps), mean = sum.z * i2 * over;
#pragma unroll
            for (int j = 0; j < EPT; ++j) {
                const float h = xo[j] * i2;
                sw_pre[j] += dn[j] * h;
                d[j] += i2 * (dn[j] * w[j] - h * mean);
            }
        }
        float dx[EPT];
#pragma unroll
        for (int j = 0; j < EPT; ++j) dx[j] = a.skip * d[j];
        st_cols<EPT, FOUR>(a.d_x + r * cols, team, tid, cols, dx);
        if (a.post) {
            const float i1 = 1.0f / sqrtf(sum.x * over + a.eps);
            if (a.w_post) ld_cols<EPT, FOUR>(a.w_post, team, tid, cols, w);
            float q = 0.0f;
#pragma unroll
            for (int j = 0; j < EPT; ++j) {
                if (!a.w_post) w[j] = 1.0f;
                y[j] *= i1;
                d[j] *= a.branch;
                sg[j] += d[j] * (y[j] * w[j]);
                d[j] *= g[j];
                sw_post[j] += d[j] * y[j];
                d[j] *= w[j];
                q += d[j] * y[j];
            }
            const float mean = team_sum<WARP>(make_float3(q, 0.0f, 0.0f), red, turn).x * over;
#pragma unroll
            for (int j = 0; j < EPT; ++j) d[j] = i1 * (d[j] - y[j] * mean);
        } else {
#pragma unroll
            for (int j = 0; j < EPT; ++j) {
                d[j] *= a.branch;
                sg[j] += d[j] * y[j];
                d[j] *= g[j];
            }
        }
        st_cols<EPT, FOUR>(static_cast<T*>(a.d_y) + r * cols, team, tid, cols, d);
        if (a.d_gate) {
            const int64_t first = group * a.gate_rows, end = min(first + a.gate_rows, a.rows);
            if (r + 1 == end || r + 1 == r1) {
                if (first >= r0 && end <= r1) put_sum<EPT, FOUR>(a.d_gate + group * cols, team, tid, cols, sg, a.accumulate);
                else st_cols<EPT, FOUR>(a.part_g + (2 * s + (first < r0 ? 0 : 1)) * cols, team, tid, cols, sg);
#pragma unroll
                for (int j = 0; j < EPT; ++j) sg[j] = 0.0f;
            }
        }
    }
    // the CTA's sums of the gains
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        if (which == 0 ? !a.d_w_pre : !a.d_w_post) continue;
        float* out = a.part_w + (2 * (int64_t)blockIdx.x + which) * cols;
        if constexpr (WARP) {
            __syncthreads();
#pragma unroll
            for (int j = 0; j < EPT; ++j) {
                const int c = col_of<FOUR>(j, team, tid);
                warp_part[(threadIdx.x >> 5) * 32 * EPT + c] = which == 0 ? sw_pre[j] : sw_post[j];
            }
            __syncthreads();
            for (int c = threadIdx.x; c < cols; c += 256) {
                float v = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) v += warp_part[i * 32 * EPT + c];
                out[c] = v;
            }
        } else if (which == 0) st_cols<EPT, FOUR>(out, team, tid, cols, sw_pre);
        else st_cols<EPT, FOUR>(out, team, tid, cols, sw_post);
    }
}

// Adds what the strips left: blockIdx.y = 0, 1 the gains over all CTAs; behind them a gate's groups that reach over several strips.
// 32 columns a block, blockDim.y lanes a column, each every blockDim.y-th part.
__global__ void __launch_bounds__(1024) join_sums_kernel(const Join a, int ctas) {
    __shared__ float sh[32][33];
    const int c = blockIdx.x * 32 + threadIdx.x, y = threadIdx.y, cols = a.cols;
    float* out;
    float v = 0.0f;
    if (blockIdx.y < 2) {
        out = blockIdx.y == 0 ? a.d_w_pre : a.d_w_post;
        if (!out) return;
        if (c < cols) {
#pragma unroll 8
            for (int i = y; i < ctas; i += blockDim.y) v += a.part_w[(2 * (int64_t)i + blockIdx.y) * cols + c];
        }
    } else {
        const int64_t group = blockIdx.y - 2, first = group * a.gate_rows, end = min(first + a.gate_rows, a.rows);
        const int64_t s0 = first / a.strip, s1 = (end - 1) / a.strip;
        if (s0 == s1) return;   // (written by the strip)
        out = a.d_gate + group * cols;
        if (c < cols) {
            // a group that begins where its first strip does is that strip's sum to the right as well
#pragma unroll 8
            for (int64_t i = s0 + y; i <= s1; i += blockDim.y) v += a.part_g[(2 * i + (i == s0 ? 1 : 0)) * cols + c];
        }
    }
    sh[y][threadIdx.x] = v;
    __syncthreads();
    if (y == 0 && c < cols) {
        float t = 0.0f;
        for (int i = 0; i < (int)blockDim.y; ++i) t += sh[i][threadIdx.x];
        out[c] = a.accumulate ? out[c] + t : t;
    }
}

// Threads of a team: 32 = warp teams (eight a CTA).
inline int team_threads(int64_t cols) { return cols <= 256 ? 32 : (int)ceil_div64(cols, 256) * 32; }

struct Strips {
    int64_t strip, strips, ctas;
    // gate_rows 0: the most strips that any gate_rows gives
    Strips(const asca_ctx* ctx, int64_t rows, int64_t cols, int64_t gate_rows) {
        const int team = team_threads(cols);
        const int64_t teams = team == 32 ? (int64_t)ctx->sm_count * 16 : (int64_t)ctx->sm_count * std::max(1, 1024 / team);
        strip = std::max<int64_t>(team == 32 ? 4 : 1, ceil_div64(rows, teams));
        if (gate_rows > 0 && gate_rows <= 2 * strip) strip = ceil_div64(strip, gate_rows) * gate_rows;
        strips = ceil_div64(rows, strip);
        ctas = team == 32 ? ceil_div64(strips, 8) : strips;
    }
    size_t part_w(int64_t cols) const { return ((size_t)ctas * 2 * cols * 4 + 255) & ~(size_t)255; }
    size_t part_g(int64_t cols) const { return (size_t)strips * 2 * cols * 4; }
};

int check(asca_ctx* ctx, const char* who, const Join& a, int64_t cols, int dtype) {
    ASCA_REQUIRE(ctx, a.rows >= 0 && cols > 0, "%s: bad shape", who);
    if (cols > MAX_COLS) return asca_fail(ctx, ASCA_ERR_UNSUPPORTED, "%s: at most %d columns", who, MAX_COLS);
    ASCA_REQUIRE(ctx, a.rows < ((int64_t)1 << 31), "%s: at most 2^31 - 1 rows", who);
    ASCA_REQUIRE(ctx, asca_known_dtype(dtype), "%s: unknown dtype", who);
    ASCA_REQUIRE(ctx, a.gate_rows > 0 || (!a.gate && !a.d_gate), "%s: a gate needs gate_rows", who);
    ASCA_REQUIRE(ctx, a.post || (!a.w_post && !a.d_w_post), "%s: w_post without the norm after the block", who);
    return ASCA_OK;
}

// MOST: threads of a CTA at most, which is what bounds its registers
template <template <typename, int, bool, bool, int> class K>
void launch(const asca_ctx* ctx, const Join& a, int dtype, bool four, int64_t units) {
    const int team = team_threads(a.cols);
    auto with = [&](auto t) {
        using T = decltype(t);
        const dim3 warps((unsigned)ceil_div64(units, 8)), ctas((unsigned)units);
        if (team == 32 && a.cols <= 128) {
            if (four) K<T, 4, true, true, 256>::go(warps, 256, ctx->stream, a);
            else K<T, 4, false, true, 256>::go(warps, 256, ctx->stream, a);
        } else if (team == 32) {
            if (four) K<T, 8, true, true, 256>::go(warps, 256, ctx->stream, a);
            else K<T, 8, false, true, 256>::go(warps, 256, ctx->stream, a);
        } else if (team <= 256) {
            if (four) K<T, 8, true, false, 256>::go(ctas, team, ctx->stream, a);
            else K<T, 8, false, false, 256>::go(ctas, team, ctx->stream, a);
        } else if (four) K<T, 8, true, false, 1024>::go(ctas, team, ctx->stream, a);
        else K<T, 8, false, false, 1024>::go(ctas, team, ctx->stream, a);
    };
    if (dtype == ASCA_BF16) with(__nv_bfloat16());
    else with(0.0f);
}
template <typename T, int EPT, bool FOUR, bool WARP, int MOST>
struct Fwd {
    static void go(dim3 grid, int threads, cudaStream_t s, const Join& a) { join_fwd_kernel<T, EPT, FOUR, WARP, MOST><<<grid, threads, 0, s>>>(a); }
};
template <typename T, int EPT, bool FOUR, bool WARP, int MOST>
struct Bwd {
    static void go(dim3 grid, int threads, cudaStream_t s, const Join& a) { join_bwd_kernel<T, EPT, FOUR, WARP, MOST><<<grid, threads, 0, s>>>(a); }
};

}  // namespace

extern "C" {

int asca_gated_residual_rmsnorm_fwd(asca_ctx* ctx, const void* y, const float* x, const float* w_post, const float* gate, int64_t gate_rows,
                                    const float* w_pre, int post_norm, float skip_scale, float branch_scale, float eps, int64_t rows, int64_t cols,
                                    int dtype, float* x_out, void* xn) {
    if (!ctx) return ASCA_ERR_ARG;
    Join a{};
    a.y = y; a.x = x; a.w_post = w_post; a.gate = gate; a.gate_rows = gate_rows; a.w_pre = w_pre; a.post = post_norm != 0;
    a.skip = skip_scale; a.branch = branch_scale; a.eps = eps; a.rows = rows; a.cols = (int)cols; a.x_out = x_out; a.xn = xn;
    ASCA_TRY(check(ctx, "gated_residual_rmsnorm_fwd", a, cols, dtype));
    if (rows == 0) return ASCA_OK;
    ASCA_REQUIRE(ctx, y && x && x_out, "gated_residual_rmsnorm_fwd: null pointer");
    asca_device_scope on(ctx);
    const bool four = asca_rows_by_four(y, cols, dtype) && asca_rows_by_four(xn, cols, dtype) && asca_aligned(x, 16) && asca_aligned(x_out, 16) &&
                      asca_aligned(w_post, 16) && asca_aligned(gate, 16) && asca_aligned(w_pre, 16);
    launch<Fwd>(ctx, a, dtype, four, rows);
    ASCA_CHECK_LAUNCH(ctx);
    return ASCA_OK;
}

int64_t asca_gated_residual_rmsnorm_bwd_ws(asca_ctx* ctx, int64_t rows, int64_t cols) {
    if (!ctx || rows < 0 || cols <= 0 || cols > MAX_COLS) return ASCA_ERR_ARG;
    const Strips s(ctx, rows, cols, 0);
    return (int64_t)(s.part_w(cols) + s.part_g(cols) + 256);
}

int asca_gated_residual_rmsnorm_bwd(asca_ctx* ctx, const void* y, const float* x_out, const void* d_xn, const float* d_out, const float* w_post,
                                    const float* gate, int64_t gate_rows, const float* w_pre, int post_norm, float skip_scale, float branch_scale,
                                    float eps, int64_t rows, int64_t cols, int dtype, int accumulate, float* d_x, void* d_y, float* d_w_post,
                                    float* d_gate, float* d_w_pre, void* ws, size_t ws_bytes) {
    if (!ctx) return ASCA_ERR_ARG;
    Join a{};
    a.y = y; a.x_out = const_cast<float*>(x_out); a.d_xn = d_xn; a.d_out = d_out; a.w_post = w_post; a.gate = gate;
    a.gate_rows = gate_rows > 0 ? gate_rows : (gate || d_gate ? 0 : 1);
    a.w_pre = w_pre; a.post = post_norm != 0; a.skip = skip_scale; a.branch = branch_scale; a.eps = eps; a.rows = rows; a.cols = (int)cols;
    a.accumulate = accumulate; a.d_x = d_x; a.d_y = d_y; a.d_w_post = d_w_post; a.d_gate = d_gate; a.d_w_pre = d_w_pre;
    const char* who = "gated_residual_rmsnorm_bwd";
    ASCA_TRY(check(ctx, who, a, cols, dtype));
    ASCA_REQUIRE(ctx, d_xn || d_out || rows == 0, "%s: needs d_xn or d_out", who);
    asca_device_scope on(ctx);
    if (rows == 0) {   // (no rows: the sums are zero)
        if (!accumulate)
            for (float* p : {d_w_post, d_w_pre})
                if (p) ASCA_CUDA(ctx, cudaMemsetAsync(p, 0, (size_t)cols * 4, ctx->stream));
        return ASCA_OK;
    }
    ASCA_REQUIRE(ctx, y && x_out && d_x && d_y && ws, "%s: null pointer", who);
    const Strips s(ctx, rows, cols, d_gate ? a.gate_rows : 0);
    ASCA_REQUIRE(ctx, asca_aligned(ws, 256) && ws_bytes >= (size_t)asca_gated_residual_rmsnorm_bwd_ws(ctx, rows, cols),
                 "%s: the workspace has to have asca_gated_residual_rmsnorm_bwd_ws bytes, 256-byte aligned", who);
    a.strip = s.strip;
    a.strips = s.strips;
    a.part_w = (float*)ws;
    a.part_g = (float*)((char*)ws + s.part_w(cols));
    const bool four = asca_rows_by_four(y, cols, dtype) && asca_rows_by_four(d_xn, cols, dtype) && asca_rows_by_four(d_y, cols, dtype) &&
                      asca_aligned(x_out, 16) && asca_aligned(d_out, 16) && asca_aligned(d_x, 16) && asca_aligned(w_post, 16) &&
                      asca_aligned(gate, 16) && asca_aligned(w_pre, 16) && asca_aligned(d_gate, 16);
    launch<Bwd>(ctx, a, dtype, four, s.strips);
    ASCA_CHECK_LAUNCH(ctx);
    const bool gates = d_gate && a.gate_rows > s.strip;   // (else every group lies in one strip)
    if (d_w_post || d_w_pre || gates) {
        const int64_t groups = gates ? ceil_div64(rows, a.gate_rows) : 0, most = std::max(s.ctas, gates ? a.gate_rows / s.strip : 0);
        const dim3 block(32, most >= 64 ? 32 : 8);
        join_sums_kernel<<<dim3((unsigned)ceil_div64(cols, 32), (unsigned)(2 + groups)), block, 0, ctx->stream>>>(a, (int)s.ctas);
        ASCA_CHECK_LAUNCH(ctx);
    }
    return ASCA_OK;
}

}  // extern "C"

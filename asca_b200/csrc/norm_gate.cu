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
// Backward, the row's six sums are taken at once: with a = branch gate w_post y, the mean of u y r1 is r1 times the mean of
// a d_out + r2 a t + c a x_out, c being what d has of x_out, so that the second mean needs no second round through the team
// (its three parts are as large as what a gradient's rounding is measured by: |d_out| + r2 (|t| + |x_out r2| mean|t x_out r2|)).
// And inside a group of rows with one gate, d_gate and the group's share of d_w_post are both S = sum of d y r1 times constants.
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
constexpr int EPT = 8;   // columns a thread

// Columns of thread `tid` of a team of `team`: groups of four, `team` groups apart, or single columns `team` apart.
template <bool FOUR>
__device__ __forceinline__ int col_of(int j, int team, int tid) { return FOUR ? ((j >> 2) * team + tid) * 4 + (j & 3) : j * team + tid; }

template <bool FOUR, typename T>
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
// a gain or a gate that is not given is ones
template <bool FOUR>
__device__ __forceinline__ void ld_gain(const float* p, int team, int tid, int cols, float (&v)[EPT]) {
    if (p) ld_cols<FOUR>(p, team, tid, cols, v, 1.0f);
    else {
#pragma unroll
        for (int j = 0; j < EPT; ++j) v[j] = 1.0f;
    }
}
template <bool FOUR, typename T>
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

// Sums of N values over a team, the same in all its threads. LANES: the team's part of a warp (8, 16, 32), or 0 for a whole CTA, which
// alternates between two halves of `red` (`turn`), so that one barrier is enough: who writes a half again has passed the barrier of
// the other, behind everybody's reading of this one.
template <int LANES, int N>
__device__ __forceinline__ void team_sum(float (&v)[N], float (*red)[32][8], int& turn) {
    static_assert(N <= 8, "a warp's place holds eight");
#pragma unroll
    for (int o = (LANES ? LANES : 32) / 2; o > 0; o >>= 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
    if constexpr (LANES == 0) {
        float(*r)[8] = red[turn];
        turn ^= 1;
        const int nw = blockDim.x >> 5;
        if ((threadIdx.x & 31) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) r[threadIdx.x >> 5][i] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = 0.0f;
        for (int w = 0; w < nw; ++w) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += r[w][i];
        }
    }
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

template <typename T, bool FOUR, int LANES, int MOST>
__global__ void __launch_bounds__(MOST, 2048 / MOST) join_fwd_kernel(const Join a) {
    __shared__ __align__(16) float red[2][32][8];
    constexpr int TEAMS = LANES ? 256 / (LANES ? LANES : 1) : 1;   // a CTA's
    const int team = LANES ? LANES : blockDim.x, tid = LANES ? threadIdx.x % (LANES ? LANES : 1) : threadIdx.x;
    const int64_t r0 = LANES ? (int64_t)blockIdx.x * TEAMS + threadIdx.x / (LANES ? LANES : 1) : blockIdx.x;
    const bool live = r0 < a.rows;
    const int64_t r = live ? r0 : a.rows - 1;   // (a warp's shuffles stay whole)
    int turn = 0;
    const int cols = a.cols;
    float y[EPT], x[EPT], w[EPT];
    ld_cols<FOUR>(static_cast<const T*>(a.y) + r * cols, team, tid, cols, y);
    ld_cols<FOUR>(a.x + r * cols, team, tid, cols, x);
    float s[1] = {0.0f};
    if (a.post) {
#pragma unroll
        for (int j = 0; j < EPT; ++j) s[0] += y[j] * y[j];
        team_sum<LANES>(s, red, turn);
        const float r1 = 1.0f / sqrtf(s[0] / (float)cols + a.eps);
        ld_gain<FOUR>(a.w_post, team, tid, cols, w);
#pragma unroll
        for (int j = 0; j < EPT; ++j) y[j] = y[j] * r1 * w[j];
    }
    if (a.gate) {
        ld_cols<FOUR>(a.gate + r / a.gate_rows * cols, team, tid, cols, w);
#pragma unroll
        for (int j = 0; j < EPT; ++j) y[j] *= w[j];
    }
    s[0] = 0.0f;
#pragma unroll
    for (int j = 0; j < EPT; ++j) {
        x[j] = a.skip * x[j] + a.branch * y[j];
        s[0] += x[j] * x[j];
    }
    if (live) st_cols<FOUR>(a.x_out + r * cols, team, tid, cols, x);
    if (!a.xn) return;
    team_sum<LANES>(s, red, turn);
    const float r2 = 1.0f / sqrtf(s[0] / (float)cols + a.eps);
    ld_gain<FOUR>(a.w_pre, team, tid, cols, w);
#pragma unroll
    for (int j = 0; j < EPT; ++j) x[j] = x[j] * r2 * w[j];
    if (live) st_cols<FOUR>(static_cast<T*>(a.xn) + r * cols, team, tid, cols, x);
}

template <bool FOUR>
__device__ __forceinline__ void put_sum(float* p, int team, int tid, int cols, float (&v)[EPT], int accumulate) {
    if (accumulate) {
        float o[EPT];
        ld_cols<FOUR>(p, team, tid, cols, o);
#pragma unroll
        for (int j = 0; j < EPT; ++j) v[j] += o[j];
    }
    st_cols<FOUR>(p, team, tid, cols, v);
}

// Rows ahead. A thread copies the columns that it will itself read (no barrier), asynchronously into its places in shared memory:
// [stage][EPT columns][thread], a place of 16 bytes for four f32, 8 for four bf16, 4 for one f32. Single bf16 columns, which are too
// small for such a copy, are read straight when their row's turn comes.
// STAGES: rows in flight and in work, 0: every row is read straight.
template <bool FOUR, int STAGES, typename T>
constexpr bool ahead() { return STAGES > 0 && (FOUR || sizeof(T) == 4); }
template <int BYTES>
__device__ __forceinline__ void copy_ahead(void* dst, const void* src) {
    const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(d), "l"(src), "n"(BYTES) : "memory");
}
template <bool FOUR, int STAGES, typename T>
__device__ __forceinline__ void ask_row(T* place, const T* row, int team, int tid, int cols) {
    if constexpr (ahead<FOUR, STAGES, T>()) {
        constexpr int V = FOUR ? 4 : 1;
#pragma unroll
        for (int q = 0; q < EPT / V; ++q) {
            const int c = (q * team + tid) * V;
            if (c < cols) copy_ahead<V * sizeof(T)>(place + ((size_t)q * blockDim.x + threadIdx.x) * V, row + c);
        }
    }
}
template <bool FOUR, int STAGES, typename T>
__device__ __forceinline__ void take_row(const T* place, const T* row, int team, int tid, int cols, float (&v)[EPT]) {
    if constexpr (ahead<FOUR, STAGES, T>()) {
        constexpr int V = FOUR ? 4 : 1;
#pragma unroll
        for (int q = 0; q < EPT / V; ++q) {
            float t[V];
            ld_row<V>(place + ((size_t)q * blockDim.x + threadIdx.x) * V, t);
            const bool in = (q * team + tid) * V < cols;
#pragma unroll
            for (int i = 0; i < V; ++i) v[q * V + i] = in ? t[i] : 0.0f;
        }
    } else ld_cols<FOUR>(row, team, tid, cols, v);
}

template <typename T>
constexpr size_t stage_bytes(int threads) { return (size_t)threads * EPT * (8 + 2 * sizeof(T)); }

template <typename T, bool FOUR, int LANES, int MOST, int STAGES>
__global__ void __launch_bounds__(MOST, MOST <= 256 ? 2 : 1) join_bwd_kernel(const Join a) {
    extern __shared__ __align__(16) char smem[];
    pdl_launch_dependents();
    __shared__ __align__(16) float red[2][32][8];
    constexpr int L = LANES ? LANES : 1, TEAMS = LANES ? 256 / L : 1;
    const int team = LANES ? LANES : blockDim.x, tid = LANES ? threadIdx.x % L : threadIdx.x, cols = a.cols;
    const int64_t s = (int64_t)blockIdx.x * TEAMS + (LANES ? threadIdx.x / L : 0);   // the strip
    const int64_t r0 = min(s * a.strip, a.rows), r1 = min(r0 + a.strip, a.rows);
    const int n = (int)(r1 - r0);
    int turn = 0;
    const float over = 1.0f / (float)cols;
    const int per = blockDim.x * EPT;   // elements of one matrix in a stage
    auto place = [&](int i) { return smem + (size_t)(STAGES > 0 ? i % (STAGES > 0 ? STAGES : 1) : 0) * stage_bytes<T>(blockDim.x); };
    auto ask = [&](int i) {
        if (i < n) {
            char* p = place(i);
            const int64_t at = (r0 + i) * cols;
            ask_row<FOUR, STAGES>(reinterpret_cast<float*>(p), a.x_out + at, team, tid, cols);
            if (a.d_out) ask_row<FOUR, STAGES>(reinterpret_cast<float*>(p) + per, a.d_out + at, team, tid, cols);
            T* t = reinterpret_cast<T*>(p + (size_t)per * 8);
            ask_row<FOUR, STAGES>(t, static_cast<const T*>(a.y) + at, team, tid, cols);
            if (a.d_xn) ask_row<FOUR, STAGES>(t + per, static_cast<const T*>(a.d_xn) + at, team, tid, cols);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) ask(i);
    float w_pre[EPT], u[EPT], sw_pre[EPT] = {}, sw_post[EPT] = {}, sum_g[EPT] = {};
    ld_gain<FOUR>(a.w_pre, team, tid, cols, w_pre);
    int64_t group = r0 / a.gate_rows, first = group * a.gate_rows, end = first + min(a.gate_rows, a.rows - first);
    auto load_u = [&]() {   // branch gate w_post
        float w[EPT];
        ld_gain<FOUR>(a.w_post, team, tid, cols, w);
        ld_gain<FOUR>(a.gate && n > 0 ? a.gate + group * cols : nullptr, team, tid, cols, u);
#pragma unroll
        for (int j = 0; j < EPT; ++j) u[j] = a.branch * u[j] * w[j];
    };
    load_u();
    // (teams that share a warp take the same number of turns)
    for (int i = 0; i < (LANES ? (int)a.strip : n); ++i) {
        const bool live = LANES == 0 || i < n;
        const int64_t r = r0 + i, at = (live ? r : 0) * cols;
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES > 2 ? STAGES - 2 : 0) : "memory");
        float y[EPT], xo[EPT], dn[EPT], d[EPT];
        {
            const char* p = place(i);
            take_row<FOUR, STAGES>(reinterpret_cast<const float*>(p), a.x_out + at, team, tid, cols, xo);
            const T* t = reinterpret_cast<const T*>(p + (size_t)per * 8);
            take_row<FOUR, STAGES>(t, static_cast<const T*>(a.y) + at, team, tid, cols, y);
            if (a.d_out) take_row<FOUR, STAGES>(reinterpret_cast<const float*>(p) + per, a.d_out + at, team, tid, cols, d);
            if (a.d_xn) take_row<FOUR, STAGES>(t + per, static_cast<const T*>(a.d_xn) + at, team, tid, cols, dn);
        }
        if (STAGES > 0) ask(i + STAGES - 1);   // into the places of the row before
        float sum[6] = {};
#pragma unroll
        for (int j = 0; j < EPT; ++j) {
            if (!a.d_out) d[j] = 0.0f;
            if (!a.d_xn) dn[j] = 0.0f;
            const float t = dn[j] * w_pre[j], v = u[j] * y[j];
            sum[0] = fmaf(y[j], y[j], sum[0]);
            sum[1] = fmaf(xo[j], xo[j], sum[1]);
            sum[2] = fmaf(t, xo[j], sum[2]);
            sum[3] = fmaf(v, d[j], sum[3]);
            sum[4] = fmaf(v, t, sum[4]);
            sum[5] = fmaf(v, xo[j], sum[5]);
        }
        team_sum<LANES>(sum, red, turn);
        // d = d_out + i2 t + c2 x_out; d_y = i1 u d + c1 y
        const float i2 = 1.0f / sqrtf(sum[1] * over + a.eps), c2 = -i2 * (i2 * (sum[2] * i2 * over));
        const float i1 = a.post ? 1.0f / sqrtf(sum[0] * over + a.eps) : 1.0f;
        const float c1 = a.post ? -i1 * (i1 * (i1 * over * (sum[3] + i2 * sum[4] + c2 * sum[5]))) : 0.0f;
        float dx[EPT];
#pragma unroll
        for (int j = 0; j < EPT; ++j) {
            if (live) sw_pre[j] = fmaf(dn[j] * xo[j], i2, sw_pre[j]);
            d[j] = fmaf(i2, dn[j] * w_pre[j], fmaf(c2, xo[j], d[j]));
            dx[j] = a.skip * d[j];
            if (live) sum_g[j] = fmaf(d[j] * y[j], i1, sum_g[j]);
            y[j] = fmaf(c1, y[j], i1 * (u[j] * d[j]));
        }
        if (!live) continue;
        st_cols<FOUR>(a.d_x + at, team, tid, cols, dx);
        st_cols<FOUR>(static_cast<T*>(a.d_y) + at, team, tid, cols, y);
        if (r + 1 == end || r + 1 == r1) {   // the last row of the gate's group, or of the strip
            float w[EPT];
            if (a.d_w_post) {
                ld_gain<FOUR>(a.gate ? a.gate + group * cols : nullptr, team, tid, cols, w);
#pragma unroll
                for (int j = 0; j < EPT; ++j) sw_post[j] = fmaf(a.branch * w[j], sum_g[j], sw_post[j]);
            }
            if (a.d_gate) {
                ld_gain<FOUR>(a.w_post, team, tid, cols, w);
#pragma unroll
                for (int j = 0; j < EPT; ++j) w[j] *= a.branch * sum_g[j];
                if (first >= r0 && end <= r1) put_sum<FOUR>(a.d_gate + group * cols, team, tid, cols, w, a.accumulate);
                else st_cols<FOUR>(a.part_g + (2 * s + (first < r0 ? 0 : 1)) * cols, team, tid, cols, w);
            }
#pragma unroll
            for (int j = 0; j < EPT; ++j) sum_g[j] = 0.0f;
            if (r + 1 < r1) {
                ++group;
                first = end;
                end = first + min(a.gate_rows, a.rows - first);
                if (a.gate) load_u();
            }
        }
    }
    // the CTA's sums of the gains
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        if (which == 0 ? !a.d_w_pre : !a.d_w_post) continue;
        float* out = a.part_w + (2 * (int64_t)blockIdx.x + which) * cols;
        if constexpr (LANES != 0) {
            float* part = reinterpret_cast<float*>(smem);   // [team][columns]: no more than a stage
            constexpr int WIDE = L * EPT;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < EPT; ++j) part[threadIdx.x / L * WIDE + col_of<FOUR>(j, team, tid)] = which == 0 ? sw_pre[j] : sw_post[j];
            __syncthreads();
            for (int c = threadIdx.x; c < cols; c += 256) {
                float v = 0.0f;
#pragma unroll
                for (int i = 0; i < TEAMS; ++i) v += part[i * WIDE + c];
                out[c] = v;
            }
        } else if (which == 0) st_cols<FOUR>(out, team, tid, cols, sw_pre);
        else st_cols<FOUR>(out, team, tid, cols, sw_post);
    }
}

// Adds what the strips left: blockIdx.y = 0, 1 the gains over all CTAs; behind them a gate's groups that reach over several strips.
// 32 columns a block, blockDim.y lanes a column, each every blockDim.y-th part.
__global__ void __launch_bounds__(1024) join_sums_kernel(const Join a, int ctas) {
    __shared__ float sh[32][33];
    pdl_wait();
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

// Lanes of a warp that make a team (0: a team is a CTA), and the team's threads.
inline int team_lanes(int64_t cols) { return cols <= 64 ? 8 : cols <= 128 ? 16 : cols <= 256 ? 32 : 0; }
inline int team_threads(int64_t cols) { return team_lanes(cols) ? team_lanes(cols) : (int)ceil_div64(cols, 32 * EPT) * 32; }

struct Strips {
    int64_t strip, strips, ctas;
    // gate_rows 0: the most strips that any gate_rows gives
    Strips(const asca_ctx* ctx, int64_t rows, int64_t cols, int64_t gate_rows) {
        const int team = team_threads(cols);
        const int64_t teams = (int64_t)ctx->sm_count * std::max(1, 512 / team);   // what is resident at once: 128 registers a thread
        strip = std::max<int64_t>(1, ceil_div64(rows, teams));
        if (gate_rows > 0 && gate_rows <= 2 * strip) strip = ceil_div64(strip, gate_rows) * gate_rows;
        strips = ceil_div64(rows, strip);
        ctas = team_lanes(cols) ? ceil_div64(strips, 256 / team) : strips;
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
template <template <typename, bool, int, int> class K>
int launch(asca_ctx* ctx, const Join& a, int dtype, bool four, int64_t teams) {
    const int lanes = team_lanes(a.cols), threads = lanes ? 256 : team_threads(a.cols);
    const dim3 grid((unsigned)(lanes ? ceil_div64(teams, 256 / lanes) : teams));
    cudaError_t e = cudaSuccess;
    auto with = [&](auto t, auto f) {
        using T = decltype(t);
        constexpr bool FOUR = decltype(f)::value;
        if (lanes == 8) e = K<T, FOUR, 8, 256>::go(grid, threads, ctx->stream, a);
        else if (lanes == 16) e = K<T, FOUR, 16, 256>::go(grid, threads, ctx->stream, a);
        else if (lanes == 32) e = K<T, FOUR, 32, 256>::go(grid, threads, ctx->stream, a);
        else if (threads <= 256) e = K<T, FOUR, 0, 256>::go(grid, threads, ctx->stream, a);
        else if (threads <= 512) e = K<T, FOUR, 0, 512>::go(grid, threads, ctx->stream, a);
        else e = K<T, FOUR, 0, 1024>::go(grid, threads, ctx->stream, a);
    };
    auto typed = [&](auto t) {
        if (four) with(t, std::true_type());
        else with(t, std::false_type());
    };
    if (dtype == ASCA_BF16) typed(__nv_bfloat16());
    else typed(0.0f);
    ASCA_CUDA(ctx, e);
    ASCA_CHECK_LAUNCH(ctx);
    return ASCA_OK;
}
template <typename T, bool FOUR, int LANES, int MOST>
struct Fwd {
    static cudaError_t go(dim3 grid, int threads, cudaStream_t s, const Join& a) {
        join_fwd_kernel<T, FOUR, LANES, MOST><<<grid, threads, 0, s>>>(a);
        return cudaSuccess;
    }
};
template <typename T, bool FOUR, int LANES, int MOST>
struct Bwd {
    static cudaError_t go(dim3 grid, int threads, cudaStream_t s, const Join& a) {
        // three rows' places fit twice into an SM up to 256 threads and once up to 512; above that two of bf16, none of f32
        constexpr int STAGES = MOST <= 512 ? 3 : sizeof(T) == 2 ? 2 : 0;
        auto kern = join_bwd_kernel<T, FOUR, LANES, MOST, STAGES>;
        const size_t smem = STAGES * stage_bytes<T>(threads);
        const cudaError_t e = smem > 40 * 1024 ? cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) : cudaSuccess;
        if (e == cudaSuccess) kern<<<grid, threads, smem, s>>>(a);
        return e;
    }
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
    const bool four = asca_rows_by(4, y, cols, dtype) && asca_rows_by(4, xn, cols, dtype) && asca_aligned(x, 16) && asca_aligned(x_out, 16) &&
                      asca_aligned(w_post, 16) && asca_aligned(gate, 16) && asca_aligned(w_pre, 16);
    return launch<Fwd>(ctx, a, dtype, four, rows);
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
    const bool four = asca_rows_by(4, y, cols, dtype) && asca_rows_by(4, d_xn, cols, dtype) && asca_rows_by(4, d_y, cols, dtype) &&
                      asca_aligned(x_out, 16) && asca_aligned(d_out, 16) && asca_aligned(d_x, 16) && asca_aligned(w_post, 16) &&
                      asca_aligned(gate, 16) && asca_aligned(w_pre, 16) && asca_aligned(d_gate, 16);
    ASCA_TRY(launch<Bwd>(ctx, a, dtype, four, s.strips));
    const bool gates = d_gate && a.gate_rows > s.strip;   // (else every group lies in one strip)
    if (d_w_post || d_w_pre || gates) {
        const int64_t groups = gates ? ceil_div64(rows, a.gate_rows) : 0, most = std::max(s.ctas, gates ? a.gate_rows / s.strip : 0);
        const dim3 block(32, most >= 64 ? 32 : 8);
        ASCA_CUDA(ctx, asca_launch_after(ctx, join_sums_kernel, dim3((unsigned)ceil_div64(cols, 32), (unsigned)(2 + groups)), block, 0, a, (int)s.ctas));
        ctx->launches++;
    }
    return ASCA_OK;
}

}  // extern "C"

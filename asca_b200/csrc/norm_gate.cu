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
// A row belongs to a team: lanes of a warp up to 256 columns, else a CTA with eight columns a thread (backward, above 4096 columns, the
// two CTAs of a cluster, because the column sums take 128 registers a thread); the row stays in registers between its two reductions,
// so every matrix passes HBM once, which is what bounds both directions: 32,768 x 2048 with bf16 y 120 us forward (6.7 TB/s), 196
// backward (6.2 TB/s), 157 and 285 with a gate a row. Rows of 64 columns take the backward pass 64 us for 200,000 (3.6 TB/s: a
// reduction for every 64 columns), rows of 8192 180 us for 4096 (3.4 TB/s; 188 with f32 y, 4.3 TB/s: the cluster's barrier waits for the
// row's stores; a CTA of 1024 threads, with half of the registers, takes 212 with bf16 y). The statistics are taken again in the
// backward pass, whose rows are in registers anyway: nothing is kept for it.
//
// Backward, a team owns a strip of consecutive rows and the same columns in all of them, so that the column sums stay in its
// registers; a strip's sums of the gains go out once, a gate's once for every group of rows in the strip, and a second launch adds
// the strips in a fixed order. A group of rows up to two strips long gets strips that end where groups end: its gate's gradient is
// then written at once. That pays where the strips become little longer by it and costs where they leave CTAs without one: 32,768 x 2048
// bf16, strips of 111 rows, one gate for all 194 us; groups of 112 rows 194 (210 with the strips as they are), of 128 219 (207), of 200
// 334 (203), of 222 277 (200), of 300, beyond the rule, 200.
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

// Two columns at a time: half the instructions of the element-wise work, which is what the backward pass waits for next after HBM.
using pair_t = unsigned long long;
__device__ __forceinline__ pair_t pair(float a, float b) {
    pair_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ pair_t pair(float a) { return pair(a, a); }
__device__ __forceinline__ float2 two(pair_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ pair_t mul2(pair_t a, pair_t b) {
    pair_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ pair_t fma2(pair_t a, pair_t b, pair_t c) {
    pair_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// Sums over a team, the same in all its threads. LANES: the team's part of a warp (8, 16, 32), or 0 for a whole CTA, which alternates
// between two halves of `red` (`turn`), so that one barrier is enough: who writes a half again has passed the barrier of the other,
// behind everybody's reading of this one.
template <int LANES>
__device__ __forceinline__ float team_sum(float v, float (*red)[32], int& turn) {
#pragma unroll
    for (int o = (LANES ? LANES : 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (LANES == 0) {
        float* r = red[turn];
        turn ^= 1;
        const int lane = threadIdx.x & 31;
        if (lane == 0) r[threadIdx.x >> 5] = v;
        __syncthreads();
        v = lane < (int)(blockDim.x >> 5) ? r[lane] : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    return v;
}
// Six sums. The first three steps halve what a lane has (it keeps the sums that three bits of its number name), so that six sums take
// 7 shuffles and more where one takes 5; the way back to all lanes is one shuffle a sum. PAIR: the team is the two CTAs of a cluster, each
// of which gets the other's warps' sums too, and the barrier is the cluster's.
template <int LANES, bool PAIR>
__device__ __forceinline__ void team_sums(float (&v)[6], float (*red)[32][8], int& turn) {
    constexpr int L = LANES ? LANES : 32;
    const int lane = threadIdx.x & 31;
    float a[4], b[2], c;
    const bool hi = lane & (L / 2), mid = lane & (L / 4), low = lane & (L / 8);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float high = i + 4 < 6 ? v[(i + 4) % 6] : 0.0f;   // (v[6], v[7] are not there)
        const float got = __shfl_xor_sync(0xffffffffu, hi ? v[i] : high, L / 2);
        a[i] = (hi ? high : v[i]) + got;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) b[i] = (mid ? a[i + 2] : a[i]) + __shfl_xor_sync(0xffffffffu, mid ? a[i] : a[i + 2], L / 4);
    c = (low ? b[1] : b[0]) + __shfl_xor_sync(0xffffffffu, low ? b[0] : b[1], L / 8);
#pragma unroll
    for (int o = L / 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
    if constexpr (LANES == 0) {
        // every warp adds the warps' sums: lane l those of its pair l % 4 and of every eighth warp from l / 4 on
        float(*r)[8] = red[turn];
        turn ^= 1;
        int warps = blockDim.x >> 5, w0 = threadIdx.x >> 5;
        if (PAIR) {
            const uint32_t me = blockIdx.x & 1;
            w0 += me * warps;
            warps *= 2;
            if ((lane & 3) == 0) {
                float* to = &r[w0][lane >> 2];
                uint32_t there;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"((uint32_t)__cvta_generic_to_shared(to)), "r"(me ^ 1u));
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(there), "f"(c) : "memory");
                *to = c;
            }
            asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        } else {
            if ((lane & 3) == 0) r[w0][lane >> 2] = c;
            __syncthreads();
        }
        float2 s = make_float2(0.0f, 0.0f);
        for (int w = lane >> 2; w < warps; w += 8) {
            const float2 x = *reinterpret_cast<const float2*>(&r[w][(lane & 3) * 2]);
            s.x += x.x; s.y += x.y;
        }
#pragma unroll
        for (int o = 16; o >= 4; o >>= 1) {
            s.x += __shfl_xor_sync(0xffffffffu, s.x, o);
            s.y += __shfl_xor_sync(0xffffffffu, s.y, o);
        }
#pragma unroll
        for (int i = 0; i < 6; ++i) v[i] = __shfl_sync(0xffffffffu, i & 1 ? s.y : s.x, i >> 1);
    } else {
#pragma unroll
        for (int i = 0; i < 6; ++i) v[i] = __shfl_sync(0xffffffffu, c, (i >> 2 & 1) * (L / 2) + (i >> 1 & 1) * (L / 4) + (i & 1) * (L / 8), L);
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
    __shared__ float red[2][32];
    constexpr int TEAMS = LANES ? 256 / (LANES ? LANES : 1) : 1;   // a CTA's
    const int team = LANES ? LANES : blockDim.x, tid = LANES ? threadIdx.x % (LANES ? LANES : 1) : threadIdx.x;
    const int64_t r0 = LANES ? (int64_t)blockIdx.x * TEAMS + threadIdx.x / (LANES ? LANES : 1) : blockIdx.x;
    const bool live = LANES == 0 || r0 < a.rows;
    const int64_t r = live ? r0 : 0;
    int turn = 0;
    const int cols = a.cols, there = live ? cols : 0;   // (a team without a row reads none, which may be written over, and shuffles with its warp)
    float y[EPT], x[EPT], w[EPT];
    ld_cols<FOUR>(static_cast<const T*>(a.y) + r * cols, team, tid, there, y);
    ld_cols<FOUR>(a.x + r * cols, team, tid, there, x);
    const float over = 1.0f / (float)cols;
    float s = 0.0f;
    if (a.post) {
#pragma unroll
        for (int j = 0; j < EPT; ++j) s += y[j] * y[j];
        const float r1 = rsqrtf(team_sum<LANES>(s, red, turn) * over + a.eps);
        ld_gain<FOUR>(a.w_post, team, tid, cols, w);
#pragma unroll
        for (int j = 0; j < EPT; ++j) y[j] = y[j] * r1 * w[j];
    }
    if (a.gate) {
        // (a 32-bit division is soon done, and the gate then asked for between the row's own loads: 124 us for 32,768 x 2048 where this takes 121)
        ld_cols<FOUR>(a.gate + r / a.gate_rows * cols, team, tid, cols, w);
#pragma unroll
        for (int j = 0; j < EPT; ++j) y[j] *= w[j];
    }
    s = 0.0f;
#pragma unroll
    for (int j = 0; j < EPT; ++j) {
        x[j] = a.skip * x[j] + a.branch * y[j];
        s += x[j] * x[j];
    }
    if (live) st_cols<FOUR>(a.x_out + r * cols, team, tid, cols, x);
    if (!a.xn) return;
    const float r2 = rsqrtf(team_sum<LANES>(s, red, turn) * over + a.eps);
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
// STAGES: rows in flight and in work. Three fit twice into an SM up to 256 threads and once up to 512.
constexpr int STAGES = 3;
template <bool FOUR, typename T>
constexpr bool ahead() { return FOUR || sizeof(T) == 4; }
template <int BYTES>
__device__ __forceinline__ void copy_ahead(uint32_t dst, const void* src) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
// place: of this thread's first columns; row: its first columns'
template <bool FOUR, typename T>
__device__ __forceinline__ void ask_row(uint32_t place, const T* row, int team, int left) {
    if constexpr (ahead<FOUR, T>()) {
        constexpr int V = FOUR ? 4 : 1;
#pragma unroll
        for (int q = 0; q < EPT / V; ++q)
            if (q * team * V < left) copy_ahead<V * sizeof(T)>(place + q * blockDim.x * (uint32_t)(V * sizeof(T)), row + q * team * V);
    }
}
template <bool FOUR, typename T>
__device__ __forceinline__ void take_row(const T* place, const T* row, int team, int left, float (&v)[EPT]) {
    constexpr int V = FOUR ? 4 : 1;
#pragma unroll
    for (int q = 0; q < EPT / V; ++q) {
        float t[V] = {};
        if (q * team * V < left) ld_row<V>(ahead<FOUR, T>() ? place + q * blockDim.x * V : row + q * team * V, t);
#pragma unroll
        for (int i = 0; i < V; ++i) v[q * V + i] = t[i];
    }
}

template <typename T>
constexpr size_t stage_bytes(int threads) { return (size_t)threads * EPT * (8 + 2 * sizeof(T)); }

// EACH: every row has a gate of its own, which is asked for a row ahead. (In the other form that costs a shared gate 9 % of the pass;
// without it a gate a row waits for its gate in every row: 351 us for 32,768 x 2048 where this form took 297 beside it.)
template <typename T, bool FOUR, int LANES, int MOST, bool PAIR, bool EACH>
__global__ void __launch_bounds__(MOST, MOST <= 256 ? 2 : 1) join_bwd_kernel(const Join a) {
    extern __shared__ __align__(16) char smem[];
    // Both CTAs of a pair have started before either writes into the other's shared memory (team_sums): arrived at here, waited for in
    // front of the rows.
    if (PAIR) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    pdl_wait();   // (the context may launch it early)
    pdl_launch_dependents();
    __shared__ __align__(16) float red[2][32][8];
    constexpr int L = LANES ? LANES : 1, TEAMS = LANES ? 256 / L : 1, V = FOUR ? 4 : 1;
    const int team = LANES ? LANES : PAIR ? 2 * blockDim.x : blockDim.x, cols = a.cols;
    const int tid = LANES ? threadIdx.x % L : threadIdx.x + (PAIR ? (blockIdx.x & 1) * blockDim.x : 0);
    const int64_t s = (int64_t)(PAIR ? blockIdx.x >> 1 : blockIdx.x) * TEAMS + (LANES ? threadIdx.x / L : 0);   // the strip
    const int64_t r0 = min(s * a.strip, a.rows), r1 = min(r0 + a.strip, a.rows);
    const int n = (int)(r1 - r0), left = n > 0 ? cols - tid * V : 0;   // columns from this thread's first one on
    int turn = 0;
    const float over = 1.0f / (float)cols;
    // rows ahead: the next row to ask for, and this thread's places, [x_out, d_out in f32; y, d_xn][columns][thread] a stage
    const int per = blockDim.x * EPT;
    const uint32_t stage = (uint32_t)stage_bytes<T>(blockDim.x);
    int asked = 0, to = 0, from = 0;   // rows asked for; the stages that the next one goes to and the current one comes from
    int64_t ask_at = r0 * cols + tid * V;
    char* mine = smem + threadIdx.x * V * 4;
    const uint32_t mine32 = (uint32_t)__cvta_generic_to_shared(mine);
    auto half = [&](auto p) { return p - threadIdx.x * V * (4 - sizeof(T)) + (size_t)per * 8; };   // the place of a T column in front of an f32 one's
    auto ask = [&]() {
        if (asked < n) {
            const uint32_t p = mine32 + to * stage;
            ask_row<FOUR>(p, a.x_out + ask_at, team, left);
            if (a.d_out) ask_row<FOUR>(p + per * 4, a.d_out + ask_at, team, left);
            const uint32_t t = half(p);
            ask_row<FOUR>(t, static_cast<const T*>(a.y) + ask_at, team, left);
            if (a.d_xn) ask_row<FOUR>(t + per * (uint32_t)sizeof(T), static_cast<const T*>(a.d_xn) + ask_at, team, left);
            ask_at += cols;
        }
        ++asked;
        to = to + 1 == STAGES ? 0 : to + 1;
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) ask();
    pair_t w_pre[EPT / 2], u[EPT / 2], sw_pre[EPT / 2] = {}, sum_g[EPT / 2] = {};   // (all-zero bits are two zeros)
    float sw_post[EPT] = {};
    {
        float t[EPT];
        ld_gain<FOUR>(a.w_pre, team, tid, cols, t);
#pragma unroll
        for (int j = 0; j < EPT / 2; ++j) w_pre[j] = pair(t[2 * j], t[2 * j + 1]);
    }
    int64_t group = (uint32_t)r0 / (uint32_t)a.gate_rows, first = group * a.gate_rows, end = first + min(a.gate_rows, a.rows - first);
    auto set_u = [&](const float (&gate)[EPT], const float (&w)[EPT]) {   // branch gate w_post
#pragma unroll
        for (int j = 0; j < EPT / 2; ++j)
            u[j] = pair(a.branch * gate[2 * j] * w[2 * j], a.branch * gate[2 * j + 1] * w[2 * j + 1]);
    };
    float g[EPT];
    {
        float w[EPT];
        ld_gain<FOUR>(a.w_post, team, tid, cols, w);
        ld_gain<FOUR>(a.gate && n > 0 ? a.gate + group * cols : nullptr, team, tid, cols, g);
        set_u(g, w);
    }
    if (PAIR) {
        __syncwarp();
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    // (teams that share a warp take the same number of turns)
    for (int i = 0; i < (LANES ? (int)a.strip : n); ++i) {
        const bool live = LANES == 0 || i < n;
        const int64_t r = r0 + i, at = (live ? r : r1 - 1) * cols, mine_at = at + tid * V;   // (behind its strip a team goes on at its last row)
        float next_g[EPT];
        if (EACH) ld_gain<FOUR>(a.gate && r + 1 < r1 ? a.gate + (r + 1) * cols : nullptr, team, tid, cols, next_g);
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
        pair_t y[EPT / 2], xo[EPT / 2], dn[EPT / 2], d[EPT / 2];
        {
            const char* p = mine + from * stage;
            const T* t = reinterpret_cast<const T*>(half(p));
            auto take = [&](auto place, auto row, pair_t (&v)[EPT / 2]) {
                float f[EPT];
                take_row<FOUR>(place, row, team, left, f);
#pragma unroll
                for (int j = 0; j < EPT / 2; ++j) v[j] = pair(f[2 * j], f[2 * j + 1]);
            };
            take(reinterpret_cast<const float*>(p), a.x_out + mine_at, xo);
            take(t, static_cast<const T*>(a.y) + mine_at, y);
            if (a.d_out) take(reinterpret_cast<const float*>(p) + per, a.d_out + mine_at, d);
            if (a.d_xn) take(t + per, static_cast<const T*>(a.d_xn) + mine_at, dn);
            from = from + 1 == STAGES ? 0 : from + 1;
        }
        ask();   // into the places of the row before
        pair_t sum2[6] = {};
#pragma unroll
        for (int j = 0; j < EPT / 2; ++j) {
            if (!a.d_out) d[j] = 0;
            if (!a.d_xn) dn[j] = 0;
            const pair_t t = mul2(dn[j], w_pre[j]), v = mul2(u[j], y[j]);
            sum2[0] = fma2(y[j], y[j], sum2[0]);
            sum2[1] = fma2(xo[j], xo[j], sum2[1]);
            sum2[2] = fma2(t, xo[j], sum2[2]);
            sum2[3] = fma2(v, d[j], sum2[3]);
            sum2[4] = fma2(v, t, sum2[4]);
            sum2[5] = fma2(v, xo[j], sum2[5]);
        }
        float sum[6];
#pragma unroll
        for (int j = 0; j < 6; ++j) {
            const float2 t = two(sum2[j]);
            sum[j] = t.x + t.y;
        }
        team_sums<LANES, PAIR>(sum, red, turn);
        // d = d_out + i2 t + c2 x_out; d_y = i1 u d + c1 y
        const float i2 = rsqrtf(sum[1] * over + a.eps), c2 = -i2 * (i2 * (sum[2] * i2 * over));
        const float i1 = a.post ? rsqrtf(sum[0] * over + a.eps) : 1.0f;
        const float c1 = a.post ? -i1 * (i1 * (i1 * over * (sum[3] + i2 * sum[4] + c2 * sum[5]))) : 0.0f;
        const pair_t I1 = pair(i1), I2 = pair(i2), C1 = pair(c1), C2 = pair(c2);
        float dx[EPT], dy[EPT];
#pragma unroll
        for (int j = 0; j < EPT / 2; ++j) {
            if (live) sw_pre[j] = fma2(mul2(dn[j], xo[j]), I2, sw_pre[j]);
            d[j] = fma2(I2, mul2(dn[j], w_pre[j]), fma2(C2, xo[j], d[j]));
            if (live) sum_g[j] = fma2(mul2(d[j], y[j]), I1, sum_g[j]);
            const float2 x2 = two(mul2(pair(a.skip), d[j])), y2 = two(fma2(C1, y[j], mul2(I1, mul2(u[j], d[j]))));
            dx[2 * j] = x2.x; dx[2 * j + 1] = x2.y;
            dy[2 * j] = y2.x; dy[2 * j + 1] = y2.y;
        }
        if (!live) continue;
        st_cols<FOUR>(a.d_x + at, team, tid, cols, dx);
        st_cols<FOUR>(static_cast<T*>(a.d_y) + at, team, tid, cols, dy);
        if (EACH || r + 1 == end || r + 1 == r1) {   // the last row of the gate's group, or of the strip
            float w[EPT], sg[EPT];
            if (!EACH) ld_gain<FOUR>(a.gate ? a.gate + group * cols : nullptr, team, tid, cols, g);
            ld_gain<FOUR>(a.w_post, team, tid, cols, w);
#pragma unroll
            for (int j = 0; j < EPT / 2; ++j) {
                const float2 t = two(sum_g[j]);
                sg[2 * j] = a.branch * t.x; sg[2 * j + 1] = a.branch * t.y;
                sum_g[j] = 0;
            }
#pragma unroll
            for (int j = 0; j < EPT; ++j) {
                sw_post[j] = fmaf(g[j], sg[j], sw_post[j]);
                sg[j] *= w[j];
            }
            if (a.d_gate) {
                if (EACH) put_sum<FOUR>(a.d_gate + at, team, tid, cols, sg, a.accumulate);
                else if (first >= r0 && end <= r1) put_sum<FOUR>(a.d_gate + group * cols, team, tid, cols, sg, a.accumulate);
                else st_cols<FOUR>(a.part_g + (2 * s + (first < r0 ? 0 : 1)) * cols, team, tid, cols, sg);
            }
            if (EACH) {
                set_u(next_g, w);
#pragma unroll
                for (int j = 0; j < EPT; ++j) g[j] = next_g[j];
            } else if (r + 1 < r1) {
                ++group;
                first = end;
                end = first + min(a.gate_rows, a.rows - first);
                if (a.gate) {
                    ld_cols<FOUR>(a.gate + group * cols, team, tid, cols, g, 1.0f);
                    set_u(g, w);
                }
            }
        }
    }
    float sums_pre[EPT];
#pragma unroll
    for (int j = 0; j < EPT / 2; ++j) {
        const float2 t = two(sw_pre[j]);
        sums_pre[2 * j] = t.x; sums_pre[2 * j + 1] = t.y;
    }
    // the CTA's sums of the gains
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        if (which == 0 ? !a.d_w_pre : !a.d_w_post) continue;
        float* out = a.part_w + (2 * (int64_t)(PAIR ? blockIdx.x >> 1 : blockIdx.x) + which) * cols;
        if constexpr (LANES != 0) {
            float* part = reinterpret_cast<float*>(smem);   // [team][columns]: no more than a stage
            constexpr int WIDE = L * EPT;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < EPT; ++j) part[threadIdx.x / L * WIDE + col_of<FOUR>(j, team, tid)] = which == 0 ? sums_pre[j] : sw_post[j];
            __syncthreads();
            for (int c = threadIdx.x; c < cols; c += 256) {
                float v = 0.0f;
#pragma unroll
                for (int i = 0; i < TEAMS; ++i) v += part[i * WIDE + c];
                out[c] = v;
            }
        } else if (which == 0) st_cols<FOUR>(out, team, tid, cols, sums_pre);
        else st_cols<FOUR>(out, team, tid, cols, sw_post);
    }
}

// Adds what the strips left: blockIdx.y = 0, 1 the gains over all CTAs; behind them a gate's groups that reach over several strips,
// as many of them a block as leave each 2^lanes_log lanes. A block owns eight columns (a 32-byte sector of every part), 128 lanes a column,
// each of which takes every so many-th part.
constexpr int SUM_COLS = 8, SUM_LANES = 128;
__global__ void __launch_bounds__(SUM_COLS * SUM_LANES) join_sums_kernel(const Join a, int ctas, uint32_t lanes_log) {
    __shared__ float sh[SUM_LANES / 4][SUM_COLS];   // [warp]
    pdl_wait();
    const int c = blockIdx.x * SUM_COLS + threadIdx.x % SUM_COLS, y = threadIdx.x / SUM_COLS, w = threadIdx.x >> 5, lane = threadIdx.x & 31, cols = a.cols;
    const bool gains = blockIdx.y < 2;
    if (gains && !(blockIdx.y == 0 ? a.d_w_pre : a.d_w_post)) return;
    const uint32_t log = gains ? 7 : lanes_log, per = 1u << log, rows = (uint32_t)a.rows, gate_rows = (uint32_t)a.gate_rows, strip = (uint32_t)a.strip;
    const uint32_t group0 = (blockIdx.y - 2) << (7 - log);
    static_assert(SUM_LANES == 1 << 7, "lanes are powers of two");
    float v = 0.0f;
    if (gains) {
        if (c < cols) {
#pragma unroll 8
            for (int i = y; i < ctas; i += SUM_LANES) v += a.part_w[(2 * (int64_t)i + blockIdx.y) * cols + c];
        }
    } else {
        const uint64_t first = (uint64_t)(group0 + (y >> log)) * gate_rows;   // (32-bit divisions below: rows are)
        if (first < rows) {
            const uint32_t end = min(gate_rows, rows - (uint32_t)first) + (uint32_t)first, s0 = (uint32_t)first / strip, s1 = (end - 1) / strip, k = y & (per - 1);
            if (s0 < s1 && c < cols) {   // (a group in one strip: written there)
                // the group begins in its first strip, whose sum goes to the right, and comes into the others from the left
                if (k == 0) v = a.part_g[(2 * (int64_t)s0 + 1) * cols + c];
#pragma unroll 8
                for (uint32_t i = s0 + 1 + k; i <= s1; i += per) v += a.part_g[2 * (int64_t)i * cols + c];
            }
        }
    }
    v += __shfl_xor_sync(0xffffffffu, v, 8);
    v += __shfl_xor_sync(0xffffffffu, v, 16);
    if (lane < SUM_COLS) sh[w][lane] = v;
    __syncthreads();
    if (y >= SUM_LANES >> log || c >= cols) return;
    float* out = gains ? (blockIdx.y == 0 ? a.d_w_pre : a.d_w_post) : a.d_gate + (int64_t)(group0 + y) * cols;
    if (!gains) {
        const uint64_t first = (uint64_t)(group0 + y) * gate_rows;
        if (first >= rows || (uint32_t)first / strip == (min(gate_rows, rows - (uint32_t)first) + (uint32_t)first - 1) / strip) return;
    }
    v = 0.0f;
#pragma unroll 8
    for (uint32_t i = 0; i < per / 4; ++i) v += sh[y * (per / 4) + i][threadIdx.x % SUM_COLS];
    out[c] = a.accumulate ? out[c] + v : v;
}

// Lanes of a warp that make a team (0: a team is a CTA), and the team's threads.
inline int team_lanes(int64_t cols) { return cols <= 64 ? 8 : cols <= 128 ? 16 : cols <= 256 ? 32 : 0; }
inline int team_threads(int64_t cols) { return team_lanes(cols) ? team_lanes(cols) : (int)ceil_div64(cols, 32 * EPT) * 32; }

struct Strips {
    int64_t strip, strips, ctas;
    // gate_rows 0: the most strips that any gate_rows gives
    Strips(const asca_ctx* ctx, int64_t rows, int64_t cols, int64_t gate_rows) {
        const int team = team_threads(cols);
        const int64_t teams = team > 512 ? ctx->sm_count / 2 : (int64_t)ctx->sm_count * (512 / team);   // what is resident at once: 128 registers a thread
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

// MOST: threads of a team at most, which is what bounds its registers
template <template <typename, bool, int, int> class K>
int launch(asca_ctx* ctx, const Join& a, int dtype, bool four, int64_t teams) {
    const int lanes = team_lanes(a.cols), threads = lanes ? 256 : team_threads(a.cols);
    const dim3 grid((unsigned)(lanes ? ceil_div64(teams, 256 / lanes) : teams));
    cudaError_t e = cudaSuccess;
    auto with = [&](auto t, auto f) {
        using T = decltype(t);
        constexpr bool FOUR = decltype(f)::value;
        if (lanes == 8) e = K<T, FOUR, 8, 256>::go(ctx, grid, threads, a);
        else if (lanes == 16) e = K<T, FOUR, 16, 256>::go(ctx, grid, threads, a);
        else if (lanes == 32) e = K<T, FOUR, 32, 256>::go(ctx, grid, threads, a);
        else if (threads <= 256) e = K<T, FOUR, 0, 256>::go(ctx, grid, threads, a);
        else if (threads <= 512) e = K<T, FOUR, 0, 512>::go(ctx, grid, threads, a);
        else e = K<T, FOUR, 0, 1024>::go(ctx, grid, threads, a);
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
    static cudaError_t go(asca_ctx* ctx, dim3 grid, int threads, const Join& a) {
        join_fwd_kernel<T, FOUR, LANES, MOST><<<grid, threads, 0, ctx->stream>>>(a);
        return cudaSuccess;
    }
};
template <typename T, bool FOUR, int LANES, int MOST>
struct Bwd {
    static cudaError_t go(asca_ctx* ctx, dim3 grid, int threads, const Join& a) {
        constexpr bool PAIR = MOST > 512;   // (a thread of a larger CTA would have half of the registers that it needs)
        constexpr int CTA = PAIR ? MOST / 2 : MOST;
        const int cta = PAIR ? (threads + 63) / 64 * 32 : threads;
        auto kern = a.gate && a.gate_rows == 1 ? join_bwd_kernel<T, FOUR, LANES, CTA, PAIR, true> : join_bwd_kernel<T, FOUR, LANES, CTA, PAIR, false>;
        const size_t smem = STAGES * stage_bytes<T>(cta);
        const cudaError_t e = asca_allow_smem(kern, smem, STAGES * stage_bytes<T>(CTA));
        if (e != cudaSuccess) return e;
        if (PAIR) return asca_launch_cluster(ctx, kern, dim3(2 * grid.x), dim3(cta), smem, 2, a);
        kern<<<grid, cta, smem, ctx->stream>>>(a);
        return cudaSuccess;
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
    a.gate_rows = std::min(gate_rows, rows);   // (32 bits)
    const int64_t n = rows * cols;
    const size_t size = asca_dtype_size(dtype);
    const asca_span_of in[2] = {{y, n, size}, {x, n, 4}}, out[2] = {{x_out, n, 4}, {xn, n, size}};
    const asca_span_of par[3] = {{w_post, cols, 4}, {gate, ceil_div64(rows, std::max<int64_t>(a.gate_rows, 1)) * cols, 4}, {w_pre, cols, 4}};
    for (const auto& o : out) {
        for (const auto& i : in) ASCA_REQUIRE(ctx, asca_in_place(o, i), "gated_residual_rmsnorm_fwd: an output lies over an input");
        for (const auto& i : par) ASCA_REQUIRE(ctx, asca_apart(o, i), "gated_residual_rmsnorm_fwd: an output lies over a gain or gate");
    }
    ASCA_REQUIRE(ctx, asca_apart(out[0], out[1]), "gated_residual_rmsnorm_fwd: x_out and xn overlap");
    asca_device_scope on(ctx);
    const bool four = asca_rows_by(4, y, cols, dtype) && asca_rows_by(4, xn, cols, dtype) && asca_aligned(x, 16) && asca_aligned(x_out, 16) &&
                      asca_aligned(w_post, 16) && asca_aligned(gate, 16) && asca_aligned(w_pre, 16);
    return launch<Fwd>(ctx, a, dtype, four, rows);
}

int64_t asca_gated_residual_rmsnorm_bwd_ws(asca_ctx* ctx, int64_t rows, int64_t cols) {
    if (!ctx || rows < 0 || rows >= ((int64_t)1 << 31) || cols <= 0 || cols > MAX_COLS) return ASCA_ERR_ARG;
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
    a.gate_rows = std::min(a.gate_rows, rows);   // (32 bits)
    const Strips s(ctx, rows, cols, d_gate ? a.gate_rows : 0);
    ASCA_REQUIRE(ctx, asca_aligned(ws, 256) && ws_bytes >= (size_t)asca_gated_residual_rmsnorm_bwd_ws(ctx, rows, cols),
                 "%s: the workspace has to have asca_gated_residual_rmsnorm_bwd_ws bytes, 256-byte aligned", who);
    const int64_t n = rows * cols, groups_all = ceil_div64(rows, a.gate_rows);
    const size_t size = asca_dtype_size(dtype);
    const asca_span_of in[4] = {{y, n, size}, {x_out, n, 4}, {d_xn, n, size}, {d_out, n, 4}};
    const asca_span_of par[3] = {{w_post, cols, 4}, {gate, groups_all * cols, 4}, {w_pre, cols, 4}};
    const asca_span_of out[5] = {{d_x, n, 4}, {d_y, n, size}, {d_w_post, cols, 4}, {d_w_pre, cols, 4}, {d_gate, groups_all * cols, 4}};
    for (int o = 0; o < 5; ++o) {
        for (const auto& i : in) ASCA_REQUIRE(ctx, asca_in_place(out[o], i), "%s: an output lies over an input", who);
        for (const auto& i : par) ASCA_REQUIRE(ctx, asca_apart(out[o], i), "%s: an output lies over a gain or gate", who);
        for (int p = 0; p < o; ++p) ASCA_REQUIRE(ctx, asca_apart(out[o], out[p]), "%s: two outputs overlap", who);
    }
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
        const int64_t groups = gates ? ceil_div64(rows, a.gate_rows) : 0, strips = gates ? ceil_div64(a.gate_rows, s.strip) : 1;   // a group's
        uint32_t log = 2;
        while (log < 7 && (1 << log) < strips) ++log;
        const dim3 grid((unsigned)ceil_div64(cols, SUM_COLS), (unsigned)(2 + ceil_div64(groups, SUM_LANES >> log)));
        ASCA_CUDA(ctx, asca_launch_after(ctx, join_sums_kernel, grid, dim3(SUM_COLS * SUM_LANES), 0, a, (int)s.ctas, log));
        ctx->launches++;
    }
    return ASCA_OK;
}

}  // extern "C"

// Rows of f32 or bf16 read and written as f32 values, four at a time or one at a time, and the device scope of an entry point.
#pragma once
#include "common.cuh"

#include <algorithm>
#include <type_traits>

// Makes the context's device current while an entry point launches, for callers that have another one current.
struct asca_device_scope {
    int was = -1;
    explicit asca_device_scope(const asca_ctx* ctx) {
        int cur = -1;
        if (cudaGetDevice(&cur) == cudaSuccess && cur != ctx->device && cudaSetDevice(ctx->device) == cudaSuccess) was = cur;
    }
    ~asca_device_scope() {
        if (was >= 0) cudaSetDevice(was);
    }
};

inline bool asca_known_dtype(int dtype) { return dtype == ASCA_F32 || dtype == ASCA_BF16; }
inline size_t asca_dtype_size(int dtype) { return dtype == ASCA_BF16 ? 2 : 4; }
inline bool asca_aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
// v (4 or 8) elements of a row of `cols` can be moved at once at every multiple of v columns (a null pointer has no rows)
inline bool asca_rows_by(int v, const void* p, int64_t cols, int dtype) {
    return cols % v == 0 && asca_aligned(p, v * asca_dtype_size(dtype));
}

// Memory that a call writes and other memory of it: apart, or (asca_in_place) the same elements in the same places, which is sound where
// whoever writes an element has read it before.
struct asca_span_of {
    uintptr_t at;
    size_t bytes;
    asca_span_of(const void* p, int64_t n, size_t size) : at(reinterpret_cast<uintptr_t>(p)), bytes(p ? (size_t)n * size : 0) {}
};
inline bool asca_apart(const asca_span_of& a, const asca_span_of& b) { return a.at + a.bytes <= b.at || b.at + b.bytes <= a.at || !a.bytes || !b.bytes; }
inline bool asca_in_place(const asca_span_of& a, const asca_span_of& b) { return (a.at == b.at && a.bytes == b.bytes) || asca_apart(a, b); }

// f(pointer of the type that `dtype` names); a const pointer stays const
template <typename F>
inline void asca_with_dtype(const void* p, int dtype, F f) {
    if (dtype == ASCA_BF16) f(static_cast<const __nv_bfloat16*>(p));
    else f(static_cast<const float*>(p));
}
template <typename F>
inline void asca_with_dtype(void* p, int dtype, F f) {
    if (dtype == ASCA_BF16) f(static_cast<__nv_bfloat16*>(p));
    else f(static_cast<float*>(p));
}

// How a thread moves its columns between rows of two types (frag below): 8 together where a bf16 side then moves 16 bytes, else 4, else
// (1) single columns; and f(std::integral_constant of that), eight only for pairs of types that have it.
inline int asca_row_width(int64_t cols, const void* a, int a_dtype, const void* b, int b_dtype) {
    if ((a_dtype == ASCA_BF16 || b_dtype == ASCA_BF16) && asca_rows_by(8, a, cols, a_dtype) && asca_rows_by(8, b, cols, b_dtype)) return 8;
    return asca_rows_by(4, a, cols, a_dtype) && asca_rows_by(4, b, cols, b_dtype) ? 4 : 1;
}
inline int64_t asca_row_frags(int64_t cols, int width) { return ceil_div64(cols, width == 1 ? 4 : width); }
#ifdef __CUDACC__
// A block of at most `threads` (a power of two) with a power of two or whole warps of lanes a row of `frags` groups of columns, as few
// rounds as that allows, the lanes spread evenly over them; and the rows beside each other.
inline dim3 asca_row_block(int64_t frags, int threads) {
    int tx = 1;
    while (tx < frags && tx < 32) tx *= 2;
    if (frags > 32) tx = (int)ceil_div64(ceil_div64(frags, ceil_div64(frags, threads)), 32) * 32;
    return dim3(tx, threads / tx);
}
#endif
// f(std::integral_constant of 8, 16 or 32): the lanes of a warp that a row of `frags` groups of columns gets
template <typename F>
inline void asca_with_lanes(int64_t frags, F f) {
    if (frags <= 8) f(std::integral_constant<int, 8>());
    else if (frags <= 16) f(std::integral_constant<int, 16>());
    else f(std::integral_constant<int, 32>());
}
// Blocks of 256 that share a row's columns, where `blocks` alone do not fill the SMs (8000 rows of 4096 bf16 looked up: 19.8 us by one
// block a row, 14.5 shared).
inline unsigned asca_column_blocks(const asca_ctx* ctx, int64_t blocks, int64_t frags, int lanes) {
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>(ceil_div64(frags, lanes), 8 * ctx->sm_count / std::max<int64_t>(blocks, 1)));
}
template <typename A, typename B, typename F>
inline void asca_with_width(int v, F f) {
    if constexpr (sizeof(A) == 2 || sizeof(B) == 2)
        if (v == 8) return f(std::integral_constant<int, 8>());
    if (v == 4) f(std::integral_constant<int, 4>());
    else f(std::integral_constant<int, 1>());
}

#ifdef __CUDACC__
// Lets a kernel have `smem` bytes of dynamic shared memory where that may be more than the 48 KiB that it has anyway, its static arrays
// (24 KiB at most here) among them. The limit belongs to the kernel on the device, not to a context or a call: `most` is the largest
// size that any call of the kernel has, so that no call of another context on another thread lowers it in front of this one's launch.
template <typename K>
inline cudaError_t asca_allow_smem(K kern, size_t smem, size_t most) {
    return smem > 24 * 1024 ? cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most) : cudaSuccess;
}
// Launches a kernel that begins with pdl_wait() behind the one before it on the stream without waiting for that one's end to be
// scheduled: a second or third launch of one call then costs about a microsecond less.
template <typename... KArgs, typename... Args>
inline cudaError_t asca_launch_after(asca_ctx* ctx, void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, KArgs(args)...);
}
__device__ __forceinline__ float2 bf16x2_f32(uint32_t u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
__device__ __forceinline__ uint32_t f32_bf16x2(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float4 ld4(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 ld4(const __nv_bfloat16* p) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const float2 a = bf16x2_f32(u.x), b = bf16x2_f32(u.y);
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void st4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void st4(__nv_bfloat16* p, float4 v) { *reinterpret_cast<uint2*>(p) = make_uint2(f32_bf16x2(v.x, v.y), f32_bf16x2(v.z, v.w)); }

// V consecutive elements as they lie in memory, for loads that wait their turn in half the registers or move on unchanged
template <int V, typename T>
struct raw_row {
    T v;
};
template <>
struct raw_row<4, float> {
    float4 v;
};
template <>
struct raw_row<8, float> {
    float4 v, w;
};
template <>
struct raw_row<4, __nv_bfloat16> {
    uint2 v;
};
template <>
struct raw_row<8, __nv_bfloat16> {
    uint4 v;
};
// V consecutive elements of a row, in one access each
// Eight f32 go in one 32-byte access: two of 16 bytes would each touch half of every sector, twice the sectors for the same bytes.
__device__ __forceinline__ void ld8(const float* p, float4& a, float4& b) {
    asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=f"(a.x), "=f"(a.y), "=f"(a.z), "=f"(a.w), "=f"(b.x), "=f"(b.y), "=f"(b.z), "=f"(b.w)
                 : "l"(__cvta_generic_to_global(p)));
}
__device__ __forceinline__ void st8(float* p, float4 a, float4 b) {
    asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(__cvta_generic_to_global(p)), "f"(a.x), "f"(a.y), "f"(a.z), "f"(a.w), "f"(b.x), "f"(b.y), "f"(b.z),
                 "f"(b.w)
                 : "memory");
}
template <int V, typename T>
__device__ __forceinline__ raw_row<V, T> ld_raw(const T* p) {
    raw_row<V, T> r;
    if constexpr (V == 8 && sizeof(T) == 4) ld8(p, r.v, r.w);
    else r.v = *reinterpret_cast<const decltype(r.v)*>(p);
    return r;
}
template <int V, typename T>
__device__ __forceinline__ void st_raw(T* p, const raw_row<V, T>& r) {
    if constexpr (V == 8 && sizeof(T) == 4) st8(p, r.v, r.w);
    else *reinterpret_cast<std::remove_const_t<decltype(r.v)>*>(p) = r.v;
}
__device__ __forceinline__ void unpack(const raw_row<1, float>& r, float (&v)[1]) { v[0] = r.v; }
__device__ __forceinline__ void unpack(const raw_row<1, __nv_bfloat16>& r, float (&v)[1]) { v[0] = __bfloat162float(r.v); }
__device__ __forceinline__ void unpack4(const float4& x, float* v) { v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w; }
__device__ __forceinline__ void unpack(const raw_row<4, float>& r, float (&v)[4]) { unpack4(r.v, v); }
__device__ __forceinline__ void unpack(const raw_row<8, float>& r, float (&v)[8]) { unpack4(r.v, v); unpack4(r.w, v + 4); }
__device__ __forceinline__ void unpack2(uint32_t u, float* v) {
    const float2 x = bf16x2_f32(u);
    v[0] = x.x; v[1] = x.y;
}
__device__ __forceinline__ void unpack(const raw_row<4, __nv_bfloat16>& r, float (&v)[4]) { unpack2(r.v.x, v); unpack2(r.v.y, v + 2); }
__device__ __forceinline__ void unpack(const raw_row<8, __nv_bfloat16>& r, float (&v)[8]) {
    unpack2(r.v.x, v); unpack2(r.v.y, v + 2); unpack2(r.v.z, v + 4); unpack2(r.v.w, v + 6);
}
template <int V, typename T>
__device__ __forceinline__ void ld_row(const T* p, float (&v)[V]) { unpack(ld_raw<V>(p), v); }
template <int V, typename T>
__device__ __forceinline__ void st_row(T* p, const float (&v)[V]) {
    if constexpr (V == 8 && sizeof(T) == 4) st8(p, make_float4(v[0], v[1], v[2], v[3]), make_float4(v[4], v[5], v[6], v[7]));
    else if constexpr (V == 8) {
        *reinterpret_cast<uint4*>(p) = make_uint4(f32_bf16x2(v[0], v[1]), f32_bf16x2(v[2], v[3]), f32_bf16x2(v[4], v[5]), f32_bf16x2(v[6], v[7]));
    } else if constexpr (V % 4 == 0) {
#pragma unroll
        for (int i = 0; i < V; i += 4) st4(p + i, make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]));
    } else *p = from_f32<T>(v[0]);
}

// A thread's columns of a row that `lanes` threads share: W = 8 or 4 together, or W = 1: four single ones, `lanes` apart. Thread x begins at
// frag_first(x) and goes on by lanes * frag<W, T>::E.
template <int W, typename T>
struct frag {
    static constexpr int E = W;
    raw_row<W, T> r;
    __device__ __forceinline__ void load(const T* row, int c, int, int) { r = ld_raw<W>(row + c); }
    __device__ __forceinline__ void store(T* row, int c, int, int) const { st_raw<W>(row + c, r); }
    __device__ __forceinline__ void get(float (&v)[E]) const { unpack(r, v); }
    static __device__ __forceinline__ void put(T* row, int c, int, int, const float (&v)[E]) { st_row<W>(row + c, v); }
};
template <typename T>
struct frag<1, T> {
    static constexpr int E = 4;
    T r[4];
    __device__ __forceinline__ void load(const T* row, int c, int lanes, int cols) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c + i * lanes < cols) r[i] = row[c + i * lanes];
    }
    __device__ __forceinline__ void store(T* row, int c, int lanes, int cols) const {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c + i * lanes < cols) row[c + i * lanes] = r[i];
    }
    __device__ __forceinline__ void get(float (&v)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = to_f32<T>(r[i]);
    }
    static __device__ __forceinline__ void put(T* row, int c, int lanes, int cols, const float (&v)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c + i * lanes < cols) row[c + i * lanes] = from_f32<T>(v[i]);
    }
};
template <int W>
__device__ __forceinline__ int frag_first(int x) { return W == 1 ? x : x * W; }
#endif

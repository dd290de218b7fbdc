// Rows of f32 or bf16 read and written as f32 values, four at a time or one at a time, and the device scope of an entry point.
#pragma once
#include "common.cuh"

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
// four elements of a row of `cols` can be moved at once at every multiple of four columns (a null pointer has no rows)
inline bool asca_rows_by_four(const void* p, int64_t cols, int dtype) { return (cols & 3) == 0 && asca_aligned(p, 4 * asca_dtype_size(dtype)); }

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

#ifdef __CUDACC__
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

// V consecutive elements: V = 4 through the vector forms, V = 1 for rows off their grid or of a width that four does not divide
template <int V, typename T>
__device__ __forceinline__ void ld_row(const T* p, float (&v)[V]) {
    if constexpr (V == 4) {
        const float4 x = ld4(p);
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    } else {
        static_assert(V == 1, "four or one");
        v[0] = to_f32<T>(*p);
    }
}
template <int V, typename T>
__device__ __forceinline__ void st_row(T* p, const float (&v)[V]) {
    if constexpr (V == 4) st4(p, make_float4(v[0], v[1], v[2], v[3]));
    else *p = from_f32<T>(v[0]);
}
#endif

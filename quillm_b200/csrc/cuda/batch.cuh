// Shared by the operators of batched decoding (rope_rows.cu, attn_prefix.cu, beam.cu): element types, chunks of
// elements moved with one access, and the checks of the caller's cache.
#pragma once

#include <cuda_bf16.h>

#include <initializer_list>

#include "common.cuh"

namespace qmc {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
// one rounding to nearest even
__device__ __forceinline__ void from_f32(float v, float *o) { *o = v; }
__device__ __forceinline__ void from_f32(float v, __half *o) { *o = __float2half_rn(v); }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16 *o) { *o = __float2bfloat16_rn(v); }

// two elements at once
__device__ __forceinline__ float2 to_f32x2(__half2 v) { return __half22float2(v); }
__device__ __forceinline__ float2 to_f32x2(__nv_bfloat162 v) { return __bfloat1622float2(v); }
__device__ __forceinline__ float2 to_f32x2(float2 v) { return v; }
__device__ __forceinline__ void from_f32x2(float x, float y, __half2 *o) { *o = __floats2half2_rn(x, y); }
__device__ __forceinline__ void from_f32x2(float x, float y, __nv_bfloat162 *o) { *o = __floats2bfloat162_rn(x, y); }
__device__ __forceinline__ void from_f32x2(float x, float y, float2 *o) { *o = make_float2(x, y); }
template <typename T>
struct Two;
template <>
struct Two<float> {
    using type = float2;
};
template <>
struct Two<__half> {
    using type = __half2;
};
template <>
struct Two<__nv_bfloat16> {
    using type = __nv_bfloat162;
};

// C consecutive elements as they lie in memory, moved in pieces of up to 16 bytes: an address is aligned to
// min(16, C * sizeof(T)) bytes
template <typename T, int C>
struct alignas(C * sizeof(T) >= 16 ? 16 : C * sizeof(T)) Chunk {
    T e[C];
};
template <typename T, int C>
__device__ __forceinline__ void widen(const Chunk<T, C> &c, float (&v)[C]) {
    if constexpr (C % 2 == 0) {
        using T2 = typename Two<T>::type;
#pragma unroll
        for (int i = 0; i < C; i += 2) {
            const float2 f = to_f32x2(*(const T2 *)&c.e[i]);
            v[i] = f.x, v[i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < C; i++) v[i] = to_f32(c.e[i]);
    }
}
template <typename T, int C>
__device__ __forceinline__ void load_chunk(const T *p, float (&v)[C]) {
    const Chunk<T, C> c = *(const Chunk<T, C> *)p;
    widen(c, v);
}
template <typename T, int C>
__device__ __forceinline__ void store_chunk(T *p, const float (&v)[C]) {
    Chunk<T, C> c;
    if constexpr (C % 2 == 0) {
        using T2 = typename Two<T>::type;
#pragma unroll
        for (int i = 0; i < C; i += 2) from_f32x2(v[i], v[i + 1], (T2 *)&c.e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < C; i++) from_f32(v[i], &c.e[i]);
    }
    *(Chunk<T, C> *)p = c;
}

__device__ __forceinline__ float ex2(float x) {  // 2^x, relative error about 2^-22; below 2^-126 it is 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

inline bool is_row_dtype(int d) { return d == QMC_F32 || d == QMC_F16 || d == QMC_BF16; }
inline int dtype_size(int d) { return d == QMC_F32 ? 4 : 2; }
// arrays of 4-byte elements
inline bool misaligned(std::initializer_list<const void *> arrays) {
    for (const void *p : arrays)
        if ((uintptr_t)p % 4) return true;
    return false;
}
// the caller's cache: QMC_OK, or QMC_EINVAL with `op` in the message
int check_cache(const qmc_paged_cache *c, const char *op);
// elements of one layer of a pool
inline int64_t layer_elems(const qmc_paged_cache *c) {
    return (int64_t)c->n_pages * c->page_size * c->n_kv_heads * c->head_dim;
}

}  // namespace qmc

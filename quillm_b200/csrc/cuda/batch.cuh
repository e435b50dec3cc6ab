// Shared by the operators of batched decoding (rope_rows.cu, attn_prefix.cu, beam.cu): element types, chunks of
// elements moved with one access, and the checks of the caller's cache.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace qmc {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
// one rounding to nearest even
__device__ __forceinline__ void from_f32(float v, float *o) { *o = v; }
__device__ __forceinline__ void from_f32(float v, __half *o) { *o = __float2half_rn(v); }
__device__ __forceinline__ void from_f32(float v, __nv_bfloat16 *o) { *o = __float2bfloat16_rn(v); }

// C consecutive elements, moved in pieces of up to 16 bytes; p is aligned to min(16, C * sizeof(T)) bytes
template <typename T, int C>
__device__ __forceinline__ void load_chunk(const T *p, float (&v)[C]) {
    constexpr int B = C * (int)sizeof(T);
    alignas(16) T e[C];
    if constexpr (B >= 16) {
#pragma unroll
        for (int i = 0; i < B / 16; i++) ((uint4 *)e)[i] = ((const uint4 *)p)[i];
    } else if constexpr (B == 8) {
        *(uint2 *)e = *(const uint2 *)p;
    } else if constexpr (B == 4) {
        *(uint32_t *)e = *(const uint32_t *)p;
    } else {
        e[0] = p[0];
    }
#pragma unroll
    for (int i = 0; i < C; i++) v[i] = to_f32(e[i]);
}
template <typename T, int C>
__device__ __forceinline__ void store_chunk(T *p, const float (&v)[C]) {
    constexpr int B = C * (int)sizeof(T);
    alignas(16) T e[C];
#pragma unroll
    for (int i = 0; i < C; i++) from_f32(v[i], &e[i]);
    if constexpr (B >= 16) {
#pragma unroll
        for (int i = 0; i < B / 16; i++) ((uint4 *)p)[i] = ((const uint4 *)e)[i];
    } else if constexpr (B == 8) {
        *(uint2 *)p = *(const uint2 *)e;
    } else if constexpr (B == 4) {
        *(uint32_t *)p = *(const uint32_t *)e;
    } else {
        p[0] = e[0];
    }
}

inline bool is_row_dtype(int d) { return d == QMC_F32 || d == QMC_F16 || d == QMC_BF16; }
inline int dtype_size(int d) { return d == QMC_F32 ? 4 : 2; }
// the caller's cache: QMC_OK, or QMC_EINVAL with `op` in the message
int check_cache(const qmc_paged_cache *c, const char *op);
// elements of one layer of a pool
inline int64_t layer_elems(const qmc_paged_cache *c) {
    return (int64_t)c->n_pages * c->page_size * c->n_kv_heads * c->head_dim;
}

}  // namespace qmc

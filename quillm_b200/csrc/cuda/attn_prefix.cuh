// Work of the shared-prefix attention (attn_prefix.cu), for its kernels: the jobs of a launch and where their parts go.
#pragma once

#include <atomic>

#include "batch.cuh"

namespace qmc {

struct AttnArgs {
    const void *q, *kc, *vc;  // kc, vc: the layer's pools
    void *out;
    int64_t ldq, ldo;
    const int *prefix_pages, *table, *lens;
    int *err;
    float2 *ml;
    float *po;
    int n_seq, heads, kv, group, hd, page_size, n_pages, ld_table, prefix;
    int rows, ptiles, psplit, gtiles, osplit;
    int pparts;   // parts that the prefix leaves of each row (psplit of its own launch); the own ones follow
    float scale;  // times log2(e): scores and maxima are exponents of two
};

// the part of one job: rows [r0, r0 + nr) of KV head h, positions [p0, p1), and where its results go
struct Job {
    int h, r0, nr, p0, p1, part, b;  // b: the sequence of an own job, -1 for the prefix
};

__device__ __forceinline__ int own_len(const AttnArgs &a, int b) {
    return min(max(a.lens[b], a.prefix), a.ld_table * a.page_size) - a.prefix;
}

// jobs: prefix [h][tile][split], then own [b][h][group tile][split]; ranges of positions are multiples of `quantum`
__device__ __forceinline__ Job job_of(const AttnArgs &a, unsigned i, int ptile, int otile, int quantum) {
    Job j;
    const unsigned np = (unsigned)(a.kv * a.ptiles * a.psplit);
    if (i < np) {
        const int sp = i % a.psplit, t = i / a.psplit % a.ptiles;
        j.h = i / a.psplit / a.ptiles;
        j.r0 = t * ptile, j.nr = min(ptile, a.rows - j.r0);
        const int64_t chunk = (((int64_t)a.prefix + a.psplit - 1) / a.psplit + quantum - 1) / quantum * quantum;
        j.p0 = (int)min((int64_t)a.prefix, sp * chunk), j.p1 = (int)min((int64_t)a.prefix, sp * chunk + chunk);
        j.part = sp, j.b = -1;
        return j;
    }
    i -= np;
    const int sp = i % a.osplit, t = i / a.osplit % a.gtiles;
    j.h = i / a.osplit / a.gtiles % a.kv;
    j.b = i / a.osplit / a.gtiles / a.kv;
    j.r0 = j.b * a.group + t * otile, j.nr = min(otile, a.group - t * otile);
    const int64_t n = own_len(a, j.b), chunk = ((n + a.osplit - 1) / a.osplit + quantum - 1) / quantum * quantum;
    j.p0 = a.prefix + (int)min(n, sp * chunk), j.p1 = a.prefix + (int)min(n, sp * chunk + chunk);
    j.part = a.pparts + sp;
    return j;
}

// slot of position p, -1 (and the error word) for a page outside the pool
__device__ __forceinline__ int64_t slot_of(const AttnArgs &a, int b, int p) {
    const int e = p / a.page_size, page = b < 0 ? a.prefix_pages[e] : a.table[(int64_t)b * a.ld_table + e];
    if (page < 0 || page >= a.n_pages) {
        raise_error(a.err, kErrBadIndex);
        return -1;
    }
    return (int64_t)page * a.page_size + p % a.page_size;
}

// row r of a KV head: sequence r / group, query head h * group + r % group; its place among all batch * heads rows
__device__ __forceinline__ int64_t out_row(const AttnArgs &a, int h, int r) {
    return (int64_t)(r / a.group) * a.heads + h * a.group + r % a.group;
}

// The reference m of a row's softmax weights 2^(s - m), where these are rounded to CT for the second product.  m moves, and o and the
// sum of weights with it, only when a tile's largest score leaves a window around it.
//   bf16 has float's range: m is a score that was the row's largest, weights stay below 2^kLift.
//   fp16 keeps a weight's 11 bits from 2^-14 to 2^16: m lies kTop below the score that set it, so that weights reach into the upper
//   range, and it follows the scores down too.  Else everything beside one score far above (a sink) would lose its bits, and vanish 2^25 below
//   it, while the float sum still counts it; with a small value at the sink that is the whole output.  o and the sum are floats and lose
//   nothing by factors above one; m goes down by at most 2^kFar from its highest, below which nothing counts and o could overflow.
// A tile's largest weight so lies between 2^kDrop and 2^kLift, and the others of that tile are off by 2^-25 at least.  With kTop at 12 the
// normal scores of 64 sequences behind 32768 positions left the window often enough to cost 2.5 us of 88.7.
template <typename CT>
struct Window {
    static constexpr bool kHalf = __is_same(CT, __half);
    static constexpr float kTop = kHalf ? 10.0f : 0.0f, kLift = kHalf ? 15.5f : 8.0f, kDrop = -2.0f, kFar = 48.0f;
    __device__ static __forceinline__ bool left_by(float m, float top) {
        return top > m + kLift || (kHalf && top > -INFINITY && top < m + kDrop);
    }
    // the reference after a tile whose largest score is `top` (-inf: it has none); hi: the highest so far, kept for fp16.  At first
    // both are -inf
    __device__ static __forceinline__ float moved(float m, float top, float &hi, float lift = kLift) {
        if constexpr (kHalf) {
            if (top - m > lift || (top > -INFINITY && top - m < kDrop)) m = fmaxf(top - kTop, hi - kFar);
            hi = fmaxf(hi, m);
            return m;
        } else {
            return fmaxf(m, top);
        }
    }
};

__device__ __forceinline__ void mma16(__half, float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(__nv_bfloat16, float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// two floats as a pair of 16-bit elements, the first in the low half; lo: what the rounding left over
__device__ __forceinline__ uint32_t pack2(__half, float x, float y, float *lo = nullptr) {
    const __half2 h = __floats2half2_rn(x, y);
    if (lo) lo[0] = x - __low2float(h), lo[1] = y - __high2float(h);
    return *(const uint32_t *)&h;
}
__device__ __forceinline__ uint32_t pack2(__nv_bfloat16, float x, float y, float *lo = nullptr) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    if (lo) lo[0] = x - __low2float(h), lo[1] = y - __high2float(h);
    return *(const uint32_t *)&h;
}

// the kernel's dynamic shared memory limit, raised once per device (twice where two threads make the first call)
template <typename F>
int raise_smem(F fn, int bytes, std::atomic<bool> (&done)[64]) {
    int dev = 0;
    QMC_CUDA(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return set_error(QMC_EINVAL, "attn_prefix: device %d out of range", dev);
    if (!done[dev]) {
        QMC_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        done[dev] = true;
    }
    return QMC_OK;
}

// a launch that may start before the kernel before it in the stream has ended (`after`); the kernel calls pdl_wait
template <typename... A>
int launch_after(void (*fn)(A...), dim3 grid, int threads, int smem, cudaStream_t s, bool after, A... args) {
    cudaLaunchConfig_t c = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    c.gridDim = grid, c.blockDim = dim3(threads), c.dynamicSmemBytes = smem, c.stream = s;
    c.attrs = attr, c.numAttrs = after ? 1 : 0;
    QMC_CUDA(cudaLaunchKernelEx(&c, fn, args...));
    return QMC_OK;
}

// the matrix-instruction kernel (attn_mma.cu), for 16-bit caches whose rows are whole 16-byte chunks
int attn_mma_tile(int rows);  // query rows of a prefix job, for `rows` of them per KV head; own jobs take 16
// after: the kernel may start before the one before it in the stream has ended, and ends after it
int launch_attn_mma(const AttnArgs &a, int dtype, int cdt, bool after, cudaStream_t s);

// up to 16 rows a tile, straight from global memory into the matrix instructions (attn_warp.cu): such caches with head_dim <= 128.  Up
// to 16 rows it is ahead of the tensor-core kernel (whole calls over 8192 shared positions of 8 heads: 8 rows 18.5 and 20.3 us, 16
// rows 20.5 both ways), with more it reads them again (24 rows 24.6 and 20.5 us; over 32768 49 and 38)
constexpr int kWarpRows = 16;
int launch_attn_warp(const AttnArgs &a, int dtype, int cdt, bool after, cudaStream_t s);

// caches of floats, heads of whole 16-byte chunks (attn_vec.cu): tiles of 1, 4 or 8 rows, the smallest that takes the rows of a
// group, and of the prefix if 8 do (4 rows of 8 heads over 4096 positions 18.5 us with tiles of 4, 28.9 with 1; 16 rows
// 29.3 us with 8, 35.0 with 4)
int attn_vec_tile(int rows);
int launch_attn_vec(const AttnArgs &a, int tile, cudaStream_t s);

// the tensor-core kernel (attn_tc.cu): the prefix jobs of such a cache with rows of its own type, head_dim <= 128, pages of a
// multiple of 8 positions and under 2^31 slots, for many rows
int attn_tc_box(int page_size);  // positions of one copy
int attn_tc_tile(int rows);
int launch_attn_tc(const AttnArgs &a, int cdt, cudaStream_t s);

}  // namespace qmc

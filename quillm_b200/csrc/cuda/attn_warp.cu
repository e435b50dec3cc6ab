// Shared-prefix attention for up to 16 query rows per tile over caches of 16-bit elements: own positions (a group's heads) and the
// prefix of a few sequences.  HBM bound: with so few rows the products cost little, so keys and values go from global memory
// straight into the registers that the matrix instructions (m16n8k16, float accumulators) take, no shared memory, no barrier; the
// group after the next is on its way to L2.  Measured: 4 rows of 32 heads over 32768 shared positions 86 us (6.3 TB/s), 16 rows of 8
// heads 31 us (4.4 TB/s; short ranges), 64 sequences of up to 1024 own positions 41 us with cold caches, 16 of up to 8192 65 us a call
// (without the way to L2 it took 13 us more; through shared memory, two or three groups ahead, 20 us).
//
// Every warp of a block takes 16 positions at a time, every fourth group of the job's range.  Of the two operand layouts only the
// dimensions' order is free, and that is enough: with g = lane / 4 and t = lane % 4,
//   K (second operand of Q K^T, column = position g): thread (g, t) holds 16-byte chunks t, t + 4, ... of position g's key; two
//   products of 16 dimensions use one chunk, Q's chunks are held the same way;
//   V (second operand of P V, rows = positions 2t, 2t + 1, 2t + 8, 2t + 9): it holds chunk g (and g + 8) of those positions' values, and
//   element j of each is column g of product j, so that a product's 8 columns are dimensions j, 8 + j, ..., 56 + j.
// A row's accumulators are rescaled only when its scores leave the window around its reference (Window); the four warps' parts are joined
// through shared memory at the end.
//
// Float queries over an fp16 cache: a row is scaled by a power of two and split in two halves q = qh + ql, the weights likewise, and
// each product is taken twice.  A score is off by 2^-21 of sum |q k|, a weight by 2^-22 of itself or 2^-25 in the window's scale, 2^-23
// of the largest of its 16 positions at most.
#include "attn_prefix.cuh"

namespace qmc {
namespace {

// streamed once: not kept in the first-level cache
__device__ __forceinline__ uint4 load_stream(const void *p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// HDP: head_dim rounded up to 64 or 128
template <typename T, typename CT, int HDP>
__global__ void __launch_bounds__(128, 2) attn_warp_kernel(const AttnArgs a) {
    constexpr bool SPLIT = sizeof(T) == 4;
    constexpr int H = SPLIT ? 2 : 1, NU = HDP / 32, NC = HDP / 64;  // chunks of K and of V a thread holds per position
    extern __shared__ __align__(16) float part[];                  // [4 warps][16][HDP]
    __shared__ float m_s[4][16], l_s[4][16];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const Job jb = job_of(a, blockIdx.x, 16, 16, 16);
    pdl_launch_dependents();
    const int hd = a.hd, nch = hd / 8;

    // the next group's keys are loaded as soon as this one's scores are formed, its values as soon as this one's are used
    auto locate = [&](int p0) {  // elements from the pool's start of position p0 + lane % 16, -1: none
        const int64_t slot = p0 + (lane & 15) < jb.p1 ? slot_of(a, jb.b, p0 + (lane & 15)) : -1;
        return slot >= 0 ? (slot * a.kv + jb.h) * hd : (int64_t)-1;
    };
    uint4 k[2][NU], v[4][NC];
    auto load_k = [&](int64_t at) {
#pragma unroll
        for (int n = 0; n < 2; n++) {
            const int64_t s = __shfl_sync(0xffffffffu, at, g + 8 * n);
#pragma unroll
            for (int u = 0; u < NU; u++)
                k[n][u] = s >= 0 && t + 4 * u < nch ? load_stream((const CT *)a.kc + s + 8 * (t + 4 * u)) : make_uint4(0, 0, 0, 0);
        }
    };
    auto load_v = [&](int64_t at) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int64_t s = __shfl_sync(0xffffffffu, at, 2 * t + (i & 1) + 4 * (i & 2));
#pragma unroll
            for (int c = 0; c < NC; c++)
                v[i][c] = s >= 0 && g + 8 * c < nch ? load_stream((const CT *)a.vc + s + 8 * (g + 8 * c)) : make_uint4(0, 0, 0, 0);
        }
    };
    // the group after that is on its way to the second-level cache: lanes 0-15 ask for the keys, the others for the values
    const uint8_t *const half = (const uint8_t *)(lane < 16 ? a.kc : a.vc);
    auto fetch = [&](int64_t at) {
        if (at < 0) return;
#pragma unroll
        for (int i = 0; i < HDP / 64; i++)
            if (64 * i < hd) asm volatile("prefetch.global.L2 [%0];" ::"l"(half + 2 * (at + 64 * i)));
    };
    int64_t at = locate(jb.p0 + 16 * warp), next = locate(jb.p0 + 16 * warp + 64);
    load_k(at);
    load_v(at);
    fetch(next);
    at = next, next = locate(jb.p0 + 16 * warp + 128);

    uint32_t q[H][2 * NU][4];
    float scale[2];  // of rows g and g + 8
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int r = g + 8 * i, rr = jb.r0 + r;
        const T *src = (const T *)a.q + (rr / a.group) * a.ldq + (int64_t)(jb.h * a.group + rr % a.group) * hd;
        float v[NU][8], mx = 0.0f, up = 1.0f;
#pragma unroll
        for (int u = 0; u < NU; u++)
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const int d = 8 * (t + 4 * u) + k;
                v[u][k] = r < jb.nr && d < hd ? to_f32(src[d]) : 0.0f;
                mx = fmaxf(mx, fabsf(v[u][k]));
            }
        if (SPLIT) {  // times 2^-e, 2^e the power of two at or below the row's largest element: both halves stay normal
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const int e = min(126, max(-126, (__float_as_int(mx) >> 23) - 127));
            const float down = __int_as_float((127 - e) << 23);
            up = __int_as_float((127 + e) << 23);
#pragma unroll
            for (int u = 0; u < NU; u++)
#pragma unroll
                for (int k = 0; k < 8; k++) v[u][k] *= down;
        }
        scale[i] = up * a.scale;
#pragma unroll
        for (int u = 0; u < NU; u++)
#pragma unroll
            for (int k = 0; k < 8; k += 2) {  // elements 0 1 | 2 3 of a chunk: one product's first and second half, 4 5 | 6 7 the next's
                float lo[2];
                q[0][2 * u + k / 4][i + (k & 2)] = pack2(CT(), v[u][k], v[u][k + 1], lo);
                if (SPLIT) q[H - 1][2 * u + k / 4][i + (k & 2)] = pack2(CT(), lo[0], lo[1]);
            }
    }

    using W = Window<CT>;
    float o[NC][8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, high[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int c = 0; c < NC; c++)
#pragma unroll
        for (int j = 0; j < 8; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[c][j][i] = 0.0f;
    for (int p0 = jb.p0 + 16 * warp; p0 < jb.p1; p0 += 64) {
        fetch(next);
        float s[2][4] = {};
#pragma unroll
        for (int u = 0; u < NU; u++)
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int h = 0; h < H; h++) {
                    mma16(CT(), s[n], q[h][2 * u], k[n][u].x, k[n][u].y);
                    mma16(CT(), s[n], q[h][2 * u + 1], k[n][u].z, k[n][u].w);
                }
        load_k(at);
        const int left = jb.p1 - p0;
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[n][i] = 8 * n + 2 * t + (i & 1) < left ? s[n][i] * scale[i >> 1] : -INFINITY;
                mx[i >> 1] = fmaxf(mx[i >> 1], s[n][i]);
            }
        bool move = __any_sync(0xffffffffu, mx[0] > m[0] + W::kLift || mx[1] > m[1] + W::kLift);
        if constexpr (W::kHalf) {  // is a row's every score below the window?  Four lanes hold a row
            const unsigned in0 = __ballot_sync(0xffffffffu, mx[0] >= m[0] + W::kDrop), in1 = __ballot_sync(0xffffffffu, mx[1] >= m[1] + W::kDrop);
            const unsigned x = in0 | in0 >> 1, y = in1 | in1 >> 1;
            move = move || (((x | x >> 2) & (y | y >> 2)) & 0x11111111u) != 0x11111111u;
        }
        if (move) {  // the first time, and rarely again
#pragma unroll
            for (int i = 0; i < 2; i++) {
                mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
                mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
                const float to = W::moved(m[i], mx[i], high[i]), by = to == -INFINITY ? 1.0f : ex2(m[i] - to);
                m[i] = to, l[i] *= by;
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int j = 0; j < 8; j++) o[c][j][2 * i] *= by, o[c][j][2 * i + 1] *= by;
            }
        }
        uint32_t p[H][4];
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float ref = m[i] == -INFINITY ? 0.0f : m[i];
                const float x = ex2(s[n][2 * i] - ref), y = ex2(s[n][2 * i + 1] - ref);
                float lo[2];
                l[i] += x + y;
                p[0][2 * n + i] = pack2(CT(), x, y, lo);
                if (SPLIT) p[H - 1][2 * n + i] = pack2(CT(), lo[0], lo[1]);
            }
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const uint32_t r0[4] = {v[0][c].x, v[0][c].y, v[0][c].z, v[0][c].w}, r1[4] = {v[1][c].x, v[1][c].y, v[1][c].z, v[1][c].w};
            const uint32_t r2[4] = {v[2][c].x, v[2][c].y, v[2][c].z, v[2][c].w}, r3[4] = {v[3][c].x, v[3][c].y, v[3][c].z, v[3][c].w};
#pragma unroll
            for (int j = 0; j < 8; j++) {  // element j of the four positions' chunks
                const uint32_t pick = j & 1 ? 0x7632u : 0x5410u;
                const uint32_t b0 = __byte_perm(r0[j / 2], r1[j / 2], pick), b1 = __byte_perm(r2[j / 2], r3[j / 2], pick);
#pragma unroll
                for (int h = 0; h < H; h++) mma16(CT(), o[c][j], p[h], b0, b1);
            }
        }
        load_v(at);
        at = next, next = locate(p0 + 192);
    }

    // join the four warps: maxima and sums first, then the rescaled accumulators; the columns of row r are rotated by 8 r
#pragma unroll
    for (int i = 0; i < 2; i++) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        if (t == 0) m_s[warp][g + 8 * i] = m[i], l_s[warp][g + 8 * i] = l[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int r = g + 8 * i;
        if (r >= jb.nr) continue;
        const float M = fmaxf(fmaxf(m_s[0][r], m_s[1][r]), fmaxf(m_s[2][r], m_s[3][r]));
        const float down = M == -INFINITY ? 0.0f : ex2(m[i] - M);
        float *dst = part + (warp * 16 + r) * HDP;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int e = 0; e < 2; e++) {  // columns 2t + e of the eight products: eight dimensions in a row
                const int d = (8 * (2 * t + e + 8 * c) + 8 * r) % HDP;
#pragma unroll
                for (int j = 0; j < 8; j += 4)
                    *(float4 *)(dst + d + j) = make_float4(o[c][j][2 * i + e] * down, o[c][j + 1][2 * i + e] * down,
                                                           o[c][j + 2][2 * i + e] * down, o[c][j + 3][2 * i + e] * down);
            }
    }
    __syncthreads();
    const int64_t all = (int64_t)a.n_seq * a.heads;
    for (int i = tid; i < jb.nr * (HDP / 4); i += 128) {
        const int r = i / (HDP / 4), d = i % (HDP / 4) * 4;
        if (d >= hd) continue;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float4 y = *(const float4 *)(part + (w * 16 + r) * HDP + (d + 8 * r) % HDP);
            x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
        }
        const int64_t to = jb.part * all + out_row(a, jb.h, jb.r0 + r);
        *(float4 *)(a.po + to * hd + d) = x;
        if (d == 0) {
            const float M = fmaxf(fmaxf(m_s[0][r], m_s[1][r]), fmaxf(m_s[2][r], m_s[3][r]));
            float sum = 0.0f;
            if (M > -INFINITY)
#pragma unroll
                for (int w = 0; w < 4; w++) sum += l_s[w][r] * ex2(m_s[w][r] - M);
            a.ml[to] = make_float2(M, sum);
        }
    }
    // launched beside the prefix's kernel, this grid ends after it, which the join relies on: one block waits, the others make room
    if (blockIdx.x == 0) pdl_wait();
}

template <typename T, typename CT, int HDP>
int launch_t(const AttnArgs &a, bool after, cudaStream_t s) {
    const int64_t jobs = (int64_t)a.kv * a.ptiles * a.psplit + (int64_t)a.n_seq * a.kv * a.gtiles * a.osplit;
    if (jobs > INT32_MAX) return set_error(QMC_EINVAL, "attn_prefix: too many blocks");
    return jobs ? launch_after(attn_warp_kernel<T, CT, HDP>, dim3((unsigned)jobs), 128, 4 * 16 * HDP * 4, s, after, a) : QMC_OK;
}
template <typename T, typename CT>
int launch_h(const AttnArgs &a, bool after, cudaStream_t s) {
    return a.hd <= 64 ? launch_t<T, CT, 64>(a, after, s) : launch_t<T, CT, 128>(a, after, s);
}

}  // namespace

int launch_attn_warp(const AttnArgs &a, int dtype, int cdt, bool after, cudaStream_t s) {
    if (dtype == QMC_F32) return launch_h<float, __half>(a, after, s);
    return cdt == QMC_F16 ? launch_h<__half, __half>(a, after, s) : launch_h<__nv_bfloat16, __nv_bfloat16>(a, after, s);
}

}  // namespace qmc

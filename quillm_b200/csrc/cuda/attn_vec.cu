// Shared-prefix attention over caches of floats, for heads of whole 16-byte chunks: own positions and prefixes, up to 8 query rows
// per tile, on the CUDA cores.
//
// L lanes share a position, each with HDP / L of its dimensions: a warp scores 32 / L positions at a time for all rows of the tile, the
// dimensions' sums meet in log2(L) shuffles, and each group of L lanes keeps a running maximum, sum and o of its own for every
// row, so that nothing else passes between lanes before the end.  Keys and values go from global memory to registers, 8 chunks of
// each on their way per lane while the group before is used; no shared memory, no barrier.  A row's accumulators are rescaled only
// when a score passes its reference by more than 2^kLift.
//
// HBM bound with few rows: one row of 32 heads over 4096 positions 28 us (4.7 TB/s), 8 sequences of up to 4096 95 us (5.6 TB/s).  With
// many rows each tile of 8 reads the prefix again, from L2, and the instructions bound it, about 14 a row and position: 128 rows of
// 8 heads over 2048 positions 81 us (staged through shared memory, 16 rows a block, 174 us).  All sums of a step's rows are formed
// side by side: row by row the shuffles' latency made that 155 us.
#include "attn_prefix.cuh"

namespace qmc {
namespace {

constexpr float kLift = 8.0f;

// not kept in the first-level cache; as floats from the start (through a common load of four words: 128 rows 84.5 -> 88.6 us)
__device__ __forceinline__ float4 load_stream(const float *p) {
    float4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
    return v;
}

// R rows of a tile; HDP: head_dim rounded up to 64, 128 or 256
template <int R, int HDP>
__global__ void __launch_bounds__(128, R == 1 ? 3 : 2) attn_vec_kernel(const AttnArgs a) {
    constexpr int L = R == 8 ? HDP / 8 : HDP / 16, NC = HDP / 4 / L, U = R == 8 ? 2 : 8 / NC, P = 32 / L, PU = P * U;
    __shared__ float part[4][R][HDP];
    __shared__ float m_s[4][R], l_s[4][R];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, t = lane % L, sub = lane / L;
    const Job jb = job_of(a, blockIdx.x, R, R, PU);
    pdl_launch_dependents();
    const int hd = a.hd, nch = hd / 4, nr = jb.nr;
    const float *const kc = (const float *)a.kc, *const vc = (const float *)a.vc;

    auto locate = [&](int p0) {  // elements from the pool's start of position p0 + lane % PU, -1: none
        const int64_t slot = p0 + lane % PU < jb.p1 ? slot_of(a, jb.b, p0 + lane % PU) : -1;
        return slot >= 0 ? (slot * a.kv + jb.h) * hd : (int64_t)-1;
    };
    float4 k[U][NC], v[U][NC];
    auto load = [&](const float *pool, float4 (&x)[U][NC], int64_t at) {  // chunk t + L c of position P u + sub
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int64_t s = __shfl_sync(0xffffffffu, at, P * u + sub);
#pragma unroll
            for (int c = 0; c < NC; c++)
                x[u][c] = s >= 0 && t + L * c < nch ? load_stream(pool + s + 4 * (t + L * c)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
    };
    // the group after that is on its way to the second-level cache: one or two lines of 128 bytes a lane
    const int line = lane / PU;
    auto fetch = [&](int64_t at) {
        if (at < 0) return;
        const float *pool = line & 1 ? vc : kc;
#pragma unroll
        for (int i = 0; i < HDP * PU / 512; i++) {
            const int d = 32 * (HDP * PU / 512 * (line >> 1) + i);
            if (d < hd) asm volatile("prefetch.global.L2 [%0];" ::"l"(pool + at + d));
        }
    };
    int64_t at = locate(jb.p0 + PU * warp), next = locate(jb.p0 + PU * (warp + 4));
    load(kc, k, at);
    load(vc, v, at);
    fetch(next);
    at = next, next = locate(jb.p0 + PU * (warp + 8));

    float4 q[R][NC], o[R][NC];
    float m[R], l[R];
#pragma unroll
    for (int j = 0; j < R; j++) {
        m[j] = -INFINITY, l[j] = 0.0f;
        const int rr = jb.r0 + j;
        const float *src = (const float *)a.q + (rr / a.group) * a.ldq + (int64_t)(jb.h * a.group + rr % a.group) * hd;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            const int d = 4 * (t + L * c);
            const bool live = j < nr && d < hd;
            q[j][c] = live ? make_float4(src[d], src[d + 1], src[d + 2], src[d + 3]) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            o[j][c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
    }
    for (int p0 = jb.p0 + PU * warp; p0 < jb.p1; p0 += 4 * PU) {
        fetch(next);
        float s[R][U];  // rows past the last have zeros for queries: without a branch the sums of all rows are under way together
#pragma unroll
        for (int j = 0; j < R; j++)
#pragma unroll
            for (int u = 0; u < U; u++) {
                float x = 0.0f, y = 0.0f;
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    x = fmaf(q[j][c].x, k[u][c].x, fmaf(q[j][c].y, k[u][c].y, x));
                    y = fmaf(q[j][c].z, k[u][c].z, fmaf(q[j][c].w, k[u][c].w, y));
                }
                s[j][u] = x + y;
            }
        load(kc, k, at);
#pragma unroll
        for (int b = 1; b < L; b *= 2)
#pragma unroll
            for (int j = 0; j < R; j++)
#pragma unroll
                for (int u = 0; u < U; u++) s[j][u] += __shfl_xor_sync(0xffffffffu, s[j][u], b);
        bool lift = false;
#pragma unroll
        for (int j = 0; j < R; j++)
#pragma unroll
            for (int u = 0; u < U; u++) {
                s[j][u] = p0 + P * u + sub < jb.p1 ? s[j][u] * a.scale : -INFINITY;
                lift = lift || s[j][u] > m[j] + kLift;
            }
        if (__any_sync(0xffffffffu, lift)) {  // the first time, and rarely again
#pragma unroll
            for (int j = 0; j < R; j++) {
                float to = m[j];
#pragma unroll
                for (int u = 0; u < U; u++) to = fmaxf(to, s[j][u]);
                const float down = to == -INFINITY ? 1.0f : ex2(m[j] - to);
                m[j] = to, l[j] *= down;
#pragma unroll
                for (int c = 0; c < NC; c++) o[j][c].x *= down, o[j][c].y *= down, o[j][c].z *= down, o[j][c].w *= down;
            }
        }
#pragma unroll
        for (int j = 0; j < R; j++) {
            const float ref = m[j] == -INFINITY ? 0.0f : m[j];
#pragma unroll
            for (int u = 0; u < U; u++) {
                const float e = ex2(s[j][u] - ref);
                l[j] += e;
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    o[j][c].x = fmaf(e, v[u][c].x, o[j][c].x), o[j][c].y = fmaf(e, v[u][c].y, o[j][c].y);
                    o[j][c].z = fmaf(e, v[u][c].z, o[j][c].z), o[j][c].w = fmaf(e, v[u][c].w, o[j][c].w);
                }
            }
        }
        load(vc, v, at);
        at = next, next = locate(p0 + 12 * PU);
    }

    // join the groups of lanes, then the four warps
#pragma unroll
    for (int j = 0; j < R; j++) {
        if (j >= nr) break;
        float M = m[j];
#pragma unroll
        for (int b = L; b < 32; b *= 2) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, b));
        const float down = M == -INFINITY ? 0.0f : ex2(m[j] - M);
        float x = l[j] * down;
#pragma unroll
        for (int b = L; b < 32; b *= 2) x += __shfl_xor_sync(0xffffffffu, x, b);
        if (lane == 0) m_s[warp][j] = M, l_s[warp][j] = x;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            float4 y = make_float4(o[j][c].x * down, o[j][c].y * down, o[j][c].z * down, o[j][c].w * down);
#pragma unroll
            for (int b = L; b < 32; b *= 2) {
                y.x += __shfl_xor_sync(0xffffffffu, y.x, b), y.y += __shfl_xor_sync(0xffffffffu, y.y, b);
                y.z += __shfl_xor_sync(0xffffffffu, y.z, b), y.w += __shfl_xor_sync(0xffffffffu, y.w, b);
            }
            if (sub == 0) *(float4 *)&part[warp][j][4 * (t + L * c)] = y;
        }
    }
    __syncthreads();
    const int64_t all = (int64_t)a.n_seq * a.heads;
    for (int i = tid; i < nr * nch; i += 128) {
        const int j = i / nch, d = i % nch * 4;
        const float M = fmaxf(fmaxf(m_s[0][j], m_s[1][j]), fmaxf(m_s[2][j], m_s[3][j]));
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float sum = 0.0f;
        if (M > -INFINITY)
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float f = ex2(m_s[w][j] - M);
                const float4 y = *(const float4 *)&part[w][j][d];
                sum = fmaf(f, l_s[w][j], sum);
                x.x = fmaf(f, y.x, x.x), x.y = fmaf(f, y.y, x.y), x.z = fmaf(f, y.z, x.z), x.w = fmaf(f, y.w, x.w);
            }
        const int64_t to = jb.part * all + out_row(a, jb.h, jb.r0 + j);
        *(float4 *)(a.po + to * hd + d) = x;
        if (d == 0) a.ml[to] = make_float2(M, sum);
    }
}

template <int R>
int launch_r(const AttnArgs &a, unsigned jobs, cudaStream_t s) {
    if (a.hd <= 64) attn_vec_kernel<R, 64><<<jobs, 128, 0, s>>>(a);
    else if (a.hd <= 128) attn_vec_kernel<R, 128><<<jobs, 128, 0, s>>>(a);
    else attn_vec_kernel<R, 256><<<jobs, 128, 0, s>>>(a);
    QMC_LAUNCH_CHECK();
    return QMC_OK;
}

}  // namespace

int attn_vec_tile(int rows) { return rows == 1 ? 1 : rows <= 4 ? 4 : 8; }

int launch_attn_vec(const AttnArgs &a, int tile, cudaStream_t s) {
    const int64_t jobs = (int64_t)a.kv * a.ptiles * a.psplit + (int64_t)a.n_seq * a.kv * a.gtiles * a.osplit;
    if (jobs > INT32_MAX) return set_error(QMC_EINVAL, "attn_prefix: too many blocks");
    if (!jobs) return QMC_OK;
    return tile == 1 ? launch_r<1>(a, (unsigned)jobs, s) : tile == 4 ? launch_r<4>(a, (unsigned)jobs, s) : launch_r<8>(a, (unsigned)jobs, s);
}

}  // namespace qmc

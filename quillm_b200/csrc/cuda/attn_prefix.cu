// Attention of one token per sequence over a shared prefix and own pages (qmc_attn_prefix).
//
// For row (b, head): o = sum_p e^(s_p - M) v_p / sum_p e^(s_p - M), s_p = scale q . k_p, over the prefix's positions
// and the sequence's own.  The prefix's keys and values are the same for every sequence, so its part is one
// product of all batch * group query rows of a KV head with them: a block takes a tile of those rows and a range
// of positions, and the prefix is read once per row tile, not once per sequence.  Own positions are read once per (sequence, KV
// head), shared by the group's heads.  Each job leaves its rows' running maximum m, sum l and unnormalised o in the workspace, and
// a last launch joins the parts of every row: o = sum_j e^(m_j - M) o_j / sum_j e^(m_j - M) l_j.
//
// Kernels of the jobs, by what they measured alone with cold caches (us; 8 KV heads of 128, fp16, 32768 shared positions, floor
// 20.5, unless stated):
//   attn_tc    more than 16 rows per KV head, rows of the cache's 16-bit type, head_dim <= 128, pages of a multiple of 8:
//              32 rows 30.5, 64 32.5, 128 32.9, 256 48, 512 (two tiles of 256) 77
//   attn_warp  up to 16 rows and all own positions, 16-bit caches, head_dim <= 128: 16 rows 31, and 64 sequences of <= 1024
//              own positions 41 (floor 21)
//   attn_mma   the other 16-bit caches of whole 16-byte chunks: pages of 20, 32 rows 45, 64 54, 512 311; float rows 512 474
//   attn_vec   float caches of whole 16-byte chunks: 128 rows over 2048 positions 81, one row of 32 heads over 4096 28 (floor 20.5)
//   this file  what is left, any head_dim up to 256 and any alignment: fp16 heads of 100, 128 rows over 2048 positions 125, float
//              heads of 50, 8 rows of 32 heads over 1024 33
// Where two of them serve a call, they run beside each other: prefix blocks first, own jobs on the SMs that they leave.
#include <algorithm>
#include <cmath>

#include "attn_prefix.cuh"

namespace qmc {
namespace {

enum { kRowsKernel, kWarpKernel, kMmaKernel, kTcKernel, kVecKernel };

struct Plan {
    int rows;                 // query rows of a KV head over the whole batch: n_seq * group
    int ptiles, psplit;       // prefix: row tiles and position ranges
    int gtiles, osplit;       // own positions: row tiles of a group and position ranges
    int pkind, okind;         // the kernels of the prefix and of own positions
    int pparts;
    int vtile;                // rows of a job of kVecKernel
    int64_t ml_bytes, bytes;  // workspace: [parts][n_seq * n_heads] float2 (m, l), then [parts][...][hd] floats
};

constexpr int kQR = 16;  // query rows per block (4 per warp)
constexpr int kPT = 32;  // positions per staged tile (one per lane)

// The general kernel, in float on the CUDA cores: any head_dim up to 256, any types, strides and alignments.  Per row and tile of
// 32 positions lane p scores position p, the warp updates the row's maximum and sum once, and each lane
// accumulates four of the head's dimensions (eight above 128).  Bound by the shared-memory reads of both products: 8 rows of 32
// heads of 50 over 1024 positions 33 us.
template <typename T, typename CT, int NG>
__global__ void __launch_bounds__(128) attn_rows_kernel(const AttnArgs a, bool vec) {
    extern __shared__ __align__(16) float smf[];
    const int hd = a.hd, hd4 = (hd + 3) & ~3;
    float *Kt = smf;               // [hd4 / 4][kPT][4]
    float *Vs = Kt + hd4 * kPT;    // [kPT][hd4]
    float *Qs = Vs + kPT * hd4;    // [kQR][hd4]
    __shared__ int64_t slot_s[kPT];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const Job jb = job_of(a, blockIdx.x, kQR, kQR, kPT);
    pdl_launch_dependents();
    for (int i = tid; i < kQR * hd4; i += 128) {
        const int r = i / hd4, d = i % hd4, rr = jb.r0 + r;
        Qs[i] = (r < jb.nr && d < hd)
                    ? to_f32(((const T *)a.q)[(rr / a.group) * a.ldq + (int64_t)(jb.h * a.group + rr % a.group) * hd + d])
                    : 0.0f;
    }
    constexpr int TW = kQR / 4;
    float m[TW], l[TW], o[TW][NG][4];
#pragma unroll
    for (int j = 0; j < TW; j++) {
        m[j] = -INFINITY, l[j] = 0.0f;
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[j][g][i] = 0.0f;
    }
    const CT *kc = (const CT *)a.kc, *vc = (const CT *)a.vc;
    for (int p0 = jb.p0; p0 < jb.p1; p0 += kPT) {
        __syncthreads();  // the previous tile is no longer read
        if (tid < kPT) slot_s[tid] = p0 + tid < jb.p1 ? slot_of(a, jb.b, p0 + tid) : -1;
        __syncthreads();
        for (int i = tid; i < kPT * (hd4 / 4); i += 128) {  // positions vary fastest: conflict-free transposed stores
            const int pp = i % kPT, c = i / kPT;
            float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (slot_s[pp] >= 0) {
                const CT *p = kc + (slot_s[pp] * a.kv + jb.h) * hd + 4 * c;
                if (sizeof(CT) == 2 && vec) load_chunk<CT, 4>(p, v);  // aligned floats have a kernel of their own
                else
                    for (int k = 0; k < 4; k++) v[k] = 4 * c + k < hd ? to_f32(p[k]) : 0.0f;
            }
            *(float4 *)(Kt + (c * kPT + pp) * 4) = make_float4(v[0], v[1], v[2], v[3]);
        }
        for (int i = tid; i < kPT * (hd4 / 4); i += 128) {
            const int c = i % (hd4 / 4), pp = i / (hd4 / 4);
            float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (slot_s[pp] >= 0) {
                const CT *p = vc + (slot_s[pp] * a.kv + jb.h) * hd + 4 * c;
                if (sizeof(CT) == 2 && vec) load_chunk<CT, 4>(p, v);
                else
                    for (int k = 0; k < 4; k++) v[k] = 4 * c + k < hd ? to_f32(p[k]) : 0.0f;
            }
            *(float4 *)(Vs + pp * hd4 + 4 * c) = make_float4(v[0], v[1], v[2], v[3]);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < TW; j++) {
            const int r = 4 * j + warp;  // few rows spread over the warps
            if (r >= jb.nr) break;
            const float *q = Qs + r * hd4;
            float s4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int c = 0; c < hd4 / 4; c++) {
                const float4 k4 = *(const float4 *)(Kt + (c * kPT + lane) * 4), q4 = *(const float4 *)(q + 4 * c);
                s4[0] = fmaf(q4.x, k4.x, s4[0]), s4[1] = fmaf(q4.y, k4.y, s4[1]);
                s4[2] = fmaf(q4.z, k4.z, s4[2]), s4[3] = fmaf(q4.w, k4.w, s4[3]);
            }
            const float sc = p0 + lane < jb.p1 ? ((s4[0] + s4[1]) + (s4[2] + s4[3])) * a.scale : -INFINITY;
            const float mn = fmaxf(m[j], warp_max(sc));
            const float ref = mn == -INFINITY ? 0.0f : mn;
            const float corr = exp2f(m[j] - ref), e = exp2f(sc - ref);
            l[j] = l[j] * corr + warp_sum(e);
            m[j] = mn;
#pragma unroll
            for (int g = 0; g < NG; g++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[j][g][i] *= corr;
            for (int pp = 0; pp < kPT; pp++) {
                const float ep = __shfl_sync(0xffffffffu, e, pp);
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    if (128 * g + 4 * lane < hd4) {
                        const float4 v4 = *(const float4 *)(Vs + pp * hd4 + 128 * g + 4 * lane);
                        o[j][g][0] = fmaf(ep, v4.x, o[j][g][0]), o[j][g][1] = fmaf(ep, v4.y, o[j][g][1]);
                        o[j][g][2] = fmaf(ep, v4.z, o[j][g][2]), o[j][g][3] = fmaf(ep, v4.w, o[j][g][3]);
                    }
                }
            }
        }
    }
    const int64_t all = (int64_t)a.n_seq * a.heads;
#pragma unroll
    for (int j = 0; j < TW; j++) {
        const int r = 4 * j + warp;  // few rows spread over the warps
        if (r >= jb.nr) break;
        const int64_t at = jb.part * all + out_row(a, jb.h, jb.r0 + r);
        if (lane == 0) a.ml[at] = make_float2(m[j], l[j]);
        if (l[j] == 0.0f) continue;  // the join skips it
#pragma unroll
        for (int g = 0; g < NG; g++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int d = 128 * g + 4 * lane + i;
                if (d < hd) a.po[at * hd + d] = o[j][g][i];
            }
    }
}

constexpr int kMostSplits = 64;

// Joins the parts of a row, W warps each: a warp takes the factors 2^(m_j - M) of all parts, a lane each, and sums every W-th
// part over the row's dimensions, V (once, twice above 128, as often as needed one by one) a lane, with loads that do not
// wait for one another.  Bound by latency: the lengths, the statistics, the parts and the warps' sums follow on one another
// (with cold caches 30 to 128 rows 4.5 to 5.3 us, 1024 rows of 9 parts 6.3 us).
template <typename T, int V, int W>
__global__ void __launch_bounds__(128) attn_join_kernel(const AttnArgs a, int parts) {
    constexpr int NV = 256 / 32 / V, NB = 2 * kMostSplits / 32;
    __shared__ float sum_s[W][256];
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) % W;
    const int64_t all = (int64_t)a.n_seq * a.heads, row = (int64_t)blockIdx.x * (4 / W) + (threadIdx.x >> 5) / W;
    const int b = (int)(row / a.heads), h = (int)(row % a.heads);
    pdl_wait();
    if (row >= all) return;  // W == 1
    const int n = a.lens[b];
    if (lane == 0 && ((n != 0 && n < a.prefix) || n > (int64_t)a.ld_table * a.page_size)) raise_error(a.err, kErrBadIndex);
    float2 st[NB];
    float M = -INFINITY;
#pragma unroll
    for (int i = 0; i < NB; i++) {
        st[i] = n > 0 && lane + 32 * i < parts ? a.ml[(lane + 32 * i) * all + row] : make_float2(-INFINITY, 0.0f);
        M = fmaxf(M, st[i].x);
    }
    M = warp_max(M);
    const float ref = M == -INFINITY ? 0.0f : M;
    float w[NB], l = 0.0f, o[NV][V];
#pragma unroll
    for (int i = 0; i < NB; i++) {  // a part without weights is not read
        w[i] = st[i].y != 0.0f ? exp2f(st[i].x - ref) : 0.0f;
        l = st[i].y != 0.0f ? fmaf(w[i], st[i].y, l) : l;
    }
    l = warp_sum(l);
#pragma unroll
    for (int i = 0; i < NV; i++)
#pragma unroll
        for (int k = 0; k < V; k++) o[i][k] = 0.0f;
#pragma unroll
    for (int i = 0; i < NB; i++) {
        const int here = min(32, parts - 32 * i);
#pragma unroll 4
        for (int j = warp; j < here; j += W) {
            const float wj = __shfl_sync(0xffffffffu, w[i], j);
            const bool live = wj != 0.0f;  // NaN included
            const float *src = a.po + ((32 * i + j) * all + row) * a.hd;
#pragma unroll
            for (int e = 0; e < NV; e++) {
                const int d = V * (lane + 32 * e);
                float v[V];
#pragma unroll
                for (int k = 0; k < V; k++) v[k] = 0.0f;
                if (live && d < a.hd) load_chunk<float, V>(src + d, v);
#pragma unroll
                for (int k = 0; k < V; k++) o[e][k] = fmaf(wj, v[k], o[e][k]);
            }
        }
    }
    const float rl = l > 0.0f ? 1.0f / l : (l == l ? 0.0f : l);  // an empty row gives zeros
    T *out = (T *)a.out + b * a.ldo + (int64_t)h * a.hd;
    if constexpr (W == 1) {
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int k = 0; k < V; k++) {
                const int d = V * (lane + 32 * i) + k;
                if (d < a.hd) from_f32(o[i][k] * rl, &out[d]);
            }
    } else {
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int k = 0; k < V; k++) sum_s[warp][V * (lane + 32 * i) + k] = o[i][k];
        __syncthreads();
        for (int d = threadIdx.x; d < a.hd; d += 128) {
            float x = 0.0f;
#pragma unroll
            for (int i = 0; i < W; i++) x += sum_s[i][d];
            from_f32(x * rl, &out[d]);
        }
    }
}

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// 16-bit rows of whole 16-byte chunks go to the matrix instructions
bool takes_mma(const qmc_paged_cache *c) {
    return c->dtype != QMC_F32 && c->head_dim % 8 == 0 && (((uintptr_t)c->k | (uintptr_t)c->v) & 15) == 0;
}

// The time of a call whose prefix blocks and own jobs are split into n and m position ranges, in the microseconds that one block takes
// while its SM runs as many as fit.  The prefix's blocks come first; own jobs take the places that these leave, and all places
// once they are done.  Sequences are taken to be half as long as the table allows, the last job as long as the longest.  The constants
// come from sweeps of both numbers over a dozen shapes; the numbers it picks are within 10 % of the best of each sweep (16 sequences
// behind 8192 positions: 8 ranges and 1, 29.6 us; 6: 30.9, 12: 38, 16: 46; 64 behind 32768: 7 ranges 90, 6: 100, 9: 101).
struct Work {
    double start, tile;  // of a block: its start, end and parts' way through memory, and each tile of positions
    int64_t units;       // row tiles
    int tiles, take;     // tiles of positions, places that a block takes
};
double time_of(const Work &pre, const Work &own, int n, int m, int64_t places) {
    double done = 0.0, here = 0.0;  // when the prefix's last round ends, and its length
    int64_t left = places;
    if (n) {
        const int64_t blocks = pre.units * n * pre.take, rounds = (blocks + places - 1) / places;
        here = pre.start + pre.tile * ((pre.tiles + n - 1) / n);
        done = rounds * here, left = rounds * places - blocks;
    }
    if (!m) return done;
    const int64_t jobs = own.units * m;
    const double half = own.tile * 0.5 * ((own.tiles + m - 1) / m), job = own.start + half;
    if (!n) return (jobs + places - 1) / places * job + half;
    const int64_t beside = left * (int64_t)ceil(here / job);
    if (jobs <= beside) return std::max(done, done - here + (jobs + left - 1) / left * job + half);
    return done + (jobs - beside + places - 1) / places * job + half;
}

Plan plan_for(const qmc_paged_cache *c, int dtype, int n_seq, int n_heads, int prefix, int ld_table, int sms) {
    Plan p{};
    const int group = n_heads / c->n_kv_heads, kv = c->n_kv_heads;
    const int64_t own = std::max<int64_t>(0, (int64_t)ld_table * c->page_size - prefix);
    p.rows = n_seq * group;
    const bool mma = takes_mma(c), narrow = mma && c->head_dim <= 128;
    const bool vec = c->dtype == QMC_F32 && c->head_dim % 4 == 0 && (((uintptr_t)c->k | (uintptr_t)c->v) & 15) == 0;
    p.okind = narrow ? kWarpKernel : mma ? kMmaKernel : vec ? kVecKernel : kRowsKernel;
    p.pkind = p.okind;
    if (narrow && p.rows > kWarpRows)
        p.pkind = dtype == c->dtype && c->page_size % 8 == 0 && (int64_t)c->n_pages * c->page_size <= INT32_MAX ? kTcKernel : kMmaKernel;
    struct Shape {
        int ptile, otile, quantum, blocks;  // rows of a prefix and of an own job, positions of a tile, blocks an SM runs at once
        double start, tile;                 // see Work
    };
    const int vtile = attn_vec_tile(prefix ? std::max(p.rows, group) : group);
    const Shape shape[5] = {{kQR, kQR, kPT, 4, 5.0, 4.0}, {kWarpRows, kWarpRows, 64, 2, 5.0, 2.2},
                            {attn_mma_tile(p.rows), 16, 64, 2, 6.0, 2.2}, {attn_tc_tile(p.rows), 0, 128, 1, 6.0, 2.0},
                            {vtile, vtile, 32, vtile == 1 ? 3 : 2, 5.0, 1.8}};
    const Shape &ps = shape[p.pkind], &os = shape[p.okind];
    p.ptiles = ceil_div(p.rows, ps.ptile);
    p.gtiles = ceil_div(group, os.otile);
    const Work pre{ps.start, ps.tile, (int64_t)kv * p.ptiles, ceil_div(prefix, ps.quantum), std::max(1, os.blocks / ps.blocks)};
    const Work mine{os.start, os.tile, (int64_t)n_seq * kv * p.gtiles, ceil_div(own, os.quantum), 1};
    // one at a time, from the own jobs by themselves: two rounds end within 15 % of the best pair for 99 of 100 shapes
    auto best = [&](int tiles, auto time) {
        int at = 0;
        double least = 0.0;
        for (int n = 1; n <= std::min(kMostSplits, tiles); n++) {
            if (n > 1 && (tiles + n - 1) / n == (tiles + n - 2) / (n - 1)) continue;  // no range gets shorter
            const double t = time(n);
            if (!at || t < least) least = t, at = n;
        }
        return at;
    };
    const int64_t places = (int64_t)os.blocks * sms;
    if (own) p.osplit = best(mine.tiles, [&](int m) { return time_of(pre, mine, 0, m, places); });
    for (int i = 0; prefix && i < 2; i++) {
        p.psplit = best(pre.tiles, [&](int n) { return time_of(pre, mine, n, p.osplit, places); });
        if (own) p.osplit = best(mine.tiles, [&](int m) { return time_of(pre, mine, p.psplit, m, places); });
    }
    p.vtile = vtile;
    p.pparts = p.psplit;
    const int64_t parts = p.pparts + p.osplit, all = (int64_t)n_seq * n_heads;
    p.ml_bytes = (parts * all * 8 + 255) / 256 * 256;
    p.bytes = p.ml_bytes + parts * all * c->head_dim * 4 + 256;
    return p;
}

template <typename T, typename CT, int NG>
int launch_rows(const AttnArgs &a, int64_t jobs, bool vec, cudaStream_t s) {
    const int hd4 = (a.hd + 3) & ~3;
    auto fn = attn_rows_kernel<T, CT, NG>;
    const int smem = (2 * kPT + kQR) * hd4 * 4;
    static std::atomic<bool> done[64];
    if (const int rc = raise_smem(fn, (2 * kPT + kQR) * 256 * 4, done)) return rc;
    fn<<<(unsigned)jobs, 128, smem, s>>>(a, vec);
    QMC_LAUNCH_CHECK();
    return QMC_OK;
}

template <typename T, typename CT>
int launch_attn(const AttnArgs &a, const Plan &p, int dtype, int cdt, int sms, cudaStream_t s) {
    const int64_t jobs = (int64_t)a.kv * a.ptiles * a.psplit + (int64_t)a.n_seq * a.kv * a.gtiles * a.osplit;
    if (jobs > INT32_MAX) return set_error(QMC_EINVAL, "attn_prefix: too many blocks");
    auto launch = [&](int kind, const AttnArgs &x, bool after) {
        if (kind == kTcKernel) return launch_attn_tc(x, cdt, s);
        if (kind == kMmaKernel) return launch_attn_mma(x, dtype, cdt, after, s);
        if (kind == kWarpKernel) return launch_attn_warp(x, dtype, cdt, after, s);
        if (kind == kVecKernel) return launch_attn_vec(x, p.vtile, s);
        const int64_t n = (int64_t)x.kv * x.ptiles * x.psplit + (int64_t)x.n_seq * x.kv * x.gtiles * x.osplit;
        const size_t al = 4 * sizeof(CT);
        const bool vec = x.hd % 4 == 0 && (uintptr_t)x.kc % al == 0 && (uintptr_t)x.vc % al == 0;
        return x.hd <= 128 ? launch_rows<T, CT, 1>(x, n, vec, s) : launch_rows<T, CT, 2>(x, n, vec, s);
    };
    int rc = QMC_OK;
    if (jobs && p.pkind == p.okind) {
        rc = launch(p.okind, a, false);
    } else if (jobs) {  // own positions beside the prefix: their blocks take the SMs that the other's leave
        AttnArgs first = a, second = a;
        first.osplit = 0, second.psplit = 0;
        if (a.psplit) rc = launch(p.pkind, first, false);
        if (!rc && a.osplit) rc = launch(p.okind, second, a.psplit > 0);
    }
    if (rc) return rc;
    // the join may start while the last parts are written; it waits for them before it reads
    const int64_t all = (int64_t)a.n_seq * a.heads;
    auto join = [&](auto fn, int rows) { return launch_after(fn, dim3((unsigned)((all + rows - 1) / rows)), 128, 0, s, jobs > 0, a, a.pparts + a.osplit); };
    // four warps a row while the SMs hold all rows' blocks at once (1024 rows: 3.6 us less than with one warp each; 1536: 2 us more,
    // 4096: 3 us more)
    const bool wide = all <= 8 * (int64_t)sms;
    if (a.hd % 4 == 0) return wide ? join(attn_join_kernel<T, 4, 4>, 1) : join(attn_join_kernel<T, 4, 1>, 4);
    return wide ? join(attn_join_kernel<T, 1, 4>, 1) : join(attn_join_kernel<T, 1, 1>, 4);
}

int check_attn(const char *op, int dtype, const qmc_paged_cache *c, int n_seq, int n_heads, int prefix, int ld_table) {
    if (const int rc = check_cache(c, op)) return rc;
    const bool ok = (dtype == QMC_F32 && (c->dtype == QMC_F32 || c->dtype == QMC_F16)) ||
                    (dtype == c->dtype && (dtype == QMC_F16 || dtype == QMC_BF16));
    if (!ok) return set_error(QMC_EINVAL, "%s: rows of dtype %d over a cache of dtype %d", op, dtype, c->dtype);
    if (c->head_dim > 256) return set_error(QMC_EINVAL, "%s: head_dim %d is above 256", op, c->head_dim);
    if (n_seq < 0 || n_heads < 1 || n_heads % c->n_kv_heads || prefix < 0 || ld_table < 1)
        return set_error(QMC_EINVAL, "%s: %d sequences, %d heads over %d, prefix %d, table %d wide", op, n_seq, n_heads,
                         c->n_kv_heads, prefix, ld_table);
    if ((int64_t)ld_table * c->page_size > INT32_MAX - 1024 || (int64_t)n_seq * n_heads > INT32_MAX)  // a position past the last is counted too
        return set_error(QMC_EINVAL, "%s: more than 2^31 - 1025 positions or 2^31 - 1 rows", op);
    if (prefix > (int64_t)ld_table * c->page_size)
        return set_error(QMC_EINVAL, "%s: prefix of %d past a table of %d pages of %d", op, prefix, ld_table, c->page_size);
    return QMC_OK;
}

}  // namespace
}  // namespace qmc

using namespace qmc;

extern "C" {

int qmc_attn_prefix_workspace(int dtype, const qmc_paged_cache *cache, int32_t n_seq, int32_t n_heads,
                              int32_t prefix_len, int32_t ld_table, size_t *bytes) {
    if (!bytes) return set_error(QMC_EINVAL, "attn_prefix_workspace: null argument");
    *bytes = 0;
    if (const int rc = check_attn("attn_prefix_workspace", dtype, cache, n_seq, n_heads, prefix_len, ld_table)) return rc;
    if (n_seq == 0) return QMC_OK;  // nothing to plan
    DevCtx *c = ctx();
    if (!c) return QMC_ECUDA;
    *bytes = (size_t)plan_for(cache, dtype, n_seq, n_heads, prefix_len, ld_table, c->num_sms).bytes;
    return QMC_OK;
}

int qmc_attn_prefix(const qmc_paged_cache *cache, int32_t layer, int dtype, const void *q, int64_t ldq, void *out,
                    int64_t ldo, int32_t n_heads, int32_t n_seq, float scale, const int32_t *prefix_pages,
                    int32_t prefix_len, const int32_t *page_table, int32_t ld_table, const int32_t *seq_lens,
                    void *workspace, size_t workspace_bytes, void *stream) {
    const char *op = "attn_prefix";
    if (const int rc = check_attn(op, dtype, cache, n_seq, n_heads, prefix_len, ld_table)) return rc;
    if (layer < 0 || layer >= cache->n_layers) return set_error(QMC_EINVAL, "%s: layer %d of %d", op, layer, cache->n_layers);
    const int64_t n = (int64_t)n_heads * cache->head_dim;
    if (ldq < n || ldo < n || ldq > (int64_t)1 << 40 || ldo > (int64_t)1 << 40)
        return set_error(QMC_EINVAL, "%s: rows of %lld elements are %lld and %lld apart", op, (long long)n, (long long)ldq, (long long)ldo);
    const float scale2 = scale * 1.4426950408889634f;  // scores as exponents of two
    if (!(scale >= 0.0f) || scale2 - scale2 != 0.0f) return set_error(QMC_EINVAL, "%s: scale %g", op, scale);
    if (n_seq == 0) return QMC_OK;
    if (!q || !out || !page_table || !seq_lens || !workspace || (prefix_len && !prefix_pages))
        return set_error(QMC_EINVAL, "%s: null argument", op);
    if ((uintptr_t)q % dtype_size(dtype) || (uintptr_t)out % dtype_size(dtype))
        return set_error(QMC_EINVAL, "%s: misaligned q or out", op);
    if (misaligned({prefix_len ? prefix_pages : nullptr, page_table, seq_lens})) return set_error(QMC_EINVAL, "%s: misaligned pages or lengths", op);
    DevCtx *c = ctx();
    if (!c) return QMC_ECUDA;
    const Plan p = plan_for(cache, dtype, n_seq, n_heads, prefix_len, ld_table, c->num_sms);
    if (workspace_bytes < (size_t)p.bytes)
        return set_error(QMC_EINVAL, "%s: workspace of %zu bytes, %zu needed", op, workspace_bytes, (size_t)p.bytes);
    AttnArgs a{};
    a.q = q, a.out = out, a.ldq = ldq, a.ldo = ldo;
    const int64_t off = layer * layer_elems(cache) * dtype_size(cache->dtype);
    a.kc = (const uint8_t *)cache->k + off, a.vc = (const uint8_t *)cache->v + off;
    a.prefix_pages = prefix_pages, a.table = page_table, a.lens = seq_lens, a.err = c->err;
    uint8_t *w = (uint8_t *)(((uintptr_t)workspace + 255) / 256 * 256);
    a.ml = (float2 *)w, a.po = (float *)(w + p.ml_bytes);
    a.n_seq = n_seq, a.heads = n_heads, a.kv = cache->n_kv_heads, a.group = n_heads / cache->n_kv_heads;
    a.hd = cache->head_dim, a.page_size = cache->page_size, a.n_pages = cache->n_pages, a.ld_table = ld_table;
    a.prefix = prefix_len, a.rows = p.rows, a.ptiles = p.ptiles, a.psplit = p.psplit, a.gtiles = p.gtiles, a.osplit = p.osplit, a.pparts = p.pparts;
    a.scale = scale2;
    cudaStream_t s = pick_stream(stream);
    const int cdt = cache->dtype;
    if (dtype == QMC_F32 && cdt == QMC_F32) return launch_attn<float, float>(a, p, dtype, cdt, c->num_sms, s);
    if (dtype == QMC_F32) return launch_attn<float, __half>(a, p, dtype, cdt, c->num_sms, s);
    if (dtype == QMC_F16) return launch_attn<__half, __half>(a, p, dtype, cdt, c->num_sms, s);
    return launch_attn<__nv_bfloat16, __nv_bfloat16>(a, p, dtype, cdt, c->num_sms, s);
}

}  // extern "C"

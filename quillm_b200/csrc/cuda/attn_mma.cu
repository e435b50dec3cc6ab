// Shared-prefix attention with matrix instructions (m16n8k16, float accumulators) over caches of 16-bit elements.
//
// A block of four warps takes a job's tile of 16, 32 or 64 query rows and streams its positions in tiles of kTP through a ring
// of kStages stages: 16-byte asynchronous copies, each position's row found through its page, slots past the range
// written as zeros and masked.  WM = tile / 16 warps cover the rows and WN = 4 / WM share a tile's positions, so that
// with few rows (own positions: a group's heads; a few beams) every warp has positions of its own; their maxima, sums
// and accumulators are joined through shared memory at the end.  Rows of K, V and Q lie in shared memory with 16-byte
// chunk c of row r at c ^ (r & 7): the eight rows of one matrix load hit distinct banks.
//
// Bound by the matrix instructions' issue and the loads from shared memory between them (512 rows over 32768 positions: 311 us, 221
// TFLOP/s; float rows, of twice the products each way, 474 us), with few rows by the copies (32 rows 45 us, 3.0 TB/s).  Its cases are
// those that the faster two cannot take: pages that are no multiple of 8, float rows in number, heads above 128.
//
// Weights are rounded to the cache's type for the second product: bf16 by half a step each at most, as the outputs are, fp16 likewise down to
// 2^-12 of the largest of its tile (Window).  Float queries over an fp16 cache: a row is scaled by a power of two and split in two halves
// q = qh + ql, the weights likewise, and each product is taken twice.  A score is off by 2^-21 of sum |q k|, a weight by 2^-22 of itself
// or 2^-23 of the largest of its tile.
#include "attn_prefix.cuh"

namespace qmc {
namespace {

constexpr int kTP = 64;  // positions per tile
template <int HDP>
__host__ __device__ constexpr int stages() {
    return HDP == 256 ? 2 : 3;
}

__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void ldm4t(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a)
                 : "memory");
}
// 16 bytes from global to shared memory, or zeros
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {  // all but the last N groups have landed
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <int HDP>
__host__ __device__ constexpr int stage_bytes() {
    return 2 * kTP * HDP * 2;
}
// query fragments stay in registers
template <int HDP, bool SPLIT>
__host__ __device__ constexpr bool q_in_registers() {
    return HDP * (SPLIT ? 2 : 1) <= 256;
}
// the ring; the query tile (two halves when split) lies behind it, or, where it is read into registers once, in the last
// stage, which the first tiles do not use.  The join at the end reuses the ring.
template <int HDP, int MT, bool SPLIT>
__host__ __device__ constexpr int smem_bytes() {
    return stages<HDP>() * stage_bytes<HDP>() + (q_in_registers<HDP, SPLIT>() ? 0 : (SPLIT ? 2 : 1) * MT * HDP * 2);
}

struct Scratch {
    int64_t slots[4][kTP];
    float qscale[64];  // what a row's scores are multiplied with
    float m[4][16], l[4][16];
};

// HDP: head_dim rounded up to 64, 128 or 256
template <typename T, typename CT, int HDP, int WM>
__device__ __forceinline__ void mma_job(const AttnArgs &a, const Job &jb, uint8_t *sm, Scratch &sc) {
    constexpr bool SPLIT = sizeof(T) == 4;
    constexpr int WN = 4 / WM, PW = kTP / WN, NT = PW / 8, KS = HDP / 16, CH = HDP / 8, RB = HDP * 2;
    constexpr int SB = stage_bytes<HDP>(), QB = 16 * WM * RB;
    constexpr bool QREG = q_in_registers<HDP, SPLIT>();
    constexpr int kStages = stages<HDP>(), QF = QREG ? KS : 1;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wm = warp / WN, wn = warp % WN;
    const int hd = a.hd, nch = hd / 8;  // chunks of a row in memory
    const uint32_t sm0 = smem_u32(sm), smq = sm0 + (QREG ? kStages - 1 : kStages) * SB;
    static_assert(!QREG || (SPLIT ? 2 : 1) * QB <= SB, "the query tile fits a stage");
    const int ntile = (jb.p1 - jb.p0 + kTP - 1) / kTP;
    auto place = [&](int row, int chunk) { return row * RB + ((chunk ^ (row & 7)) << 4); };

    auto find_slots = [&](int t) {
        if (tid < kTP) {
            const int p = jb.p0 + t * kTP + tid;
            sc.slots[t % (kStages + 1)][tid] = p < jb.p1 ? slot_of(a, jb.b, p) : -1;
        }
    };
    auto load_tile = [&](int t) {
        const uint32_t st = sm0 + (t % kStages) * SB;
        const int64_t *sl = sc.slots[t % (kStages + 1)];
        for (int i = tid; i < kTP * CH; i += 128) {
            const int row = i / CH, c = i % CH;
            if (c < nch) {
                const int64_t s = sl[row], off = s >= 0 ? (s * a.kv + jb.h) * hd + 8 * c : 0;
                copy16(st + place(row, c), (const CT *)a.kc + off, s >= 0);
                copy16(st + kTP * RB + place(row, c), (const CT *)a.vc + off, s >= 0);
            }
        }
    };
    // slots two tiles before they are loaded, tiles kStages - 1 before they are used; every tile commits a group, empty or not
#pragma unroll
    for (int t = 0; t < kStages; t++)
        if (t < ntile) find_slots(t);
    if (nch < CH)  // chunks past the head: zeros in every stage, never written again (rows of all stages follow one another)
        for (int i = tid; i < kStages * 2 * kTP * (CH - nch); i += 128)
            *(uint4 *)(sm + place(i / (CH - nch), nch + i % (CH - nch))) = make_uint4(0, 0, 0, 0);
    __syncthreads();
#pragma unroll
    for (int t = 0; t < kStages - 1; t++) {
        if (t < ntile) load_tile(t);
        copy_commit();
    }
    for (int r = warp; r < 16 * WM; r += 4) {  // the query tile
        const int rr = jb.r0 + r;
        const T *src = (const T *)a.q + (rr / a.group) * a.ldq + (int64_t)(jb.h * a.group + rr % a.group) * hd;
        float v[HDP / 32], mx = 0.0f, up = 1.0f;
#pragma unroll
        for (int i = 0; i < HDP / 32; i++) {
            v[i] = r < jb.nr && lane + 32 * i < hd ? to_f32(src[lane + 32 * i]) : 0.0f;
            mx = fmaxf(mx, fabsf(v[i]));
        }
        if (SPLIT) {  // times 2^-e, 2^e the power of two at or below the row's largest element: both halves stay normal
            const int e = min(126, max(-126, (__float_as_int(warp_max(mx)) >> 23) - 127));
            const float down = __int_as_float((127 - e) << 23);
            up = __int_as_float((127 + e) << 23);
#pragma unroll
            for (int i = 0; i < HDP / 32; i++) v[i] *= down;
        }
        if (lane == 0) sc.qscale[r] = up * a.scale;
#pragma unroll
        for (int i = 0; i < HDP / 32; i++) {
            const int d = lane + 32 * i;
            uint8_t *o = sm + (smq - sm0) + place(r, d / 8) + (d % 8) * 2;
            CT hi, lo;
            from_f32(v[i], &hi);
            *(CT *)o = hi;
            if (SPLIT) from_f32(v[i] - to_f32(hi), &lo), *(CT *)(o + QB) = lo;
        }
    }

    using W = Window<CT>;
    float o[HDP / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f}, high[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int d = 0; d < HDP / 8; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) o[d][i] = 0.0f;
    uint32_t qf[SPLIT ? 2 : 1][QF][4];
    // address parts of the matrix loads: A (rows lane % 16, column half lane / 16), B of K (rows by lane bits 0-2 and 4, column
    // half by bit 3), B of V transposed (rows lane % 16, column half lane / 16)
    const int ar = lane & 15, ac = lane >> 4, kr = (lane & 7) + ((lane >> 4) << 3), kc = (lane >> 3) & 1;
    float qs[2] = {0.0f, 0.0f};

    for (int t = 0; t < ntile; t++) {
        copy_wait<kStages - 2>();
        __syncthreads();  // tile t has landed for all; tile t - 1 is no longer read
        if (t == 0) {
            qs[0] = sc.qscale[16 * wm + (lane >> 2)], qs[1] = sc.qscale[16 * wm + (lane >> 2) + 8];
            if constexpr (QREG) {
#pragma unroll
                for (int h = 0; h < (SPLIT ? 2 : 1); h++)
#pragma unroll
                    for (int k = 0; k < KS; k++) ldm4(qf[h][k], smq + h * QB + place(16 * wm + ar, 2 * k + ac));
                __syncthreads();  // before the last stage is loaded
            }
        }
        if (t + kStages - 1 < ntile) load_tile(t + kStages - 1);
        copy_commit();
        if (t + kStages < ntile) find_slots(t + kStages);
        const uint32_t st = sm0 + (t % kStages) * SB;
        float s[NT][4];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[n][i] = 0.0f;
#pragma unroll
        for (int k = 0; k < KS; k++) {
            if constexpr (!QREG) {
#pragma unroll
                for (int h = 0; h < (SPLIT ? 2 : 1); h++) ldm4(qf[h][0], smq + h * QB + place(16 * wm + ar, 2 * k + ac));
            }
#pragma unroll
            for (int n = 0; n < NT; n += 2) {
                uint32_t b[4];
                ldm4(b, st + place(PW * wn + 8 * n + kr, 2 * k + kc));
                mma16(CT(), s[n], qf[0][QREG ? k : 0], b[0], b[1]);
                mma16(CT(), s[n + 1], qf[0][QREG ? k : 0], b[2], b[3]);
                if (SPLIT) {
                    mma16(CT(), s[n], qf[SPLIT][QREG ? k : 0], b[0], b[1]);
                    mma16(CT(), s[n + 1], qf[SPLIT][QREG ? k : 0], b[2], b[3]);
                }
            }
        }
        const int left = jb.p1 - jb.p0 - t * kTP - PW * wn;  // positions of this warp's part that exist
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[n][i] = 8 * n + 2 * (lane & 3) + (i & 1) < left ? s[n][i] * qs[i >> 1] : -INFINITY;
                mx[i >> 1] = fmaxf(mx[i >> 1], s[n][i]);
            }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
            mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
        }
        if (__any_sync(0xffffffffu, W::left_by(m[0], mx[0]) || W::left_by(m[1], mx[1]))) {  // the first time, and rarely again
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const float to = W::moved(m[i], mx[i], high[i]), by = to == -INFINITY ? 1.0f : ex2(m[i] - to);
                m[i] = to, l[i] *= by;
#pragma unroll
                for (int d = 0; d < HDP / 8; d++) o[d][2 * i] *= by, o[d][2 * i + 1] *= by;
            }
        }
        const float ref[2] = {m[0] == -INFINITY ? 0.0f : m[0], m[1] == -INFINITY ? 0.0f : m[1]};
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[n][i] = ex2(s[n][i] - ref[i >> 1]);
                l[i >> 1] += s[n][i];
            }
#pragma unroll
        for (int n = 0; n < NT; n += 2) {  // 16 positions: two score tiles are one A operand
            uint32_t p[4], pl[4];
            if constexpr (SPLIT) {
                float r[8];
                p[0] = pack2(CT(), s[n][0], s[n][1], &r[0]), p[1] = pack2(CT(), s[n][2], s[n][3], &r[2]);
                p[2] = pack2(CT(), s[n + 1][0], s[n + 1][1], &r[4]);
                p[3] = pack2(CT(), s[n + 1][2], s[n + 1][3], &r[6]);
#pragma unroll
                for (int i = 0; i < 4; i++) pl[i] = pack2(CT(), r[2 * i], r[2 * i + 1]);
            } else {
                p[0] = pack2(CT(), s[n][0], s[n][1]), p[1] = pack2(CT(), s[n][2], s[n][3]);
                p[2] = pack2(CT(), s[n + 1][0], s[n + 1][1]), p[3] = pack2(CT(), s[n + 1][2], s[n + 1][3]);
            }
#pragma unroll
            for (int d = 0; d < HDP / 8; d += 2) {
                uint32_t b[4];
                ldm4t(b, st + kTP * RB + place(PW * wn + 8 * n + ar, d + ac));
                mma16(CT(), o[d], p, b[0], b[1]);
                mma16(CT(), o[d + 1], p, b[2], b[3]);
                if constexpr (SPLIT) {
                    mma16(CT(), o[d], pl, b[0], b[1]);
                    mma16(CT(), o[d + 1], pl, b[2], b[3]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    }
    const int64_t all = (int64_t)a.n_seq * a.heads;
    if constexpr (WN > 1) {  // join the warps that share rows: maxima and sums first, then the rescaled accumulators
        copy_wait<0>();
        __syncthreads();  // the ring is no longer read or written
#pragma unroll
        for (int i = 0; i < 2; i++)
            if ((lane & 3) == 0) sc.m[warp][(lane >> 2) + 8 * i] = m[i], sc.l[warp][(lane >> 2) + 8 * i] = l[i];
        __syncthreads();
        float *part = (float *)sm;  // [4 warps][16][HDP], the columns rotated by 8 a row
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int r = (lane >> 2) + 8 * i;
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < WN; w++) M = fmaxf(M, sc.m[wm * WN + w][r]);
            const float c = M == -INFINITY ? 0.0f : ex2(m[i] - M);
#pragma unroll
            for (int d = 0; d < HDP / 8; d++) {
                const int col = (8 * d + 2 * (lane & 3) + 8 * r) % HDP;
                *(float2 *)(part + (warp * 16 + r) * HDP + col) = make_float2(o[d][2 * i] * c, o[d][2 * i + 1] * c);
            }
        }
        __syncthreads();
        for (int i = tid; i < 16 * WM * HDP; i += 128) {
            const int row = i / HDP, d = i % HDP, g = row / 16, r = row % 16;
            if (row >= jb.nr || d >= hd) continue;
            float M = -INFINITY, x = 0.0f, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < WN; w++) {
                M = fmaxf(M, sc.m[g * WN + w][r]);
                x += part[((g * WN + w) * 16 + r) * HDP + (d + 8 * r) % HDP];
            }
            const int64_t to = jb.part * all + out_row(a, jb.h, jb.r0 + row);
            a.po[to * hd + d] = x;
            if (d == 0) {
                if (M > -INFINITY)
#pragma unroll
                    for (int w = 0; w < WN; w++) sum += sc.l[g * WN + w][r] * ex2(sc.m[g * WN + w][r] - M);
                a.ml[to] = make_float2(M, sum);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int row = 16 * wm + (lane >> 2) + 8 * i;
            if (row >= jb.nr) continue;
            const int64_t to = jb.part * all + out_row(a, jb.h, jb.r0 + row);
            if ((lane & 3) == 0) a.ml[to] = make_float2(m[i], l[i]);
#pragma unroll
            for (int d = 0; d < HDP / 8; d++) {
                const int col = 8 * d + 2 * (lane & 3);
                if (col < hd) *(float2 *)(a.po + to * hd + col) = make_float2(o[d][2 * i], o[d][2 * i + 1]);
            }
        }
    }
}

// WM: 16-row groups of a prefix job's tile; own jobs, which come here with heads above 128 alone, have one
template <typename T, typename CT, int HDP, int WM>
__global__ void __launch_bounds__(128, 2) attn_mma_kernel(const AttnArgs a) {
    extern __shared__ __align__(128) uint8_t sm[];
    __shared__ Scratch sc;
    const Job jb = job_of(a, blockIdx.x, 16 * WM, 16, kTP);
    pdl_launch_dependents();
    if (HDP <= 128 || (WM > 1 && jb.b < 0)) mma_job<T, CT, HDP, WM>(a, jb, sm, sc);
    else mma_job<T, CT, HDP, 1>(a, jb, sm, sc);
    // launched beside the prefix's kernel, this grid ends after it, which the join relies on: one block waits, the others make room
    if (blockIdx.x == 0) pdl_wait();
}

template <typename T, typename CT, int HDP, int WM>
int launch_t(const AttnArgs &a, bool after, cudaStream_t s) {
    auto fn = attn_mma_kernel<T, CT, HDP, WM>;
    constexpr int smem = smem_bytes<HDP, 16 * WM, sizeof(T) == 4>();
    static_assert(4 * 16 * HDP * 4 <= stages<HDP>() * stage_bytes<HDP>(), "the join fits the ring");
    static std::atomic<bool> done[64];
    if (const int rc = raise_smem(fn, smem, done)) return rc;
    const int64_t jobs = (int64_t)a.kv * a.ptiles * a.psplit + (int64_t)a.n_seq * a.kv * a.gtiles * a.osplit;
    if (jobs > INT32_MAX) return set_error(QMC_EINVAL, "attn_prefix: too many blocks");
    return jobs ? launch_after(fn, dim3((unsigned)jobs), 128, smem, s, after, a) : QMC_OK;
}
template <typename T, typename CT, int HDP>
int launch_m(const AttnArgs &a, bool after, cudaStream_t s) {
    const int tile = attn_mma_tile(a.rows);
    if constexpr (HDP > 128)  // narrower heads of so few rows go to attn_warp
        if (tile == 16) return launch_t<T, CT, HDP, 1>(a, after, s);
    return tile == 32 ? launch_t<T, CT, HDP, 2>(a, after, s) : launch_t<T, CT, HDP, 4>(a, after, s);
}
template <typename T, typename CT>
int launch_h(const AttnArgs &a, bool after, cudaStream_t s) {
    if (a.hd <= 64) return launch_m<T, CT, 64>(a, after, s);
    if (a.hd <= 128) return launch_m<T, CT, 128>(a, after, s);
    return launch_m<T, CT, 256>(a, after, s);
}

}  // namespace

int attn_mma_tile(int rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

int launch_attn_mma(const AttnArgs &a, int dtype, int cdt, bool after, cudaStream_t s) {
    if (dtype == QMC_F32) return launch_h<float, __half>(a, after, s);
    return cdt == QMC_F16 ? launch_h<__half, __half>(a, after, s) : launch_h<__nv_bfloat16, __nv_bfloat16>(a, after, s);
}

}  // namespace qmc

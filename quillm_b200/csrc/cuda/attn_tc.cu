// The prefix part of the shared-prefix attention on the 5th-generation tensor cores, for many query rows per KV head:
// tcgen05.mma with scores and accumulators in tensor memory (TMEM).
//
// Per 128 query rows and 128 positions: S = Q K^T (M = 128 rows, N = 128 positions) into 128 TMEM columns; eight warps, two
// threads per row with 64 positions each, turn S into weights P = 2^(scale S - m) and write them over S as 16-bit pairs;
// O += P V with P read from TMEM as the A operand and V from shared memory as it lies in the cache ([position][dim], an
// MN-major operand).  A row's reference m moves only when a thread's weights show that the scores have left the window around it
// (Window): sums above what its type or l can hold, or, in fp16, too small to keep a weight's bits.  Then the row's two warps rescale
// its O in TMEM and take the tile again, which after a row's first tile is rare, so O normally stays where it is until the end.
//
// A block runs two streams of such tiles, so that the tensor cores work on one while the other's warps take its exponentials.
// PAIR: the streams are two row tiles over the same positions (each K and V tile is read once for 256 rows).  Otherwise, with
// at most 128 rows, they take the range's position tiles in turn and are joined at the end.
//
// Bound by the chain of a stream, scores 500 cycles, weights 1300, product 500 and the waits between (3500 cycles for the two tiles
// of PAIR, in which the tensor cores have 2050 to do), and before that by the start and the end of a block, 5 us together.
// 512 rows of 8 heads over 32768 positions in 8 ranges: 77 us, 890 TFLOP/s of the measured 1613; beside own jobs, in 7: 84 us.  128
// rows 33 us, 4.1 TB/s.  Tried and not kept, each against the 80 us or 83 us of its day: four threads a row (84 us), copies by threads
// instead of TMA (192 us), one wait with a lane for each barrier (97 us).
//
// Warps 0-15: weights; 16: TMA; 17: one lane issues the MMAs.  A box is a run of rows within a page (the largest power of two that
// divides the page size, 8 to 128 of them) and 64 dimensions wide, the 128-byte swizzle's row.  Dimensions past the head are the next
// head's, or zeros: for the scores Q has zeros there, in O they are not stored.  Rows past the range, which a box may bring along, are
// masked in the scores and overwritten with zeros in the last V tile, since what lies there need not be finite.
// Every wait is bounded: after a timeout a role raises the error word and falls through to the end, where the copies and MMAs in
// flight are waited for (bounded) and the TMEM is freed.  A role that has stopped leaves the others to their own timeouts.
#include <algorithm>

#include "attn_prefix.cuh"
#include "matmul_tc.cuh"

namespace qmc {
namespace {

constexpr int kM = 128, kN = 128;  // rows and positions of a tile
constexpr int kCopyWarp = 16, kMmaWarp = 17, kThreads = 18 * 32;  // warps 0-15: weights
// what a thread's weights may add up to, in bf16 the 64 of a tile, in fp16 each eight, of which none then passes the type's largest (level
// scores at the reference's 2^10: 2^13); and in fp16 the least that a tile's must
template <typename CT>
__host__ __device__ constexpr float most_of() {
    return Window<CT>::kHalf ? 65504.0f : 256.0f;
}
constexpr float kLeast = 0.25f;
constexpr float kLiftSum = 12.5f;  // fp16: a tile whose eight weights pass 65504 has one at 2^12.99 or above

template <int HDP>
__host__ __device__ constexpr int tile_bytes() {  // of Q, K or V
    return 128 * HDP * 2;
}
// tiles of the ring, K and V in turn: what is left of shared memory beside the query tiles
template <int HDP, bool PAIR>
__host__ __device__ constexpr int ring() {
    return PAIR ? 5 : 6;
}
template <int HDP, bool PAIR>
__host__ __device__ constexpr int smem_bytes() {
    return 1024 + ((PAIR ? 2 : 1) + ring<HDP, PAIR>()) * tile_bytes<HDP>();
}

__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap *map, int x, int y, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
        "l"((uint64_t)map), "r"(x), "r"(y), "r"(smem_u32(bar))
        : "memory");
}

// shared-memory operand descriptors, 128-byte swizzle, from the address in 16-byte units.  K-major (rows of 64 elements, eight-row
// groups 1024 bytes apart); MN-major (64 elements of M or N a row, eight-row groups of K 1024 bytes apart, the next 64
// elements a panel further).  Only the low word holds an address, so the next operand is an addition to it.
__device__ __forceinline__ uint64_t desc(uint32_t low) {
    constexpr uint32_t kHigh = (1024 >> 4) | (1u << 14) | (2u << 29);
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(low), "n"(kHigh));
    return d;
}
constexpr uint32_t kLowK = 1u << 16, kLowMN = (uint32_t)(128 * 128 >> 4) << 16;
// float accumulator, A and B of one 16-bit type; bmn: B is MN-major
__device__ __forceinline__ constexpr uint32_t idesc(int n, bool bmn, bool bf16) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((bmn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(kM >> 4) << 24);
}
__device__ __forceinline__ bool elect_one() {  // true for one lane of a converged warp
    uint32_t p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.b32 %0, 1, 0, p;\n}\n" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t ad, uint64_t bd, uint32_t id, uint32_t acc) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
                 "l"(ad), "l"(bd), "r"(id), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t at, uint64_t bd, uint32_t id, uint32_t acc) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
                 "r"(at), "l"(bd), "r"(id), "r"(acc)
                 : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// 32 consecutive TMEM columns of this thread's lane; the load and its wait are one statement, so that nothing reads the
// registers between the two
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t *r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
        "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
        "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// a bit for each of the 32 positions from `at` that are among the first `left`
__device__ __forceinline__ uint32_t live_bits(int left, int at) {
    return left >= at + 32 ? 0xffffffffu : left <= at ? 0u : (1u << (left - at)) - 1u;
}
// pairs of floats, one instruction each
__device__ __forceinline__ uint64_t pair_of(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void of_pair(uint64_t v, float &x, float &y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// x * y + c held in [0, 1]
__device__ __forceinline__ float fma_sat(float x, float y, float c) {
    float r;
    asm("fma.rn.sat.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(c));
    return r;
}
// 2^t of a pair without the special-function unit.  t comes as x = (t + 112) / 128, held in [0, 1] by the instruction that forms it: below
// 2^-112 a weight counts for nothing, and 2^16 is above what a tile's sum may reach, so that the reference moves (beyond 127 the
// exponent would run into the sign).  x is off by 2^-25, the result by 2^-18.5 of itself.  n = t rounded to an integer (as the low
// bits of t + 1.5 * 2^23), 2^(t - n) by the minimax polynomial of the relative error on [-1/2, 1/2] (degree 4: 2^-18.5; one of degree 3,
// 2^-13.7, would do for bf16 weights but not for their float sum), n added to its exponent
constexpr float kSpan = 128.0f, kBelow = 112.0f;
__device__ __forceinline__ void ex2_pair(uint64_t x, float &p0, float &p1) {
    const float kRnd = 12582912.0f;
    const uint64_t span = pair_of(kSpan, kSpan), rnd = pair_of(kRnd - kBelow, kRnd - kBelow);
    const uint64_t up = fma2(x, span, rnd), f = fma2(x, span, fma2(up, pair_of(-1.0f, -1.0f), rnd));
    uint64_t v = fma2(f, pair_of(0.00957010220736f, 0.00957010220736f), pair_of(0.05591785907745f, 0.05591785907745f));
    v = fma2(f, v, pair_of(0.24024744331837f, 0.24024744331837f));
    v = fma2(f, v, pair_of(0.69312179088593f, 0.69312179088593f));
    v = fma2(f, v, pair_of(0.99999928474426f, 0.99999928474426f));
    float u0, u1, v0, v1;
    of_pair(up, u0, u1);
    of_pair(v, v0, v1);
    p0 = __int_as_float(__float_as_int(v0) + (__float_as_int(u0) << 23));
    p1 = __int_as_float(__float_as_int(v1) + (__float_as_int(u1) << 23));
}
// a thread's 32 scores of a row: 2^(scale s - m) as 16-bit pairs in pk, and their sum before rounding; most: the largest sum of eight of
// them.  The special-function unit gives 16 results a cycle and SM: three of every eight pairs, spread among the others, go to the FMA
// pipe instead.  MASK: only the first `left` positions exist
template <typename CT, bool MASK>
__device__ __forceinline__ float row_weights(const uint32_t (&x)[32], uint32_t *pk, float scale, float m, int left, float &most) {
    const uint64_t sc = pair_of(scale, scale), mm = pair_of(-m, -m);
    const float part = scale * (1.0f / kSpan), from = (kBelow - m) * (1.0f / kSpan);
    const uint32_t live = MASK ? live_bits(left, 0) : 0xffffffffu;
    uint64_t sum[2] = {0, 0};
#pragma unroll
    for (int k = 0; k < 32; k += 2) {
        const float s0 = __uint_as_float(x[k]), s1 = __uint_as_float(x[k + 1]);
        float p0, p1;
        if (!MASK && (k >> 1) % 8 % 3 == 1) {
            ex2_pair(pair_of(fma_sat(s0, part, from), fma_sat(s1, part, from)), p0, p1);
        } else {
            float t0, t1;
            of_pair(fma2(pair_of(s0, s1), sc, mm), t0, t1);
            if (MASK) {
                t0 = live >> k & 1u ? t0 : -INFINITY;
                t1 = live >> (k + 1) & 1u ? t1 : -INFINITY;
            }
            p0 = ex2(t0), p1 = ex2(t1);
        }
        sum[(k >> 1) & 1] = add2(sum[(k >> 1) & 1], pair_of(p0, p1));
        pk[k / 2] = pack2(CT(), p0, p1);
    }
    float s0, s1;
    if constexpr (Window<CT>::kHalf) {
        float s2, s3;
        of_pair(sum[0], s0, s1), of_pair(sum[1], s2, s3);
        asm("max.f32 %0, %0, %1, %2;" : "+f"(most) : "f"(s0), "f"(s1));
        asm("max.f32 %0, %0, %1, %2;" : "+f"(most) : "f"(s2), "f"(s3));
    }
    of_pair(add2(sum[0], sum[1]), s0, s1);
    return s0 + s1;
}
// barrier `id` of the two warps of 32 rows: the or of their verdicts
__device__ __forceinline__ bool rows_any(int id, bool v) {
    int r;
    asm volatile(
        "{\n .reg .pred p, q;\n setp.ne.b32 p, %1, 0;\n barrier.cta.red.or.pred q, %2, 64, p;\n selp.s32 %0, 1, 0, q;\n}\n"
        : "=r"(r)
        : "r"((int)v), "r"(id)
        : "memory");
    return r != 0;
}
struct Shared {
    uint64_t full[6], empty[6], sfull[2], pfull[2], ofin[2], qready, vlast, drain;
    float top[2][kM];  // the larger of a row's two threads
    uint32_t tmem;
};

template <typename CT, int HDP, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1) attn_tc_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const AttnArgs a, int box) {
    extern __shared__ __align__(128) uint8_t sm_raw[];
    __shared__ Shared sh;
    constexpr int NS = ring<HDP, PAIR>(), TB = tile_bytes<HDP>(), CH = HDP / 8, PANEL = 128 * 128;  // chunks of a row; bytes of 64 dimensions
    constexpr bool BF = !(sizeof(CT) == 2 && __is_same(CT, __half));
    const uint32_t smq = (smem_u32(sm_raw) + 1023) & ~1023u, smk = smq + (PAIR ? 2 : 1) * TB;
    uint8_t *const base = sm_raw + (smq - smem_u32(sm_raw));
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int hd = a.hd, nch = hd / 8;
    const Job jb = job_of(a, blockIdx.x, PAIR ? 2 * kM : kM, 0, kN);
    const int ntile = (jb.p1 - jb.p0 + kN - 1) / kN;
    // the copy warp's lane i finds the pages of box i of a tile; the first tile's are on their way before anything else
    const int groups = kN / box;
    auto page_at = [&](int p) { return p < jb.p1 ? a.prefix_pages[p / a.page_size] : -1; };
    const int first = warp == kCopyWarp ? page_at(jb.p0 + lane % groups * box) : -1;
    // chunk c of row r of a tile, 128-byte swizzle
    auto place = [](int r, int c) { return (c >> 3) * PANEL + r * 128 + (((c & 7) ^ (r & 7)) << 4); };

    if (tid == 0) {
        for (int i = 0; i < NS; i++) {
            mbar_init(&sh.full[i], 1);   // the expected bytes
            mbar_init(&sh.empty[i], 1);  // a commit
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.sfull[i], 1);
            mbar_init(&sh.pfull[i], 8);  // the stream's warps
            mbar_init(&sh.ofin[i], 1);
        }
        mbar_init(&sh.qready, 32 * kCopyWarp);
        mbar_init(&sh.vlast, 1);
        mbar_init(&sh.drain, 1);
        fence_mbar_init();
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    __syncthreads();  // the barriers
    pdl_launch_dependents();
    // all 512 columns are this block's, so they start at 0: S (and P) of stream w at 128 w, O at 256 + HDP w

    if (warp == kCopyWarp) {  // ---------------------------------------------------------------- TMA
        // one lane issues the copies: lanes that each issue their own take 90 cycles apiece
        const int g = lane % groups;
        const bool lead = elect_one();
        int issued = 0, page = first;
        auto issue = [&](int row, int left, int u, const CUtensorMap *map) {  // tile u of the sequence K0 V0 K1 V1 ...
            const int at = u % NS, here = min(groups, (left + box - 1) / box);
            if (u >= NS && __any_sync(0xffffffffu, !mbar_wait(&sh.empty[at], (u / NS - 1) & 1))) {
                if (lane == 0) raise_error(a.err, kErrMbarTimeout);
                return false;
            }
            if (lead) mbar_arrive_tx(&sh.full[at], here * (HDP / 64) * box * 128);
#pragma unroll 4
            for (int i = 0; i < here; i++) {
                const int y = __shfl_sync(0xffffffffu, row, i);
                if (lead)
#pragma unroll
                    for (int k = 0; k < HDP / 64; k++)
                        tma_2d(smk + at * TB + k * PANEL + i * box * 128, map, jb.h * hd + 64 * k, y, &sh.full[at]);
            }
            issued = u + 1;
            return true;
        };
        for (int j = 0; j < ntile; j++) {
            const int p = jb.p0 + j * kN + g * box, left = jb.p1 - jb.p0 - j * kN;
            int row = -kN;  // a page outside the pool: rows that do not exist read as zeros
            if (p < jb.p1) {
                if (page >= 0 && page < a.n_pages) row = page * a.page_size + p % a.page_size;
                else raise_error(a.err, kErrBadIndex);
            }
            page = page_at(p + kN);
            if (!issue(row, left, 2 * j, &kmap) || !issue(row, left, 2 * j + 1, &vmap)) break;
            if (left < kN) {  // the last V tile: zeros behind the range, once its copies have landed
                const int u = 2 * j + 1, at = u % NS;
                if (__any_sync(0xffffffffu, !mbar_wait(&sh.full[at], (u / NS) & 1))) {
                    if (lane == 0) raise_error(a.err, kErrMbarTimeout);
                    break;
                }
                for (int i = lane; i < (kN - left) * CH; i += 32)
                    *(uint4 *)(base + (smk - smq) + at * TB + place(left + i / CH, i % CH)) = make_uint4(0, 0, 0, 0);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.vlast);
            }
        }
        // no copy may still be landing when the block exits
        const long long t0 = clock64();
        for (int u = max(0, issued - NS); u < issued; u++)
            if (!mbar_wait_since(&sh.full[u % NS], (u / NS) & 1, t0)) {
                if (lane == 0) raise_error(a.err, kErrMbarTimeout);
                break;
            }
        __syncwarp();
    } else if (warp == kMmaWarp) {  // ---------------------------------------------------------------- MMA issuer
        // the whole warp runs this, one lane issues: addresses and descriptors stay uniform, where a lone lane would move each
        // of them to the uniform registers that the instruction takes.  It shares its issue slots with four busy warps: a wait that
        // is over costs a few instructions, and the ring's places are counted along, not divided for.
        const bool lead = elect_one();
        auto wait = [&](uint64_t *bar, uint32_t parity) {
            if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
            const bool ok = __all_sync(0xffffffffu, mbar_wait(bar, parity));
            if (!ok && lane == 0) raise_error(a.err, kErrMbarTimeout);
            return ok;
        };
        struct Place {  // of the next K or V tile in the ring
            uint32_t at, parity;
        } k{0, 0}, v{1, 0};
        auto advance = [&](Place &p) {
            p.at += 2;
            if (p.at >= NS) p.at -= NS, p.parity ^= 1;
        };
        const bool cut = (jb.p1 - jb.p0) % kN != 0;  // the last V tile waits for its zeros too
        auto v_landed = [&](int j) { return wait(&sh.full[v.at], v.parity) && (!cut || j < ntile - 1 || wait(&sh.vlast, 0)); };
        auto scores = [&](int w) {  // S_w = Q_w K^T
            const uint32_t qd = (smq + (PAIR ? w : 0) * TB) / 16 | kLowK, kd = (smk + k.at * TB) / 16 | kLowK;
            if (lead) {
#pragma unroll
                for (int i = 0; i < HDP / 16; i++) {
                    const uint32_t off = ((i >> 2) * PANEL + (i & 3) * 32) / 16;
                    mma_ss(128 * w, desc(qd + off), desc(kd + off), idesc(kN, false, BF), i > 0);
                }
                mma_commit(&sh.sfull[w]);
                if (!PAIR || w == 1) mma_commit(&sh.empty[k.at]);
            }
            if (!PAIR || w == 1) advance(k);
        };
        auto weigh = [&](int w, bool first) {  // O_w += P_w V
            const uint32_t vd = (smk + v.at * TB) / 16 | kLowMN;
            if (lead) {
#pragma unroll
                for (int i = 0; i < kN / 16; i++)
                    mma_ts(256 + HDP * w, 128 * w + 8 * i, desc(vd + i * (16 * 128 / 16)), idesc(HDP, true, BF), !first || i > 0);
                if (!PAIR || w == 1) mma_commit(&sh.empty[v.at]);
            }
            if (!PAIR || w == 1) advance(v);
        };
        constexpr int step = PAIR ? 1 : 2;  // tiles from one of a stream's to its next
        bool ok = wait(&sh.qready, 0);
        for (int w = 0; w < 2 && ok; w++) {
            if ((PAIR ? 0 : w) >= ntile) continue;
            ok = wait(&sh.full[k.at], k.parity);
            if (ok) scores(w);
        }
        ok = ok && (ntile == 0 || v_landed(0));
        for (int i = 0; i * step < ntile && ok; i++)
#pragma unroll
            for (int w = 0; w < 2; w++) {
                const int j = PAIR ? i : 2 * i + w;
                if (!ok || j >= ntile) break;
                ok = wait(&sh.pfull[w], i & 1u);
                if (!ok) break;
                tc_fence_after();
                weigh(w, i == 0);
                // the tiles of what follows, waited for while the tensor cores have these products to do: the V tile of the next
                // step (PAIR: with the second stream), then the K tile of the scores
                if ((!PAIR || w == 1) && j + 1 < ntile && !(ok = v_landed(j + 1))) break;
                if (j + step < ntile) {
                    if ((!PAIR || w == 0) && !(ok = wait(&sh.full[k.at], k.parity))) break;
                    scores(w);
                } else if (lead) {
                    mma_commit(&sh.ofin[w]);
                }
            }
        // nothing may be in flight when the TMEM is freed
        if (lead) mma_commit(&sh.drain);
        if (!mbar_wait(&sh.drain, 0) && lane == 0) raise_error(a.err, kErrMbarTimeout);
        __syncwarp();
    } else {  // ---------------------------------------------------------------- weights
        // the query tiles first; rows past the last and chunks past the head are zeros
        const bool vec = a.ldq % 8 == 0 && (uintptr_t)a.q % 16 == 0;
        constexpr int NQ = (PAIR ? 2 : 1) * kM * CH / (32 * kCopyWarp);  // chunks of a thread, all on their way at once
        uint4 x[NQ];
        const CT *const q0 = (const CT *)a.q + (int64_t)jb.h * a.group * hd + 8 * (tid % CH);
#pragma unroll
        for (int u = 0; u < NQ; u++) {
            const int r = tid / CH + u * (32 * kCopyWarp / CH), b = (jb.r0 + r) / a.group, g = (jb.r0 + r) - b * a.group;
            const CT *src = q0 + b * a.ldq + (int64_t)g * hd;
            x[u] = make_uint4(0, 0, 0, 0);
            if (r < jb.nr && tid % CH < nch) {
                if (vec) {
                    x[u] = *(const uint4 *)src;
                } else {
                    const uint16_t *e = (const uint16_t *)src;
                    x[u] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < NQ; u++) {
            const int r = tid / CH + u * (32 * kCopyWarp / CH);
            *(uint4 *)(base + (r / kM) * TB + place(r % kM, tid % CH)) = x[u];
        }
        fence_proxy_async();
        mbar_arrive(&sh.qready);

        // warp 8 w + 4 half + q: stream w, rows 32 q .. + 31 (the TMEM lanes it may access), half of the positions of each tile.
        // The two warps of a row meet once a tile: before either writes weights over scores that the other reads, and to
        // agree on the row's reference.  A warp whose wait has expired goes on through the barriers without touching TMEM.
        const int w = warp >> 3, half = (warp >> 2) & 1, row = 32 * (warp & 3) + lane, id = 1 + 4 * w + (warp & 3);
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16, ts = lanes + 128 * w, to = lanes + 256 + HDP * w + HDP / 2 * half;
        const int mine = PAIR ? ntile : (ntile - w + 1) / 2;
        auto largest = [&](float v) {
            rows_any(id, false);  // both have read what it held
            if (half == 0) sh.top[w][row] = v;
            rows_any(id, false);
            if (half == 1) sh.top[w][row] = v = fmaxf(v, sh.top[w][row]);
            rows_any(id, false);
            return sh.top[w][row];
        };
        using W = Window<CT>;
        float m = 0.0f, l = 0.0f, high = -INFINITY;
        bool ok = true;
        for (int i = 0; i < mine; i++) {
            const int j = PAIR ? i : 2 * i + w, left = jb.p1 - jb.p0 - j * kN - 64 * half;  // of this thread's positions
            if (ok && __any_sync(0xffffffffu, !mbar_wait(&sh.sfull[w], i & 1u))) {
                if (lane == 0) raise_error(a.err, kErrMbarTimeout);
                ok = false;
            }
            tc_fence_after();
            uint32_t pk[32];
            float sum = 0.0f, most = 0.0f;
            for (int again = i == 0 ? -1 : 0;; again++) {  // -1: no reference yet
                if (ok && again >= 0) {
                    sum = most = 0.0f;
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        uint32_t x[32];
                        tmem_ld32(ts + 64 * half + 32 * c, x);
                        sum += left >= 64 ? row_weights<CT, false>(x, pk + 16 * c, a.scale, m, left, most)
                                          : row_weights<CT, true>(x, pk + 16 * c, a.scale, m, left - 32 * c, most);
                    }
                }
                // both have read the scores; does a row leave its window (NaN sums count as that)?  After a move none does
                bool out;
                if constexpr (W::kHalf) out = !(most <= most_of<CT>()) || !(sum == sum) || (sum < kLeast && left > 0);
                else out = !(sum <= most_of<CT>());
                if (!rows_any(id, again < 0 || (again == 0 && i > 0 && out))) break;
                float top = -INFINITY;
                if (ok)
#pragma unroll 1
                    for (int c = 0; c < 2; c++) {
                        uint32_t x[32];
                        tmem_ld32(ts + 64 * half + 32 * c, x);
                        const uint32_t live = live_bits(left, 32 * c);
#pragma unroll
                        for (int k = 0; k < 32; k++) top = fmaxf(top, live >> k & 1u ? __uint_as_float(x[k]) : -INFINITY);
                    }
                top = largest(top) * a.scale;
                if (again < 0) {
                    m = high = top == -INFINITY ? 0.0f : top - W::kTop;
                    continue;
                }
                // O (half of its columns each) holds the tiles before this one, whose product is complete (this tile's scores
                // were committed after it)
                const float to_m = W::moved(m, top, high, kLiftSum), by = ex2(m - to_m);
                m = to_m, l *= by;
                if (ok)
#pragma unroll 1
                    for (int c = 0; c < HDP / 64; c++) {
                        uint32_t x[32];
                        tmem_ld32(to + 32 * c, x);
#pragma unroll
                        for (int k = 0; k < 32; k++) x[k] = __float_as_uint(__uint_as_float(x[k]) * by);
                        tmem_st32(to + 32 * c, x);
                    }
            }
            l += sum;
            if (ok) {
                tmem_st32(ts + 32 * half, pk);
                tmem_wait_st();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.pfull[w]);
        }
        if (ok && mine > 0 && __any_sync(0xffffffffu, !mbar_wait(&sh.ofin[w], 0))) {
            if (lane == 0) raise_error(a.err, kErrMbarTimeout);
            ok = false;
        }
        tc_fence_after();
        // The last products of both streams are complete, so the ring is free: m and l of the rows, and O, so that it leaves in
        // whole lines.  16-byte chunk c of row r lies at c ^ (r & 7).
        asm volatile("bar.sync 9, 512;" ::: "memory");
        float *const ml = (float *)(base + (smk - smq));  // [stream][m, l of either half][row]
        uint8_t *const rows = (uint8_t *)(ml + 2 * 3 * kM), *const own = rows + w * (kM * HDP * 4);
        if (half == 0) ml[3 * w * kM + row] = mine > 0 && ok ? m : -INFINITY;
        ml[(3 * w + 1 + half) * kM + row] = mine > 0 && ok ? l : 0.0f;
#pragma unroll 1
        for (int c = 0; c < HDP / 64; c++) {
            uint32_t x[32];
            if (ok && mine > 0) {
                tmem_ld32(to + 32 * c, x);
            } else {
#pragma unroll
                for (int k = 0; k < 32; k++) x[k] = 0;
            }
#pragma unroll
            for (int k = 0; k < 8; k++)
                *(uint4 *)(own + row * (HDP * 4) + (((HDP / 8 * half + 8 * c + k) ^ (row & 7)) << 4)) =
                    make_uint4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]);
        }
        asm volatile("bar.sync 9, 512;" ::: "memory");
        // lane i: the place and the factors of the warp's row i
        constexpr int RW = (PAIR ? 2 : 1) * kM / 16;  // rows a warp stores
        const int64_t all = (int64_t)a.n_seq * a.heads;
        const int r0 = RW * warp, here = min(RW, jb.nr - r0), s = PAIR ? r0 / kM : 0;
        int64_t at = 0;
        float c0 = 1.0f, c1 = 0.0f;
        if (lane < here) {
            at = jb.part * all + out_row(a, jb.h, jb.r0 + r0 + lane);
            const float *h = ml + 3 * s * kM + (r0 + lane) % kM;
            float M = h[0], L = h[kM] + h[2 * kM];
            if (!PAIR) {  // the two streams' parts of the row as one
                const float m0 = M, m1 = h[3 * kM];
                M = fmaxf(m0, m1);
                if (M > -INFINITY) c0 = ex2(m0 - M), c1 = ex2(m1 - M);
                L = L * c0 + (h[4 * kM] + h[5 * kM]) * c1;
            }
            a.ml[at] = make_float2(M, L);
        }
#pragma unroll 4
        for (int k = 0; k < RW; k++) {
            const int64_t to = __shfl_sync(0xffffffffu, at, k);
            const float f0 = __shfl_sync(0xffffffffu, c0, k), f1 = __shfl_sync(0xffffffffu, c1, k);
            if (k < here && 4 * lane < hd) {
                const int rr = (r0 + k) % kM, o = rr * (HDP * 4) + ((lane ^ (rr & 7)) << 4);
                float4 v = *(const float4 *)(rows + s * (kM * HDP * 4) + o);
                if (!PAIR) {
                    const float4 u = *(const float4 *)(rows + kM * HDP * 4 + o);
                    v = make_float4(v.x * f0 + u.x * f1, v.y * f0 + u.y * f1, v.z * f0 + u.z * f1, v.w * f0 + u.w * f1);
                }
                *(float4 *)(a.po + to * hd + 4 * lane) = v;
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(sh.tmem), "r"(512) : "memory");
    }
}

template <typename CT, int HDP, bool PAIR>
int launch_t(const AttnArgs &a, const CUtensorMap &kmap, const CUtensorMap &vmap, int box, cudaStream_t s) {
    auto fn = attn_tc_kernel<CT, HDP, PAIR>;
    constexpr int smem = smem_bytes<HDP, PAIR>();
    static_assert(smem + sizeof(Shared) <= 232448, "shared memory of a block");
    static std::atomic<bool> done[64];
    if (const int rc = raise_smem(fn, smem, done)) return rc;
    const int64_t jobs = (int64_t)a.kv * a.ptiles * a.psplit;
    if (jobs > INT32_MAX) return set_error(QMC_EINVAL, "attn_prefix: too many blocks");
    fn<<<(unsigned)jobs, kThreads, smem, s>>>(kmap, vmap, a, box);
    QMC_LAUNCH_CHECK();
    return QMC_OK;
}
template <typename CT>
int launch_h(const AttnArgs &a, CUtensorMapDataType type, cudaStream_t s) {
    const int box = attn_tc_box(a.page_size);
    const int64_t slots = (int64_t)a.n_pages * a.page_size, row = (int64_t)a.kv * a.hd;
    CUtensorMap kmap, vmap;
    int rc;
    if ((rc = make_tensor_map(&kmap, a.kc, type, row, slots, row * 2, 64, box, true)) ||
        (rc = make_tensor_map(&vmap, a.vc, type, row, slots, row * 2, 64, box, true)))
        return rc;
    const bool pair = a.rows > kM;
    if (a.hd <= 64) return pair ? launch_t<CT, 64, true>(a, kmap, vmap, box, s) : launch_t<CT, 64, false>(a, kmap, vmap, box, s);
    return pair ? launch_t<CT, 128, true>(a, kmap, vmap, box, s) : launch_t<CT, 128, false>(a, kmap, vmap, box, s);
}

}  // namespace

int attn_tc_box(int page_size) { return std::min(kN, page_size & -page_size); }
// two row tiles a block above 128 rows (the calls of their day over 32768 positions of 8 heads: 136 rows 47.5 us, 53.4 with a tile
// each; 512 rows 84 and 95; over 4096 positions they are even)
int attn_tc_tile(int rows) { return rows > kM ? 2 * kM : kM; }

int launch_attn_tc(const AttnArgs &a, int cdt, cudaStream_t s) {
    return cdt == QMC_F16 ? launch_h<__half>(a, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, s)
                          : launch_h<__nv_bfloat16>(a, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, s);
}

}  // namespace qmc

// The prefix part of the shared-prefix attention on the 5th-generation tensor cores, for many query rows per KV head:
// tcgen05.mma with scores and accumulators in tensor memory (TMEM).
//
// Per 128 query rows and 128 positions: S = Q K^T (M = 128 rows, N = 128 positions) into 128 TMEM columns; a warpgroup,
// one thread per row, turns S into weights P = 2^(scale S - m) and writes them over S as 16-bit pairs; O += P V with P
// read from TMEM as the A operand and V from shared memory as it lies in the cache ([position][dim], an MN-major
// operand).  A row's reference m moves only when a score passes it by more than 8 (weights stay below 2^8, exact
// in the split of l and O): then the warp rescales its O rows in TMEM and takes the tile again, which after a row's first
// tile is rare, so O normally stays where it is until the end.
//
// A block runs two streams of such tiles, so that the tensor cores work on one while the other's warpgroup takes its
// exponentials (16384 of them per tile at 16 a cycle are as long as the tile's two products).  PAIR: the streams are
// two row tiles over the same positions (each K and V tile is read once for 256 rows).  Otherwise, with at most 128 rows, they
// take the range's position tiles in turn and leave a part each.
//
// Warps 0-3 and 4-7: the streams' weights (warp w may access TMEM lanes 32 (w % 4) .. + 31); 8-11: copies, 16 bytes a thread at
// a time, each position's row found through its page, into a ring of K and V tiles in the 128-byte swizzle (chunk c of
// row r at c ^ (r & 7), a panel of 128 rows for each 64 dimensions); 12: one lane issues the MMAs.  Every wait is bounded: after a
// timeout a role raises the error word and falls through to the end, where the copies and MMAs in flight are waited for
// (bounded) and the TMEM is freed.
#include "attn_prefix.cuh"

namespace qmc {
namespace {

constexpr int kM = 128, kN = 128;  // rows and positions of a tile
constexpr int kCopyWarps = 4, kMmaWarp = 8 + kCopyWarps, kThreads = (kMmaWarp + 1) * 32;
constexpr float kLift = 8.0f;      // how far a score may pass its row's reference, in powers of two

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

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack2(__half, float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *(const uint32_t *)&h;
}
__device__ __forceinline__ uint32_t pack2(__nv_bfloat16, float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *(const uint32_t *)&h;
}
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
// this thread's arrival on a barrier once its copies so far have landed
__device__ __forceinline__ void copies_arrive(uint64_t *bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void copy_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// shared-memory operand descriptors, 128-byte swizzle.  K-major (rows of 64 elements, eight-row groups 1024 bytes apart); MN-major
// (64 elements of M or N a row, eight-row groups of K 1024 bytes apart, the next 64 elements a panel further)
__device__ __forceinline__ uint64_t desc_k(uint32_t a) {
    return (uint64_t)((a >> 4) & 0x3fffu) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t a) {
    return (uint64_t)((a >> 4) & 0x3fffu) | ((uint64_t)(128 * 128 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// float accumulator, A and B of one 16-bit type; bmn: B is MN-major
__device__ __forceinline__ constexpr uint32_t idesc(int n, bool bmn, bool bf16) {
    return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((bmn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(kM >> 4) << 24);
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

// 32 or 64 consecutive TMEM columns of this thread's lane; the load and its wait are one statement, so that nothing reads the
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
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, uint32_t (&r)[64]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
        "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
        "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
          "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
          "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
          "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
          "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
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
// one row of a tile, read in halves of 64 scores: the largest, and 2^(scale s - m) as 16-bit pairs over the scores (a half's pairs
// lie on the first quarter or second quarter of the columns, which have been read by then) with their sum, before rounding.
// MASK: only the first `left` positions exist
template <bool MASK>
__device__ __forceinline__ float row_max(uint32_t ts, int left) {
    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int h = 0; h < 2; h++) {
        uint32_t x[64];
        tmem_ld64(ts + 64 * h, x);
#pragma unroll
        for (int k = 0; k < 64; k++) {
            const float s = __uint_as_float(x[k]);
            if (!MASK || (live_bits(left, 64 * h + (k & 32)) >> (k & 31) & 1u)) mx[k & 3] = fmaxf(mx[k & 3], s);
        }
    }
    return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
}
template <typename CT, bool MASK>
__device__ __forceinline__ float row_weights(uint32_t ts, float scale, float m, int left) {
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int h = 0; h < 2; h++) {
        uint32_t x[64];
        tmem_ld64(ts + 64 * h, x);
#pragma unroll
        for (int k = 0; k < 64; k += 2) {
            float t0 = fmaf(__uint_as_float(x[k]), scale, -m), t1 = fmaf(__uint_as_float(x[k + 1]), scale, -m);
            if (MASK) {
                const uint32_t live = live_bits(left, 64 * h + (k & 32)) >> (k & 31);
                t0 = live & 1u ? t0 : -INFINITY;
                t1 = live & 2u ? t1 : -INFINITY;
            }
            const float p0 = ex2(t0), p1 = ex2(t1);
            sum[k & 2] += p0, sum[(k & 2) + 1] += p1;
            x[k / 2] = pack2(CT(), p0, p1);
        }
        tmem_st32(ts + 32 * h, x);
    }
    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

struct Shared {
    uint64_t full[6], empty[6], sfull[2], pfull[2], ofin[2], drain;
    uint32_t tmem;
    int dead;
};

template <typename CT, int HDP, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1) attn_tc_kernel(const AttnArgs a) {
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
    // chunk c of row r of a tile, 128-byte swizzle
    auto place = [](int r, int c) { return (c >> 3) * PANEL + r * 128 + (((c & 7) ^ (r & 7)) << 4); };

    if (tid == 0) {
        for (int i = 0; i < NS; i++) {
            mbar_init(&sh.full[i], 32 * kCopyWarps);  // the copying threads
            mbar_init(&sh.empty[i], 1);               // a commit
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.sfull[i], 1);
            mbar_init(&sh.pfull[i], 4);    // the stream's warps
            mbar_init(&sh.ofin[i], 1);
        }
        mbar_init(&sh.drain, 1);
        sh.dead = 0;
        fence_mbar_init();
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp < 8) {  // the query tiles; rows past the last and chunks past the head are zeros
        const bool vec = a.ldq % 8 == 0 && (uintptr_t)a.q % 16 == 0;
        for (int i = tid; i < (PAIR ? 2 : 1) * kM * CH; i += 256) {
            const int r = i / CH, c = i % CH, rr = jb.r0 + r;
            alignas(16) CT e[8];
            *(uint4 *)e = make_uint4(0, 0, 0, 0);
            if (r < jb.nr && c < nch) {
                const CT *src = (const CT *)a.q + (rr / a.group) * a.ldq + (int64_t)(jb.h * a.group + rr % a.group) * hd + 8 * c;
                if (vec) *(uint4 *)e = *(const uint4 *)src;
                else
                    for (int k = 0; k < 8; k++) e[k] = src[k];
            }
            *(uint4 *)(base + (r / kM) * TB + place(r % kM, c)) = *(const uint4 *)e;
        }
    } else if (nch < CH) {  // K and V: chunks past the head, in the whole ring, never written again
        for (int i = tid - 256; i < NS * kN * (CH - nch); i += kThreads - 256) {
            const int r = i / (CH - nch), c = nch + i % (CH - nch);
            *(uint4 *)(base + (smk - smq) + (r / kN) * TB + place(r % kN, c)) = make_uint4(0, 0, 0, 0);
        }
    }
    fence_proxy_async();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;  // S (and P) of stream w at columns 128 w, O at 256 + HDP w
    volatile int *dead = &sh.dead;

    if (warp >= 8 && warp < 8 + kCopyWarps) {  // ---------------------------------------------------------------- copies
        // warp wl copies rows 32 wl .. + 31 of every tile; its lane i knows where row 32 wl + i lies, in 16-byte units from
        // the pool's start (a layer's pool is under 2^36 bytes)
        const int wl = warp - 8, c = lane % CH, rl = lane / CH;
        constexpr int RPI = 32 / CH;  // rows an instruction covers
        constexpr uint32_t kNone = 0xffffffffu;
        auto find = [&](int j) {
            const int p = jb.p0 + j * kN + 32 * wl + lane;
            const int64_t s = p < jb.p1 ? slot_of(a, -1, p) : (int64_t)-1;
            return s >= 0 ? (uint32_t)((s * a.kv + jb.h) * nch) : kNone;
        };
        uint32_t put[8 / RPI];  // this lane's place in rows rl, rl + RPI, ... of an eight-row group
#pragma unroll
        for (int i = 0; i < 8 / RPI; i++) put[i] = place(32 * wl + i * RPI + rl, c);
        auto issue = [&](uint32_t slot, int u, const uint8_t *pool) {  // tile u of the sequence K0 V0 K1 V1 ...
            const int at = u % NS;
            if (u >= NS && __any_sync(0xffffffffu, !mbar_wait(&sh.empty[at], (u / NS - 1) & 1) || *dead)) {
                if (lane == 0 && !*dead) raise_error(a.err, kErrMbarTimeout);
                *dead = 1;
                return false;
            }
            const uint32_t st = smk + at * TB;
            const uint8_t *src = pool + 16 * c;
#pragma unroll
            for (int i = 0; i < 32 / RPI; i++) {
                const uint32_t s = __shfl_sync(0xffffffffu, slot, i * RPI + rl);
                const uint32_t to = st + put[i % (8 / RPI)] + (i * RPI / 8 * 8) * 128;
                if (c < nch) copy16(to, src + (s != kNone ? (uint64_t)s * 16 : 0), s != kNone);
            }
            copies_arrive(&sh.full[at]);
            return true;
        };
        uint32_t slot = ntile > 0 ? find(0) : kNone;
        for (int j = 0; j < ntile; j++) {
            const uint32_t next = j + 1 < ntile ? find(j + 1) : kNone;
            if (!issue(slot, 2 * j, (const uint8_t *)a.kc) || !issue(slot, 2 * j + 1, (const uint8_t *)a.vc)) break;
            slot = next;
        }
        copy_wait_all();
    } else if (warp == kMmaWarp) {  // ---------------------------------------------------------------- MMA issuer
        if (lane == 0) {
            bool ok = true;
            auto wait = [&](uint64_t *bar, uint32_t parity) {
                if (ok && (!mbar_wait(bar, parity) || *dead)) {
                    if (!*dead) raise_error(a.err, kErrMbarTimeout);
                    *dead = 1;
                    ok = false;
                }
                return ok;
            };
            auto tile = [&](int u) {  // has landed; the copies are ordered before the tensor core's reads of them
                if (!wait(&sh.full[u % NS], (u / NS) & 1)) return false;
                fence_proxy_async();
                return true;
            };
            auto scores = [&](int w, int j) {  // S_w = Q_w K_j^T
                if (!tile(2 * j)) return;
                tc_fence_after();
                const uint32_t q = smq + (PAIR ? w : 0) * TB, k = smk + (2 * j) % NS * TB;
#pragma unroll
                for (int i = 0; i < HDP / 16; i++) {
                    const uint32_t off = (i >> 2) * PANEL + (i & 3) * 32;
                    mma_ss(tmem + 128 * w, desc_k(q + off), desc_k(k + off), idesc(kN, false, BF), i > 0);
                }
                mma_commit(&sh.sfull[w]);
                if (!PAIR || w == 1) mma_commit(&sh.empty[(2 * j) % NS]);
            };
            auto weigh = [&](int w, int j, int i) {  // O_w += P_w V_j, the stream's i-th tile
                if (!tile(2 * j + 1) || !wait(&sh.pfull[w], i & 1u)) return;
                tc_fence_after();
                const uint32_t v = smk + (2 * j + 1) % NS * TB;
#pragma unroll
                for (int k = 0; k < kN / 16; k++)
                    mma_ts(tmem + 256 + HDP * w, tmem + 128 * w + 8 * k, desc_mn(v + k * 16 * 128), idesc(HDP, true, BF),
                           i > 0 || k > 0);
                if (!PAIR || w == 1) mma_commit(&sh.empty[(2 * j + 1) % NS]);
            };
            constexpr int step = PAIR ? 1 : 2;  // tiles from one of a stream's to its next
            for (int w = 0; w < 2; w++) {
                const int j = PAIR ? 0 : w;
                if (j < ntile) scores(w, j);
            }
            for (int i = 0; i * step < ntile && ok; i++)
                for (int w = 0; w < 2 && ok; w++) {
                    const int j = PAIR ? i : 2 * i + w;
                    if (j >= ntile) continue;
                    weigh(w, j, i);
                    if (!ok) break;
                    if (j + step < ntile) scores(w, j + step);
                    else mma_commit(&sh.ofin[w]);
                }
            // nothing may be in flight when the TMEM is freed
            mma_commit(&sh.drain);
            if (!mbar_wait(&sh.drain, 0)) raise_error(a.err, kErrMbarTimeout);
        }
        __syncwarp();
    } else {  // ---------------------------------------------------------------- weights
        const int w = warp >> 2, row = 32 * (warp & 3) + lane, r = (PAIR ? w * kM : 0) + row;
        const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16), ts = lanes + 128 * w, to = lanes + 256 + HDP * w;
        const int mine = PAIR ? ntile : (ntile - w + 1) / 2;
        float m = 0.0f, l = 0.0f;
        bool ok = true;
        for (int i = 0; i < mine; i++) {
            const int j = PAIR ? i : 2 * i + w, left = jb.p1 - jb.p0 - j * kN;
            if (__any_sync(0xffffffffu, !mbar_wait(&sh.sfull[w], i & 1u) || *dead)) {
                if (lane == 0 && !*dead) raise_error(a.err, kErrMbarTimeout);
                *dead = 1;
                ok = false;
                break;
            }
            tc_fence_after();
            const bool whole = left >= kN;
            const float top = whole ? row_max<false>(ts, left) : row_max<true>(ts, left), mx = top * a.scale;
            if (i == 0) {
                m = mx == -INFINITY ? 0.0f : mx;
            } else if (__any_sync(0xffffffffu, mx > m + kLift)) {
                // lift the references of the warp's rows; O holds the tiles before this one, whose product is complete (this
                // tile's scores were committed after it)
                const float to_m = fmaxf(m, mx), down = ex2(m - to_m);
                m = to_m, l *= down;
                for (int c = 0; c < HDP / 32; c++) {
                    uint32_t x[32];
                    tmem_ld32(to + 32 * c, x);
#pragma unroll
                    for (int k = 0; k < 32; k++) x[k] = __float_as_uint(__uint_as_float(x[k]) * down);
                    tmem_st32(to + 32 * c, x);
                }
            }
            l += whole ? row_weights<CT, false>(ts, a.scale, m, left) : row_weights<CT, true>(ts, a.scale, m, left);
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.pfull[w]);
        }
        if (ok && mine > 0 && __any_sync(0xffffffffu, !mbar_wait(&sh.ofin[w], 0) || *dead)) {
            if (lane == 0 && !*dead) raise_error(a.err, kErrMbarTimeout);
            *dead = 1;
            ok = false;
        }
        tc_fence_after();
        const int64_t all = (int64_t)a.n_seq * a.heads, part = PAIR ? jb.part : 2 * jb.part + w;
        const bool real = r < jb.nr;
        const int64_t at = part * all + (real ? out_row(a, jb.h, jb.r0 + r) : 0);
        if (real) a.ml[at] = mine > 0 && ok ? make_float2(m, l) : make_float2(-INFINITY, 0.0f);
        if (ok && mine > 0)
            for (int c = 0; c < HDP / 32; c++) {
                uint32_t x[32];
                tmem_ld32(to + 32 * c, x);
                if (real)
#pragma unroll
                    for (int k = 0; k < 32; k += 4)
                        if (32 * c + k < hd)
                            *(float4 *)(a.po + at * hd + 32 * c + k) = make_float4(__uint_as_float(x[k]), __uint_as_float(x[k + 1]),
                                                                               __uint_as_float(x[k + 2]), __uint_as_float(x[k + 3]));
            }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

template <typename CT, int HDP, bool PAIR>
int launch_t(const AttnArgs &a, cudaStream_t s) {
    auto fn = attn_tc_kernel<CT, HDP, PAIR>;
    constexpr int smem = smem_bytes<HDP, PAIR>();
    QMC_CUDA(cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    const int64_t jobs = (int64_t)a.kv * a.ptiles * a.psplit;
    if (jobs > INT32_MAX) return set_error(QMC_EINVAL, "attn_prefix: too many blocks");
    fn<<<(unsigned)jobs, kThreads, smem, s>>>(a);
    QMC_LAUNCH_CHECK();
    return QMC_OK;
}
template <typename CT>
int launch_h(const AttnArgs &a, cudaStream_t s) {
    const bool pair = a.rows > kM;
    if (a.hd <= 64) return pair ? launch_t<CT, 64, true>(a, s) : launch_t<CT, 64, false>(a, s);
    return pair ? launch_t<CT, 128, true>(a, s) : launch_t<CT, 128, false>(a, s);
}

}  // namespace

int attn_tc_tile(int rows) { return rows > kM ? 2 * kM : kM; }
int attn_tc_parts(int rows) { return rows > kM ? 1 : 2; }

int launch_attn_tc(const AttnArgs &a, int cdt, cudaStream_t s) {
    return cdt == QMC_F16 ? launch_h<__half>(a, s) : launch_h<__nv_bfloat16>(a, s);
}

}  // namespace qmc

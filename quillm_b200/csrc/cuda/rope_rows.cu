// Norms of queries and keys per head and the rotary rotation, over rows at positions of their own, into rows or
// into a paged cache (qmc_qk_norm_rope, qmc_kv_append_paged).
//
// For every head x of a row:  y = x / sqrt(mean(x^2) + eps) * w  (optional), then each pair (a, b) of the first
// rot dimensions becomes (a c - b s, a s + b c) with (c, s) = m (cos, sin)(pos f_i).  The angle is formed in turns in fixed point:
// f_i / 2 pi is kept as a fraction of 2^64, and pos times it modulo 2^64 is the fraction of a turn, off by pos times the double's
// rounding of f_i (2^-36 turns at position 10^6, where a float angle would be off by a sixteenth of a radian); its upper half
// (2^-32 turns), rounded to float, goes to sincospi.
//
// HBM bound: each element is read once and written once with ~10 operations between.  8192 rows of 64 + 8 heads of 128 in bf16, with
// norms: 67 us, 4.5 TB/s of the measured 6.56, and 81 us with the append of keys and values; the issue of instructions binds
// what is left (a block that stays and loops over rows: 115 us and more).  A token's kernel takes 2.4 us, 3.6 with cold caches, its
// call from Python 6.8.
//
// A lane group of 1 to 32 lanes
// holds one head, each lane two chunks of C elements (16 bytes each where the layout allows it) that hold whole
// pairs between them: in the half layout the chunks at t C and t C + rot / 2, in the interleaved one neighbours.  So a
// rotation needs no exchange, a norm log2(lanes) shuffles, and every access is a full vector.  While the elements are in flight the
// block forms a table of its rows' pairs in shared memory, (w0 c, w1 s, w0 s, w1 c) with the pair's weights folded in, for
// queries and for keys: with r the head's 1 / sqrt(mean + eps), a' = (a w0 c - b w1 s) r and b' = (a w0 s + b w1 c) r.
#include <algorithm>
#include <cmath>
#include <new>

#include "batch.cuh"

struct qmc_rope_plan {
    int head_dim, rot_dim, layout;
    float mscale;
    uint64_t turns[128];  // f_i / 2 pi without its whole turns, times 2^64
};

namespace qmc {

int check_cache(const qmc_paged_cache *c, const char *op) {
    if (!c || !c->k || !c->v) return set_error(QMC_EINVAL, "%s: null cache", op);
    if (!is_row_dtype(c->dtype)) return set_error(QMC_EINVAL, "%s: bad cache dtype %d", op, c->dtype);
    if (c->n_layers < 1 || c->n_pages < 1 || c->page_size < 1 || c->n_kv_heads < 1 || c->head_dim < 1)
        return set_error(QMC_EINVAL, "%s: cache of %d layers, %d pages of %d, %d heads of %d", op, c->n_layers, c->n_pages,
                         c->page_size, c->n_kv_heads, c->head_dim);
    const int64_t sz = dtype_size(c->dtype);
    if ((uintptr_t)c->k % sz || (uintptr_t)c->v % sz) return set_error(QMC_EINVAL, "%s: misaligned cache", op);
    // slots of a layer are counted in 64 bits, elements of the pool must be too
    const __int128 n = (__int128)c->n_layers * c->n_pages * c->page_size * c->n_kv_heads * c->head_dim * sz;
    if (n > ((__int128)1 << 62) || (int64_t)c->n_kv_heads * c->head_dim > 1 << 28) return set_error(QMC_EINVAL, "%s: cache too large", op);
    return QMC_OK;
}

namespace {

struct RowsArgs {
    const void *q, *k, *v;
    void *qo, *ko;  // rows; ko: keys to rows (no cache)
    int64_t ldq, ldk, ldv, ldqo, ldko, rows;
    void *kc, *vc;  // one layer of the pools, or null
    const int *seq, *pos, *table;
    const float *qw, *kw;
    int *err;
    int n_seq, ld_table, page_size, n_pages;
    int heads, kv, hd, rot;
    int shift;      // log2 of a head's lanes
    int pairs;      // of the table: items times C
    bool half;
    float eps, mscale, inv_hd;
};
constexpr int kRows = 4;  // rows of a block, of many
struct Turns {
    uint64_t t[128];
};

// where item t's pair e lies among the C of its item: the 16-byte entries that eight neighbouring lanes read together fall on
// distinct banks
template <int C>
__device__ __forceinline__ int spread(int t, int e) {
    return e ^ ((t / (8 / C)) & (C - 1));
}
// (a, b) of a pair through its row of the table, times the head's factor.  A pair that stays keeps its elements apart: a product with
// the other's zero would be NaN for an infinite one
__device__ __forceinline__ void rotate(float &a, float &b, float4 r, float f, bool turns) {
    const float u = a, v = b, u0 = turns ? u : 0.0f, v0 = turns ? v : 0.0f;
    a = (u * r.x - v0 * r.y) * f;
    b = (u0 * r.z + v * r.w) * f;
}

// T rows, CT cache elements, C elements per chunk, NIT items per lane, R rows a block: their elements are all on their way before
// the rows' (c, s) and slots are formed, each by a thread of its own.  FULL: every lane has both its chunks, and a head's lanes
// and pairs are powers of two.
template <typename T, typename CT, int C, int NIT, int R, bool HALF, bool FULL>
__global__ void __launch_bounds__(288, 3) rope_rows_kernel(const __grid_constant__ RowsArgs a, const __grid_constant__ Turns f) {
    __shared__ float4 tab[2][R][128];  // [queries, keys][row][pair]
    __shared__ int64_t slot_s[R];
    const int tid = threadIdx.x, lph = 1 << a.shift, li = tid & (lph - 1), hd = a.hd;
    const int head = (int)blockIdx.y * ((int)blockDim.x >> a.shift) + (tid >> a.shift);
    const bool cache = a.kc != nullptr;
    const int kind = head < a.heads ? 0 : head < a.heads + a.kv ? 1 : 2;  // q, k, v
    const bool live = kind < 2 || (cache && head < a.heads + 2 * a.kv);
    const int h = kind == 0 ? head : kind == 1 ? head - a.heads : head - a.heads - a.kv;
    const int64_t row0 = (int64_t)blockIdx.x * R, ld = kind == 0 ? a.ldq : kind == 1 ? a.ldk : a.ldv;
    const int n = (int)(a.rows - row0 < R ? a.rows - row0 : R);

    // this lane's items: chunks at ea and eb (hd: none), which hold the pairs t C, ... of item t.  HALF: element i of one chunk
    // pairs with element i of the other; else pairs lie within a chunk, or, of one element, in the two neighbours
    const int rot_items = (a.rot >> 1) / C;
    int ea[NIT], eb[NIT];
#pragma unroll
    for (int j = 0; j < NIT; j++) {
        const int t = li + j * lph;
        ea[j] = !HALF ? 2 * t * C : t < rot_items ? t * C : a.rot + 2 * (t - rot_items) * C;
        eb[j] = ea[j] + (HALF && t < rot_items ? a.rot >> 1 : C);
        if (!FULL && (!live || ea[j] > hd)) ea[j] = hd;
        if (!FULL && (!live || eb[j] > hd)) eb[j] = hd;
    }
    auto has = [&](int e) { return FULL ? live : e < hd; };
    const T *src = (const T *)(kind == 0 ? a.q : kind == 1 ? a.k : a.v) + (live ? row0 * ld + (int64_t)h * hd : 0);
    Chunk<T, C> ca[R][NIT] = {}, cb[R][NIT] = {};
#pragma unroll
    for (int k = 0; k < R; k++)
#pragma unroll
        for (int j = 0; j < NIT; j++) {
            if (k < n && has(ea[j])) ca[k][j] = *(const Chunk<T, C> *)(src + k * ld + ea[j]);
            if (k < n && has(eb[j])) cb[k][j] = *(const Chunk<T, C> *)(src + k * ld + eb[j]);
        }
    // the lanes of a warp want different entries: read as memory, since the constant cache gives one address at a time
    const uint64_t *step = f.t;
    asm volatile("" : "+l"(step));
    for (int i = tid; i < n * a.pairs; i += blockDim.x) {
        const int k = R == 1 ? 0 : FULL ? i >> (31 - __clz(a.pairs)) : i / a.pairs, p = R == 1 ? i : FULL ? i & (a.pairs - 1) : i % a.pairs;
        const int t = p / C, d0 = !HALF ? 2 * p : t < rot_items ? p : a.rot + 2 * (t - rot_items) * C + p % C;
        const int d1 = !HALF ? 2 * p + 1 : t < rot_items ? p + (a.rot >> 1) : d0 + C;
        float s = 0.0f, c = 1.0f;
        if (HALF ? t < rot_items : d0 < a.rot) {
            const uint64_t turns = (uint64_t)(int64_t)a.pos[row0 + k] * step[p];
            sincospif((float)(int32_t)(turns >> 32) * 4.656612873077393e-10f, &s, &c);  // 2^-31: half turns in [-1, 1)
            s *= a.mscale, c *= a.mscale;
        }
#pragma unroll
        for (int q = 0; q < 2; q++) {
            const float *w = q ? a.kw : a.qw;
            const float w0 = w && d0 < hd ? w[d0] : 1.0f, w1 = w && d1 < hd ? w[d1] : 1.0f;
            tab[q][k][t * C + spread<C>(t, p % C)] = make_float4(w0 * c, w1 * s, w0 * s, w1 * c);
        }
    }
    if (const int k = (int)blockDim.x - 1 - tid; cache && k < n) {
        int64_t slot = -2;  // padding; -1: none
        const int64_t row = row0 + k;
        const int sq = a.seq ? a.seq[row] : (int)row, pos = a.pos[row];
        if (sq >= 0 && pos >= 0) {
            slot = -1;
            const int e = pos / a.page_size;
            if (sq < a.n_seq && e < a.ld_table) {
                const int page = a.table[(int64_t)sq * a.ld_table + e];
                if (page >= 0 && page < a.n_pages) slot = (int64_t)page * a.page_size + pos % a.page_size;
            }
            if (slot < 0) raise_error(a.err, kErrBadIndex);
        }
        slot_s[k] = slot;
    }
    const bool norm = live && (kind == 0 ? a.qw : kind == 1 ? a.kw : nullptr) != nullptr;
    __syncthreads();
    if (FULL && !live) return;
    const float inv_hd = a.inv_hd, eps = a.eps;
    const int row_elems = a.kv * hd;
    CT *const cbase = (kind == 1 ? (CT *)a.kc : (CT *)a.vc) + (live ? h * hd : 0);
    T *dst = (T *)(kind == 0 ? a.qo : a.ko) + (!live || (cache && kind) ? 0 : row0 * (kind == 0 ? a.ldqo : a.ldko) + (int64_t)h * hd);
    const int64_t ldo = kind == 0 ? a.ldqo : a.ldko;
    const unsigned group = (lph == 32 ? 0xffffffffu : ((1u << lph) - 1u)) << ((tid & 31) & ~(lph - 1));
#pragma unroll
    for (int k = 0; k < R; k++) {
        float xa[NIT][C], xb[NIT][C], r = 1.0f;
#pragma unroll
        for (int j = 0; j < NIT; j++) widen(ca[k][j], xa[j]), widen(cb[k][j], xb[j]);
        if (norm) {  // the same for a head's lanes; other heads of the warp may differ, so the shuffles are masked to the group
            float ss = 0.0f;  // missing chunks are zeros
#pragma unroll
            for (int j = 0; j < NIT; j++)
#pragma unroll
                for (int i = 0; i < C; i++) ss = fmaf(xa[j][i], xa[j][i], fmaf(xb[j][i], xb[j][i], ss));
            for (int o = lph >> 1; o; o >>= 1) ss += __shfl_xor_sync(group, ss, o);
            r = rsqrtf(fmaf(ss, inv_hd, eps));  // two units in the last place
        }
        if (kind != 2)
#pragma unroll
            for (int j = 0; j < NIT; j++) {
                if (!FULL && ea[j] >= hd) continue;
                const int t = li + j * lph, x = spread<C>(t, 0);
                const float4 *row = &tab[kind][k][t * C];
                // rotated pairs of this item, none of which the item has left where that is all
                const int turning = HALF ? (t < rot_items ? C : 0) : (a.rot >> 1) - t * C;
#pragma unroll
                for (int i = 0; i < C; i++) {
                    const bool turns = i < turning;
                    if (HALF || C == 1) rotate(xa[j][i], xb[j][i], row[i ^ x], r, turns);
                    else if (i < C / 2) rotate(xa[j][2 * i % C], xa[j][(2 * i + 1) % C], row[i ^ x], r, turns);
                    else rotate(xb[j][2 * i % C], xb[j][(2 * i + 1) % C], row[i ^ x], r, turns);
                }
            }
        // rows past the last, and padding, have gone through this for nothing: no branch lies between the rows' arithmetic
        const int64_t slot = cache && k < n ? slot_s[k] : 0;
        if (k >= n || slot == -2) continue;
        if (kind == 0 || !cache) {
            T *o = dst + k * ldo;
#pragma unroll
            for (int j = 0; j < NIT; j++) {
                if (FULL || ea[j] < hd) store_chunk<T, C>(o + ea[j], xa[j]);
                if (FULL || eb[j] < hd) store_chunk<T, C>(o + eb[j], xb[j]);
            }
        } else if (slot >= 0) {
            CT *o = cbase + slot * (int64_t)row_elems;
#pragma unroll
            for (int j = 0; j < NIT; j++) {
                if (FULL || ea[j] < hd) store_chunk<CT, C>(o + ea[j], xa[j]);
                if (FULL || eb[j] < hd) store_chunk<CT, C>(o + eb[j], xb[j]);
            }
        }
    }
}

template <typename T, typename CT, int C, int NIT, int R, bool FULL>
int launch_r(RowsArgs &a, const Turns &f, int64_t warps, cudaStream_t s) {
    const int64_t parts = (warps + 8) / 9, wpb = (warps + parts - 1) / parts;  // even blocks of at most nine warps, three of which an SM holds
    if (parts > 65535) return set_error(QMC_EINVAL, "rope rows: %d heads are too many", a.heads + a.kv);
    const dim3 grid((unsigned)((a.rows + R - 1) / R), (unsigned)parts);
    if (a.half) rope_rows_kernel<T, CT, C, NIT, R, true, FULL><<<grid, (unsigned)wpb * 32, 0, s>>>(a, f);
    else rope_rows_kernel<T, CT, C, NIT, R, false, FULL><<<grid, (unsigned)wpb * 32, 0, s>>>(a, f);
    QMC_LAUNCH_CHECK();
    return QMC_OK;
}

template <typename T, typename CT, int C, int NIT>
int launch_t(RowsArgs &a, const Turns &f, int64_t rows, cudaStream_t s) {
    const DevCtx *dc = ctx();
    const int64_t sms = dc ? dc->num_sms : 148;
    const int P = a.half ? (a.rot >> 1) / C : 0;
    const int chunks = a.half ? (a.hd - a.rot) / C : a.hd / C;
    const int items = P + (chunks + 1) / 2;
    a.shift = 0;
    while ((NIT << a.shift) < items) a.shift++;
    a.pairs = items * C;
    a.rows = rows, a.inv_hd = 1.0f / (float)a.hd;
    const int heads = a.heads + a.kv + (a.kc ? a.kv : 0);
    const int64_t warps = ((int64_t)heads * (1 << a.shift) + 31) / 32;
    // several rows a block once one row each fills the SMs (64 + 8 heads of 128 in bf16: 256 rows 6.8 us both ways, 512 rows 8.3 us
    // and 10.4 with one, 4096 rows 39 and 56)
    if constexpr (NIT == 1)
        if (rows * warps > 32 * sms) {
            const bool full = items == 1 << a.shift && chunks % 2 == 0 && (a.hd & (a.hd - 1)) == 0;
            return full ? launch_r<T, CT, C, NIT, kRows, true>(a, f, warps, s) : launch_r<T, CT, C, NIT, kRows, false>(a, f, warps, s);
        }
    return launch_r<T, CT, C, NIT, 1, false>(a, f, warps, s);
}

// the widest chunk that divides the head, the rotated half, the strides and every address; hd <= 256, so a lane needs at most
// 4 items of one element (128 lanes' worth of pairs), 2 of two and 1 of four or eight
template <typename T, typename CT>
int launch_c(RowsArgs &a, const Turns &f, int64_t rows, cudaStream_t s) {
    constexpr int CM = 16 / sizeof(T);
    auto fits = [&](int c) {
        auto addr = [&](const void *p, size_t elem) {
            const size_t b = c * elem < 16 ? c * elem : 16;
            return !p || (uintptr_t)p % b == 0;
        };
        const int64_t lds[5] = {a.q ? a.ldq : 0, a.k ? a.ldk : 0, a.v ? a.ldv : 0, a.q ? a.ldqo : 0, a.ko ? a.ldko : 0};
        for (int64_t ld : lds)
            if (ld % c) return false;
        return a.hd % c == 0 && (!a.half || (a.rot / 2 % c == 0 && a.rot % c == 0)) && addr(a.q, sizeof(T)) &&
               addr(a.k, sizeof(T)) && addr(a.v, sizeof(T)) && addr(a.qo, sizeof(T)) && addr(a.ko, sizeof(T)) &&
               addr(a.kc, sizeof(CT)) && addr(a.vc, sizeof(CT));
    };
    if (fits(CM)) return launch_t<T, CT, CM, 1>(a, f, rows, s);
    if (fits(2)) return launch_t<T, CT, 2, 2>(a, f, rows, s);
    return launch_t<T, CT, 1, 4>(a, f, rows, s);
}

template <typename T>
int launch_ct(RowsArgs &a, const Turns &f, int cdt, int64_t rows, cudaStream_t s) {
    if (!a.kc) return launch_c<T, T>(a, f, rows, s);
    if (cdt == QMC_F32) return launch_c<T, float>(a, f, rows, s);
    if (cdt == QMC_F16) return launch_c<T, __half>(a, f, rows, s);
    return launch_c<T, __nv_bfloat16>(a, f, rows, s);
}

int launch_rows(RowsArgs &a, const qmc_rope_plan *p, int dtype, int cdt, int64_t rows, cudaStream_t s) {
    static const Turns none{};
    Turns f = none;
    a.half = p && p->layout == QMC_ROPE_HALF;
    a.rot = p ? p->rot_dim : 0;
    a.mscale = p ? p->mscale : 1.0f;
    if (p)
        for (int i = 0; i < p->rot_dim / 2; i++) f.t[i] = p->turns[i];
    if (dtype == QMC_F32) return launch_ct<float>(a, f, cdt, rows, s);
    if (dtype == QMC_F16) return launch_ct<__half>(a, f, cdt, rows, s);
    return launch_ct<__nv_bfloat16>(a, f, cdt, rows, s);
}

constexpr int kMostHeads = 1 << 20;  // of a row, queries or keys: their elements are counted in 32 bits

// rows of `n` heads `ld` elements apart
int check_rows(const char *op, const char *name, const void *p, int64_t ld, int64_t n, int hd, int dtype) {
    if (!p) return set_error(QMC_EINVAL, "%s: null %s", op, name);
    if (n > kMostHeads) return set_error(QMC_EINVAL, "%s: %lld heads are too many", op, (long long)n);
    if (ld < n * hd) return set_error(QMC_EINVAL, "%s: %s rows of %lld elements are %lld apart", op, name, (long long)(n * hd), (long long)ld);
    if (ld > (int64_t)1 << 40) return set_error(QMC_EINVAL, "%s: ld of %s too large", op, name);
    if ((uintptr_t)p % dtype_size(dtype)) return set_error(QMC_EINVAL, "%s: misaligned %s", op, name);
    return QMC_OK;
}

}  // namespace
}  // namespace qmc

using namespace qmc;

extern "C" {

int qmc_rope_plan_create(const qmc_rope_config *c, qmc_rope_plan **out) {
    if (!c || !out) return set_error(QMC_EINVAL, "rope_plan_create: null argument");
    *out = nullptr;
    const int rot = c->rot_dim;
    if (c->head_dim < 2 || c->head_dim > 256 || (c->head_dim & 1) || rot < 2 || rot > c->head_dim || (rot & 1))
        return set_error(QMC_EINVAL, "rope_plan_create: head_dim %d, rot_dim %d", c->head_dim, rot);
    if (c->layout != QMC_ROPE_INTERLEAVED && c->layout != QMC_ROPE_HALF)
        return set_error(QMC_EINVAL, "rope_plan_create: bad layout %d", c->layout);
    if (c->scaling < QMC_ROPE_PLAIN || c->scaling > QMC_ROPE_YARN)
        return set_error(QMC_EINVAL, "rope_plan_create: bad scaling %d", c->scaling);
    if (!(c->theta > 0) || !std::isfinite(c->theta)) return set_error(QMC_EINVAL, "rope_plan_create: theta %g", c->theta);
    const bool scaled = c->scaling != QMC_ROPE_PLAIN;
    if (scaled && (!(c->factor > 0) || !std::isfinite(c->factor)))
        return set_error(QMC_EINVAL, "rope_plan_create: factor %g", c->factor);
    if (c->scaling == QMC_ROPE_BANDS && (!(c->low > 0) || !(c->high > c->low) || !std::isfinite(c->high) || c->orig_ctx < 1))
        return set_error(QMC_EINVAL, "rope_plan_create: bands %g .. %g of %d", c->low, c->high, c->orig_ctx);
    if (c->scaling == QMC_ROPE_YARN &&
        (!(c->low > 0) || !(c->high >= c->low) || !std::isfinite(c->high) || c->orig_ctx < 1 || c->theta == 1.0))
        return set_error(QMC_EINVAL, "rope_plan_create: ramp %g .. %g of %d, theta %g", c->low, c->high, c->orig_ctx, c->theta);
    qmc_rope_plan *p = new (std::nothrow) qmc_rope_plan();
    if (!p) return set_error(QMC_ENOMEM, "rope_plan_create: out of memory");
    p->head_dim = c->head_dim, p->rot_dim = rot, p->layout = c->layout;
    const double two_pi = 6.283185307179586476925286766559;
    double lo = 0, hi = 0;
    p->mscale = 1.0f;
    if (c->scaling == QMC_ROPE_YARN) {
        auto d = [&](double turns) { return rot * log(c->orig_ctx / (two_pi * turns)) / (2.0 * log(c->theta)); };
        lo = fmin(fmax(floor(d(c->high)), 0.0), rot - 1.0);
        hi = fmin(fmax(ceil(d(c->low)), 0.0), rot - 1.0);
        if (c->factor > 1.0) p->mscale = (float)(0.1 * log(c->factor) + 1.0);
    }
    for (int i = 0; i < rot / 2; i++) {
        double f = pow(c->theta, -2.0 * i / rot);
        if (c->scaling == QMC_ROPE_LINEAR) {
            f /= c->factor;
        } else if (c->scaling == QMC_ROPE_BANDS) {
            const double t = c->orig_ctx * f / two_pi;
            const double s = fmin(fmax((t - c->low) / (c->high - c->low), 0.0), 1.0);
            f = f * s + f / c->factor * (1.0 - s);
        } else if (c->scaling == QMC_ROPE_YARN) {
            const double r = fmin(fmax((i - lo) / fmax(hi - lo, 0.001), 0.0), 1.0);
            f = f / c->factor * r + f * (1.0 - r);
        }
        if (!std::isfinite(f)) {
            delete p;
            return set_error(QMC_EINVAL, "rope_plan_create: frequency %d of theta %g, factor %g is not finite", i, c->theta, c->factor);
        }
        double turns = f / two_pi;  // the whole turns go, the rest is exact
        turns -= floor(turns);
        // two halves of 32 bits: a double holds 53 bits of the fraction, none is lost
        const double hi = floor(turns * 4294967296.0);
        p->turns[i] = ((uint64_t)hi << 32) + (uint64_t)((turns * 4294967296.0 - hi) * 4294967296.0);
    }
    *out = p;
    return QMC_OK;
}

int qmc_rope_plan_free(qmc_rope_plan *p) {
    delete p;
    return QMC_OK;
}

int qmc_qk_norm_rope(const qmc_rope_plan *plan, int dtype, const void *q, int64_t ldq, void *q_out, int64_t ldqo,
                     int32_t n_heads, const void *k, int64_t ldk, void *k_out, int64_t ldko, int32_t n_kv_heads,
                     const float *q_weight, const float *k_weight, float eps, const int32_t *positions, int64_t rows,
                     void *stream) {
    const char *op = "qk_norm_rope";
    if (!plan) return set_error(QMC_EINVAL, "%s: null plan", op);
    if (!is_row_dtype(dtype)) return set_error(QMC_EINVAL, "%s: bad dtype %d", op, dtype);
    if (n_heads < 0 || n_kv_heads < 0 || rows < 0 || rows > INT32_MAX)
        return set_error(QMC_EINVAL, "%s: %d + %d heads, %lld rows", op, n_heads, n_kv_heads, (long long)rows);
    if (!(eps >= 0)) return set_error(QMC_EINVAL, "%s: eps %g", op, eps);
    if (rows == 0 || (int64_t)n_heads + n_kv_heads == 0) return QMC_OK;
    const int hd = plan->head_dim;
    int rc;
    if (n_heads && ((rc = check_rows(op, "q", q, ldq, n_heads, hd, dtype)) || (rc = check_rows(op, "q_out", q_out, ldqo, n_heads, hd, dtype))))
        return rc;
    if (n_kv_heads && ((rc = check_rows(op, "k", k, ldk, n_kv_heads, hd, dtype)) || (rc = check_rows(op, "k_out", k_out, ldko, n_kv_heads, hd, dtype))))
        return rc;
    if (!positions) return set_error(QMC_EINVAL, "%s: null positions", op);
    if (misaligned({positions, q_weight, k_weight})) return set_error(QMC_EINVAL, "%s: misaligned positions or weights", op);
    DevCtx *c = ctx();
    if (!c) return QMC_ECUDA;
    RowsArgs a{};
    if (n_heads) a.q = q, a.qo = q_out, a.ldq = ldq, a.ldqo = ldqo;
    if (n_kv_heads) a.k = k, a.ko = k_out, a.ldk = ldk, a.ldko = ldko;
    a.heads = n_heads, a.kv = n_kv_heads, a.hd = hd;
    a.qw = q_weight, a.kw = k_weight, a.eps = eps;
    a.pos = positions, a.err = c->err;
    return launch_rows(a, plan, dtype, dtype, rows, pick_stream(stream));
}

int qmc_kv_append_paged(const qmc_rope_plan *plan, const qmc_paged_cache *cache, int32_t layer, int dtype,
                        const void *q, int64_t ldq, void *q_out, int64_t ldqo, int32_t n_heads, const void *k,
                        int64_t ldk, const void *v, int64_t ldv, const float *q_weight, const float *k_weight, float eps,
                        const int32_t *seq, const int32_t *positions, const int32_t *page_table, int32_t n_seq,
                        int32_t ld_table, int64_t rows, void *stream) {
    const char *op = "kv_append_paged";
    int rc = check_cache(cache, op);
    if (rc) return rc;
    const int hd = cache->head_dim, kv = cache->n_kv_heads;
    if (hd > 256 || (hd & 1)) return set_error(QMC_EINVAL, "%s: head_dim %d is odd or above 256", op, hd);
    if (plan && plan->head_dim != hd) return set_error(QMC_EINVAL, "%s: plan for head_dim %d, cache of %d", op, plan->head_dim, hd);
    if (layer < 0 || layer >= cache->n_layers) return set_error(QMC_EINVAL, "%s: layer %d of %d", op, layer, cache->n_layers);
    if (!is_row_dtype(dtype)) return set_error(QMC_EINVAL, "%s: bad dtype %d", op, dtype);
    if (n_heads < 0 || rows < 0 || rows > INT32_MAX || n_seq < 0 || ld_table < 1)
        return set_error(QMC_EINVAL, "%s: %d heads, %lld rows, table of %d x %d", op, n_heads, (long long)rows, n_seq, ld_table);
    if (!(eps >= 0)) return set_error(QMC_EINVAL, "%s: eps %g", op, eps);
    if (!q != !n_heads) return set_error(QMC_EINVAL, "%s: %d query heads with%s q", op, n_heads, q ? "" : "out");
    if (rows == 0) return QMC_OK;
    if (n_heads && ((rc = check_rows(op, "q", q, ldq, n_heads, hd, dtype)) || (rc = check_rows(op, "q_out", q_out, ldqo, n_heads, hd, dtype))))
        return rc;
    if ((rc = check_rows(op, "k", k, ldk, kv, hd, dtype)) || (rc = check_rows(op, "v", v, ldv, kv, hd, dtype))) return rc;
    if (!positions || !page_table) return set_error(QMC_EINVAL, "%s: null positions or page table", op);
    if (misaligned({seq, positions, page_table, q_weight, k_weight}))
        return set_error(QMC_EINVAL, "%s: misaligned sequences, positions, page table or weights", op);
    if (!seq && rows > n_seq) return set_error(QMC_EINVAL, "%s: %lld rows for %d sequences", op, (long long)rows, n_seq);
    DevCtx *c = ctx();
    if (!c) return QMC_ECUDA;
    RowsArgs a{};
    if (n_heads) a.q = q, a.qo = q_out, a.ldq = ldq, a.ldqo = ldqo;
    a.k = k, a.v = v, a.ldk = ldk, a.ldv = ldv;
    const int64_t off = layer * layer_elems(cache) * dtype_size(cache->dtype);
    a.kc = (uint8_t *)cache->k + off, a.vc = (uint8_t *)cache->v + off;
    a.seq = seq, a.pos = positions, a.table = page_table;
    a.n_seq = n_seq, a.ld_table = ld_table, a.page_size = cache->page_size, a.n_pages = cache->n_pages;
    a.heads = n_heads, a.kv = kv, a.hd = hd;
    a.qw = q_weight, a.kw = k_weight, a.eps = eps;
    a.err = c->err;
    return launch_rows(a, plan, dtype, cache->dtype, rows, pick_stream(stream));
}

}  // extern "C"

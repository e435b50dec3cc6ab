// Beam search's selection over beams x vocabulary (qmc_beam_select) and the reordering of paged states
// (qmc_beam_reorder).
//
// Selection in two launches.  Both the log-sum-exp and the order need every logit once, so the first reads each row
// once, kChunk logits per block held in registers: the chunk's maximum m and sum of exp(x - m), and its n best logits.
// Within a row the order of scores is the order of logits, so n per chunk suffice whatever the row's log-sum-exp
// turns out to be.  The second, one block per prompt, joins a row's (m, sum) pairs in double, and merges the rows'
// sorted lists by score, n rounds of a block-wide maximum over the lists' heads.
//
// The n best of a chunk: the n-th largest of the 256 threads' maxima is a lower bound T that at least n elements reach, found
// by building T's bits from the top in one warp; the few elements >= T are collected in shared memory and ranked by
// counting.  Keys (logit, index) are distinct, so with all 64 bits of the key at most n threads' elements
// reach T (n * kItems, the collection's size); the first 32 bits are tried alone first and almost always enough.
#include "batch.cuh"

namespace qmc {
namespace {

constexpr int kBT = 256;               // threads
constexpr int kItems = 16;             // logits per thread
constexpr int kChunk = kBT * kItems;   // logits per block
constexpr int kMaxOut = 64;            // n_out and beams
constexpr int kCap = kMaxOut * kItems; // collected candidates

struct SelArgs {
    const void *logits;
    int64_t ld;
    int prompts, beams, vocab, n_out, eos, chunks;
    const float *scores;
    const uint8_t *finished;
    float2 *stat;              // [row][chunk] (m, sum exp(x - m))
    unsigned long long *cand;  // [row][chunk][n_out] keys, falling
    int *parents, *tokens;
    float *out_scores;
};

// order-preserving bits of a float; NaN counts as -inf, -0 as +0.  Never 0.
__device__ __forceinline__ uint32_t order_bits(float v) {
    if (v != v) v = -INFINITY;
    uint32_t u = v == 0.0f ? 0u : __float_as_uint(v);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t u) {
    return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}
__device__ __forceinline__ unsigned long long order_key(float v, int idx) {
    return ((unsigned long long)order_bits(v) << 32) | (uint32_t)~idx;
}

template <typename T>
__global__ void __launch_bounds__(kBT) beam_chunk_kernel(const SelArgs a) {
    __shared__ unsigned long long kmax[kBT], buf[kCap], T64_s;
    __shared__ float red[kBT / 32];
    __shared__ double redd[kBT / 32];
    __shared__ int cnt_s;
    const int chunk = blockIdx.x, row = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // the second kernel does not look at the lists of a finished or dead beam
    if ((a.finished && a.finished[row]) || !(a.scores[row] > -INFINITY)) return;
    const int base = chunk * kChunk, nel = min(kChunk, a.vocab - base), n = min(a.n_out, nel);
    const T *x = (const T *)a.logits + (int64_t)row * a.ld + base;

    constexpr int C = 16 / sizeof(T), NV = kItems / C;
    const bool vec = ((uintptr_t)x & 15) == 0;
    float v[kItems];
#pragma unroll
    for (int j = 0; j < NV; j++) {
        const int e0 = (j * kBT + tid) * C;
        float t[C];
        if (vec && e0 + C <= nel) {
            load_chunk<T, C>(x + e0, t);
#pragma unroll
            for (int i = 0; i < C; i++) v[j * C + i] = t[i];
        } else {
#pragma unroll
            for (int i = 0; i < C; i++) v[j * C + i] = e0 + i < nel ? to_f32(x[e0 + i]) : 0.0f;
        }
    }
    auto index = [&](int k) { return ((k / C) * kBT + tid) * C + k % C; };  // place in the chunk

    unsigned long long best = 0;
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < kItems; k++) {
        if (index(k) >= nel) continue;
        m = fmaxf(m, v[k]);  // fmaxf ignores NaN
        const unsigned long long key = order_key(v[k], base + index(k));
        best = key > best ? key : best;
    }
    kmax[tid] = best;
    m = warp_max(m);
    if (lane == 0) red[warp] = m;
    if (tid == 0) cnt_s = 0;
    __syncthreads();
    m = red[0];
#pragma unroll
    for (int w = 1; w < kBT / 32; w++) m = fmaxf(m, red[w]);
    if (warp == 0) {  // T: the n-th largest of the threads' maxima, its upper 32 bits
        uint32_t mine[kBT / 32], hi = 0, lo = 0xffffffffu;
#pragma unroll
        for (int j = 0; j < kBT / 32; j++) {
            mine[j] = (uint32_t)(kmax[lane + 32 * j] >> 32);
            hi = max(hi, mine[j]), lo = min(lo, mine[j]);
        }
        hi = __reduce_max_sync(0xffffffffu, hi), lo = __reduce_min_sync(0xffffffffu, lo);
        int bit = 31 - __clz(hi ^ lo);  // the bits above are common to all; -1: all equal
        uint32_t t = bit < 0 ? hi : hi & ~((2u << bit) - 1u);
        for (; bit >= 0; bit--) {
            const uint32_t c = t | (1u << bit);
            int k = 0;
#pragma unroll
            for (int j = 0; j < kBT / 32; j++) k += mine[j] >= c;
            k = __reduce_add_sync(0xffffffffu, k);
            if (k >= n) t = c;
            if (k == n) break;
        }
        if (lane == 0) T64_s = (unsigned long long)max(t, 1u) << 32;
    }
    float s = 0.0f;  // every thread, while the first warp looks for T
    if (m > -INFINITY) {
#pragma unroll
        for (int k = 0; k < kItems; k++)
            if (index(k) < nel && v[k] == v[k]) s += v[k] == m ? 1.0f : expf(v[k] - m);
    }
    const double sd = warp_sum_d((double)s);
    if (lane == 0) redd[warp] = sd;
    __syncthreads();
    if (tid == 0) {
        double tot = 0.0;
        for (int w = 0; w < kBT / 32; w++) tot += redd[w];
        a.stat[(int64_t)row * a.chunks + chunk] = make_float2(m, (float)tot);
    }
    auto collect = [&](unsigned long long least) {
        if (best >= least) {
#pragma unroll
            for (int k = 0; k < kItems; k++) {
                if (index(k) >= nel) continue;
                const unsigned long long key = order_key(v[k], base + index(k));
                if (key >= least) {
                    const int at = atomicAdd(&cnt_s, 1);  // places differ from run to run, ranks do not
                    if (at < kCap) buf[at] = key;
                }
            }
        }
    };
    collect(T64_s);
    __syncthreads();
    int cnt = cnt_s;
    __syncthreads();  // read by all before a second collection changes it
    if (cnt > kCap) {  // many equal logits: the rest of T's bits, over the indices
        if (warp == 0) {
            unsigned long long t = T64_s;
            for (int bit = 31; bit >= 0; bit--) {
                const unsigned long long c = t | (1ull << bit);
                int k = 0;
#pragma unroll
                for (int j = 0; j < kBT / 32; j++) k += kmax[lane + 32 * j] >= c;
                if (__reduce_add_sync(0xffffffffu, k) >= n) t = c;
            }
            if (lane == 0) T64_s = t, cnt_s = 0;
        }
        __syncthreads();
        collect(T64_s);
        __syncthreads();
        cnt = min(cnt_s, kCap);
    }
    unsigned long long *out = a.cand + ((int64_t)row * a.chunks + chunk) * a.n_out;
    for (int i = tid; i < cnt; i += kBT) {
        const unsigned long long key = buf[i];
        int rank = 0;
        for (int j = 0; j < cnt; j++) rank += buf[j] > key;
        if (rank < n) out[rank] = key;
    }
}

// the i-th of a list that does not come from the logits: a finished beam's one continuation, or none (dead); the other tokens
// follow at -inf in order
__device__ __forceinline__ int virtual_token(bool ended, int eos, int i) {
    return !ended ? i : i == 0 ? eos : i - 1 + (i - 1 >= eos);
}

struct Head {
    double score;
    int64_t flat;  // beam * vocab + token; INT64_MAX: none
};
__device__ __forceinline__ bool before(const Head &a, const Head &b) {
    return a.score > b.score || (a.score == b.score && a.flat < b.flat);
}

__global__ void __launch_bounds__(kBT) beam_merge_kernel(const SelArgs a) {
    __shared__ double lse_s[kMaxOut], cum_s[kMaxOut];
    __shared__ float top_s[kMaxOut];
    __shared__ uint8_t kind_s[kMaxOut];  // 0 logits, 1 finished, 2 dead
    __shared__ double wsc[kBT / 32];
    __shared__ int64_t wfl[kBT / 32];
    __shared__ int wth[kBT / 32];
    extern __shared__ int next_s[];  // [beams * chunks] entries taken of each list
    const int prompt = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int lists = a.beams * a.chunks;
    for (int b = warp; b < a.beams; b += kBT / 32) {
        const int row = prompt * a.beams + b;
        const float cum = a.scores[row];
        const bool dead = !(cum > -INFINITY), ended = !dead && a.finished && a.finished[row];
        float m = -INFINITY;
        double s = 0.0;
        if (!dead && !ended) {
            const float2 *st = a.stat + (int64_t)row * a.chunks;
            for (int c = lane; c < a.chunks; c += 32) m = fmaxf(m, st[c].x);
            m = warp_max(m);
            for (int c = lane; c < a.chunks; c += 32) {
                const float2 p = st[c];
                if (p.x > -INFINITY) s += (double)p.y * (p.x == m ? 1.0 : exp((double)p.x - (double)m));
            }
            s = warp_sum_d(s);
        }
        if (lane == 0) {
            cum_s[b] = cum, top_s[b] = m;
            kind_s[b] = ended ? 1 : (dead || !(m > -INFINITY)) ? 2 : 0;
            lse_s[b] = m == INFINITY ? log(s) : (double)m + log(s);
        }
    }
    for (int i = tid; i < lists; i += kBT) next_s[i] = 0;
    __syncthreads();

    auto head_of = [&](int list) {
        Head h{-INFINITY, INT64_MAX};
        const int b = list / a.chunks, c = list % a.chunks, i = next_s[list], kind = kind_s[b];
        if (kind) {
            if (c == 0 && i < min(a.n_out, a.vocab)) {
                h.flat = (int64_t)b * a.vocab + virtual_token(kind == 1, a.eos, i);
                if (kind == 1 && i == 0) h.score = cum_s[b];
            }
            return h;
        }
        const int nel = min(kChunk, a.vocab - c * kChunk);
        if (i >= min(a.n_out, nel)) return h;
        const unsigned long long key = a.cand[((int64_t)(prompt * a.beams + b) * a.chunks + c) * a.n_out + i];
        const float x = order_value((uint32_t)(key >> 32));
        h.flat = (int64_t)b * a.vocab + (int)~(uint32_t)key;
        // with an infinite maximum lse is the log of the number of infinities
        if (top_s[b] == INFINITY) h.score = x == INFINITY ? cum_s[b] - lse_s[b] : -INFINITY;
        else h.score = cum_s[b] + ((double)x - lse_s[b]);
        if (h.score != h.score) h.score = -INFINITY;
        return h;
    };
    Head mine{-INFINITY, INT64_MAX};
    int my_list = -1;
    auto scan = [&]() {
        mine = Head{-INFINITY, INT64_MAX};
        my_list = -1;
        for (int l = tid; l < lists; l += kBT) {
            const Head h = head_of(l);
            if (h.flat != INT64_MAX && (my_list < 0 || before(h, mine))) mine = h, my_list = l;
        }
    };
    scan();
    for (int r = 0; r < a.n_out; r++) {
        Head h = mine;
        int th = tid;
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            Head g;
            g.score = __shfl_xor_sync(0xffffffffu, h.score, o);
            g.flat = __shfl_xor_sync(0xffffffffu, h.flat, o);
            const int gt = __shfl_xor_sync(0xffffffffu, th, o);
            if (before(g, h)) h = g, th = gt;
        }
        if (lane == 0) wsc[warp] = h.score, wfl[warp] = h.flat, wth[warp] = th;
        __syncthreads();
        h = Head{wsc[0], wfl[0]}, th = wth[0];
#pragma unroll
        for (int w = 1; w < kBT / 32; w++) {
            const Head g{wsc[w], wfl[w]};
            if (before(g, h)) h = g, th = wth[w];
        }
        if (tid == 0) {
            const int64_t o = (int64_t)prompt * a.n_out + r;
            a.parents[o] = (int)(h.flat / a.vocab);
            a.tokens[o] = (int)(h.flat % a.vocab);
            a.out_scores[o] = (float)h.score;
        }
        if (tid == th && my_list >= 0) {
            next_s[my_list]++;
            scan();
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- reordering
struct ReorderArgs {
    uint8_t *pool[2];
    int64_t layer_bytes, page_bytes, slot_bytes;
    int n_pages, page_size, beams, ld_parents, ld_table;
    const int *parents, *lens, *tin;
    int *tout, *err;
};

// blockIdx.x: row; blockIdx.y: 2 * layer + (k or v).  Every block works out its beam's parent and pages from the prompt's
// parents; the first of a row writes the table.
__global__ void __launch_bounds__(kBT) beam_reorder_kernel(const ReorderArgs a) {
    __shared__ int par[kMaxOut];
    __shared__ uint8_t has[kMaxOut], first[kMaxOut];
    const int row = blockIdx.x, prompt = row / a.beams, j = row % a.beams, tid = threadIdx.x;
    int n = a.lens[prompt * a.beams];
    if (n < 0) {
        if (tid == 0) raise_error(a.err, kErrBadIndex);
        n = 0;
    }
    const int tail = n / a.page_size, filled = n % a.page_size;
    if (tid < a.beams) {
        int p = a.parents[(int64_t)prompt * a.ld_parents + tid];
        if (p < 0 || p >= a.beams) {
            raise_error(a.err, kErrBadIndex);
            p = tid;
        }
        par[tid] = p;
        has[tid] = 0;
    }
    __syncthreads();
    if (tid < a.beams) {
        bool f = true;
        for (int i = 0; i < tid; i++) f = f && par[i] != par[tid];
        first[tid] = f;
        has[par[tid]] = 1;
    }
    __syncthreads();
    int owner = par[j];  // the beam whose page being filled becomes this one's
    if (!first[j]) {
        int e = 0;
        for (int i = 0; i < j; i++) e += !first[i];
        // as many beams have no child as there are further children
        for (int i = 0; i < a.beams; i++)
            if (!has[i] && e-- == 0) {
                owner = i;
                break;
            }
    }
    const int *own = a.tin + (int64_t)row * a.ld_table, *from = a.tin + (int64_t)(prompt * a.beams + par[j]) * a.ld_table,
              *give = a.tin + (int64_t)(prompt * a.beams + owner) * a.ld_table;
    if (blockIdx.y == 0) {
        int *out = a.tout + (int64_t)row * a.ld_table;
        for (int i = tid; i < a.ld_table; i += kBT) out[i] = i < tail ? from[i] : i == tail ? give[i] : own[i];
    }
    if (first[j] || filled == 0) return;
    const int src = tail < a.ld_table ? from[tail] : -1, dst = tail < a.ld_table ? give[tail] : -1;
    if (src < 0 || src >= a.n_pages || dst < 0 || dst >= a.n_pages) {
        if (tid == 0) raise_error(a.err, kErrBadIndex);
        return;
    }
    uint8_t *pool = a.pool[blockIdx.y & 1] + (int64_t)(blockIdx.y >> 1) * a.layer_bytes;
    const uint8_t *s = pool + src * a.page_bytes;
    uint8_t *d = pool + dst * a.page_bytes;
    const int64_t bytes = filled * a.slot_bytes;
    if ((((uintptr_t)s | (uintptr_t)d | (uintptr_t)bytes) & 15) == 0) {
        for (int64_t i = tid; i < bytes / 16; i += kBT) ((uint4 *)d)[i] = ((const uint4 *)s)[i];
    } else {
        for (int64_t i = tid; i < bytes / 2; i += kBT) ((uint16_t *)d)[i] = ((const uint16_t *)s)[i];
    }
}

int beam_chunks(int vocab) { return (vocab + kChunk - 1) / kChunk; }
size_t beam_stat_bytes(int64_t rows, int chunks) { return ((size_t)rows * chunks * sizeof(float2) + 255) / 256 * 256; }

int check_beams(const char *op, int64_t prompts, int beams, int vocab, int n_out) {
    if (prompts < 0 || beams < 1 || beams > kMaxOut) return set_error(QMC_EINVAL, "%s: %lld prompts of %d beams", op, (long long)prompts, beams);
    if (vocab < 1) return set_error(QMC_EINVAL, "%s: vocabulary of %d", op, vocab);
    if (n_out < 1 || n_out > kMaxOut || n_out > (int64_t)beams * vocab) return set_error(QMC_EINVAL, "%s: n_out %d", op, n_out);
    if (prompts * beams > 65535) return set_error(QMC_EINVAL, "%s: %lld rows exceed 65535", op, (long long)prompts * beams);
    // the merge keeps one counter a list in shared memory
    if ((int64_t)beams * beam_chunks(vocab) > 10240)
        return set_error(QMC_EINVAL, "%s: %d beams over a vocabulary of %d are too many", op, beams, vocab);
    return QMC_OK;
}

}  // namespace
}  // namespace qmc

using namespace qmc;

extern "C" {

int qmc_beam_workspace(int32_t n_prompts, int32_t beams, int32_t n_vocab, int32_t n_out, size_t *bytes) {
    if (!bytes) return set_error(QMC_EINVAL, "beam_workspace: null argument");
    *bytes = 0;
    if (const int rc = check_beams("beam_workspace", n_prompts, beams, n_vocab, n_out)) return rc;
    const int64_t rows = (int64_t)n_prompts * beams;
    const int chunks = beam_chunks(n_vocab);
    *bytes = beam_stat_bytes(rows, chunks) + (size_t)rows * chunks * n_out * 8 + 256;
    return QMC_OK;
}

int qmc_beam_select(int dtype, const void *logits, int64_t ld, int32_t n_prompts, int32_t beams, int32_t n_vocab,
                    const float *scores, const uint8_t *finished, int32_t eos_token, int32_t n_out, int32_t *parents,
                    int32_t *tokens, float *out_scores, void *workspace, size_t workspace_bytes, void *stream) {
    const char *op = "beam_select";
    if (!is_row_dtype(dtype)) return set_error(QMC_EINVAL, "%s: bad dtype %d", op, dtype);
    if (const int rc = check_beams(op, n_prompts, beams, n_vocab, n_out)) return rc;
    if (ld < n_vocab || ld > (int64_t)1 << 40) return set_error(QMC_EINVAL, "%s: rows of %d logits are %lld apart", op, n_vocab, (long long)ld);
    if (finished && (eos_token < 0 || eos_token >= n_vocab)) return set_error(QMC_EINVAL, "%s: eos token %d", op, eos_token);
    if (n_prompts == 0) return QMC_OK;
    if (!logits || !scores || !parents || !tokens || !out_scores || !workspace)
        return set_error(QMC_EINVAL, "%s: null argument", op);
    if ((uintptr_t)logits % dtype_size(dtype)) return set_error(QMC_EINVAL, "%s: misaligned logits", op);
    size_t need = 0;
    qmc_beam_workspace(n_prompts, beams, n_vocab, n_out, &need);
    if (workspace_bytes < need) return set_error(QMC_EINVAL, "%s: workspace of %zu bytes, %zu needed", op, workspace_bytes, need);
    DevCtx *c = ctx();
    if (!c) return QMC_ECUDA;
    SelArgs a{};
    a.logits = logits, a.ld = ld, a.prompts = n_prompts, a.beams = beams, a.vocab = n_vocab, a.n_out = n_out, a.eos = eos_token;
    a.chunks = beam_chunks(n_vocab);
    a.scores = scores, a.finished = finished;
    const int64_t rows = (int64_t)n_prompts * beams;
    uint8_t *w = (uint8_t *)(((uintptr_t)workspace + 255) / 256 * 256);
    a.stat = (float2 *)w;
    a.cand = (unsigned long long *)(w + beam_stat_bytes(rows, a.chunks));
    a.parents = parents, a.tokens = tokens, a.out_scores = out_scores;
    cudaStream_t s = pick_stream(stream);
    const dim3 grid(a.chunks, (unsigned)rows);
    if (dtype == QMC_F32) beam_chunk_kernel<float><<<grid, kBT, 0, s>>>(a);
    else if (dtype == QMC_F16) beam_chunk_kernel<__half><<<grid, kBT, 0, s>>>(a);
    else beam_chunk_kernel<__nv_bfloat16><<<grid, kBT, 0, s>>>(a);
    QMC_LAUNCH_CHECK();
    beam_merge_kernel<<<n_prompts, kBT, (size_t)beams * a.chunks * 4, s>>>(a);
    QMC_LAUNCH_CHECK();
    return QMC_OK;
}

int qmc_beam_reorder(const qmc_paged_cache *cache, int32_t n_prompts, int32_t beams, const int32_t *parents,
                     int32_t ld_parents, const int32_t *seq_lens, const int32_t *page_table, int32_t *page_table_out,
                     int32_t ld_table, void *stream) {
    const char *op = "beam_reorder";
    if (const int rc = check_cache(cache, op)) return rc;
    if (n_prompts < 0 || beams < 1 || beams > kMaxOut || ld_parents < beams || ld_table < 1)
        return set_error(QMC_EINVAL, "%s: %d prompts of %d beams, parents %d apart, table %d wide", op, n_prompts, beams,
                         ld_parents, ld_table);
    if (cache->n_layers > 32767) return set_error(QMC_EINVAL, "%s: %d layers exceed the grid", op, cache->n_layers);
    if ((int64_t)n_prompts * beams > INT32_MAX) return set_error(QMC_EINVAL, "%s: too many rows", op);
    if (n_prompts == 0) return QMC_OK;
    if (!parents || !seq_lens || !page_table || !page_table_out) return set_error(QMC_EINVAL, "%s: null argument", op);
    if (page_table == page_table_out) return set_error(QMC_EINVAL, "%s: the table cannot be reordered in place", op);
    DevCtx *c = ctx();
    if (!c) return QMC_ECUDA;
    ReorderArgs a{};
    const int64_t sz = dtype_size(cache->dtype);
    a.pool[0] = (uint8_t *)cache->k, a.pool[1] = (uint8_t *)cache->v;
    a.slot_bytes = (int64_t)cache->n_kv_heads * cache->head_dim * sz;
    a.page_bytes = a.slot_bytes * cache->page_size;
    a.layer_bytes = a.page_bytes * cache->n_pages;
    a.n_pages = cache->n_pages, a.page_size = cache->page_size, a.beams = beams;
    a.ld_parents = ld_parents, a.ld_table = ld_table;
    a.parents = parents, a.lens = seq_lens, a.tin = page_table, a.tout = page_table_out, a.err = c->err;
    beam_reorder_kernel<<<dim3((unsigned)n_prompts * beams, 2u * cache->n_layers), kBT, 0, pick_stream(stream)>>>(a);
    QMC_LAUNCH_CHECK();
    return QMC_OK;
}

}  // extern "C"

// Beam search's selection over beams x vocabulary (qmc_beam_select) and the reordering of paged states
// (qmc_beam_reorder).
//
// Selection in two launches.  Both the log-sum-exp and the order need every logit once, so the first reads each row
// once, a chunk per block held in registers: the chunk's maximum m and sum of exp(x - m), and its n best logits.
// Within a row the order of scores is the order of logits, so n per chunk suffice whatever the row's log-sum-exp
// turns out to be.  The second, one block per prompt, joins a row's (m, sum) pairs and takes the n best of the rows' sorted lists.
// Exponentials are floats (2^-22), summed in float within a thread and in double over the block; a chunk's sum is stored as a float, and the
// chunks are added in double.
//
// The n best of a chunk: with w warps, the smallest of the warps' ceil(n / w)-th largest thread maxima is a lower bound T that at
// least n elements reach, found in a few warp-wide maxima (in the 32-bit order-preserving form); the few elements >= T are
// collected in shared memory and ranked by counting, with the index, so that ties go to the lower one.  Where too many reach T
// (equal logits), the exact n-th largest of the threads' maxima is built from the top bit, and its bits continued over the indices, after
// which at most n threads' elements remain.  Blocks stay and take chunk after chunk, the next one's logits on their way to registers.
// Measured with cold caches: 24 x 8 rows of 128000 bf16 logits, two of eight beams ended, 26.7 us (1.4 TB/s: the barriers and the
// warp-wide steps of a chunk bind it, three blocks an SM; spans of chunks with a running bound took longer, as did all rows in turn without
// a list of the live ones), 4 rows of 32000 floats 5.4 us; the merge 9.7 and 6.5 us; the reordering 14.4 us for 67 MB (4.7 TB/s) and 6.7 us.
// Of the lists' heads, whose beams' scores lie apart, the exact n-th largest is taken at once; where too many reach it, n rounds of a
// block-wide maximum over the heads.
#include <algorithm>

#include "attn_prefix.cuh"

namespace qmc {
namespace {

constexpr int kBT = 256;      // threads
constexpr int kMaxOut = 64;   // n_out and beams
constexpr int kGroups = 256;  // 16-byte groups of logits of a chunk that may reach the bound before it counts as one with too many
constexpr int kListed = 1024;  // rows of a call whose live ones are listed
constexpr int kLeast = 4096;  // logits of the smallest chunk
// logits per thread: 4 16-byte loads
template <typename T>
__host__ __device__ constexpr int items() {
    return 64 / sizeof(T);
}
static_assert(items<float>() * kBT == kLeast, "smallest chunk");

struct SelArgs {
    const void *logits;
    int64_t ld;
    int prompts, beams, vocab, n_out, eos, chunks, chunk;
    const float *scores;
    const uint8_t *finished;
    float2 *stat;              // [row][chunk] (m, sum exp(x - m))
    unsigned long long *cand;  // [row][chunk][n_out] keys, falling
    int *parents, *tokens;
    float *out_scores;
};

// order-preserving bits of a float, -0 as +0; no NaN comes here.  Never 0.
__device__ __forceinline__ uint32_t order_bits(float v) {
    const uint32_t u = __float_as_uint(v + 0.0f);  // -0 + 0 = +0
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t u) {
    return __uint_as_float((u & 0x80000000u) ? (u & 0x7fffffffu) : ~u);
}

// by one warp: the largest T that at least n of the 256 values reach (their n-th largest, or a value above it that exactly n
// reach), at least 1
__device__ __forceinline__ uint32_t nth_largest(const uint32_t *vals, int lane, int n) {
    uint32_t mine[kBT / 32], hi = 0, lo = 0xffffffffu;
#pragma unroll
    for (int j = 0; j < kBT / 32; j++) {
        mine[j] = vals[lane + 32 * j];
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
    return max(t, 1u);
}

// the k-th largest of the warp's values (0: there are fewer)
__device__ __forceinline__ uint32_t warp_kth(uint32_t v, int lane, int k) {
    uint32_t mx = 0;
    for (int r = 0; r < k; r++) {
        mx = __reduce_max_sync(0xffffffffu, v);
        const unsigned holders = __ballot_sync(0xffffffffu, v == mx);
        if (lane == __ffs(holders) - 1) v = 0;
    }
    return mx;
}
// how many of the warps' largest make n together, and over how many warps, when the first `threads` threads have a value; no warp: no
// bound
__device__ __forceinline__ int kth_of(int threads, int n, int &warps) {
    warps = min(threads, kBT) / 32;
    const int k = warps ? (n + warps - 1) / warps : 33;
    if (k > 32) warps = 0;
    return k;
}

template <typename T>
__global__ void __launch_bounds__(kBT, 3) beam_chunk_kernel(const SelArgs a) {
    constexpr int E = items<T>(), C = 16 / sizeof(T), CAP = kMaxOut * E;
    __shared__ uint32_t vmax[kBT], kth[kBT / 32];
    __shared__ unsigned long long buf[CAP], T64_s;
    __shared__ float gval[kGroups][C];  // 16-byte groups that reach the bound
    __shared__ int gat[kGroups], groups_s;
    __shared__ float red[kBT / 32];
    __shared__ double redd[kBT / 32];
    __shared__ int cnt_s;
    __shared__ uint16_t list_s[kListed];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_launch_dependents();
    const int rows = a.prompts * a.beams;
    int total = rows * a.chunks;
    // the second kernel does not look at the lists of a finished or dead beam
    auto live = [&](int row) {
        const bool ended = a.finished && a.finished[row];
        return a.scores[row] > -INFINITY && !ended;
    };
    // blocks with several chunks share out those of the live rows alone; where each has one, a dead row's has nothing to do
    const bool listed = total > (int)gridDim.x && rows <= kListed;
    if (listed) {
        int n = 0;
        for (int r0 = 0; r0 < rows; r0 += kBT) {
            const bool mine = r0 + tid < rows && live(r0 + tid);
            const unsigned votes = __ballot_sync(0xffffffffu, mine);
            if (lane == 0) kth[warp] = __popc(votes);
            __syncthreads();
            int at = n + __popc(votes & ((1u << lane) - 1));
            for (int w = 0; w < kBT / 32; w++) {
                if (w < warp) at += kth[w];
                n += kth[w];
            }
            if (mine) list_s[at] = (uint16_t)(r0 + tid);
            __syncthreads();
        }
        total = n * a.chunks;
    }
    auto row_of = [&](int item) { return listed ? (int)list_s[item / a.chunks] : item / a.chunks; };
    auto live_item = [&](int item) { return item < total && (listed || live(item / a.chunks)); };
    Chunk<T, C> raw[E / C] = {};
    auto fetch = [&](int item) {  // -inf past the end
        const int row = row_of(item), base = item % a.chunks * a.chunk, nel = min(a.chunk, a.vocab - base);
        const T *x = (const T *)a.logits + (int64_t)row * a.ld + base;
        const bool vec = ((uintptr_t)x & 15) == 0;
#pragma unroll
        for (int j = 0; j < E / C; j++) {
            const int e = (j * kBT + tid) * C;
            if (vec && e + C <= nel) {
                raw[j] = *(const Chunk<T, C> *)(x + e);
            } else {
#pragma unroll
                for (int i = 0; i < C; i++) {
                    if (e + i < nel) raw[j].e[i] = x[e + i];
                    else from_f32(-INFINITY, &raw[j].e[i]);
                }
            }
        }
    };
    bool here = live_item(blockIdx.x), next = live_item(blockIdx.x + gridDim.x);
    if (here) fetch(blockIdx.x);
    for (int item = blockIdx.x; item < total; item += gridDim.x) {
    const bool now = here;
    const int chunk = item % a.chunks, row = row_of(item);
    const int base = chunk * a.chunk, nel = min(a.chunk, a.vocab - base), n = min(a.n_out, nel);
    auto place = [&](int k) { return ((k / C) * kBT + tid) * C + k % C; };  // in the chunk
    float v[E];
#pragma unroll
    for (int j = 0; j < E / C; j++) {
        float t[C];
        widen(raw[j], t);
#pragma unroll
        for (int i = 0; i < C; i++) v[j * C + i] = t[i];
    }
    here = next;
    if (here) fetch(item + gridDim.x);
    next = live_item(item + 2 * gridDim.x);
    if (!now) continue;

    float top[E / C], best = -INFINITY;  // NaN counts as -inf: maxima pass it over
#pragma unroll
    for (int j = 0; j < E / C; j++) {
        top[j] = -INFINITY;
#pragma unroll
        for (int i = 0; i < C; i++) top[j] = fmaxf(top[j], v[j * C + i]);
        best = fmaxf(best, top[j]);
    }
    const uint32_t mine = place(0) < nel ? order_bits(best) : 0u;  // a thread's first element comes before its others
    int warps;
    const int k_each = kth_of((nel + C - 1) / C, n, warps);
    const uint32_t my_kth = warps ? warp_kth(mine, lane, k_each) : 0u;
    float m = warp_max(best);
    if (lane == 0) red[warp] = m, kth[warp] = my_kth;
    if (tid == 0) cnt_s = groups_s = 0;
    __syncthreads();
    m = red[0];
#pragma unroll
    for (int w = 1; w < kBT / 32; w++) m = fmaxf(m, red[w]);
    uint32_t bound = 0xffffffffu;  // T
    for (int w = 0; w < warps; w++) bound = min(bound, kth[w]);
    bound = warps ? max(bound, 1u) : 1u;
    float s4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (m == INFINITY) {  // the infinities share the probability
#pragma unroll
        for (int k = 0; k < E; k++) s4[0] += v[k] == m ? 1.0f : 0.0f;
    } else if (m > -INFINITY) {
#pragma unroll
        for (int k = 0; k < E; k++) s4[k & 3] += ex2((v[k] - m) * 1.4426950408889634f);
    }
    float s = (s4[0] + s4[1]) + (s4[2] + s4[3]);
    if (s != s) {  // some NaN among them
        s = 0.0f;
#pragma unroll
        for (int k = 0; k < E; k++) s += v[k] == v[k] ? ex2((v[k] - m) * 1.4426950408889634f) : 0.0f;
    }
    const double sd = warp_sum_d((double)s);
    if (lane == 0) redd[warp] = sd;
    __syncthreads();
    if (tid == 0) {
        double tot = 0.0;
        for (int w = 0; w < kBT / 32; w++) tot += redd[w];
        a.stat[(int64_t)row * a.chunks + chunk] = make_float2(m, (float)tot);
    }
    auto key_of = [&](int k) { return ((unsigned long long)order_bits(fmaxf(v[k], -INFINITY)) << 32) | (uint32_t)~(base + place(k)); };
    auto collect = [&](unsigned long long least) {
        if (mine >= (uint32_t)(least >> 32)) {
            // T as a float, for one comparison an element; where -inf and NaN reach it, all do
            const uint32_t bits = (uint32_t)(least >> 32);
            const bool any = bits <= order_bits(-INFINITY);
            const float value = any ? -INFINITY : order_value(bits);
#pragma unroll
            for (int j = 0; j < E / C; j++) {
                if (!(top[j] >= value)) continue;
#pragma unroll
                for (int i = 0; i < C; i++) {
                    const int k = j * C + i;
                    if (!(v[k] >= value) && !any) continue;
                    if (place(k) >= nel) continue;
                    const unsigned long long key = key_of(k);
                    if (key >= least) {
                        const int at = atomicAdd(&cnt_s, 1);  // places differ from run to run, ranks do not
                        if (at < CAP) buf[at] = key;
                    }
                }
            }
        }
    };
    // first the 16-byte groups that reach the bound, then, an element a thread, what of them does.  -inf never does: where fewer than
    // n others exist, every element is looked at below
    const float value = bound <= order_bits(-INFINITY) ? -INFINITY : order_value(bound);
    if (best >= value) {
#pragma unroll
        for (int j = 0; j < E / C; j++)
            if (top[j] >= value && place(j * C) < nel) {
                const int at = atomicAdd(&groups_s, 1);  // places differ from run to run, ranks do not
                if (at < kGroups) {
                    gat[at] = place(j * C);
#pragma unroll
                    for (int i = 0; i < C; i++) gval[at][i] = v[j * C + i];
                }
            }
    }
    __syncthreads();
    const int groups = groups_s;
    if (groups <= kGroups)
        for (int i = tid; i < groups * C; i += kBT) {
            const float y = gval[i / C][i % C];
            const int at = gat[i / C] + i % C;
            if ((y >= value || value == -INFINITY) && at < nel) {
                const int to = atomicAdd(&cnt_s, 1);
                if (to < CAP) buf[to] = ((unsigned long long)order_bits(fmaxf(y, -INFINITY)) << 32) | (uint32_t)~(base + at);
            }
        }
    __syncthreads();
    int cnt = groups <= kGroups ? cnt_s : CAP + 1;
    __syncthreads();  // read by all before a second collection changes it
    if (cnt > CAP) {
        // many equal logits: the threads' maxima with their indices are distinct; T's lower bits are built over those
        unsigned long long top = 0;
#pragma unroll
        for (int k = 0; k < E; k++)
            if (place(k) < nel) top = max(top, key_of(k));
        buf[tid] = top, vmax[tid] = mine;
        __syncthreads();
        if (warp == 0) {
            unsigned long long t = (unsigned long long)nth_largest(vmax, lane, n) << 32;
            for (int bit = 31; bit >= 0; bit--) {
                const unsigned long long c = t | (1ull << bit);
                int k = 0;
#pragma unroll
                for (int j = 0; j < kBT / 32; j++) k += buf[lane + 32 * j] >= c;
                if (__reduce_add_sync(0xffffffffu, k) >= n) t = c;
            }
            if (lane == 0) T64_s = t, cnt_s = 0;
        }
        __syncthreads();
        collect(T64_s);
        __syncthreads();
        cnt = min(cnt_s, CAP);
    }
    unsigned long long *out = a.cand + ((int64_t)row * a.chunks + chunk) * a.n_out;
    for (int i = tid; i < cnt; i += kBT) {
        const unsigned long long key = buf[i];
        int rank = 0;
        for (int j = 0; j < cnt; j++) rank += buf[j] > key;
        if (rank < n) out[rank] = key;
    }
    __syncthreads();  // before the next chunk
    }
}

// the i-th of a list that does not come from the logits: a finished beam's one continuation, or none (dead); the other tokens
// follow at -inf in order
__device__ __forceinline__ int virtual_token(bool ended, int eos, int i) {
    return !ended ? i : i == 0 ? eos : i - 1 + (i - 1 >= eos);
}

struct Head {
    double score;
    uint64_t at;  // beam << 32 | token: ordered as beam * vocab + token.  ~0: none
};
__device__ __forceinline__ bool before(const Head &a, const Head &b) {
    return a.score > b.score || (a.score == b.score && a.at < b.at);
}
constexpr int kMergeCap = 512;  // candidates that are ranked by counting

__global__ void __launch_bounds__(kBT) beam_merge_kernel(const SelArgs a) {
    __shared__ double lse_s[kMaxOut], cum_s[kMaxOut];  // lse: of the logits above the row's largest, top_s
    __shared__ float top_s[kMaxOut];
    __shared__ uint8_t kind_s[kMaxOut];  // 0 logits, 1 finished, 2 dead
    __shared__ Head buf[kMergeCap];
    __shared__ uint32_t vmax[kBT], T_s;
    __shared__ int cnt_s, wth[kBT / 32];
    extern __shared__ int next_s[];  // [beams * chunks] entries taken of each list (the rounds)
    const int prompt = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int lists = a.beams * a.chunks, offered = min(a.n_out, a.vocab);
    pdl_launch_dependents();
    pdl_wait();
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
                if (p.x > -INFINITY) s += (double)(p.y * (p.x == m ? 1.0f : ex2((p.x - m) * 1.4426950408889634f)));
            }
            s = warp_sum_d(s);
        }
        if (lane == 0) {
            cum_s[b] = cum, top_s[b] = m;
            kind_s[b] = ended ? 1 : (dead || !(m > -INFINITY)) ? 2 : 0;
            lse_s[b] = log(s);
        }
    }
    if (tid == 0) cnt_s = 0;
    __syncthreads();

    auto entry = [&](int list, int i) {  // the i-th of a list
        Head h{-INFINITY, ~0ull};
        const int b = list / a.chunks, c = list % a.chunks, kind = kind_s[b];
        if (kind) {
            if (c == 0 && i < offered) {
                h.at = (uint64_t)b << 32 | (uint32_t)virtual_token(kind == 1, a.eos, i);
                if (kind == 1 && i == 0) h.score = cum_s[b];
            }
            return h;
        }
        if (i >= min(a.n_out, a.vocab - c * a.chunk)) return h;
        if (i >= a.chunk) return h;
        const unsigned long long *const keys = a.cand + ((int64_t)(prompt * a.beams + b) * a.chunks + c) * a.n_out;
        const unsigned long long key = keys[i];
        const float x = order_value((uint32_t)(key >> 32));
        h.at = (uint64_t)b << 32 | (uint32_t)~(uint32_t)key;
        if (top_s[b] == INFINITY) {
            // lse_s is the log of the number of infinities, which come first.  All other tokens score -inf, so their order is the
            // tokens', not the logits': chunk 0's list goes on with the lowest ones that are not infinite.  The first i of
            // these end below n_out, as do the infinities that they pass over, all of which are in the list
            if (x == INFINITY) {
                h.score = cum_s[b] - lse_s[b];
            } else if (c == 0) {
                int infs = 0;
                while (infs < i && order_value((uint32_t)(keys[infs] >> 32)) == INFINITY) infs++;
                uint32_t token = (uint32_t)(i - infs);
                for (int j = 0; j < infs; j++) token += ~(uint32_t)keys[j] <= token;
                h.at = (uint64_t)b << 32 | token;
            } else {
                h.at = ~0ull;
            }
        } else {
            // the distance first: a large logit would round the logarithm away, and rows that differ by a constant are to tie
            h.score = cum_s[b] + (((double)x - (double)top_s[b]) - lse_s[b]);
        }
        if (h.score != h.score) h.score = -INFINITY;
        return h;
    };
    // the score rounded down to a float keeps the order; equal bits are settled by the whole score and the index
    auto bits = [&](const Head &h) { return h.at == ~0ull ? 0u : order_bits(__double2float_rd(h.score)); };
    auto put = [&](int r, const Head &h) {
        const int64_t o = (int64_t)prompt * a.n_out + r;
        a.parents[o] = (int)(h.at >> 32);
        a.tokens[o] = (int)(uint32_t)h.at;
        a.out_scores[o] = (float)h.score;
    };
    uint32_t best = 0;
    for (int l = tid; l < lists; l += kBT) best = max(best, bits(entry(l, 0)));
    vmax[tid] = best;
    __syncthreads();
    if (warp == 0) {
        const uint32_t t = nth_largest(vmax, lane, a.n_out);
        if (lane == 0) T_s = t;
    }
    __syncthreads();
    const uint32_t least = T_s;
    if (best >= least)
        for (int l = tid; l < lists; l += kBT)
            for (int i = 0; i < offered; i++) {
                const Head h = entry(l, i);
                if (bits(h) < least) break;
                const int at = atomicAdd(&cnt_s, 1);
                if (at < kMergeCap) buf[at] = h;
                else break;
            }
    __syncthreads();
    const int cnt = cnt_s;
    if (cnt <= kMergeCap) {
        for (int i = tid; i < cnt; i += kBT) {
            const Head h = buf[i];
            int rank = 0;
            for (int j = 0; j < cnt; j++) rank += before(buf[j], h);
            if (rank < a.n_out) put(rank, h);
        }
        return;
    }

    // many equal scores: n rounds of a maximum over the lists' heads, each thread's in registers
    for (int i = tid; i < lists; i += kBT) next_s[i] = 0;
    __syncthreads();
    Head mine{-INFINITY, ~0ull};
    int my_list = -1;
    auto scan = [&]() {
        mine = Head{-INFINITY, ~0ull};
        my_list = -1;
        for (int l = tid; l < lists; l += kBT) {
            const Head h = entry(l, next_s[l]);
            if (h.at != ~0ull && (my_list < 0 || before(h, mine))) mine = h, my_list = l;
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
            g.at = __shfl_xor_sync(0xffffffffu, h.at, o);
            const int gt = __shfl_xor_sync(0xffffffffu, th, o);
            if (before(g, h)) h = g, th = gt;
        }
        if (lane == 0) buf[warp] = h, wth[warp] = th;
        __syncthreads();
        h = buf[0], th = wth[0];
#pragma unroll
        for (int w = 1; w < kBT / 32; w++)
            if (before(buf[w], h)) h = buf[w], th = wth[w];
        if (tid == 0) put(r, h);
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
    int n_pages, page_size, beams, ld_parents, ld_table, layers;
    const int *parents, *lens, *tin;
    int *tout, *err;
};

constexpr int kPiece = 4 * 16 * kBT;  // bytes of keys, and of values, that a block copies at a time: eight loads a thread on their way

// blockIdx.x: prompt; its blocks work out all beams' pages from the prompt's parents, and share its table rows and the pieces of its
// copies evenly.  Bound by latency: length, parents, table entries and the copies follow on one another, so every block stays
// for several pieces and all run at once (192 beams of 16 layers, two of eight beams ended, with the
// selection before it: 53.1 us with a block for each beam and few layers, 52.2 so).
__global__ void __launch_bounds__(kBT) beam_reorder_kernel(const ReorderArgs a) {
    __shared__ int par[kMaxOut], owner[kMaxOut];  // owner: the beam whose page being filled becomes this one's
    __shared__ int2 copy[kMaxOut];                // pages from and to, of the further children in order
    __shared__ uint8_t has[kMaxOut], first[kMaxOut], child[kMaxOut];
    __shared__ int copies_s;
    const int prompt = blockIdx.x, tid = threadIdx.x;
    pdl_wait();
    int n = a.lens[(int64_t)prompt * a.beams];
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
    if (tid < a.beams) {
        int e = 0, o = par[tid];
        for (int i = 0; i < tid; i++) e += !first[i];
        if (tid == a.beams - 1) copies_s = e + !first[tid];
        if (!first[tid]) {
            child[e] = (uint8_t)tid;
            // as many beams have no child as there are further children
            for (int i = 0; i < a.beams; i++)
                if (!has[i] && e-- == 0) {
                    o = i;
                    break;
                }
        }
        owner[tid] = o;
    }
    __syncthreads();
    const int *const rows = a.tin + (int64_t)prompt * a.beams * a.ld_table;
    if (tid < copies_s && filled) {
        const int j = child[tid];
        int2 c = make_int2(-1, -1);
        if (tail < a.ld_table) c = make_int2(rows[(int64_t)par[j] * a.ld_table + tail], rows[(int64_t)owner[j] * a.ld_table + tail]);
        if (c.x < 0 || c.x >= a.n_pages || c.y < 0 || c.y >= a.n_pages) {
            raise_error(a.err, kErrBadIndex);
            c.x = -1;
        }
        copy[tid] = c;
    }
    for (int j = blockIdx.y; j < a.beams; j += gridDim.y) {
        const int *own = rows + (int64_t)j * a.ld_table, *from = rows + (int64_t)par[j] * a.ld_table, *give = rows + (int64_t)owner[j] * a.ld_table;
        int *out = a.tout + ((int64_t)prompt * a.beams + j) * a.ld_table;
        for (int i = tid; i < a.ld_table; i += kBT) out[i] = i < tail ? from[i] : i == tail ? give[i] : own[i];
    }
    __syncthreads();
    if (filled == 0) return;
    const int64_t bytes = filled * a.slot_bytes;
    const unsigned copies = copies_s, pieces = (unsigned)((bytes + kPiece - 1) / kPiece), units = copies * pieces * a.layers;  // below 2^31
    for (unsigned u = blockIdx.y; u < units; u += gridDim.y) {
        const int2 c = copy[u % copies];
        if (c.x < 0) continue;
        const int64_t layer = u / copies / pieces * a.layer_bytes, at = (int64_t)(u / copies % pieces) * kPiece, left = min((int64_t)kPiece, bytes - at);
        const int64_t from_at = layer + c.x * a.page_bytes + at, to_at = layer + c.y * a.page_bytes + at;
        uint8_t *const k = a.pool[0], *const v = a.pool[1];
        if ((((uintptr_t)k | (uintptr_t)v | (uintptr_t)from_at | (uintptr_t)to_at | (uintptr_t)left) & 15) == 0) {
            const uint4 *ks = (const uint4 *)(k + from_at), *vs = (const uint4 *)(v + from_at);
            uint4 *kd = (uint4 *)(k + to_at), *vd = (uint4 *)(v + to_at);
            uint4 x[4], z[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (16 * (tid + i * kBT) < left) x[i] = __ldcs(ks + tid + i * kBT), z[i] = __ldcs(vs + tid + i * kBT);
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (16 * (tid + i * kBT) < left) kd[tid + i * kBT] = x[i], vd[tid + i * kBT] = z[i];
        } else {
            for (int64_t i = tid; i < left / 2; i += kBT) {
                ((uint16_t *)(k + to_at))[i] = ((const uint16_t *)(k + from_at))[i];
                ((uint16_t *)(v + to_at))[i] = ((const uint16_t *)(v + from_at))[i];
            }
        }
    }
}

int beam_chunks(int vocab, int chunk) { return (vocab + chunk - 1) / chunk; }
size_t beam_stat_bytes(int64_t rows, int chunks) { return ((size_t)rows * chunks * sizeof(float2) + 255) / 256 * 256; }

int check_beams(const char *op, int64_t prompts, int beams, int vocab, int n_out) {
    if (prompts < 0 || beams < 1 || beams > kMaxOut) return set_error(QMC_EINVAL, "%s: %lld prompts of %d beams", op, (long long)prompts, beams);
    if (vocab < 1) return set_error(QMC_EINVAL, "%s: vocabulary of %d", op, vocab);
    if (n_out < 1 || n_out > kMaxOut || n_out > (int64_t)beams * vocab) return set_error(QMC_EINVAL, "%s: n_out %d", op, n_out);
    if (prompts * beams > 65535) return set_error(QMC_EINVAL, "%s: %lld rows exceed 65535", op, (long long)prompts * beams);
    // the merge keeps one counter a list in shared memory
    if ((int64_t)beams * beam_chunks(vocab, kLeast) > 8192)
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
    const int chunks = beam_chunks(n_vocab, kLeast);  // whatever the logits' type
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
    if (misaligned({scores, parents, tokens, out_scores})) return set_error(QMC_EINVAL, "%s: misaligned scores, parents or tokens", op);
    size_t need = 0;
    qmc_beam_workspace(n_prompts, beams, n_vocab, n_out, &need);
    if (workspace_bytes < need) return set_error(QMC_EINVAL, "%s: workspace of %zu bytes, %zu needed", op, workspace_bytes, need);
    DevCtx *c = ctx();
    if (!c) return QMC_ECUDA;
    SelArgs a{};
    a.logits = logits, a.ld = ld, a.prompts = n_prompts, a.beams = beams, a.vocab = n_vocab, a.n_out = n_out, a.eos = eos_token;
    a.chunk = dtype == QMC_F32 ? kLeast : 2 * kLeast;
    a.chunks = beam_chunks(n_vocab, a.chunk);
    a.scores = scores, a.finished = finished;
    const int64_t rows = (int64_t)n_prompts * beams;
    uint8_t *w = (uint8_t *)(((uintptr_t)workspace + 255) / 256 * 256);
    a.stat = (float2 *)w;
    a.cand = (unsigned long long *)(w + beam_stat_bytes(rows, a.chunks));
    a.parents = parents, a.tokens = tokens, a.out_scores = out_scores;
    cudaStream_t s = pick_stream(stream);
    const int grid = (int)std::min<int64_t>(rows * a.chunks, 3 * c->num_sms);
    if (dtype == QMC_F32) beam_chunk_kernel<float><<<grid, kBT, 0, s>>>(a);
    else if (dtype == QMC_F16) beam_chunk_kernel<__half><<<grid, kBT, 0, s>>>(a);
    else beam_chunk_kernel<__nv_bfloat16><<<grid, kBT, 0, s>>>(a);
    QMC_LAUNCH_CHECK();
    return launch_after(beam_merge_kernel, dim3(n_prompts), kBT, beams * a.chunks * 4, s, true, a);
}

int qmc_beam_reorder(const qmc_paged_cache *cache, int32_t n_prompts, int32_t beams, const int32_t *parents,
                     int32_t ld_parents, const int32_t *seq_lens, const int32_t *page_table, int32_t *page_table_out,
                     int32_t ld_table, void *stream) {
    const char *op = "beam_reorder";
    if (const int rc = check_cache(cache, op)) return rc;
    if (n_prompts < 0 || beams < 1 || beams > kMaxOut || ld_parents < beams || ld_table < 1)
        return set_error(QMC_EINVAL, "%s: %d prompts of %d beams, parents %d apart, table %d wide", op, n_prompts, beams,
                         ld_parents, ld_table);
    if (cache->n_layers > 1 << 20) return set_error(QMC_EINVAL, "%s: %d layers", op, cache->n_layers);
    if ((int64_t)n_prompts * beams > INT32_MAX) return set_error(QMC_EINVAL, "%s: too many rows", op);
    const int64_t page_bytes = (int64_t)cache->n_kv_heads * cache->head_dim * dtype_size(cache->dtype) * cache->page_size;
    const int64_t most = (int64_t)beams * cache->n_layers * ((page_bytes + kPiece - 1) / kPiece);  // pieces of a prompt
    if (most > INT32_MAX) return set_error(QMC_EINVAL, "%s: %d beams of %d layers of such pages are too many", op, beams, cache->n_layers);
    if (n_prompts == 0) return QMC_OK;
    if (!parents || !seq_lens || !page_table || !page_table_out) return set_error(QMC_EINVAL, "%s: null argument", op);
    if (misaligned({parents, seq_lens, page_table, page_table_out}))
        return set_error(QMC_EINVAL, "%s: misaligned parents, lengths or page table", op);
    if (page_table == page_table_out) return set_error(QMC_EINVAL, "%s: the table cannot be reordered in place", op);
    DevCtx *c = ctx();
    if (!c) return QMC_ECUDA;
    ReorderArgs a{};
    const int64_t sz = dtype_size(cache->dtype);
    a.pool[0] = (uint8_t *)cache->k, a.pool[1] = (uint8_t *)cache->v;
    a.slot_bytes = (int64_t)cache->n_kv_heads * cache->head_dim * sz;
    a.page_bytes = page_bytes;
    a.layer_bytes = a.page_bytes * cache->n_pages;
    a.n_pages = cache->n_pages, a.page_size = cache->page_size, a.beams = beams;
    a.ld_parents = ld_parents, a.ld_table = ld_table;
    a.parents = parents, a.lens = seq_lens, a.tin = page_table, a.tout = page_table_out, a.err = c->err;
    // as many blocks as run at once, as far as there are pieces.  They may start while the selection before them ends, and read
    // nothing before it has ended.
    a.layers = cache->n_layers;
    const int64_t want = (3 * c->num_sms + n_prompts - 1) / n_prompts;
    const dim3 grid((unsigned)n_prompts, (unsigned)std::min(want, most));
    return launch_after(beam_reorder_kernel, grid, kBT, 0, pick_stream(stream), true, a);
}

}  // extern "C"

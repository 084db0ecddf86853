// Which drafted tokens the target takes, and the token that follows them, from given random numbers.
//
// For one sequence: drafts x_0 .. x_{G-1}; target logits in G + 1 rows, draft logits in G rows; p_i and q_i the softmax at
// the temperature over each row's top_k largest logits (ties: the lowest index first).  Draft i is taken while
//     u_i q_i(x_i) < p_i(x_i);
// at the first that is not, the token comes from max(p_i - q_i, 0), after the last draft (or at a draft of -1, which ends
// a sequence's drafts) from p_i alone: the first index at which the running sum in the vocabulary's order passes u_G of the
// whole.  The tokens are then distributed as p's.  Greedy: a draft is taken while it is its row's first maximum.
//
// Where nothing is left of max(p - q, 0) (p and q equal) the token comes from p; where p has no mass either (a row without a
// finite logit, or one with a NaN) it is the row's first maximum, a NaN being larger than every number.
//
// Two launches.  The first reads every row once.  Without a top_k: its maximum and its sum of exp((l - max) / T), which are bound
// by the reading.  With one: the k largest logits, as a list (verify_top_kernel).  Greedy: the first maximum.  The second
// decides, a block or a cluster of blocks a sequence, and draws the token: from the lists (verify_list_kernel), or by a
// walk over the one row pair that matters, each block of the cluster its share of the vocabulary (verify_walk_kernel).
// What bounds them, on a B200: the first launch reads 704 rows of 50,257 logits (141 MB) in 27 us, 5.3 TB/s, one such launch after another;
// the walk behind it for 64 sequences takes another 47, two waves of clusters: some 33 clusters of eight go at a time (rows that are still
// in the L2, no drafts: 8 to 32 sequences 13 to 17 us, 36 to 64 21 to 25).  With a top_k of 40, 8 sequences of 4 drafts:
// 17.3 us for both, 11.9 the first, which reads 1.5, finds the floor 1.2, gathers 1.7, ranks 1, joins 2.6.
// The walk is in 64 bits, exponentials included: with 50,000 tokens in a row a running sum that is off by 1e-7 of the whole
// would give another token once in a hundred draws.  The exponentials are made by a table
// (exp_of).  Decisions about drafts are the 64-bit formula's too: the first launch's 32-bit sums decide where their error cannot matter, and
// a draft nearer than that to its border (5e-5 of it, about one in 20,000) has its two rows added up again in 64 bits.
#include "common.cuh"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace mu {

// Orders as the floats do, -0 and 0 the same; a NaN without a sign is above them all, one with a sign below.  (By whole numbers: of
// v + 0.0f the compiler takes a NaN's sign as it likes.)
__device__ __forceinline__ unsigned int order_key(float v) {
    const unsigned int b = __float_as_uint(v);
    return 0x80000000u + ((b & 0x80000000u) ? 0u - (b & 0x7FFFFFFFu) : b);
}
__device__ __forceinline__ float key_value(unsigned int k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : 0x80000000u | (0x80000000u - k));
}
// A larger logit wins, any NaN against every number; among equals the lower index.
__device__ __forceinline__ unsigned long long best_of(float v, int i) {
    return ((unsigned long long)(v != v ? 0xFFFFFFFFu : order_key(v)) << 32) | (0xFFFFFFFFu - (unsigned int)i);
}
__device__ __forceinline__ unsigned long long larger(unsigned long long a, unsigned long long b) { return a > b ? a : b; }
__device__ __forceinline__ unsigned long long warp_best(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = larger(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ double warp_total(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// exp(x) for x <= 0 in 64 bits: x = (64 m + j + f) ln2 / 64 with |f| <= 1/2, exp(x) = 2^m 2^(j / 64) exp(f ln2 / 64), the last factor by
// its series (the fifth term is below 4e-14).  The table-driven method of P. T. P. Tang, "Table-driven implementation of the
// exponential function in IEEE floating-point arithmetic" (1989), with fewer terms.  Within 1e-13 of exp; 0 below -700,
// NaN for NaN.  Nine 64-bit operations where exp takes some forty.
__device__ __forceinline__ void exp_table(double* table) {           // 64 entries of shared memory, by the block's first threads
    if (threadIdx.x < 64) table[threadIdx.x] = exp2((double)threadIdx.x / 64.0);
}
__device__ __forceinline__ double exp_of(double x, const double* table) {
    const double shift = 6755399441055744.0;                          // 1.5 * 2^52: adding it rounds to a whole number
    const double t = fma(x, 92.332482616893656877, shift);            // 64 / ln2
    const int n = __double2loint(t);
    const double r = fma(t - shift, -0.010830424696249145461, x);     // ln2 / 64
    double p = fma(r, 1.0 / 24.0, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p * r, r, r);
    const double e = table[n & 63];
    const double v = fma(e, p, e);
    const double scaled = __hiloint2double(__double2hiint(v) + ((n >> 6) << 20), __double2loint(v));
    return x >= -700.0 ? scaled : (x < -700.0 ? 0.0 : x);
}

// What the first launch says of a part of a row (a row has one part where a top_k cuts it).
struct VerifyPart {
    unsigned long long best;       // greedy and with a top_k: the part's first maximum (best_of); else only its logit
    double sum;                    // of exp((l - max) / T) over what is kept, max the part's
    unsigned int threshold;        // kept: key above it, or equal to it and an index up to last
    int last;
    float at_draft;                // the row's logit of the draft that it decides about (-inf where there is none)
    int unused;
};

struct VerifyRows {
    const float* target;           // [batch][drafts + 1][vocab], strides below
    const float* draft;            // [batch][drafts][vocab], or null (greedy)
    long long target_seq, target_row, draft_seq, draft_row;
    int batch, drafts, vocab;
    __device__ __forceinline__ const float* row(int r) const {         // rows of the targets, then those of the drafts
        const int t = batch * (drafts + 1);
        if (r < t) return target + (long long)(r / (drafts + 1)) * target_seq + (long long)(r % (drafts + 1)) * target_row;
        r -= t;
        return draft + (long long)(r / drafts) * draft_seq + (long long)(r % drafts) * draft_row;
    }
    // The logit of row r (at `row`) of the draft that it decides about.
    __device__ __forceinline__ float at_draft(int r, const float* at_row, const int* tokens) const {
        const int t = batch * (drafts + 1);
        int x = -1;
        if (r >= t) x = tokens[r - t];
        else if (r % (drafts + 1) < drafts) x = tokens[r / (drafts + 1) * drafts + r % (drafts + 1)];
        return x >= 0 && x < vocab ? at_row[x] : -INFINITY;
    }
};

constexpr int VS_THREADS = 256;

// A share [begin, end) of a row by a block's threads, sixteen logits a thread and turn in aligned pieces of four, the next turn's on
// their way while f works on this one's: f(l, index of l[0], ..) with l[4 v .. 4 v + 3] the logits index + 4 THREADS v + 0 .. 3, -inf past the
// end.  The up to three logits before the first aligned piece and behind the last one come first, one a thread: g(l, index).
template <int THREADS, typename F, typename G>
__device__ __forceinline__ void for_share(const float* row, int begin, int end, F f, G g) {
    const int tid = threadIdx.x, head = min(end - begin, (int)((16 - ((uintptr_t)(row + begin) & 15)) & 15) / 4);
    const int body = begin + head, pieces = (end - body) / 4, tail = body + 4 * pieces;
    if (tid < head) g(row[begin + tid], begin + tid);
    else if (tid >= 32 && tid - 32 < end - tail) g(row[tail + tid - 32], tail + tid - 32);
    constexpr int V = 4;
    const float4* from = reinterpret_cast<const float4*>(row + body);
    float4 next[V];
    const float4 none = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    auto ask = [&](int i) {
#pragma unroll
        for (int v = 0; v < V; ++v) next[v] = i + v * THREADS < pieces ? __ldg(from + i + v * THREADS) : none;
    };
    ask(tid);
    for (int i = tid; i < pieces; i += V * THREADS) {
        float l[4 * V];
#pragma unroll
        for (int v = 0; v < V; ++v) { l[4 * v] = next[v].x; l[4 * v + 1] = next[v].y; l[4 * v + 2] = next[v].z; l[4 * v + 3] = next[v].w; }
        ask(i + V * THREADS);
        f(l, body + 4 * i);
    }
}

// Block (r, part), greedy: the part's first maximum.
__global__ void __launch_bounds__(VS_THREADS)
verify_best_kernel(const VerifyRows rows, int parts, VerifyPart* __restrict__ out) {
    __shared__ unsigned long long best_s[VS_THREADS / 32];
    pdl_trigger();
    pdl_wait();
    const int r = blockIdx.x, part = blockIdx.y;
    const float* row = rows.row(r);
    const int begin = (int)((long long)rows.vocab * part / parts), end = (int)((long long)rows.vocab * (part + 1) / parts);
    unsigned long long best = 0;
    float high = -INFINITY;
    int at = -1;                                                      // the thread's first maximum among the pieces, which come in rising order
    bool nan = false;
    for_share<VS_THREADS>(row, begin, end, [&](const float (&l)[16], int i) {
        if (at < 0) { high = l[0]; at = i; }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            if (l[e] > high) { high = l[e]; at = i + (e / 4) * 4 * VS_THREADS + e % 4; }
            nan |= l[e] != l[e];
        }
    }, [&](float l, int i) { best = best_of(l, i); });
    if (at >= 0) best = larger(best, best_of(high, at));
    if (__syncthreads_or(nan))                                        // comparisons pass NaNs by: entry by entry
        for (int i = begin + (int)threadIdx.x; i < end; i += VS_THREADS) best = larger(best, best_of(row[i], i));
    best = warp_best(best);
    if ((threadIdx.x & 31) == 0) best_s[threadIdx.x >> 5] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < VS_THREADS / 32; ++w) best = larger(best, best_s[w]);
        out[(long long)r * parts + part] = {best, 0.0, 0u, rows.vocab, 0.0f, 0};
    }
}

// 2^x within 2^-22 of itself: for sums that decide about a draft where it is not near, not about where a draw falls.
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// How far u q has to lie from p, as a share of the larger, for the sums below to decide about a draft.  A sum's relative error, to first
// order, in units of 2^-22: an argument is made with five roundings and off by 5 x 2^-24 nats, x its distance from the top
// in nats, which under a softmax over n < 2^31 tokens averages less than ln n < 22: 28; the exponential itself and the thread's last one: 2;
// in each of a thread's turns (of 16 logits and one rescaling) 16 additions of 2^-24, one exponential, one product: 6.  Both
// rows' together, and a quarter more.  Beyond 1e30 for 1 / T the factor in 32 bits is no longer the one in 64: nothing is decided here.
__host__ inline double margin_of_sums(double inv_t, int vocab, int parts) {
    const double turns = vocab / parts / (16 * 256) + 2;
    return inv_t > 1e30 ? 4.0 : 2.5 * (30.0 + 6.0 * turns) / 4194304.0;
}

// Block (r, part): the part's maximum and its sum.  A thread takes sixteen logits at a time onto its running maximum.
__global__ void __launch_bounds__(VS_THREADS)
verify_sums_kernel(const VerifyRows rows, const int* __restrict__ drafts, float inv_t, int parts, VerifyPart* __restrict__ out) {
    __shared__ float top_s[VS_THREADS / 32];
    __shared__ double sum_s[VS_THREADS / 32];
    pdl_trigger();
    pdl_wait();
    const int r = blockIdx.x, part = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float* row = rows.row(r);
    const int begin = (int)((long long)rows.vocab * part / parts), end = (int)((long long)rows.vocab * (part + 1) / parts);
    const float at_draft = threadIdx.x == 0 ? rows.at_draft(r, row, drafts) : 0.0f;
    // exp((l - top) / T) = 2^((l - top) * scale): the difference first, which is exact near the top (l * scale - top * scale in one fma
    // would carry the rounding of top * scale, 0.3 % of a row's sum at logits of 1,000 and T = 0.01)
    const float scale = inv_t * 1.4426950408889634f;
    float top = -INFINITY, sum = 0.0f;
    for_share<VS_THREADS>(row, begin, end, [&](const float (&l)[16], int) {
        float most = top;
#pragma unroll
        for (int e = 0; e < 16; ++e) most = fmaxf(most, l[e]);
        if (most > -INFINITY) {                                       // (else there is nothing yet)
            sum *= fast_exp2((top - most) * scale);
            top = most;
#pragma unroll
            for (int e = 0; e < 16; ++e) sum += fast_exp2((l[e] - top) * scale);
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e) sum += l[e] != l[e] ? l[e] : 0.0f;            // a NaN stays one
        }
    }, [&](float l, int) { top = l; sum = l > -INFINITY ? 1.0f : l != l ? l : 0.0f; });
    const float most = warp_max(top);
    if (lane == 0) top_s[warp] = most;
    __syncthreads();
    float all_top = top_s[0];
    for (int w = 1; w < VS_THREADS / 32; ++w) all_top = fmaxf(all_top, top_s[w]);
    // each thread's sum on the part's maximum (a thread that saw nothing has none)
    double mine = top > -INFINITY ? (double)sum * (double)fast_exp2((top - all_top) * scale) : (double)sum;
    mine = warp_total(mine);
    if (lane == 0) sum_s[warp] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
        double all = 0.0;
        for (int w = 0; w < VS_THREADS / 32; ++w) all += sum_s[w];
        out[(long long)r * parts + part] = {best_of(all_top, 0), all, 0u, rows.vocab, at_draft, 0};
    }
}

constexpr int VK_THREADS = 512, VK_WARPS = VK_THREADS / 32, VK_HELD = 16;
constexpr int VK_CANDIDATES = 2048;
constexpr int VERIFY_LIST = 512;          // the largest top_k whose kept logits are handed on as a list
constexpr int VK_MERGE = 2048;            // entries that a cluster's first block ranks

constexpr unsigned int LOWEST_KEY = 0x00800000u;       // of -inf: no number has a smaller one

// The threshold of the top_k largest by counts over the whole row or share, a bit at a time: each(f) calls f(logit, index) for a
// thread's logits, `total` is a shared word.  threshold and last as VerifyPart has them; NaNs are not counted, and where there are
// fewer numbers than top_k the threshold is 0 (everything is kept).  The counts compare floats: one operation a logit.
template <typename Each>
__device__ __forceinline__ void cut_by_counts(Each each, int top_k, int vocab, int* total, unsigned int& threshold, int& last) {
    auto count_where = [&](auto test) {                    // the same for every thread
        int n = 0;
        each([&](float l, int i) { n += test(l, i); });
        __syncthreads();
        if (threadIdx.x == 0) *total = 0;
        __syncthreads();
        atomicAdd(total, n);
        __syncthreads();
        return *total;
    };
    threshold = 0;
    for (unsigned int bit = 0x80000000u; bit; bit >>= 1) {
        const unsigned int trial = threshold | bit;
        const float t = key_value(trial);                  // (above inf's key a NaN: nothing reaches it)
        if (trial >= LOWEST_KEY && count_where([&](float l, int) { return l >= t; }) >= top_k) threshold = trial;
    }
    last = vocab;
    if (threshold >= LOWEST_KEY) {
        const float t = key_value(threshold);
        const int room = top_k - count_where([&](float l, int) { return l > t; });          // of those equal to it, at least one
        int cut = 0;                                       // the largest index below which fewer than `room` are equal to it
        for (int bit = 1 << 30; bit; bit >>= 1) {
            const int trial = cut + bit;
            if (trial > cut && trial <= vocab && count_where([&](float l, int i) { return l == t && i < trial; }) < room) cut = trial;
        }
        last = cut;
    }
    __syncthreads();
}

// A cluster of blocks a row: the k <= 512 largest logits as a list, their threshold and their sum.  Every block finds the k
// largest of its share, reading it once: of its first 8,192 logits, which the threads hold in registers, at least k of the
// threads' own maxima reach the k-th largest of those maxima, so a logit below that one is not among the share's k largest.
// What is not below it, of those and of the rest as they come, is gathered (k and a few more, for every 8,192) and ranked.
// Where that is too much (equal logits) the threshold comes from counts over the share, a bit at a time.  The first block ranks
// the shares' lists.
__global__ void __launch_bounds__(VK_THREADS, 2)
verify_top_kernel(const VerifyRows rows, const int* __restrict__ drafts, double inv_t, int top_k, int blocks, VerifyPart* __restrict__ out,
                  unsigned long long* __restrict__ lists) {
    __shared__ unsigned long long list[VK_CANDIDATES], merged[VK_MERGE];
    __shared__ double sum_s[VK_WARPS];
    __shared__ double table[64];
    __shared__ int count, total;
    cg::cluster_group cluster = cg::this_cluster();
    pdl_trigger();
    exp_table(table);
    if (threadIdx.x == 0) count = 0;
    pdl_wait();
    const int r = blockIdx.x / blocks, rank = blockIdx.x % blocks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float* row = rows.row(r);
    const int begin = (int)((long long)rows.vocab * rank / blocks), end = (int)((long long)rows.vocab * (rank + 1) / blocks);
    const int first = begin + tid, behind = first + VK_HELD * VK_THREADS;
    float held[VK_HELD];
#pragma unroll
    for (int j = 0; j < VK_HELD; ++j) held[j] = first + j * VK_THREADS < end ? row[first + j * VK_THREADS] : -INFINITY;
    const float at_draft = rank == 0 && tid == 0 ? rows.at_draft(r, row, drafts) : 0.0f;
    float high = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int j = 0; j < VK_HELD; ++j) { high = fmaxf(high, held[j]); nan |= held[j] != held[j]; }
    const unsigned int mine = first < end ? order_key(nan ? __uint_as_float(0x7FFFFFFFu) : high) : 0u;
    unsigned int floor_key = 0;                            // the upper half of the k-th largest of the threads' maxima
    for (unsigned int bit = 0x80000000u; bit >= 0x10000u; bit >>= 1)
        if (__syncthreads_count(mine >= (floor_key | bit)) >= top_k) floor_key |= bit;
    // (no keys lie between those of numbers and 0: a floor below -inf's takes all)
    const float least = floor_key > order_key(-INFINITY) ? key_value(floor_key) : -INFINITY;
    auto gather = [&](float l, int i) {
        if (!(l < least)) {                                // (a NaN is among the largest)
            const int at = atomicAdd(&count, 1);
            if (at < VK_CANDIDATES) list[at] = best_of(l, i);
        }
    };
    for (int i0 = behind; i0 < end; i0 += VK_HELD * VK_THREADS) {        // the next logits are asked for before the last are looked at
        float next[VK_HELD];
#pragma unroll
        for (int j = 0; j < VK_HELD; ++j) next[j] = i0 + j * VK_THREADS < end ? row[i0 + j * VK_THREADS] : 0.0f;
#pragma unroll
        for (int j = 0; j < VK_HELD; ++j) {
            gather(held[j], i0 + (j - VK_HELD) * VK_THREADS);
            held[j] = i0 + j * VK_THREADS < end ? next[j] : __uint_as_float(0xFF800000u);
        }
    }
    {
        // the last ones held: those from the last whole turn on
        const int turns = end > first ? (end - first - 1) / (VK_HELD * VK_THREADS) : 0;
#pragma unroll
        for (int j = 0; j < VK_HELD; ++j) {
            const int i = first + (turns * VK_HELD + j) * VK_THREADS;
            if (i < end) gather(held[j], i);
        }
    }
    __syncthreads();
    const int n = count;
    const bool ranked = n <= VK_CANDIDATES;
    // puts `all` entries of `from` into the order of their rank, the first top_k of them, at `list`
    auto rank_all = [&](const unsigned long long* from, int all) {
        constexpr int EACH = VK_CANDIDATES / VK_THREADS;
        unsigned long long v[EACH];
        int place[EACH];
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            v[j] = 0;
            place[j] = 0;
            if (j * VK_THREADS < all && tid + j * VK_THREADS < all) {
                v[j] = from[tid + j * VK_THREADS];
#pragma unroll 8
                for (int o = 0; o < all; ++o) place[j] += from[o] > v[j];        // (no two are equal: the index is part of them)
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < EACH; ++j)
            if (tid + j * VK_THREADS < all && place[j] < top_k) list[place[j]] = v[j];
        __syncthreads();
    };
    if (ranked) {
        rank_all(list, n);
    } else {
        auto each = [&](auto f) { for (int i = first; i < end; i += VK_THREADS) f(row[i], i); };
        unsigned int t;
        int last;
        cut_by_counts(each, top_k, rows.vocab, &total, t, last);
        if (tid == 0) { count = 0; total = rows.vocab; }
        __syncthreads();
        const float least_kept = key_value(t);
        each([&](float l, int i) {
            if (l != l) atomicMin(&total, i);              // the first NaN
            // (fewer numbers than top_k: the first top_k entries, the first NaN among them)
            if (t >= LOWEST_KEY ? l > least_kept || (l == least_kept && i <= last) : i - begin < top_k) {
                const int at = atomicAdd(&count, 1);
                if (at < VK_CANDIDATES) list[at] = best_of(l, i);        // (exactly top_k of them)
            }
        });
        __syncthreads();
        const bool with_nan = t >= LOWEST_KEY && total < rows.vocab;
        if (with_nan && tid == 0) list[top_k] = best_of(__uint_as_float(0x7FFFFFFFu), total);
        __syncthreads();
        rank_all(list, top_k + (with_nan ? 1 : 0));
    }
    if (blocks > 1) {
        cluster.sync();
        const int all = blocks * top_k;                    // at most VK_MERGE: the host sees to it
        if (rank == 0)
            for (int c = tid; c < all; c += VK_THREADS) merged[c] = cluster.map_shared_rank(list, c / top_k)[c % top_k];
        cluster.sync();                                    // nobody's list is read any more
        if (rank != 0) return;
        // an entry's rank: its place in its own list, and in each other one how many are larger, found by halving
        for (int c = tid; c < all; c += VK_THREADS) {
            const unsigned long long v = merged[c];
            const int own = c / top_k;
            int place = c % top_k;
            for (int l = 0; l < blocks && place < top_k; ++l) {
                if (l == own) continue;
                int low = 0, high_at = top_k;              // merged[l * top_k + i] > v for all i below `low`
                while (low < high_at) {
                    const int mid = (low + high_at) / 2;
                    if (merged[l * top_k + mid] > v) low = mid + 1;
                    else high_at = mid;
                }
                place += low;
            }
            if (place < top_k) list[place] = v;
        }
        __syncthreads();
    }
    const unsigned long long best = list[0], at_k = list[top_k - 1];
    const double top = (double)key_value((unsigned int)(best >> 32));
    double sum = 0.0;
    for (int c = tid; c < top_k; c += VK_THREADS) {
        const unsigned long long v = list[c];
        sum += exp_of(((double)key_value((unsigned int)(v >> 32)) - top) * inv_t, table);
        lists[(long long)r * top_k + c] = v;
    }
    sum = warp_total(sum);
    if (lane == 0) sum_s[warp] = sum;
    __syncthreads();
    if (tid == 0) {
        double every = 0.0;
        for (int w = 0; w < VK_WARPS; ++w) every += sum_s[w];
        out[r] = {best, every, (unsigned int)(at_k >> 32), (int)(0xFFFFFFFFu - (unsigned int)(at_k & 0xFFFFFFFFull)), at_draft, 0};
    }
}

// A block a row, any top_k: the threshold, the maximum and the sum over what is kept.  (Beyond 512 kept logits: the row is read
// once for every bit of the threshold.)
__global__ void __launch_bounds__(VK_THREADS)
verify_cut_kernel(const VerifyRows rows, const int* __restrict__ drafts, double inv_t, int top_k, VerifyPart* __restrict__ out) {
    __shared__ unsigned long long best_s[VK_WARPS];
    __shared__ double sum_s[VK_WARPS];
    __shared__ double table[64];
    __shared__ int total;
    pdl_trigger();
    exp_table(table);
    pdl_wait();
    const int r = blockIdx.x, vocab = rows.vocab, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float* row = rows.row(r);
    auto each = [&](auto f) {
        constexpr int U = 8;
        for (int i0 = tid; i0 < vocab; i0 += U * VK_THREADS) {
            float l[U];
#pragma unroll
            for (int u = 0; u < U; ++u) l[u] = i0 + u * VK_THREADS < vocab ? row[i0 + u * VK_THREADS] : 0.0f;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i0 + u * VK_THREADS < vocab) f(l[u], i0 + u * VK_THREADS);
        }
    };
    unsigned long long best = 0;
    each([&](float l, int i) { best = larger(best, best_of(l, i)); });
    best = warp_best(best);
    if (lane == 0) best_s[warp] = best;
    __syncthreads();
    best = best_s[0];
    for (int w = 1; w < VK_WARPS; ++w) best = larger(best, best_s[w]);
    const double top = (double)key_value((unsigned int)(best >> 32));
    unsigned int threshold;
    int last;
    cut_by_counts(each, top_k, vocab, &total, threshold, last);
    double sum = 0.0;
    each([&](float l, int i) {
        const unsigned int k = order_key(l);
        if (k > threshold || (k == threshold && i <= last)) sum += exp_of(((double)l - top) * inv_t, table);
    });
    sum = warp_total(sum);
    if (lane == 0) sum_s[warp] = sum;
    __syncthreads();
    if (tid == 0) {
        double all = 0.0;
        for (int w = 0; w < VK_WARPS; ++w) all += sum_s[w];
        out[r] = {best, all, threshold, last, rows.at_draft(r, row, drafts), 0};
    }
}

// One row as the second launch sees it: its parts put together.
struct VerifyRow {
    const float* row;
    double top, inv_sum;
    unsigned int threshold;
    int last, first_best;          // first_best: of the greedy and the top_k launch
    float at_draft;
    __device__ __forceinline__ bool keeps(float l, int i) const {
        const unsigned int k = order_key(l);
        return k > threshold || (k == threshold && i <= last);
    }
    __device__ __forceinline__ double mass(float l, int i, double inv_t, const double* table) const {
        return keeps(l, i) ? exp_of(((double)l - top) * inv_t, table) : 0.0;
    }
};

constexpr int VERIFY_PARTS = 16;          // parts of a row, at most

// Row r by the sixteen lanes of a half warp together, a part each (all lanes of the warp take part; the other half may have
// another row).
__device__ __forceinline__ VerifyRow row_of(const VerifyRows& rows, const VerifyPart* parts_of, int r, int parts, double inv_t, const double* table) {
    const int at = threadIdx.x & 15;
    VerifyPart p = {0ull, 0.0, 0u, 0, 0.0f, 0};
    if (at < parts) p = parts_of[(long long)r * parts + at];
    unsigned long long best = p.best;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) best = larger(best, __shfl_xor_sync(0xffffffffu, best, o));
    VerifyRow v;
    v.row = rows.row(r);
    v.top = (double)key_value((unsigned int)(best >> 32));
    v.first_best = (int)(0xFFFFFFFFu - (unsigned int)(best & 0xFFFFFFFFull));
    double sum = at < parts && !(p.sum <= 0.0) ? (parts > 1 ? p.sum * exp_of(((double)key_value((unsigned int)(p.best >> 32)) - v.top) * inv_t, table) : p.sum) : 0.0;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    v.inv_sum = 1.0 / sum;
    const int first = threadIdx.x & 16;                    // the half's first lane has the first part
    v.threshold = __shfl_sync(0xffffffffu, p.threshold, first);
    v.last = __shfl_sync(0xffffffffu, p.last, first);
    v.at_draft = __shfl_sync(0xffffffffu, p.at_draft, first);
    return v;
}

constexpr int VERIFY_ROWS = 32;           // rows whose numbers a block keeps

// A block's sums of exp((l - top) / T) over all of two rows, in 64 bits; the same in every thread, and in every block that makes them.
__device__ __forceinline__ double2 sums_of_rows(const VerifyRow& p, const VerifyRow& q, int vocab, double inv_t, const double* table,
                                                double2* scratch) {
    double sp = 0.0, sq = 0.0;
    constexpr int U = 4;
    for (int i0 = threadIdx.x; i0 < vocab; i0 += U * blockDim.x) {
        float lp[U], lq[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const long long i = (long long)i0 + j * (int)blockDim.x;
            lp[j] = i < vocab ? p.row[i] : -INFINITY;
            lq[j] = i < vocab ? q.row[i] : -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const bool there = (long long)i0 + j * (int)blockDim.x < vocab;
            sp += there ? exp_of(((double)lp[j] - p.top) * inv_t, table) : 0.0;
            sq += there ? exp_of(((double)lq[j] - q.top) * inv_t, table) : 0.0;
        }
    }
    sp = warp_total(sp);
    sq = warp_total(sq);
    __syncthreads();                                       // (what the scratch held before has been read)
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = make_double2(sp, sq);
    __syncthreads();
    double2 all = make_double2(0.0, 0.0);
    for (int w = 0; w < (int)(blockDim.x >> 5); ++w) { all.x += scratch[w].x; all.y += scratch[w].y; }
    return all;
}

// Decides how many drafts of sequence b are taken, by the block's warps, a place each: one half of a warp has the target's row,
// the other the draft's.  first_s: a shared word; kept_rows: shared room for VERIFY_ROWS pairs.  Gives the number and the
// row pair (p, q) of the place behind the drafts taken; q is p where there is no draft.
// MARGIN: the rows' sums are of 32-bit exponentials (verify_sums_kernel), and where u q lies within `margin` of p, as a share of the larger,
// the place's sums are made again in 64 bits by the whole block, so that every decision is the 64-bit formula's.
template <bool MARGIN>
__device__ __forceinline__ int decide(const VerifyRows& rows, const VerifyPart* parts_of, int parts, const int* mine, const double* u, int b,
                                      double inv_t, int greedy, double margin, const double* table, int* first_s, double2* scratch,
                                      VerifyRow (*kept_rows)[2], VerifyRow& p, VerifyRow& q, bool& ended) {
    const int g = rows.drafts, lane = threadIdx.x & 31, t0 = b * (g + 1), d0 = rows.batch * (g + 1) + b * g;
    auto pair_at = [&](int i, bool both) {                 // all threads, of a place up to g
        if (i < VERIFY_ROWS) {
            p = kept_rows[i][0];
            q = kept_rows[i][1];
        } else {
            p = row_of(rows, parts_of, t0 + i, parts, inv_t, table);
            q = both ? row_of(rows, parts_of, d0 + i, parts, inv_t, table) : p;
        }
    };
    int kept = 0;
    for (int from = 0;;) {
        if (threadIdx.x == 0) *first_s = 2 * g;
        __syncthreads();
        for (int i = from + (threadIdx.x >> 5); i <= g; i += blockDim.x >> 5) {
            const int x = i < g ? mine[i] : -1;
            const bool theirs = lane >= 16 && !greedy && i < g;
            const VerifyRow v = row_of(rows, parts_of, theirs ? d0 + i : t0 + i, parts, inv_t, table);
            if ((lane & 15) == 0 && i < VERIFY_ROWS) kept_rows[i][lane >> 4] = v;
            bool taken = x >= 0 && x < rows.vocab, near = false;
            if (greedy) taken = taken && x == v.first_best;
            else {
                const double m = taken ? v.mass(v.at_draft, x, inv_t, table) * v.inv_sum : 0.0;
                const double other = u[i] * __shfl_sync(0xffffffffu, m, 16);        // (lane 0's m is p)
                near = MARGIN && taken && fabs(other - m) < margin * fmax(other, m);
                taken = taken && other < m;
            }
            if (lane == 0 && (near || !taken)) atomicMin(first_s, 2 * i + (near ? 1 : 0));
        }
        __syncthreads();
        const int first = *first_s;                        // the first place that is refused, or too near to say
        kept = first >> 1;
        if (!MARGIN || !(first & 1)) break;
        pair_at(kept, true);
        const double2 sums = sums_of_rows(p, q, rows.vocab, inv_t, table, scratch);
        const double mp = p.mass(p.at_draft, mine[kept], inv_t, table) / sums.x, mq = q.mass(q.at_draft, mine[kept], inv_t, table) / sums.y;
        if (!(u[kept] * mq < mp)) break;
        from = kept + 1;                                   // (the sums' barriers lie behind everyone's look at first_s)
    }
    ended = kept == g || mine[kept] < 0 || mine[kept] >= rows.vocab;       // no draft there: from p alone
    pair_at(kept, !ended && !greedy);
    return kept;
}
// The answer's row apart from the drawn token: the drafts taken, -1 behind the token.
__device__ __forceinline__ void write_taken(const VerifyRows& rows, const int* mine, int kept, int b, int* tokens, int* kept_out) {
    const int g = rows.drafts;
    for (int i = threadIdx.x; i <= g; i += blockDim.x)
        if (i != kept) tokens[(long long)b * (g + 1) + i] = i < kept ? mine[i] : -1;
    if (threadIdx.x == 0) kept_out[b] = kept;
}

constexpr int VL_THREADS = 256;

// A block a sequence: greedy (lists null), or from the lists of the k kept logits.
__global__ void __launch_bounds__(VL_THREADS)
verify_list_kernel(const VerifyRows rows, const VerifyPart* __restrict__ parts_of, int parts, const unsigned long long* __restrict__ lists,
                   int top_k, const int* __restrict__ drafts, const double* __restrict__ draws, double inv_t, int greedy,
                   int* __restrict__ tokens, int* __restrict__ kept_out) {
    __shared__ double table[64];
    __shared__ int first_s, found_s;
    __shared__ int p_at[VERIFY_LIST], q_at[VERIFY_LIST];
    __shared__ double p_mass[VERIFY_LIST], q_mass[VERIFY_LIST], sorted[VERIFY_LIST];
    __shared__ int sorted_at[VERIFY_LIST];
    __shared__ VerifyRow kept_rows[VERIFY_ROWS][2];
    pdl_trigger();
    exp_table(table);
    pdl_wait();
    const int b = blockIdx.x, tid = threadIdx.x, g = rows.drafts;
    const int* mine = drafts + (long long)b * g;
    const double* u = draws + (long long)b * (g + 1);
    __syncthreads();
    VerifyRow p, q;
    bool ended;
    const int kept = decide<false>(rows, parts_of, parts, mine, u, b, inv_t, greedy, 0.0, table, &first_s, nullptr, kept_rows, p, q, ended);
    write_taken(rows, mine, kept, b, tokens, kept_out);
    const int pr = b * (g + 1) + kept, qr = rows.batch * (g + 1) + b * g + kept;
    int* out = tokens + (long long)b * (g + 1) + kept;
    if (greedy) {
        if (tid == 0) *out = p.first_best;
        return;
    }
    for (int c = tid; c < top_k; c += VL_THREADS) {
        const unsigned long long v = lists[(long long)pr * top_k + c];
        p_at[c] = (int)(0xFFFFFFFFu - (unsigned int)(v & 0xFFFFFFFFull));
        p_mass[c] = exp_of(((double)key_value((unsigned int)(v >> 32)) - p.top) * inv_t, table) * p.inv_sum;
        if (!ended) {
            const unsigned long long w = lists[(long long)qr * top_k + c];
            q_at[c] = (int)(0xFFFFFFFFu - (unsigned int)(w & 0xFFFFFFFFull));
            q_mass[c] = exp_of(((double)key_value((unsigned int)(w >> 32)) - q.top) * inv_t, table) * q.inv_sum;
        }
    }
    __syncthreads();
    bool from_p = ended;
    for (int turn = 0; turn < 2; ++turn) {
        // what each kept token has, put into the vocabulary's order
        for (int c = tid; c < top_k; c += VL_THREADS) {
            double m = p_mass[c];
            int place = 0;
            const int at = p_at[c];
            for (int o = 0; o < top_k; ++o) {
                place += p_at[o] < at;
                if (!from_p && q_at[o] == at) m = fmax(m - q_mass[o], 0.0);
            }
            sorted[place] = m;
            sorted_at[place] = at;
        }
        __syncthreads();
        if (tid < 32) {                                    // one warp walks: 32 tokens at a time
            double all = 0.0;
            for (int c = tid; c < top_k; c += 32) all += sorted[c];
            all = warp_total(all);
            int found = -1;
            if (all > 0.0) {
                const double target = u[g] * all;
                double run = 0.0;
                for (int c0 = 0; c0 < top_k; c0 += 32) {
                    const double m = c0 + tid < top_k ? sorted[c0 + tid] : 0.0;
                    double upto = m;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const double left = __shfl_up_sync(0xffffffffu, upto, o);
                        if (tid >= o) upto += left;
                    }
                    const unsigned int some = __ballot_sync(0xffffffffu, m > 0.0);
                    const unsigned int passed = __ballot_sync(0xffffffffu, m > 0.0 && run + upto > target);
                    if (some) found = c0 + 31 - __clz(some);            // the last with anything in it, where rounding lets none pass
                    if (passed) { found = c0 + __ffs(passed) - 1; break; }
                    run += __shfl_sync(0xffffffffu, upto, 31);
                }
            }
            if (tid == 0) found_s = found;
        }
        __syncthreads();
        if (found_s >= 0 || from_p) break;
        from_p = true;                                     // nothing is left of max(p - q, 0)
        __syncthreads();
    }
    if (tid == 0) *out = found_s >= 0 ? sorted_at[found_s] : p.first_best;
}

constexpr int VW_THREADS = 512, VW_WARPS = VW_THREADS / 32, VW_BLOCKS = 8;

// A cluster of up to VW_BLOCKS blocks a sequence.  CUT: a top_k beyond the lists.  HELD > 0: a thread has at most that many tokens;
// it asks for all of its logits at once and keeps their masses in the block's shared memory (two doubles a token, read
// again by the thread that wrote them).  HELD 0: eight at a time, and the masses are made again where they are needed.
template <bool CUT, int HELD>
__global__ void __launch_bounds__(VW_THREADS, 2)
verify_walk_kernel(const VerifyRows rows, const VerifyPart* __restrict__ parts_of, int parts, const int* __restrict__ drafts,
                   const double* __restrict__ draws, double inv_t, double margin, int blocks, int* __restrict__ tokens, int* __restrict__ kept_out) {
    __shared__ double table[64];
    __shared__ double span_p[VW_WARPS], span_r[VW_WARPS];
    __shared__ double2 again[VW_WARPS];
    __shared__ double share[4];                            // this block's sums: p, q, then what the token is drawn from
    __shared__ unsigned long long best_s[VW_WARPS];
    __shared__ VerifyRow kept_rows[VERIFY_ROWS][2];
    __shared__ int first_s;
    extern __shared__ double2 held_masses[];               // [HELD][VW_THREADS]
    cg::cluster_group cluster = cg::this_cluster();
    pdl_trigger();
    exp_table(table);
    pdl_wait();
    const int b = blockIdx.x / blocks, rank = blockIdx.x % blocks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = rows.drafts, vocab = rows.vocab;
    const int* mine = drafts + (long long)b * g;
    const double* u = draws + (long long)b * (g + 1);
    __syncthreads();
    VerifyRow p, q;
    bool ended;
    const int kept = decide<!CUT>(rows, parts_of, parts, mine, u, b, inv_t, 0, margin, table, &first_s, again, kept_rows, p, q, ended);      // the same in every block
    if (rank == 0) write_taken(rows, mine, kept, b, tokens, kept_out);
    const int begin = (int)((long long)vocab * rank / blocks), end = (int)((long long)vocab * (rank + 1) / blocks);
    const int w0 = begin + (int)((long long)(end - begin) * warp / VW_WARPS), w1 = begin + (int)((long long)(end - begin) * (warp + 1) / VW_WARPS);
    auto mass = [&](const VerifyRow& v, float l, int i) {
        return !CUT || v.keeps(l, i) ? exp_of(((double)l - v.top) * inv_t, table) : 0.0;
    };
    // the sums of both rows, anew: the first launch's are of 32-bit exponentials
    double sp = 0.0, sq = 0.0;
    if (HELD > 0) {
        float lp[HELD > 0 ? HELD : 1], lq[HELD > 0 ? HELD : 1];
#pragma unroll
        for (int j = 0; j < HELD; ++j) {
            const int i = w0 + 32 * j + lane;
            lp[j] = i < w1 ? p.row[i] : -INFINITY;
            lq[j] = !ended && i < w1 ? q.row[i] : -INFINITY;
        }
#pragma unroll
        for (int j = 0; j < HELD; ++j) {
            const int i = w0 + 32 * j + lane;
            const double mp = i < w1 ? mass(p, lp[j], i) : 0.0, mq = !ended && i < w1 ? mass(q, lq[j], i) : 0.0;
            held_masses[j * VW_THREADS + tid] = make_double2(mp, mq);
            sp += mp;
            sq += mq;
        }
    }
    // otherwise f(first token, p's mass, q's) for 32 tokens at a time, eight times as many asked for at once
    auto each = [&](bool with_q, auto f) {
        constexpr int U = 8;
        for (int i0 = w0; i0 < w1; i0 += 32 * U) {
            float lp[U], lq[U];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int i = i0 + 32 * j + lane;
                lp[j] = i < w1 ? p.row[i] : -INFINITY;
                lq[j] = with_q && i < w1 ? q.row[i] : -INFINITY;
            }
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int i = i0 + 32 * j + lane;
                if (!f(i0 + 32 * j, i < w1 ? mass(p, lp[j], i) : 0.0, with_q && i < w1 ? mass(q, lq[j], i) : 0.0)) return;
            }
        }
    };
    if (HELD == 0) each(!ended, [&](int, double mp, double mq) { sp += mp; sq += mq; return true; });
    sp = warp_total(sp);
    sq = warp_total(sq);
    if (lane == 0) { span_p[warp] = sp; span_r[warp] = sq; }
    __syncthreads();
    if (tid == 0) {
        double a = 0.0, c = 0.0;
        for (int w = 0; w < VW_WARPS; ++w) { a += span_p[w]; c += span_r[w]; }
        share[0] = a;
        share[1] = c;
    }
    cluster.sync();
    double all_p = 0.0, all_q = 0.0;
    for (int c = 0; c < blocks; ++c) {
        const double* s = cluster.map_shared_rank(share, c);
        all_p += s[0];
        all_q += s[1];
    }
    // what the token is drawn from: max(p - q, 0) in p's unnormalised masses, or p
    const double ratio = ended ? 0.0 : all_p / all_q;      // q in p's units
    bool from_p = ended;
    double all = all_p;
    if (!ended) {
        double sr = 0.0;
        if (HELD > 0) {
#pragma unroll
            for (int j = 0; j < HELD; ++j) {
                const double2 m = held_masses[j * VW_THREADS + tid];
                const double left = fmax(m.x - m.y * ratio, 0.0);
                held_masses[j * VW_THREADS + tid].y = left;            // from here on what is left
                sr += left;
            }
        } else {
            each(true, [&](int, double mp, double mq) { sr += fmax(mp - mq * ratio, 0.0); return true; });
        }
        sr = warp_total(sr);
        __syncthreads();                                   // (thread 0 has read span_r)
        if (lane == 0) span_r[warp] = sr;
        __syncthreads();
        if (tid == 0) {
            double a = 0.0;
            for (int w = 0; w < VW_WARPS; ++w) a += span_r[w];
            share[2] = a;
        }
        cluster.sync();
        double all_r = 0.0;
        for (int c = 0; c < blocks; ++c) all_r += cluster.map_shared_rank(share, c)[2];
        if (all_r > 0.0) all = all_r;
        else from_p = true;
    }
    const int which = from_p ? 0 : 2;
    // the block whose share of the running sum passes the target, else the last with anything in it
    const double target = u[g] * all;
    int owner = -1;
    double before = 0.0, run = 0.0;
    if (all > 0.0) {
        for (int c = 0; c < blocks; ++c) {
            const double s = cluster.map_shared_rank(share, c)[which];
            if (s > 0.0) { owner = c; before = run; }
            run += s;
            if (run > target) break;
        }
    }
    cluster.sync();                                        // nobody's shares are read any more
    int* out = tokens + (long long)b * (g + 1) + kept;
    if (owner < 0) {                                       // nothing to draw from (or sums that are no numbers): the row's first maximum
        if (rank != 0) return;
        unsigned long long best = 0;
        for (int i = tid; i < vocab; i += VW_THREADS) best = larger(best, best_of(p.row[i], i));
        best = warp_best(best);
        if (lane == 0) best_s[warp] = best;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < VW_WARPS; ++w) best = larger(best, best_s[w]);
            *out = (int)(0xFFFFFFFFu - (unsigned int)(best & 0xFFFFFFFFull));
        }
        return;
    }
    if (rank != owner) return;
    const double* span = from_p ? span_p : span_r;
    int at_warp = -1;
    run = before;
    for (int w = 0; w < VW_WARPS; ++w) {
        if (span[w] > 0.0) { at_warp = w; before = run; }
        run += span[w];
        if (run > target) break;
    }
    if (warp != at_warp) return;
    run = before;
    int found = -1;
    auto step = [&](int i0, double m) {                    // 32 tokens of the running sum; false where it passes the target
        double upto = m;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double left = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += left;
        }
        const unsigned int some = __ballot_sync(0xffffffffu, m > 0.0);
        const unsigned int passed = __ballot_sync(0xffffffffu, m > 0.0 && run + upto > target);
        if (some) found = i0 + 31 - __clz(some);           // the last with anything in it, where rounding lets none pass
        if (passed) found = i0 + __ffs(passed) - 1;
        run += __shfl_sync(0xffffffffu, upto, 31);
        return passed == 0;
    };
    if (HELD > 0) {
        for (int j = 0; j < HELD && w0 + 32 * j < w1; ++j) {
            const double2 m = held_masses[j * VW_THREADS + tid];
            if (!step(w0 + 32 * j, from_p ? m.x : m.y)) break;
        }
    } else {
        each(!from_p, [&](int i0, double mp, double mq) { return step(i0, from_p ? mp : fmax(mp - mq * ratio, 0.0)); });
    }
    if (lane == 0) *out = found;
}

// `groups` clusters of `blocks` blocks each.
template <typename... KArgs, typename... Args>
static int launch_clusters(void (*kernel)(KArgs...), int groups, int blocks, int threads, size_t smem, cudaStream_t s, Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(groups * blocks));
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    unsigned n = 0;
    if (pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)blocks;
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
    cfg.attrs = attr;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...) == cudaSuccess ? MU_OK : MU_ERR_LAUNCH;
}

}  // namespace mu

// target [batch, drafts + 1, vocab] and draft [batch, drafts, vocab] float32 (strides of sequences and rows in elements;
// draft may be null where greedy); draft_tokens [batch, drafts] int32; draws [batch, drafts + 1] float64; top_k 0: all; room: 32
// bytes for each of `parts` parts of every row read (one part with a top_k, and 8 bytes for each of up to 512 kept logits of a
// row).  tokens [batch, drafts + 1] (the drafts taken, the token after them,
// then -1) and kept [batch] int32.  One packed record (q4_linear.cu says why).
struct VerifyArgs {
    const float *target, *draft;
    const int* draft_tokens;
    const double* draws;
    void* room;
    int *tokens, *kept;
    void* stream;
    long long target_seq, target_row, draft_seq, draft_row;
    double temperature;
    int batch, drafts, vocab, top_k, parts, unused;
};
static_assert(sizeof(mu::VerifyPart) == 32, "what the caller gives room for");
MU_EXPORT int mu_verify_args_size() { return (int)sizeof(VerifyArgs); }

MU_EXPORT int mu_verify_drafts(const VerifyArgs* record) {
    const VerifyArgs a = *record;
    const float *target = a.target, *draft = a.draft;
    const int* draft_tokens = a.draft_tokens;
    const double* draws = a.draws;
    void *scratch = a.room, *stream = a.stream;
    int *tokens = a.tokens, *kept = a.kept, parts = a.parts;
    const int batch = a.batch, drafts = a.drafts, vocab = a.vocab, top_k = a.top_k;
    const double temperature = a.temperature;
    if (batch <= 0) return MU_OK;
    const bool greedy = !(temperature > 0.0) || top_k == 1;
    if (!target || drafts < 0 || vocab <= 0 || (drafts > 0 && !draft_tokens) || !draws || !scratch || !tokens || !kept || top_k < 0 ||
        parts < 1 || parts > mu::VERIFY_PARTS || (!greedy && drafts > 0 && !draft))
        return MU_ERR_BAD_ARGUMENT;
    const long long n_rows = (long long)batch * (drafts + 1) + (greedy ? 0 : (long long)batch * drafts);
    if (n_rows > 2147483647ll || (long long)batch * mu::VW_BLOCKS > 2147483647ll) return MU_ERR_UNSUPPORTED_SIZE;
    if ((uintptr_t)scratch & 7) return MU_ERR_ALIGNMENT;
    const mu::VerifyRows rows = {target, draft, a.target_seq, a.target_row, a.draft_seq, a.draft_row, batch, drafts, vocab};
    cudaStream_t s = (cudaStream_t)stream;
    const bool cuts = !greedy && top_k > 0 && top_k < vocab, listed = cuts && top_k <= mu::VERIFY_LIST;
    const double inv_t = greedy ? 1.0 : fmin(1.0 / temperature, 1e300);       // finite: the maximum's own difference of 0 stays 0
    mu::VerifyPart* p = (mu::VerifyPart*)scratch;
    unsigned long long* lists = listed ? (unsigned long long*)(p + n_rows) : nullptr;
    int code;
    if (listed) {
        // blocks a row: as many as keep what a share gathers near 1,000 (top_k for every 8,192 logits), and more where there are few
        // rows, while every SM gets one at most and a share fills its threads' registers (8,192 logits); their lists together are
        // what the first of them ranks.  Microseconds with 1, 2, 4, 8 blocks a row, both launches, rows of 50,257 and a top_k of 40:
        // 9 rows 19.3, 16.4, 15.2, 15.7; 36 rows 19.1, 17.3, 16.0, 21.0; 72 rows 19.7, 17.4, 21.5, 27.5; 288 rows 28, 34, 48, 73; a top_k
        // of 200, 72 rows: 112, 51, 48, 57.
        const int sms = mu::sm_count();
        if (sms <= 0) return MU_ERR_LAUNCH;
        parts = 1;
        int blocks = 1;
        while (blocks < 8 && 2 * blocks * top_k <= mu::VK_MERGE && vocab / (2 * blocks) >= 2 * top_k &&
               ((long long)vocab / blocks * top_k > 1000ll * 8192 || (n_rows * 2 * blocks <= sms && vocab / (2 * blocks) >= mu::VK_HELD * mu::VK_THREADS)))
            blocks *= 2;
        if (n_rows * blocks > 2147483647ll) return MU_ERR_UNSUPPORTED_SIZE;
        code = mu::launch_clusters(mu::verify_top_kernel, (int)n_rows, blocks, mu::VK_THREADS, 0, s, rows, draft_tokens, inv_t, top_k, blocks, p, lists);
    } else if (cuts) {
        parts = 1;
        code = mu::launch_pdl(mu::verify_cut_kernel, dim3((unsigned)n_rows), dim3(mu::VK_THREADS), 0, s, 1, rows, draft_tokens, inv_t, top_k, p);
    } else {
        const dim3 grid((unsigned)n_rows, (unsigned)parts), block(mu::VS_THREADS);
        if (greedy) code = mu::launch_pdl(mu::verify_best_kernel, grid, block, 0, s, 1, rows, parts, p);
        else code = mu::launch_pdl(mu::verify_sums_kernel, grid, block, 0, s, 1, rows, draft_tokens, (float)fmin(inv_t, 1e38), parts, p);
    }
    if (code != MU_OK) return code;
    if (greedy || listed)
        return mu::launch_pdl(mu::verify_list_kernel, dim3((unsigned)batch), dim3(mu::VL_THREADS), 0, s, 1, rows, (const mu::VerifyPart*)p, parts,
                              (const unsigned long long*)lists, top_k, draft_tokens, draws, inv_t, (int)greedy, tokens, kept);
    const double margin = cuts ? 0.0 : mu::margin_of_sums(inv_t, vocab, parts);
    // Eight blocks a sequence hold the masses of 53,000 tokens in their shared memory (104 KB, two on an SM); a larger vocabulary
    // is read in each pass.
    const int blocks = mu::VW_BLOCKS, held = (vocab / blocks / mu::VW_WARPS + 1 + 31) / 32;
#define MU_WALK(CUT, HELD)                                                                                                          \
    do {                                                                                                                            \
        constexpr size_t smem = (size_t)(HELD) * mu::VW_THREADS * 16;                                                               \
        auto kernel = mu::verify_walk_kernel<CUT, HELD>;                                                                            \
        if (!mu::allow_shared(reinterpret_cast<const void*>(kernel), smem)) return MU_ERR_LAUNCH;                                   \
        return mu::launch_clusters(kernel, batch, blocks, mu::VW_THREADS, smem, s, rows, (const mu::VerifyPart*)p, parts, draft_tokens, draws, \
                                   inv_t, margin, blocks, tokens, kept);                                                                    \
    } while (0)
    if (cuts) {
        if (held <= 13) MU_WALK(true, 13);
        MU_WALK(true, 0);
    }
    if (held <= 4) MU_WALK(false, 4);
    if (held <= 13) MU_WALK(false, 13);
    MU_WALK(false, 0);
#undef MU_WALK
}

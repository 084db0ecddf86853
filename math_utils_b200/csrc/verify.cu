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
// finite logit) it is the row's first maximum.
//
// Two launches.  The first reads every row once: its first maximum, its sum of exp((l - max) / T) and, with a top_k, the
// k-th largest logit.  The second is a cluster of blocks a sequence: all of them make the same decisions from the first
// launch's numbers, then walk the one row pair that matters, each block its share of the vocabulary.  The walk is in 64
// bits, exponentials included: with 50,000 tokens in a row a running sum that is off by 1e-7 of the whole would give
// another token once in a hundred draws.
#include "common.cuh"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace mu {

__device__ __forceinline__ unsigned int order_key(float v) {          // orders as the floats do
    const unsigned int b = __float_as_uint(v + 0.0f);                 // (-0 is 0)
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(unsigned int k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}
__device__ __forceinline__ unsigned long long best_of(float v, int i) {       // a larger logit wins, among equals the lower index
    return ((unsigned long long)order_key(v) << 32) | (0xFFFFFFFFu - (unsigned int)i);
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

// What the first launch says of a part of a row (a row has one part where a top_k cuts it).
struct VerifyPart {
    unsigned long long best;       // the part's first maximum (best_of)
    double sum;                    // of exp((l - max) / T) over what is kept, max the part's
    unsigned int threshold;        // kept: key above it, or equal to it and an index up to last
    int last;
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
};

constexpr int VS_THREADS = 512;

// Block (r, part): the part's maximum and, unless greedy, its sum.
__global__ void __launch_bounds__(VS_THREADS)
verify_sums_kernel(const VerifyRows rows, float inv_t, int greedy, int parts, VerifyPart* __restrict__ out) {
    __shared__ unsigned long long best_s[VS_THREADS / 32];
    __shared__ double sum_s[VS_THREADS / 32];
    __shared__ float top_s;
    pdl_trigger();
    pdl_wait();
    const int r = blockIdx.x, part = blockIdx.y;
    const float* row = rows.row(r);
    const int begin = (int)((long long)rows.vocab * part / parts), end = (int)((long long)rows.vocab * (part + 1) / parts);
    constexpr int U = 8;
    unsigned long long best = 0;
    float top = -INFINITY, sum = 0.0f;
    for (int i0 = begin + threadIdx.x; i0 < end; i0 += U * VS_THREADS) {
        float l[U];
#pragma unroll
        for (int u = 0; u < U; ++u) l[u] = i0 + u * VS_THREADS < end ? row[i0 + u * VS_THREADS] : -INFINITY;
        float most = top;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i0 + u * VS_THREADS < end) best = larger(best, best_of(l[u], i0 + u * VS_THREADS));
            most = fmaxf(most, l[u]);
        }
        if (!greedy && most > -INFINITY) {
            sum *= expf((top - most) * inv_t);
            top = most;
#pragma unroll
            for (int u = 0; u < U; ++u) sum += expf((l[u] - top) * inv_t);
        }
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    best = warp_best(best);
    if (lane == 0) best_s[warp] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < VS_THREADS / 32; ++w) best = larger(best, best_s[w]);
        best_s[0] = best;
        top_s = key_value((unsigned int)(best >> 32));
    }
    __syncthreads();
    // each thread's sum on the part's maximum (a thread that saw nothing has none)
    double mine = 0.0;
    if (!greedy && top > -INFINITY) mine = (double)sum * exp(((double)top - (double)top_s) * (double)inv_t);
    mine = warp_total(mine);
    if (lane == 0) sum_s[warp] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
        double all = 0.0;
        for (int w = 0; w < VS_THREADS / 32; ++w) all += sum_s[w];
        VerifyPart p;
        p.best = best_s[0];
        p.sum = all;
        p.threshold = 0;
        p.last = rows.vocab;
        out[(long long)r * parts + part] = p;
    }
}

constexpr int VK_THREADS = 1024;
constexpr int VK_CANDIDATES = 2048;

// A block a row: the k-th largest logit, and the maximum and the sum over the k largest.  At least k of the threads'
// own maxima reach the k-th largest of them, so a logit below that one is not among the k largest: what is not below it is
// gathered (k and a few more, of an ordinary row) and ranked.  Where that is too much (equal logits, a k beyond the number
// of threads) the threshold comes from counts over the whole row, a bit at a time.
__global__ void __launch_bounds__(VK_THREADS)
verify_top_kernel(const VerifyRows rows, float inv_t, int top_k, VerifyPart* __restrict__ out) {
    __shared__ unsigned long long list[VK_CANDIDATES];
    __shared__ float kept_value[VK_CANDIDATES];
    __shared__ unsigned long long best_s[VK_THREADS / 32];
    __shared__ double sum_s[VK_THREADS / 32];
    __shared__ int count, total;
    __shared__ unsigned long long at_k;
    pdl_trigger();
    pdl_wait();
    const int r = blockIdx.x, vocab = rows.vocab, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const float* row = rows.row(r);
    if (tid == 0) count = 0;
    constexpr int U = 8;
    unsigned long long best = 0;
    for (int i0 = tid; i0 < vocab; i0 += U * VK_THREADS) {
        float l[U];
#pragma unroll
        for (int u = 0; u < U; ++u) l[u] = i0 + u * VK_THREADS < vocab ? row[i0 + u * VK_THREADS] : 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + u * VK_THREADS < vocab) best = larger(best, best_of(l[u], i0 + u * VK_THREADS));
    }
    const unsigned int mine = (unsigned int)(best >> 32);
    best = warp_best(best);
    if (lane == 0) best_s[warp] = best;
    __syncthreads();
    best = best_s[0];
    for (int w = 1; w < VK_THREADS / 32; ++w) best = larger(best, best_s[w]);
    const float top = key_value((unsigned int)(best >> 32));

    unsigned int threshold = 0;
    int last = vocab;
    bool ranked = false;
    double sum = 0.0;
    if (top_k <= VK_THREADS) {
        unsigned int floor_key = 0;                        // the upper half of the k-th largest of the threads' maxima
        for (unsigned int bit = 0x80000000u; bit >= 0x10000u; bit >>= 1)
            if (__syncthreads_count(mine >= (floor_key | bit)) >= top_k) floor_key |= bit;
        for (int i0 = tid; i0 < vocab; i0 += U * VK_THREADS) {
            float l[U];
#pragma unroll
            for (int u = 0; u < U; ++u) l[u] = i0 + u * VK_THREADS < vocab ? row[i0 + u * VK_THREADS] : 0.0f;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + u * VK_THREADS;
                if (i < vocab && order_key(l[u]) >= floor_key) {
                    const int at = atomicAdd(&count, 1);
                    if (at < VK_CANDIDATES) list[at] = best_of(l[u], i);
                }
            }
        }
        __syncthreads();
        const int n = count;
        if (n >= top_k && n <= VK_CANDIDATES) {
            for (int c = tid; c < n; c += VK_THREADS) {
                const unsigned long long v = list[c];
                int rank = 0;
                for (int o = 0; o < n; ++o) rank += list[o] > v;           // (no two are equal: the index is part of them)
                if (rank < top_k) kept_value[rank] = key_value((unsigned int)(v >> 32));
                if (rank == top_k - 1) at_k = v;
            }
            __syncthreads();
            threshold = (unsigned int)(at_k >> 32);
            last = (int)(0xFFFFFFFFu - (unsigned int)(at_k & 0xFFFFFFFFull));
            for (int c = tid; c < top_k; c += VK_THREADS) sum += (double)expf((kept_value[c] - top) * inv_t);
            ranked = true;
        }
    }
    if (!ranked) {
        auto count_where = [&](auto test) {                // over the row, the same for every thread
            int n = 0;
            for (int i = tid; i < vocab; i += VK_THREADS) n += test(order_key(row[i]), i);
            __syncthreads();
            if (tid == 0) total = 0;
            __syncthreads();
            atomicAdd(&total, n);
            __syncthreads();
            return total;
        };
        for (unsigned int bit = 0x80000000u; bit; bit >>= 1) {
            const unsigned int trial = threshold | bit;
            if (count_where([&](unsigned int k, int) { return k >= trial; }) >= top_k) threshold = trial;
        }
        const unsigned int t = threshold;
        const int room = top_k - count_where([&](unsigned int k, int) { return k > t; });      // of those equal to it, at least one
        int cut = 0;                                       // the largest index below which fewer than `room` are equal to it
        for (int bit = 1 << 30; bit; bit >>= 1) {
            const int trial = cut + bit;
            if (trial > cut && trial <= vocab && count_where([&](unsigned int k, int i) { return k == t && i < trial; }) < room) cut = trial;
        }
        last = cut;
        for (int i = tid; i < vocab; i += VK_THREADS) {
            const unsigned int k = order_key(row[i]);
            if (k > t || (k == t && i <= last)) sum += (double)expf((row[i] - top) * inv_t);
        }
    }
    sum = warp_total(sum);
    if (lane == 0) sum_s[warp] = sum;
    __syncthreads();
    if (tid == 0) {
        double all = 0.0;
        for (int w = 0; w < VK_THREADS / 32; ++w) all += sum_s[w];
        VerifyPart p;
        p.best = best;
        p.sum = all;
        p.threshold = threshold;
        p.last = last;
        out[r] = p;
    }
}

constexpr int VW_THREADS = 512, VW_WARPS = VW_THREADS / 32, VW_BLOCKS = 8;

// One row as the second launch sees it: its parts put together.
struct VerifyRow {
    const float* row;
    double top, inv_sum;
    unsigned int threshold;
    int last, first_best;
    __device__ __forceinline__ bool keeps(float l, int i) const {
        const unsigned int k = order_key(l);
        return k > threshold || (k == threshold && i <= last);
    }
    __device__ __forceinline__ double mass(float l, int i, double inv_t) const {
        return keeps(l, i) ? exp(((double)l - top) * inv_t) : 0.0;
    }
};

__device__ __forceinline__ VerifyRow row_of(const VerifyRows& rows, const VerifyPart* parts_of, int r, int parts, double inv_t) {
    VerifyRow v;
    v.row = rows.row(r);
    const VerifyPart* p = parts_of + (long long)r * parts;
    unsigned long long best = p[0].best;
    for (int i = 1; i < parts; ++i) best = larger(best, p[i].best);
    v.top = (double)key_value((unsigned int)(best >> 32));
    v.first_best = (int)(0xFFFFFFFFu - (unsigned int)(best & 0xFFFFFFFFull));
    double sum = 0.0;
    for (int i = 0; i < parts; ++i) {
        const double top = (double)key_value((unsigned int)(p[i].best >> 32));
        if (p[i].sum > 0.0) sum += p[i].sum * exp((top - v.top) * inv_t);
    }
    v.inv_sum = 1.0 / sum;
    v.threshold = p[0].threshold;
    v.last = p[0].last;
    return v;
}

// A cluster of VW_BLOCKS blocks a sequence.
__global__ void __launch_bounds__(VW_THREADS)
verify_walk_kernel(const VerifyRows rows, const VerifyPart* __restrict__ parts_of, int parts, const int* __restrict__ drafts,
                   const double* __restrict__ draws, double inv_t, int greedy, int* __restrict__ tokens, int* __restrict__ kept_out) {
    __shared__ double span_p[VW_WARPS], span_r[VW_WARPS];
    __shared__ double share[4];                            // this block's sums: p, q, then what the token is drawn from
    __shared__ int kept_s;
    cg::cluster_group cluster = cg::this_cluster();
    pdl_trigger();
    pdl_wait();
    const int b = blockIdx.x / VW_BLOCKS, rank = (int)cluster.block_rank(), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = rows.drafts, vocab = rows.vocab;
    const int* mine = drafts + (long long)b * g;
    const double* u = draws + (long long)b * (g + 1);
    const int target0 = b * (g + 1), draft0 = rows.batch * (g + 1) + b * g;
    // how many drafts are taken: every block of the cluster finds the same number
    if (tid == 0) kept_s = g;
    __syncthreads();
    for (int i = tid; i < g; i += VW_THREADS) {
        const int x = mine[i];
        bool taken = x >= 0 && x < vocab;
        if (taken) {
            const VerifyRow p = row_of(rows, parts_of, target0 + i, parts, inv_t);
            if (greedy) taken = x == p.first_best;
            else {
                const VerifyRow q = row_of(rows, parts_of, draft0 + i, parts, inv_t);
                taken = u[i] * (q.mass(q.row[x], x, inv_t) * q.inv_sum) < p.mass(p.row[x], x, inv_t) * p.inv_sum;
            }
        }
        if (!taken) atomicMin(&kept_s, i);
    }
    __syncthreads();
    const int kept = kept_s;
    const bool ended = kept == g || mine[kept] < 0 || mine[kept] >= vocab;       // no draft there: from p alone
    const VerifyRow p = row_of(rows, parts_of, target0 + kept, parts, inv_t);
    if (rank == 0) {
        for (int i = tid; i <= g; i += VW_THREADS)
            if (i != kept) tokens[(long long)b * (g + 1) + i] = i < kept ? mine[i] : -1;
        if (tid == 0) kept_out[b] = kept;
    }
    if (greedy) {
        if (rank == 0 && tid == 0) tokens[(long long)b * (g + 1) + kept] = p.first_best;
        return;                                            // (every block of the cluster: none waits for another)
    }
    VerifyRow q = p;
    if (!ended) q = row_of(rows, parts_of, draft0 + kept, parts, inv_t);
    const int begin = (int)((long long)vocab * rank / VW_BLOCKS), end = (int)((long long)vocab * (rank + 1) / VW_BLOCKS);
    const int w0 = begin + (int)((long long)(end - begin) * warp / VW_WARPS), w1 = begin + (int)((long long)(end - begin) * (warp + 1) / VW_WARPS);

    // the sums of both rows, anew: the first launch's are of 32-bit exponentials
    double sp = 0.0, sq = 0.0;
    for (int i = w0 + lane; i < w1; i += 32) {
        sp += p.mass(p.row[i], i, inv_t);
        if (!ended) sq += q.mass(q.row[i], i, inv_t);
    }
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
    for (int c = 0; c < VW_BLOCKS; ++c) {
        const double* s = cluster.map_shared_rank(share, c);
        all_p += s[0];
        all_q += s[1];
    }
    // what the token is drawn from: max(p - q, 0) in p's unnormalised masses, or p
    const double ratio = ended ? 0.0 : all_p / all_q;      // q in p's units
    auto rest = [&](int i, bool from_p) {
        const double m = p.mass(p.row[i], i, inv_t);
        return from_p ? m : fmax(m - q.mass(q.row[i], i, inv_t) * ratio, 0.0);
    };
    bool from_p = ended;
    double all = all_p;
    if (!ended) {
        double sr = 0.0;
        for (int i = w0 + lane; i < w1; i += 32) sr += rest(i, false);
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
        for (int c = 0; c < VW_BLOCKS; ++c) all_r += cluster.map_shared_rank(share, c)[2];
        if (all_r > 0.0) all = all_r;
        else from_p = true;
    }
    const int which = from_p ? 0 : 2;
    // the block whose share of the running sum passes the target, else the last with anything in it
    const double target = u[g] * all;
    int owner = -1;
    double before = 0.0, run = 0.0;
    if (all > 0.0) {
        for (int c = 0; c < VW_BLOCKS; ++c) {
            const double s = cluster.map_shared_rank(share, c)[which];
            if (s > 0.0) { owner = c; before = run; }
            run += s;
            if (run > target) break;
        }
    }
    cluster.sync();                                        // nobody's shares are read any more
    int* out = tokens + (long long)b * (g + 1) + kept;
    if (owner < 0) {                                       // nothing to draw from (or sums that are no numbers)
        if (rank == 0 && tid == 0) *out = p.first_best;
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
    for (int i0 = w0; i0 < w1; i0 += 32) {
        const int i = i0 + lane;
        const double m = i < w1 ? rest(i, from_p) : 0.0;
        double upto = m;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double left = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += left;
        }
        const unsigned int some = __ballot_sync(0xffffffffu, m > 0.0);
        const unsigned int passed = __ballot_sync(0xffffffffu, m > 0.0 && run + upto > target);
        if (some) found = i0 + 31 - __clz(some);           // the last with anything in it, where rounding lets none pass
        if (passed) { found = i0 + __ffs(passed) - 1; break; }
        run += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (lane == 0) *out = found >= 0 ? found : p.first_best;
}

}  // namespace mu

// target [batch, drafts + 1, vocab] and draft [batch, drafts, vocab] float32 (strides of sequences and rows in elements;
// draft may be null where greedy); draft_tokens [batch, drafts] int32; draws [batch, drafts + 1] float64; top_k 0: all; room: 24
// bytes for each of `parts` parts of every row read.  tokens [batch, drafts + 1] (the drafts taken, the token after them,
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
static_assert(sizeof(mu::VerifyPart) == 24, "what the caller gives room for");
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
        parts < 1 || parts > 64 || (!greedy && drafts > 0 && !draft))
        return MU_ERR_BAD_ARGUMENT;
    const long long n_rows = (long long)batch * (drafts + 1) + (greedy ? 0 : (long long)batch * drafts);
    if (n_rows > 2147483647ll || (long long)batch * mu::VW_BLOCKS > 2147483647ll) return MU_ERR_UNSUPPORTED_SIZE;
    if ((uintptr_t)scratch & 7) return MU_ERR_ALIGNMENT;
    const mu::VerifyRows rows = {target, draft, a.target_seq, a.target_row, a.draft_seq, a.draft_row, batch, drafts, vocab};
    cudaStream_t s = (cudaStream_t)stream;
    const bool cuts = !greedy && top_k > 0 && top_k < vocab;
    const double inv_td = greedy ? 1.0 : 1.0 / temperature;
    const float inv_t = (float)inv_td;
    if (cuts) parts = 1;
    mu::VerifyPart* p = (mu::VerifyPart*)scratch;
    int code;
    if (cuts) code = mu::launch_pdl(mu::verify_top_kernel, dim3((unsigned)n_rows), dim3(mu::VK_THREADS), 0, s, 1, rows, inv_t, top_k, p);
    else code = mu::launch_pdl(mu::verify_sums_kernel, dim3((unsigned)n_rows, (unsigned)parts), dim3(mu::VS_THREADS), 0, s, 1, rows, inv_t,
                               (int)greedy, parts, p);
    if (code != MU_OK) return code;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(batch * mu::VW_BLOCKS));
    cfg.blockDim = dim3(mu::VW_THREADS);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    unsigned n = 0;
    if (mu::pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = mu::VW_BLOCKS;
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
    cfg.attrs = attr;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, mu::verify_walk_kernel, rows, (const mu::VerifyPart*)p, parts, draft_tokens, draws, inv_td, (int)greedy,
                              tokens, kept) == cudaSuccess ? MU_OK : MU_ERR_LAUNCH;
}

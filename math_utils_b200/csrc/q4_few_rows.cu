// C[M, N] = act(X[M, K] . W[N, K]^T + bias) (+ residual) for up to 64 rows, W in 4 bits, X in 8 bits (block_scaled.cuh),
// the WEIGHTS as the 128-row operand of tcgen05.mma and the batch as its narrow side.
//
// A step of single tokens reads each weight once, 17 bytes for 32 of them, and does almost no arithmetic.  The codes go
// from HBM to the tensor cores without passing a register: TMA spreads them to 16 per 16 bytes of shared memory, the
// instruction multiplies e2m1 by e4m3 and applies both exponents.  Expanding 4-bit codes in registers would cost two
// instructions a code where an SM takes in 46 codes a clock.
//   * a tile is 128 rows of W (128 output columns) by all M rows of X: D[128, NB] = W_tile . X^T, NB = M rounded up to 8, 16,
//     32 or 64; a stage is 128 of k: 8 KB of codes, 512 bytes of exponents, and the rows' share;
//   * K is cut over the blocks of a cluster (any number up to 8) so that tiles x splits fill the SMs; the partial tiles
//     meet in distributed shared memory and are added in rank order.  They lie on the stages, which nothing reads once
//     every block of the cluster has its accumulator;
//   * bfloat16 rows are two pieces, each e4m3, that together hold them (block_scaled.cuh says how exactly): they lie one behind the other,
//     one instruction multiplies both (up to 32 columns take the instruction 40 cycles, however few they are), and their
//     accumulators are added where they are read.  Up to 8 rows are cut here, by eight warps, two a stage (every block cuts its own share of k: 1.2 us a
//     launch at 8 rows, 3.5 at 16, where a launch before costs 1.4); more rows come cut by a launch of their own
//     (q8_rows.cu).
//   * the blocks of a tile begin at different places of k (each tile one 128 further on): every block reads the same rows,
//     and blocks in step would all ask for the same lines at once.
// Warp 0 copies the weights, warp 6 the rows (or warps 2-9 cut them), warp 1 owns the tensor memory and issues the products,
// warps 2-5 read the accumulators.
// Waits are bounded as everywhere: one that runs out sets the status word, and the blocks leave together.
#include "block_scaled_mma.cuh"

namespace mu {

constexpr int QF_THREADS = 224, QF_THREADS_CUT = 320;
constexpr int QF_BN = 128, QF_BK = 128;
constexpr int QF_MAX_SPLIT = 8;               // blocks of a cluster
constexpr int QF_MAX_CUT = 8;                 // bfloat16 rows that are cut here
constexpr uint32_t QF_W_BYTES = QF_BN * QF_BK;            // in shared memory: a byte a code
constexpr uint32_t QF_W_COPIED = QF_BN * QF_BK / 2;       // what the copy of them counts on its barrier: the packed codes

__device__ __forceinline__ uint32_t qf_cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void qf_cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void qf_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// COUNT columns of tensor memory, this warp's 32 lanes.
template <int COUNT> __device__ __forceinline__ void qf_load_columns(uint32_t taddr, uint32_t (&r)[COUNT]) {
    if constexpr (COUNT == 8) {
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr));
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    } else if constexpr (COUNT == 16) {
        asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
              "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
            : "r"(taddr));
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
    } else {
        tmem_ld_32x32(taddr, r);
    }
}

template <int ACT> __device__ __forceinline__ float qf_act(float x, bool to_bf16) { return to_bf16 ? apply_act_bf16(x, ACT) : apply_act(x, ACT); }

// The activation is the same for a whole launch: f(the activation as a constant), outside the loops over the elements (inside
// them every activation is evaluated for every element: 75 cycles a row and warp).
template <int A> struct QfAct { static constexpr int value = A; };
template <typename F> __device__ __forceinline__ void qf_with_act(int act, F f) {
    if (act == ACT_GELU_NEW) f(QfAct<ACT_GELU_NEW>());
    else if (act == ACT_GELU_ERF) f(QfAct<ACT_GELU_ERF>());
    else if (act == ACT_RELU2) f(QfAct<ACT_RELU2>());
    else f(QfAct<ACT_NONE>());
}

// How the rows come: in 8 bits, as two pieces of a launch before (the second NB rows behind the first, in one matrix), or in
// bfloat16 and cut into two pieces here.
// QF_NORMED: the rows are LayerNorms, made here: bfloat16((x - mean) / sqrt(var + eps) * gamma + beta) of float32 rows x, cut as any.
constexpr int QF_EIGHT = 0, QF_PIECES = 1, QF_SIXTEEN = 2, QF_NORMED = 3;
__host__ __device__ constexpr bool qf_cuts(int mode) { return mode >= QF_SIXTEEN; }

struct QfRows {
    const unsigned char* scales;      // of the rows, or of their pieces: one tile of 128 rows, [kb][512]
    const __nv_bfloat16* x;           // QF_SIXTEEN: [M, K] (ldx)
    long long ldx;
    int K, vec;                       // vec: rows in whole, aligned 16-byte pieces
    // QF_NORMED: float32 rows norm_x [.][K] (ldx), those that `pick` names (or 0 .. M - 1), all in whole, aligned 16-byte pieces
    const float *norm_x, *gamma, *beta;
    const int* pick;
    float eps;
};

// Eight entries of a normed row, rounded to bfloat16; gamma and beta from the block's shared memory.
__device__ __forceinline__ uint4 qf_normed_eight(const float4 (&x)[2], const float* gamma, const float* beta, float mean, float inv) {
    unsigned int w[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float4 g = reinterpret_cast<const float4*>(gamma)[h], b = reinterpret_cast<const float4*>(beta)[h];
        const __nv_bfloat162 lo = __floats2bfloat162_rn((x[h].x - mean) * inv * g.x + b.x, (x[h].y - mean) * inv * g.y + b.y);
        const __nv_bfloat162 hi = __floats2bfloat162_rn((x[h].z - mean) * inv * g.z + b.z, (x[h].w - mean) * inv * g.w + b.w);
        w[2 * h] = *reinterpret_cast<const unsigned int*>(&lo);
        w[2 * h + 1] = *reinterpret_cast<const unsigned int*>(&hi);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Eight bfloat16 of a row from column c on; columns from K on are zeros.
__device__ __forceinline__ uint4 qf_load_eight(const QfRows& rows, int row, int c) {
    const __nv_bfloat16* p = rows.x + (long long)row * rows.ldx + c;
    if (rows.vec) return c < rows.K ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
    unsigned int w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned int lo = c + 2 * i < rows.K ? __bfloat16_as_ushort(p[2 * i]) : 0u;
        const unsigned int hi = c + 2 * i + 1 < rows.K ? __bfloat16_as_ushort(p[2 * i + 1]) : 0u;
        w[i] = lo | hi << 16;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// grid.x = tiles * splits: the blocks of a cluster (along x) share a tile and cut K.  Dynamic shared memory, 1,024-byte
// aligned: per stage W 16 KB and PIECES x (NB x 128 bytes), then per stage the exponents (512 bytes a tile).  With splits > 1
// this block's partial tile and the shares it is sent lie on the stages when they are no longer read.
template <int NB, int MODE, typename TC>
__global__ void __launch_bounds__(qf_cuts(MODE) ? QF_THREADS_CUT : QF_THREADS)
q4_few_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const unsigned char* __restrict__ w_scales, const QfRows rows,
                   const float* __restrict__ bias, const float* residual, TC* C, int M, int N, int kb_all, long long ldc,
                   long long ldr, int act, int* status, int splits, int stages, int fixed) {
    constexpr int PIECES = MODE == QF_EIGHT ? 1 : 2;
    constexpr int NX = PIECES * NB;                       // rows as the instruction sees them: the pieces one behind the other
    constexpr uint32_t X_PIECE = NB * QF_BK, STAGE = QF_W_BYTES + PIECES * X_PIECE;
    constexpr uint32_t SCALE_STAGE = 2 * BS_TILE_BYTES;   // a tile of exponents each
    constexpr uint32_t ACC_COLS = NX < 32 ? 32 : NX, SCALE_COLS = 8;
    constexpr uint32_t TMEM_COLS = ACC_COLS + 2 * SCALE_COLS <= 64 ? 64 : ACC_COLS + 2 * SCALE_COLS <= 128 ? 128 : 256;
    constexpr int CHUNK = NB < 32 ? NB : 32;
    extern __shared__ unsigned char qf_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>(((uintptr_t)qf_raw + 1023) & ~(uintptr_t)1023);
    unsigned char* scale_smem = base + (size_t)stages * STAGE;
    float* outbox = reinterpret_cast<float*>(base);
    __shared__ uint64_t full[16], empty[16], acc_full, parts_in;
    __shared__ uint32_t tmem_slot;
    __shared__ float bias_s[QF_BN];
    __shared__ float stat_s[2][QF_MAX_CUT];               // QF_NORMED: a row's mean and inverse deviation

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rank = splits > 1 ? (int)qf_cluster_rank() : 0;
    const int tile = blockIdx.x / splits;
    const int n0 = tile * QF_BN;
    const int kb_begin = (int)((long long)kb_all * rank / splits), kb_end = (int)((long long)kb_all * (rank + 1) / splits);
    const int my_kb = kb_end - kb_begin;                  // at least one: the host keeps splits <= kb_all
    bool ok = true;

    if (threadIdx.x == 0) {
        tma_prefetch_map(&map_w);
        if (!qf_cuts(MODE)) tma_prefetch_map(&map_x);
        for (int s = 0; s < stages; ++s) { mbar_init(&full[s], qf_cuts(MODE) ? 3 : 2); mbar_init(&empty[s], 1); }
        mbar_init(&acc_full, 1);
        mbar_init(&parts_in, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (!fixed) pdl_wait();                               // weights, bias, gamma and beta may be the work of earlier kernels
    if (threadIdx.x >= 64 && threadIdx.x < 192) {
        const int n = n0 + (int)threadIdx.x - 64;
        bias_s[threadIdx.x - 64] = (bias && n < N) ? bias[n] : 0.0f;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_acc = tmem_slot;
    pdl_trigger();
    // The two issuing threads run alone on their warps, where every dependent instruction costs its whole latency: stages and
    // phases are counted on instead of divided out, and addresses and descriptors are added to.  (With i % stages and
    // descriptors made anew a stage took its loader and its issuer about 500 cycles each, more than its bytes.)
    const int turned = tile % my_kb;                      // where this block begins in its share of k
    if (warp == 0 || (!qf_cuts(MODE) && warp == 6)) {
        const bool weights = warp == 0;
        if (lane == 0) {
            int kb = turned;
            auto load = [&](int s) {
                const int k = kb_begin + kb;
                if (weights) {
                    mbar_expect_tx(&full[s], QF_W_COPIED + BS_TILE_BYTES);
                    tma_load_2d(base + s * STAGE, &map_w, k * QF_BK, n0, &full[s]);
                    bulk_load(scale_smem + s * SCALE_STAGE, w_scales + ((long long)tile * kb_all + k) * BS_TILE_BYTES, BS_TILE_BYTES, &full[s]);
                } else {
                    mbar_expect_tx(&full[s], PIECES * X_PIECE + BS_TILE_BYTES);
                    tma_load_2d(base + s * STAGE + QF_W_BYTES, &map_x, k * QF_BK, 0, &full[s]);
                    bulk_load(scale_smem + s * SCALE_STAGE + BS_TILE_BYTES, rows.scales + (long long)k * BS_TILE_BYTES, BS_TILE_BYTES, &full[s]);
                }
                if (++kb == my_kb) kb = 0;
            };
            if (!weights) pdl_wait();                     // (the weights: above, unless they are fixed)
            const int first = my_kb < stages ? my_kb : stages;
            for (int i = 0; i < first; ++i) load(i);
            int issued = first, s = 0;
            uint32_t phase = 0;
            for (int i = first; i < my_kb; ++i) {
                ok = mbar_wait(&empty[s], phase);
                if (!ok) break;
                load(s);
                issued = i + 1;
                if (++s == stages) { s = 0; phase ^= 1; }
            }
            if (!ok) {
                atomicExch(status, 1);
                for (int j = issued > stages ? issued - stages : 0; j < issued; ++j)      // copies under way land first
                    mbar_wait(&full[j % stages], (uint32_t)((j / stages) & 1));
            }
        }
    } else if (warp == 1) {
        const bool one = elect_one();
        constexpr uint32_t idesc = idesc_block_scaled(BM_E2M1, BM_E4M3, QF_BN, NX);
        const uint64_t w_desc0 = smem_desc_sw128(smem_u32(base)), s_desc0 = scales_desc(smem_u32(scale_smem));
        uint64_t w_desc = w_desc0, s_desc = s_desc0;
        int s = 0;
        uint32_t phase = 0;
        for (int i = 0; i < my_kb; ++i) {
            ok = mbar_wait(&full[s], phase);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (one) {
                const uint32_t tmem_s = tmem_acc + ACC_COLS + (i & 1) * SCALE_COLS;      // two sets, in turn
                copy_scales(tmem_s, s_desc);
                copy_scales(tmem_s + 4, s_desc + BS_TILE_BYTES / 16);
#pragma unroll
                for (int j = 0; j < QF_BK / 32; ++j)
                    umma_block_scaled(tmem_acc, w_desc + 2 * j, w_desc + QF_W_BYTES / 16 + 2 * j, idesc | idesc_scale_byte(j), tmem_s, tmem_s + 4,
                                      i > 0 || j > 0 ? 1u : 0u);
                umma_commit(&empty[s]);
            }
            __syncwarp();
            w_desc += STAGE / 16;
            s_desc += SCALE_STAGE / 16;
            if (++s == stages) { s = 0; phase ^= 1; w_desc = w_desc0; s_desc = s_desc0; }
        }
        if (ok && one) umma_commit(&acc_full);
        if (!ok && one) atomicExch(status, 2);
    } else {
        const int quad = warp & 3, col = quad * 32 + lane;        // a lane is an output column: n0 + col
        const bool to_bf16 = sizeof(TC) == 2;
        if (qf_cuts(MODE)) {
            // Two warps take every fourth stage, every other pair of its rows each, a lane eight entries at a time, four neighbours
            // a group of 32: 16 lanes a row.
            constexpr int PAIRS = NB / 4;                          // of rows, a warp
            const int turn = (warp - 2) & 3, pair0 = (warp - 2) >> 2;
            const int half = lane >> 4, c8 = lane & 15;
            // QF_NORMED: gamma and beta of this block's share of k to shared memory (before the wait where they are fixed), then a row's mean and
            // inverse deviation by a warp each
            float* gamma_s = reinterpret_cast<float*>(scale_smem + (size_t)stages * SCALE_STAGE);
            float* beta_s = gamma_s + my_kb * QF_BK;
            if (MODE == QF_NORMED) {
                for (int j = 4 * ((int)threadIdx.x - 64); j < my_kb * QF_BK; j += 4 * (QF_THREADS_CUT - 64)) {
                    const int k = kb_begin * QF_BK + j;
                    const float4 none = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    *reinterpret_cast<float4*>(gamma_s + j) = k < rows.K ? *reinterpret_cast<const float4*>(rows.gamma + k) : none;
                    *reinterpret_cast<float4*>(beta_s + j) = rows.beta && k < rows.K ? *reinterpret_cast<const float4*>(rows.beta + k) : none;
                }
            }
            pdl_wait();                                            // the rows are the work of earlier kernels
            if (MODE == QF_NORMED) {
                const int m = warp - 2;
                if (m < M) {
                    const float4* src = reinterpret_cast<const float4*>(rows.norm_x + (long long)(rows.pick ? rows.pick[m] : m) * rows.ldx);
                    const int n4 = rows.K / 4;
                    constexpr int KEEP = 13;                       // pieces a lane keeps between the two sums: rows of up to 1,664
                    float4 v[KEEP];
                    float sum = 0.0f;
#pragma unroll
                    for (int i = 0; i < KEEP; ++i) v[i] = lane + 32 * i < n4 ? src[lane + 32 * i] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                    for (int i = 0; i < KEEP; ++i) sum += (v[i].x + v[i].y) + (v[i].z + v[i].w);
                    for (int i = lane + 32 * KEEP; i < n4; i += 32) { const float4 x = src[i]; sum += (x.x + x.y) + (x.z + x.w); }
                    const float mean = warp_sum(sum) / (float)rows.K;
                    float sq = 0.0f;
                    auto add = [&](const float4& x) {
                        const float a = x.x - mean, b = x.y - mean, c = x.z - mean, d = x.w - mean;
                        sq += (a * a + b * b) + (c * c + d * d);
                    };
#pragma unroll
                    for (int i = 0; i < KEEP; ++i) if (lane + 32 * i < n4) add(v[i]);
                    for (int i = lane + 32 * KEEP; i < n4; i += 32) add(src[i]);
                    const float inv = 1.0f / sqrtf(warp_sum(sq) / (float)rows.K + rows.eps);
                    if (lane == 0) { stat_s[0][m] = mean; stat_s[1][m] = inv; }
                }
                asm volatile("bar.sync 2, %0;" ::"n"(QF_THREADS_CUT - 64) : "memory");
            }
            // Two stages' rows are on their way while a third's are cut.
            constexpr int WORDS = MODE == QF_NORMED ? 2 : 1;       // 16-byte pieces of eight entries
            uint4 raw[2][PAIRS][WORDS];
            auto ask = [&](int i, int e, uint4 (&to)[WORDS]) {
                const int row = 2 * (2 * e + pair0) + half;
                const int k = (kb_begin + (i + turned < my_kb ? i + turned : i + turned - my_kb)) * QF_BK + 8 * c8;
                const bool there = i < my_kb && row < M;
                if (MODE == QF_NORMED) {
                    const float* src = there ? rows.norm_x + (long long)(rows.pick ? rows.pick[row] : row) * rows.ldx : nullptr;
#pragma unroll
                    for (int h = 0; h < WORDS; ++h)
                        to[h] = there && k < rows.K ? *reinterpret_cast<const uint4*>(src + k + 4 * h) : make_uint4(0, 0, 0, 0);
                } else {
                    to[0] = there ? qf_load_eight(rows, row, k) : make_uint4(0, 0, 0, 0);
                }
            };
            // (a ring of four stages or more, or of all of them: a warp four stages on then waits for the phase before its own)
            int s = turn % stages;
            uint32_t phase = (uint32_t)(turn / stages) & 1u;
            auto cut = [&](int i, uint4 (&mine)[PAIRS][WORDS]) {
                if (i >= stages) ok = mbar_wait(&empty[s], phase ^ 1u);
                if (!__all_sync(0xffffffffu, ok)) { ok = false; return; }
                unsigned char* x0 = base + s * STAGE + QF_W_BYTES;
                unsigned char* sx = scale_smem + s * SCALE_STAGE + BS_TILE_BYTES;
#pragma unroll
                for (int e = 0; e < PAIRS; ++e) {
                    if (2 * (2 * e + pair0) >= M) break;           // rows past M are left as they are: their columns go nowhere
                    const int row = 2 * (2 * e + pair0) + half;
                    uint4 eight = mine[e][0];
                    if (MODE == QF_NORMED) {
                        const int j = (i + turned < my_kb ? i + turned : i + turned - my_kb) * QF_BK + 8 * c8, at_row = row < M ? row : 0;
                        const float4 x[2] = {make_float4(__uint_as_float(mine[e][0].x), __uint_as_float(mine[e][0].y), __uint_as_float(mine[e][0].z), __uint_as_float(mine[e][0].w)),
                                             make_float4(__uint_as_float(mine[e][WORDS - 1].x), __uint_as_float(mine[e][WORDS - 1].y), __uint_as_float(mine[e][WORDS - 1].z), __uint_as_float(mine[e][WORDS - 1].w))};
                        // (columns past K have gamma and beta of 0, whatever the row's mean)
                        eight = qf_normed_eight(x, gamma_s + j, beta_s + j, stat_s[0][at_row], stat_s[1][at_row]);
                    }
                    const unsigned int w[4] = {eight.x, eight.y, eight.z, eight.w};
                    ask(i + 8, e, mine[e]);
                    const unsigned int top = group_top_bf16(w);
                    const bool fine = top < 0x7F80u;
                    const int b = fine ? exponent_e4m3_bf16(top) : 127;
                    uint2 hi, lo;
                    e4m3_pieces_of_eight(w, b, hi, lo);
                    if (!fine) hi = lo = make_uint2(E4M3_NAN4, E4M3_NAN4);
                    // the copies' layout: 16-byte pieces of a 128-byte row, swapped by the row's place among eight
                    const int at = row * 128 + (((c8 >> 1) ^ (row & 7)) << 4) + (c8 & 1) * 8;
                    *reinterpret_cast<uint2*>(x0 + at) = hi;
                    *reinterpret_cast<uint2*>(x0 + X_PIECE + at) = lo;
                    if ((c8 & 3) == 0) {
                        sx[row * 16 + c8 / 4] = (unsigned char)b;
                        sx[(row + NB) * 16 + c8 / 4] = (unsigned char)low_exponent(b);
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");        // the tensor cores read what was stored here
                __syncwarp();
                if (lane == 0) mbar_arrive(&full[s]);
                for (int step = 0; step < 4; ++step)
                    if (++s == stages) { s = 0; phase ^= 1; }
            };
#pragma unroll
            for (int e = 0; e < PAIRS; ++e) { ask(turn, e, raw[0][e]); ask(turn + 4, e, raw[1][e]); }
            for (int i = turn; i < my_kb && ok; i += 8) {
                cut(i, raw[0]);
                if (i + 4 < my_kb && ok) cut(i + 4, raw[1]);
            }
            if (!ok && lane == 0) atomicExch(status, 1);
            __syncwarp();
        }
        if (warp < 6) {
        ok = mbar_wait(&acc_full, 0);
        if (!ok && lane == 0) atomicExch(status, 3);
        __syncwarp();
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t acc_addr = tmem_acc + ((uint32_t)(quad * 32) << 16);
        if (splits == 1) {
            const int n = n0 + col;
            pdl_wait();                                           // the residual is the work of earlier kernels
            if (ok) {
#pragma unroll
                for (int c0 = 0; c0 < NB; c0 += CHUNK) {
                    if (c0 >= M) break;
                    uint32_t r[CHUNK];
                    qf_load_columns<CHUNK>(acc_addr + c0, r);
                    if (PIECES == 2) {
                        uint32_t low[CHUNK];
                        qf_load_columns<CHUNK>(acc_addr + NB + c0, low);
#pragma unroll
                        for (int e = 0; e < CHUNK; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) + __uint_as_float(low[e]));
                    }
                    if (n < N) {
                        float res[CHUNK];                         // all asked for before anything is stored: it may be C itself
#pragma unroll
                        for (int e = 0; e < CHUNK; ++e) res[e] = (residual && c0 + e < M) ? residual[(long long)(c0 + e) * ldr + n] : 0.0f;
                        qf_with_act(act, [&](auto a) {
#pragma unroll
                            for (int e = 0; e < CHUNK; ++e)
                                if (c0 + e < M)
                                    C[(long long)(c0 + e) * ldc + n] = from_float<TC>(qf_act<decltype(a)::value>(__uint_as_float(r[e]) + bias_s[col], to_bf16) + res[e]);
                        });
                    }
                    __syncwarp();                                 // the lanes are together for the next load
                }
            }
        } else {
            // block r finishes the tile's columns [128 r / splits, 128 (r + 1) / splits)
            auto first_of = [&](int r) { return QF_BN * r / splits; };
            const int groups = (M + 3) / 4;                       // batch rows travel four at a time
            const int pitch = 4 * groups + 4;
            const int mine0 = first_of(rank), cols = first_of(rank + 1) - mine0;
            float* part = outbox + (size_t)QF_BN * pitch;         // [splits][cols][pitch]: what this block is sent
            {
                float* mine = outbox + (size_t)col * pitch;
#pragma unroll
                for (int c0 = 0; c0 < NB; c0 += CHUNK) {
                    if (c0 >= M) break;
                    uint32_t r[CHUNK];
                    qf_load_columns<CHUNK>(acc_addr + c0, r);
                    if (PIECES == 2) {
                        uint32_t low[CHUNK];
                        qf_load_columns<CHUNK>(acc_addr + NB + c0, low);
#pragma unroll
                        for (int e = 0; e < CHUNK; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) + __uint_as_float(low[e]));
                    }
#pragma unroll
                    for (int g = 0; g < CHUNK / 4; ++g)
                        if (c0 / 4 + g < groups)
                            *reinterpret_cast<float4*>(mine + c0 + 4 * g) =
                                make_float4(__uint_as_float(r[4 * g]), __uint_as_float(r[4 * g + 1]), __uint_as_float(r[4 * g + 2]), __uint_as_float(r[4 * g + 3]));
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");        // the copies below read what was stored here
            asm volatile("bar.sync 1, 128;" ::: "memory");
            __syncwarp();
            qf_cluster_arrive();                                  // this block's stages are no longer read ...
            qf_cluster_wait();                                    // ... nor any other's
            if (threadIdx.x == 64) {
                mbar_expect_tx(&parts_in, (uint32_t)((splits - 1) * cols * pitch) * 4u);
                for (int step = 1; step < splits; ++step) {
                    const int owner = (rank + step) % splits;     // not everyone at the same owner first
                    const int from = first_of(owner), count = first_of(owner + 1) - from;
                    uint32_t dst, bar;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                                 : "=r"(dst) : "r"(smem_u32(part + (size_t)rank * count * pitch)), "r"(owner));
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(bar) : "r"(smem_u32(&parts_in)), "r"(owner));
                    asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                                 ::"r"(dst), "r"(smem_u32(outbox + (size_t)from * pitch)), "r"((uint32_t)(count * pitch) * 4u), "r"(bar)
                                 : "memory");
                }
            }
            const bool arrived = mbar_wait(&parts_in, 0);
            if (!arrived && lane == 0) atomicExch(status, 3);
            __syncwarp();
            qf_cluster_arrive();
            pdl_wait();
            const int who = (int)threadIdx.x - 64, total = groups * cols;
            qf_with_act(act, [&](auto a) {
            for (int idx = who; idx < total && arrived; idx += 128) {
                const int g = idx / cols, i = idx - g * cols;
                const int c = mine0 + i, n = n0 + c;
                if (n >= N) continue;
                float res[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    res[e] = (residual && 4 * g + e < M) ? residual[(long long)(4 * g + e) * ldr + n] : 0.0f;
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                for (int r = 0; r < splits; ++r) {                // in rank order, whoever sent when
                    const float* src = r == rank ? outbox + (size_t)c * pitch : part + ((size_t)r * cols + i) * pitch;
                    const float4 p = *reinterpret_cast<const float4*>(src + 4 * g);
                    v.x += p.x; v.y += p.y; v.z += p.z; v.w += p.w;
                }
                const float out4[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (4 * g + e < M)
                        C[(long long)(4 * g + e) * ldc + n] = from_float<TC>(qf_act<decltype(a)::value>(out4[e] + bias_s[c], to_bf16) + res[e]);
            }
            });
            __syncwarp();
            qf_cluster_wait();                                    // nobody leaves while a copy may still read its outbox
        }
        }
    }
    if (splits > 1 && (warp < 2 || warp >= 6)) {                                 // the same two cluster barriers as the epilogue warps
        __syncwarp();
        qf_cluster_arrive();
        qf_cluster_wait();
        qf_cluster_arrive();
        qf_cluster_wait();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_acc), "r"(TMEM_COLS) : "memory");
}

template <int NB, int MODE, typename TC>
static int launch_few(const CUtensorMap& map_w, const CUtensorMap& map_x, const unsigned char* w_scales,
                      const QfRows& rows, const float* bias, const float* residual, TC* C, int M, int N, int kb_all, long long ldc,
                      long long ldr, int act, int* status, int splits, int stages, int fixed, size_t smem, cudaStream_t s) {
    auto kernel = q4_few_rows_kernel<NB, MODE, TC>;
    if (!allow_shared(reinterpret_cast<const void*>(kernel), 224 * 1024)) return MU_ERR_LAUNCH;
    const int tiles = (N + QF_BN - 1) / QF_BN;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * splits));
    cfg.blockDim = dim3(qf_cuts(MODE) ? QF_THREADS_CUT : QF_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    unsigned n = 0;
    if (pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    if (splits > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = (unsigned)splits;
        attr[n].val.clusterDim.y = 1;
        attr[n].val.clusterDim.z = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, kernel, map_w, map_x, w_scales, rows, bias, residual, C, M, N, kb_all, ldc, ldr, act,
                              status, splits, stages, fixed) == cudaSuccess ? MU_OK : MU_ERR_LAUNCH;
}

static bool tensor_map_codes(CUtensorMap* map, CUtensorMapDataType type, const void* base, long long rows, int kp, long long row_bytes,
                             int box_rows) {
    static EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)kp, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)row_bytes};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
    const cuuint32_t elem[2] = {1, 1};
    return fn(map, type, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool tensor_map_boxes(CUtensorMap* map, const void* base, long long rows, int cols, long long ld, int is_bf16) {
    static EncodeTiledFn fn = encode_tiled_fn();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)ld * (is_bf16 ? 2 : 4)};
    const cuuint32_t box[2] = {32, 32};
    const cuuint32_t elem[2] = {1, 1};
    return fn(map, is_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<void*>(base), dims, strides, box,
              elem, CU_TENSOR_MAP_INTERLEAVE_NONE, is_bf16 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
bool tensor_map_q4(CUtensorMap* map, const void* base, long long rows, int kp, int box_rows) {
    return tensor_map_codes(map, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, base, rows, kp, kp / 2, box_rows);
}
bool tensor_map_q8(CUtensorMap* map, const void* base, long long rows, int kp, int box_rows) {
    return tensor_map_codes(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, rows, kp, kp, box_rows);
}

// How many blocks share a tile, in hundredths of a stage of a block alone on its SM (some 0.25 us).  Two blocks on an SM fill each
// other's waits: their stages take two thirds of that each, but the ring is half as long (three stages more).  The exchange of parts
// costs five stages, one more for every block that takes part and one for 8 rows.  A cluster lies within one part of the chip: of three to six
// blocks they fill some 7 of 8 SMs at once, of seven and eight 3 of 4 (16 of eight took 11.6 us where 16 of six took 7.1).
// Microseconds on a B200, 8-bit rows: 1 x 6,400 x 1,600 uncut 4.0, by 2 4.6, by 4 4.8; 8 x 1,600 x 6,400 uncut 13.4, by 2 8.2, by
// 5 5.2, by 8 5.8; 8 x 4,096 x 2,048 uncut 4.8, by 2 4.5, by 4 4.6; 48 x 11,264 x 2,048 uncut 8.6, by 2 9.4, by 4 13.4; 8 x 16,384 x
// 8,192 uncut 18.4, by 2 15.1, by 4 19.8; 8 x 8,192 x 8,192 uncut 17.4, by 2 11.4, by 4 10.2; 8 x 28,672 x 4,096 uncut 13.0, by 2 18.4.
static int choose_splits(long long tiles, int kb_all, int rows, int sms) {
    int best = 1;
    long long least = 1ll << 60;
    for (int s = 1; s <= QF_MAX_SPLIT && s <= kb_all; ++s) {
        const int filled = s <= 2 ? sms : s <= 6 ? sms * 7 / 8 : sms * 3 / 4;
        long long per_sm = (tiles * s + filled - 1) / filled;                 // blocks that an SM runs, two at a time
        if (per_sm > 1) per_sm = (per_sm + 1) / 2 * 2;
        const long long stages = per_sm * ((kb_all + s - 1) / s);
        const long long cost = (per_sm > 1 ? 66 * stages + 300 : 100 * stages) + (s > 1 ? 100 * (5 + s + rows / 8) : 0);
        if (cost < least) { least = cost; best = s; }
    }
    return best;
}

// The rows of a batch in whole 8s, 16s, 32s or 64s: how far behind the first piece the second one's rows lie.
int q4_few_rows_tile(int M, bool cut_here) { return cut_here ? 8 : M <= 16 ? 16 : M <= 32 ? 32 : 64; }

// W: codes [N, kp / 2] and exponents (pointers and strides as mu_linear_q4 has checked them); M <= 64.  The rows: 8-bit codes x
// [M, kp] with one tile of exponents; with two_pieces the second piece's rows q4_few_rows_tile() behind the first's; or
// (scales null) bfloat16 x [M, K] (ldx), M <= 8; or (norm not null) the LayerNorms of float32 x [.][K] (ldx), M <= 8.  splits: blocks that share a tile and cut K (up to 8; 0: chosen here).
int launch_q4_few_rows(const void* x, const void* x_scales, bool two_pieces, long long ldx, int K, const void* w, const void* w_scales,
                       const float* bias, const float* residual, void* C, int M, int N, int kp, long long ldc, long long ldr, int act,
                       int out_bf16, int splits, const RowNorm* norm, int fixed, int* status, void* stream) {
    const int mode = norm ? QF_NORMED : !x_scales ? QF_SIXTEEN : two_pieces ? QF_PIECES : QF_EIGHT;
    if (M > (qf_cuts(mode) ? QF_MAX_CUT : 64)) return MU_ERR_UNSUPPORTED_SIZE;
    if (splits < 0 || splits > QF_MAX_SPLIT) return MU_ERR_BAD_ARGUMENT;
    const int sms = sm_count();
    if (sms <= 0) return MU_ERR_LAUNCH;
    const long long tiles = ((long long)N + 127) / 128;
    const int kb_all = kp / 128, pieces = mode == QF_EIGHT ? 1 : 2;
    if (tiles * QF_MAX_SPLIT > 2147483647ll) return MU_ERR_UNSUPPORTED_SIZE;
    if (splits == 0) splits = choose_splits(tiles, kb_all, M, sms);
    if (splits > kb_all) splits = kb_all;
    const int nb = q4_few_rows_tile(M, qf_cuts(mode));
    const size_t operands = QF_W_BYTES + (size_t)pieces * nb * 128, stage_bytes = operands + 2 * 512;
    // the ring: half of an SM's room where there are blocks for two on one and it leaves each three stages; at least what the
    // partial tiles take
    const size_t parts_bytes = splits > 1 ? (size_t)((M + 3) / 4 * 4 + 4) * 4 * (128 + splits * (128 / splits + 1)) : 0;
    const int per_block = (kb_all + splits - 1) / splits, least = (int)((parts_bytes + operands - 1) / operands);
    const size_t norm_bytes = mode == QF_NORMED ? (size_t)per_block * QF_BK * 8 : 0;       // gamma and beta
    const size_t ring = (qf_cuts(mode) ? 4 : 3) * stage_bytes;
    const size_t room = 1024 + norm_bytes + ring <= 111 * 1024 && tiles * splits > sms ? 111 * 1024 : 220 * 1024;
    if (1024 + norm_bytes + ring > room) return MU_ERR_UNSUPPORTED_SIZE;
    int stages = (int)((room - 1024 - norm_bytes) / stage_bytes);
    if (stages > per_block) stages = per_block;
    if (stages < least) stages = least;
    if (stages > 16) stages = 16;
    if (stages < 1) stages = 1;
    const size_t smem = 1024 + (size_t)stages * stage_bytes + norm_bytes;
    if (smem > 224 * 1024 || parts_bytes > (size_t)stages * operands || (qf_cuts(mode) && stages < 4 && stages < per_block))
        return MU_ERR_UNSUPPORTED_SIZE;
    CUtensorMap map_w, map_x = {};
    if (!tensor_map_q4(&map_w, w, N, kp, 128)) return MU_ERR_LAUNCH;
    if (!qf_cuts(mode) && !tensor_map_q8(&map_x, x, mode == QF_PIECES ? 2 * nb : M, kp, pieces * nb)) return MU_ERR_LAUNCH;
    QfRows rows = {(const unsigned char*)x_scales, (const __nv_bfloat16*)x, ldx, K,
                   K % 8 == 0 && ((uintptr_t)x & 15) == 0 && (M == 1 || ldx % 8 == 0), nullptr, nullptr, nullptr, nullptr, 0.0f};
    if (norm) {
        rows.norm_x = (const float*)x;
        rows.gamma = norm->gamma;
        rows.beta = norm->beta;
        rows.pick = norm->pick;
        rows.eps = norm->eps;
    }
    cudaStream_t s = (cudaStream_t)stream;
#define MU_FEW(NB, MODE)                                                                                                            \
    (out_bf16 ? launch_few<NB, MODE, __nv_bfloat16>(map_w, map_x, (const unsigned char*)w_scales, rows, bias, residual, \
                                                        (__nv_bfloat16*)C, M, N, kb_all, ldc, ldr, act, status, splits, stages, fixed, smem, s) \
              : launch_few<NB, MODE, float>(map_w, map_x, (const unsigned char*)w_scales, rows, bias, residual, (float*)C, \
                                                M, N, kb_all, ldc, ldr, act, status, splits, stages, fixed, smem, s))
#define MU_FEW_BOTH(NB) (mode == QF_PIECES ? MU_FEW(NB, QF_PIECES) : MU_FEW(NB, QF_EIGHT))
    if (mode == QF_NORMED) return MU_FEW(8, QF_NORMED);
    if (mode == QF_SIXTEEN) return MU_FEW(8, QF_SIXTEEN);
    if (nb == 16) return MU_FEW_BOTH(16);
    if (nb == 32) return MU_FEW_BOTH(32);
    return MU_FEW_BOTH(64);
#undef MU_FEW_BOTH
#undef MU_FEW
}

}  // namespace mu

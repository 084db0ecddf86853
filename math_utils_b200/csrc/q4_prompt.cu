// C[M, N] = act(X[M, K] . W[N, K]^T + bias) (+ residual) for many rows, W in 4 bits, X in 8 bits (block_scaled.cuh): tiles of
// 128 rows by BN columns, the ROWS as the 128-row operand of tcgen05.mma.
//
// The instruction multiplies e4m3 by e2m1 at the 8-bit rate, 128 x 192 x 32 in 96 cycles, and applies both exponents, so the
// weights are never expanded: TMA spreads the packed codes in shared memory, 12 KB of L2 for 192 columns of 128 of k.
// bfloat16 rows come as two 8-bit pieces that together hold them (block_scaled.cuh says how exactly): two products a step into one
// accumulator, the rate of a bfloat16 product.
//
// Persistent: a block an SM walks over the tiles; the ring of stages runs on across tiles, two accumulators in tensor memory
// take turns, so a tile is read out and stored while the next is multiplied.  (Tiles of 256 columns have one: two would
// leave no tensor memory for the exponents.)  What bounds large products is what an SM takes in from the L2.  Warp 0 copies the rows, warp 10 the weights (one thread cannot issue both in a
// stage's 384 cycles), warp 1 owns the tensor memory and issues the products, warps 2-9 finish the tiles as in
// gemm_tc_kernel.cuh.  Waits are bounded as there.
#include "block_scaled_mma.cuh"
#include "gemm_tc_kernel.cuh"

namespace mu {

constexpr int QP_BK = 128, QP_THREADS = TC_THREADS + 32;

template <int BN, int PIECES, int STAGES>
struct QpSmem {
    unsigned char x[STAGES][PIECES][TC_BM * QP_BK];           // each 1,024-byte aligned
    unsigned char w[STAGES][BN * QP_BK];
    unsigned char scales[STAGES][PIECES + (BN > 128 ? 2 : 1)][BS_TILE_BYTES];     // of the rows' pieces, then the weights
    alignas(128) float patch[TC_EPI_WARPS][32 * TC_PATCH_PITCH];
    uint64_t full[STAGES], empty[STAGES], acc_full[2], acc_empty[2];
    uint32_t tmem_base;
};

struct QpScales { const unsigned char* x[2]; const unsigned char* w; };

template <int BN, int PIECES, int STAGES, typename TC>
__global__ void __launch_bounds__(QP_THREADS, 1)
q4_prompt_kernel(const __grid_constant__ CUtensorMap map_x0, const __grid_constant__ CUtensorMap map_x1,
                 const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_c, const QpScales scales,
                 const float* __restrict__ bias, const float* residual, TC* C, int M, int N, int kb_all, long long ldc, long long ldr,
                 int act, int* status, int bulk_out, int fixed) {
    extern __shared__ unsigned char qp_raw[];
    typedef QpSmem<BN, PIECES, STAGES> Smem;
    Smem& sm = *reinterpret_cast<Smem*>(((uintptr_t)qp_raw + 1023) & ~(uintptr_t)1023);
    constexpr int W_BLOCKS = BN > 128 ? 2 : 1;                // tiles of exponents that BN columns touch
    constexpr int ACCS = BN > 192 ? 1 : 2;                    // accumulators that tensor memory holds beside the exponents
    constexpr uint32_t SCALE_COLS = 4 * (PIECES + W_BLOCKS), TMEM_COLS = ACCS * BN + 2 * SCALE_COLS <= 256 ? 256 : 512;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int m_tiles = (M + TC_BM - 1) / TC_BM, n_tiles = (N + BN - 1) / BN, tiles = m_tiles * n_tiles;
    bool ok = true;

    if (threadIdx.x == 0) {
        tma_prefetch_map(&map_x0);
        tma_prefetch_map(&map_w);
        for (int s = 0; s < STAGES; ++s) { mbar_init(&sm.full[s], 2); mbar_init(&sm.empty[s], 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(&sm.acc_full[b], 1); mbar_init(&sm.acc_empty[b], TC_EPI_WARPS); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&sm.tmem_base)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = sm.tmem_base;
    pdl_trigger();

    if (warp == 0 || warp == 10) {
        if (lane == 0) {
            const bool rows = warp == 0;
            if (rows || !fixed) pdl_wait();                   // (fixed weights are written by no kernel)
            long long issued = 0;
            int s = 0;
            uint32_t phase = 1;                               // an empty ring's stages count as given back
            for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
                const int mt = tile % m_tiles, m0 = mt * TC_BM, n0 = (tile / m_tiles) * BN;
                const unsigned char* sx0 = scales.x[0] + (long long)mt * kb_all * BS_TILE_BYTES;
                const unsigned char* sx1 = PIECES == 2 ? scales.x[1] + (long long)mt * kb_all * BS_TILE_BYTES : nullptr;
                const int wb = n0 / BS_TILE, wb_last = (N - 1) / BS_TILE;
                const unsigned char* sw0 = scales.w + (long long)wb * kb_all * BS_TILE_BYTES;
                const unsigned char* sw1 = scales.w + (long long)(wb < wb_last ? wb + 1 : wb_last) * kb_all * BS_TILE_BYTES;
                for (int kb = 0; kb < kb_all; ++kb) {
                    ok = mbar_wait(&sm.empty[s], phase);
                    if (!ok) break;
                    const long long at = (long long)kb * BS_TILE_BYTES;
                    if (rows) {
                        mbar_expect_tx(&sm.full[s], PIECES * (TC_BM * QP_BK + BS_TILE_BYTES));
                        tma_load_2d(sm.x[s][0], &map_x0, kb * QP_BK, m0, &sm.full[s]);
                        bulk_load(sm.scales[s][0], sx0 + at, BS_TILE_BYTES, &sm.full[s]);
                        if (PIECES == 2) {
                            tma_load_2d(sm.x[s][PIECES - 1], &map_x1, kb * QP_BK, m0, &sm.full[s]);
                            bulk_load(sm.scales[s][1], sx1 + at, BS_TILE_BYTES, &sm.full[s]);
                        }
                    } else {
                        // (the copy of 4-bit codes counts its packed bytes)
                        mbar_expect_tx(&sm.full[s], BN * QP_BK / 2 + W_BLOCKS * BS_TILE_BYTES);
                        tma_load_2d(sm.w[s], &map_w, kb * QP_BK, n0, &sm.full[s]);
                        bulk_load(sm.scales[s][PIECES], sw0 + at, BS_TILE_BYTES, &sm.full[s]);
                        if (W_BLOCKS == 2) bulk_load(sm.scales[s][PIECES + W_BLOCKS - 1], sw1 + at, BS_TILE_BYTES, &sm.full[s]);
                    }
                    ++issued;
                    if (++s == STAGES) { s = 0; phase ^= 1; }
                }
            }
            if (!ok) {
                atomicExch(status, 1);                        // copies under way land before the block goes away
                for (long long j = issued > STAGES ? issued - STAGES : 0; j < issued; ++j)
                    mbar_wait(&sm.full[j % STAGES], (uint32_t)((j / STAGES) & 1));
            }
        }
    } else if (warp == 1) {
        constexpr uint32_t idesc = idesc_block_scaled(BM_E4M3, BM_E2M1, TC_BM, BN);
        constexpr uint32_t X_STAGE = PIECES * TC_BM * QP_BK / 16, X_PIECE = TC_BM * QP_BK / 16, W_STAGE = BN * QP_BK / 16;
        constexpr uint32_t S_STAGE = (PIECES + W_BLOCKS) * BS_TILE_BYTES / 16;
        const bool one = elect_one();
        const uint64_t x_desc0 = smem_desc_sw128(smem_u32(sm.x[0][0])), w_desc0 = smem_desc_sw128(smem_u32(sm.w[0]));
        const uint64_t s_desc0 = scales_desc(smem_u32(sm.scales[0][0]));
        uint64_t x_desc = x_desc0, w_desc = w_desc0, s_desc = s_desc0;
        int s = 0, local = 0;
        uint32_t phase = 0, set = 0;
        for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++local) {
            const int buf = ACCS == 2 ? local & 1 : 0, turn = ACCS == 2 ? local >> 1 : local;
            // which of the exponents' columns this tile's weights begin at: a tile may begin half-way into 128 rows of W
            const uint32_t w_from = BN % 128 ? (uint32_t)((tile / m_tiles) * BN % BS_TILE / 32) : 0u;
            ok = mbar_wait(&sm.acc_empty[buf], (uint32_t)((turn & 1) ^ 1));
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t tmem_d = tmem_base + (uint32_t)(buf * BN);
            for (int kb = 0; kb < kb_all; ++kb) {
                ok = mbar_wait(&sm.full[s], phase);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (one) {
                    const uint32_t tmem_s = tmem_base + ACCS * BN + set * SCALE_COLS;        // two sets, in turn
#pragma unroll
                    for (int p = 0; p < PIECES + W_BLOCKS; ++p) copy_scales(tmem_s + 4 * p, s_desc + p * (BS_TILE_BYTES / 16));
#pragma unroll
                    for (int j = 0; j < QP_BK / 32; ++j)
#pragma unroll
                        for (int p = 0; p < PIECES; ++p)
                            umma_block_scaled(tmem_d, x_desc + p * X_PIECE + 2 * j, w_desc + 2 * j, idesc | idesc_scale_byte(j), tmem_s + 4 * p,
                                              tmem_s + 4 * PIECES + w_from, kb > 0 || j > 0 || p > 0 ? 1u : 0u);
                    umma_commit(&sm.empty[s]);
                }
                __syncwarp();
                set ^= 1;
                x_desc += X_STAGE;
                w_desc += W_STAGE;
                s_desc += S_STAGE;
                if (++s == STAGES) { s = 0; phase ^= 1; x_desc = x_desc0; w_desc = w_desc0; s_desc = s_desc0; }
            }
            if (ok && one) umma_commit(&sm.acc_full[buf]);
            __syncwarp();
        }
        if (!ok && one) atomicExch(status, 2);
    } else {
        const int quad = warp & 3, half = (warp - 2) / 4;
        constexpr int COLS = BN / 2, CHUNKS = COLS / 32;
        float* patch = sm.patch[warp - 2];
        const bool vec_ok = sizeof(TC) == 2 && ((ldc * sizeof(TC)) % 16 == 0) && (((uintptr_t)C) % 16 == 0) && !residual &&
                            (((uintptr_t)bias) % 16 == 0);
        pdl_wait();                                           // the residual is the work of earlier kernels, and C may be read by them
        int local = 0;
        for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++local) {
            const int buf = ACCS == 2 ? local & 1 : 0, turn = ACCS == 2 ? local >> 1 : local;
            const int row0 = (tile % m_tiles) * TC_BM + quad * 32, n0 = (tile / m_tiles) * BN;
            ok = mbar_wait(&sm.acc_full[buf], (uint32_t)(turn & 1));
            if (!ok) {
                if (lane == 0) atomicExch(status, 3);
                break;
            }
            __syncwarp();
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint32_t acc_addr = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(buf * BN + half * COLS);
#pragma unroll
            for (int q = 0; q < CHUNKS; ++q) {
                const int nb = n0 + half * COLS + 32 * q;
                uint32_t r[32];
                tmem_ld_32x32(acc_addr + 32 * q, r);
                if (q == CHUNKS - 1) {
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    if (lane == 0) mbar_arrive(&sm.acc_empty[buf]);
                    __syncwarp();
                }
                if (row0 >= M || nb >= N) continue;           // the same for the whole warp
                if (bulk_out) {
                    if (act == ACT_GELU_NEW) tc_finish_block_bulk<ACT_GELU_NEW, TC>(r, patch, lane, bias, &map_c, N, row0, nb, bulk_out == 2, true);
                    else if (act == ACT_GELU_ERF) tc_finish_block_bulk<ACT_GELU_ERF, TC>(r, patch, lane, bias, &map_c, N, row0, nb, bulk_out == 2, true);
                    else if (act == ACT_RELU2) tc_finish_block_bulk<ACT_RELU2, TC>(r, patch, lane, bias, &map_c, N, row0, nb, bulk_out == 2, true);
                    else tc_finish_block_bulk<0, TC>(r, patch, lane, bias, &map_c, N, row0, nb, bulk_out == 2, true);
                    continue;
                }
                const bool packed = vec_ok && nb + 32 <= N;
                float bias_col[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int n = packed ? nb + 8 * (lane & 3) + e : nb + lane;
                    bias_col[e] = bias && n < N ? bias[n] : 0.0f;
                }
                if (act == ACT_GELU_NEW) tc_finish_block<ACT_GELU_NEW, TC>(r, patch, lane, bias, bias_col, residual, C, M, N, row0, nb, ldc, ldr, packed);
                else if (act == ACT_GELU_ERF) tc_finish_block<ACT_GELU_ERF, TC>(r, patch, lane, bias, bias_col, residual, C, M, N, row0, nb, ldc, ldr, packed);
                else if (act == ACT_RELU2) tc_finish_block<ACT_RELU2, TC>(r, patch, lane, bias, bias_col, residual, C, M, N, row0, nb, ldc, ldr, packed);
                else tc_finish_block<0, TC>(r, patch, lane, bias, bias_col, residual, C, M, N, row0, nb, ldc, ldr, packed);
            }
        }
        if (bulk_out && lane == 0) tma_store_wait_all();
        __syncwarp();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLS) : "memory");
}

template <int BN, int PIECES, int STAGES, typename TC>
static int launch_prompt(const void* x0, const void* x1, const void* w, const QpScales& scales, const float* bias, const float* residual,
                         TC* C, int M, int N, int kp, long long ldc, long long ldr, int act, int fixed, int* status, cudaStream_t s) {
    CUtensorMap map_x0, map_x1, map_w, map_c;
    if (!tensor_map_q8(&map_x0, x0, M, kp, TC_BM) || !tensor_map_q4(&map_w, w, N, kp, BN)) return MU_ERR_LAUNCH;
    map_x1 = map_x0;
    if (PIECES == 2 && !tensor_map_q8(&map_x1, x1, M, kp, TC_BM)) return MU_ERR_LAUNCH;
    int bulk_out = 0;                                         // as in launch_tc
    if ((((uintptr_t)C) & 15) == 0 && (ldc * (long long)sizeof(TC)) % 16 == 0 &&
        (residual == nullptr || (sizeof(TC) == 4 && (const void*)residual == (const void*)C && ldr == ldc)) &&
        tensor_map_boxes(&map_c, C, M, N, ldc, sizeof(TC) == 2))
        bulk_out = residual ? 2 : 1;
    if (!bulk_out) map_c = map_x0;
    auto kernel = q4_prompt_kernel<BN, PIECES, STAGES, TC>;
    const size_t smem = sizeof(QpSmem<BN, PIECES, STAGES>) + 1024;
    static_assert(sizeof(QpSmem<BN, PIECES, STAGES>) + 1024 <= 227 * 1024, "a block's shared memory");
    if (!allow_shared(reinterpret_cast<const void*>(kernel), smem)) return MU_ERR_LAUNCH;
    prefer_shared_memory(reinterpret_cast<const void*>(kernel));
    const int sms = sm_count();
    if (sms <= 0) return MU_ERR_LAUNCH;
    const long long tiles = (long long)((N + BN - 1) / BN) * ((M + TC_BM - 1) / TC_BM);
    if (tiles > 2147483647ll - sms) return MU_ERR_UNSUPPORTED_SIZE;
    return launch_pdl(kernel, dim3((unsigned)(tiles < sms ? tiles : sms)), dim3(QP_THREADS), smem, s, 1, map_x0, map_x1, map_w, map_c, scales,
                      bias, residual, C, M, N, kp / QP_BK, ldc, ldr, act, status, bulk_out, fixed);
}

// The columns of a tile, by the cycles of the waves that its tiles make, which rank the widths and do not foretell times (2,048 x 4,096 x
// 1,024, bfloat16 rows: 11 us counted, 21 measured): a stage of 128 of k takes its products (2 cycles a column
// and piece) or what it brings in from the L2 (16 KB a piece of rows, 64 bytes a column, the exponents; 55 bytes a cycle
// and SM), a tile some 300 cycles more, and 1,800 where it is 256 wide: its one accumulator is read out before the next
// tile's products begin (and with two pieces its ring has two stages).  Microseconds on a B200 for 128, 192 and 256 columns, 8-bit
// rows: 777 x 4,800 x 1,600 10.1, 11.9, 8.8; 512 x 4,096 x 2,048 7.3, 8.6, 9.3; 1,000 x 6,400 x 1,600 13.6, 12.4, 14.2;
// 4,096 x 16,384 x 4,096 232, 208, 210; bfloat16 rows: 1,000 x 6,400 x 1,600 22.8, 21.3, 26.7; 4,096 x 16,384 x 4,096 428, 372, 435.
static int choose_columns(int M, int N, int kb, int pieces, int sms) {
    int best = 64;
    long long least = 1ll << 62;
    for (int b = 64; b <= 256; b += 64) {
        const long long tiles = (((long long)N + b - 1) / b) * (((long long)M + 127) / 128);
        const long long products = 2ll * b * pieces, bytes = 16384ll * pieces + 64ll * b + 512ll * (pieces + (b > 128 ? 2 : 1));
        long long stage = products > bytes / 55 ? products : bytes / 55;
        if (b == 256 && pieces == 2) stage += stage / 5;
        const long long cost = (tiles + sms - 1) / sms * (kb * stage + (b == 256 ? 1800 : 300));
        if (cost < least) { least = cost; best = b; }
    }
    return best;
}

// Rows and weights as launch_q4_few_rows has them (8 bits, or two pieces); any M.  bn: columns of a tile (64, 128, 192, 256; 0:
// chosen here).
int launch_q4_prompt(const void* x0, const void* x0_scales, const void* x1, const void* x1_scales, const void* w, const void* w_scales,
                           const float* bias, const float* residual, void* C, int M, int N, int kp, long long ldc, long long ldr, int act,
                           int out_bf16, int bn, int fixed, int* status, void* stream) {
    const QpScales scales = {{(const unsigned char*)x0_scales, (const unsigned char*)x1_scales}, (const unsigned char*)w_scales};
    const int sms = sm_count();
    if (sms <= 0) return MU_ERR_LAUNCH;
    if (bn == 0) bn = choose_columns(M, N, kp / QP_BK, x1 ? 2 : 1, sms);
    cudaStream_t s = (cudaStream_t)stream;
#define MU_QP(BN, P, ST)                                                                                                            \
    (out_bf16 ? launch_prompt<BN, P, ST, __nv_bfloat16>(x0, x1, w, scales, bias, residual, (__nv_bfloat16*)C, M, N, kp, ldc, ldr, act, fixed, status, s) \
              : launch_prompt<BN, P, ST, float>(x0, x1, w, scales, bias, residual, (float*)C, M, N, kp, ldc, ldr, act, fixed, status, s))
    if (bn == 256) return x1 ? MU_QP(256, 2, 2) : MU_QP(256, 1, 3);
    if (bn == 192) return x1 ? MU_QP(192, 2, 3) : MU_QP(192, 1, 4);
    if (bn == 128) return x1 ? MU_QP(128, 2, 3) : MU_QP(128, 1, 5);
    if (bn == 64) return x1 ? MU_QP(64, 2, 4) : MU_QP(64, 1, 6);
#undef MU_QP
    return MU_ERR_BAD_ARGUMENT;
}

}  // namespace mu

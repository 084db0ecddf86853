// C[M, N] = act(X[M, K] . W[N, K]^T + bias) (+ residual) for up to 128 rows, W in 4 bits, X in 8 bits (block_scaled.cuh),
// the WEIGHTS as the 128-row operand of tcgen05.mma and the batch as its narrow side.
//
// A step of single tokens reads each weight once, 17 bytes for 32 of them, and does almost no arithmetic.  The codes go
// from HBM to the tensor cores without passing a register: TMA spreads them to 16 per 16 bytes of shared memory, the
// instruction multiplies e2m1 by e4m3 and applies both exponents.  Expanding 4-bit codes in registers would cost two
// instructions a code where an SM takes in 46 codes a clock.
//   * a tile is 128 rows of W (128 output columns) by all M rows of X: D[128, NB] = W_tile . X^T, NB = M rounded up to 16,
//     32, 64 or 128; a stage is 128 of k: 8 KB of codes, 512 bytes of exponents, and the rows' share;
//   * K is cut over the blocks of a cluster (up to 16) so that tiles x splits fill the SMs; the partial tiles meet in
//     distributed shared memory and are added in rank order (as in gemm_rows.cu);
//   * bfloat16 rows come as two pieces, each e4m3, that together hold them exactly: two products a step into one
//     accumulator.
// Warp 0 issues the copies, warp 1 owns the tensor memory and issues the products, warps 2-5 read the accumulators.
// Waits are bounded as everywhere: one that runs out sets the status word, and the blocks leave together.
#include "block_scaled_mma.cuh"

namespace mu {

constexpr int QF_THREADS = 192;
constexpr int QF_BN = 128, QF_BK = 128;
constexpr int QF_MAX_SPLIT = 16;
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
    if constexpr (COUNT == 16) {
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

__device__ __forceinline__ float qf_act(float x, int act, bool to_bf16) { return to_bf16 ? apply_act_bf16(x, act) : apply_act(x, act); }

struct QfRows {                       // the rows' codes and exponents: one piece, or two
    const unsigned char* scales[2];   // [tiles of 128 rows][kb][512]
};

// grid.x = tiles * splits: the blocks of a cluster (along x) share a tile and cut K.  Dynamic shared memory, 1,024-byte
// aligned: per stage W 16 KB and PIECES x (NB x 128 bytes), then per stage the exponents (512 bytes each), then, with
// splits > 1, the shares this block is sent and its own partial tile (on the stages, when they are no longer read).
template <int NB, int PIECES, typename TC>
__global__ void __launch_bounds__(QF_THREADS)
q4_few_rows_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x0,
                   const __grid_constant__ CUtensorMap map_x1, const unsigned char* __restrict__ w_scales, const QfRows rows,
                   const float* __restrict__ bias, const float* residual, TC* C, int M, int N, int kb_all, long long ldc,
                   long long ldr, int act, int* status, int splits, int stages) {
    constexpr uint32_t X_BYTES = NB * QF_BK, STAGE = QF_W_BYTES + PIECES * X_BYTES;
    constexpr uint32_t SCALE_STAGE = (1 + PIECES) * BS_TILE_BYTES, ALL_BYTES = QF_W_COPIED + PIECES * X_BYTES + SCALE_STAGE;
    constexpr uint32_t ACC_COLS = NB < 32 ? 32 : NB, SCALE_COLS = 4 * (1 + PIECES);
    constexpr uint32_t TMEM_COLS = ACC_COLS + 2 * SCALE_COLS <= 64 ? 64 : ACC_COLS + 2 * SCALE_COLS <= 128 ? 128 : 256;
    constexpr int CHUNK = NB < 32 ? 16 : 32;
    extern __shared__ unsigned char qf_raw[];
    unsigned char* base = reinterpret_cast<unsigned char*>(((uintptr_t)qf_raw + 1023) & ~(uintptr_t)1023);
    unsigned char* scale_smem = base + (size_t)stages * STAGE;
    float* part = reinterpret_cast<float*>(scale_smem + (size_t)stages * SCALE_STAGE);
    float* outbox = reinterpret_cast<float*>(base);
    __shared__ uint64_t full[16], empty[16], acc_full, parts_in;
    __shared__ uint32_t tmem_slot;
    __shared__ float bias_s[QF_BN];

    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rank = splits > 1 ? (int)qf_cluster_rank() : 0;
    const int tile = blockIdx.x / splits;
    const int n0 = tile * QF_BN;
    const int kb_begin = (int)((long long)kb_all * rank / splits), kb_end = (int)((long long)kb_all * (rank + 1) / splits);
    const int my_kb = kb_end - kb_begin;                  // at least one: the host keeps splits <= kb_all
    bool ok = true;

    if (threadIdx.x == 0) {
        tma_prefetch_map(&map_w);
        tma_prefetch_map(&map_x0);
        if (PIECES == 2) tma_prefetch_map(&map_x1);
        for (int s = 0; s < stages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
        mbar_init(&acc_full, 1);
        mbar_init(&parts_in, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&tmem_slot)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (threadIdx.x >= 64) {
        const int n = n0 + (int)threadIdx.x - 64;
        bias_s[threadIdx.x - 64] = (bias && n < N) ? bias[n] : 0.0f;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_acc = tmem_slot;
    pdl_trigger();
    if (splits > 1) qf_cluster_arrive();                  // every block runs before anyone writes into another's shared memory

    if (warp == 0) {
        if (lane == 0) {
            auto load_weights = [&](int i, int s) {
                mbar_expect_tx(&full[s], ALL_BYTES);
                tma_load_2d(base + (size_t)s * STAGE, &map_w, (kb_begin + i) * QF_BK, n0, &full[s]);
                bulk_load(scale_smem + (size_t)s * SCALE_STAGE, w_scales + ((long long)tile * kb_all + kb_begin + i) * BS_TILE_BYTES,
                          BS_TILE_BYTES, &full[s]);
            };
            auto load_rows = [&](int i, int s) {
#pragma unroll
                for (int p = 0; p < PIECES; ++p) {
                    tma_load_2d(base + (size_t)s * STAGE + QF_W_BYTES + p * X_BYTES, p == 0 ? &map_x0 : &map_x1, (kb_begin + i) * QF_BK, 0, &full[s]);
                    bulk_load(scale_smem + (size_t)s * SCALE_STAGE + (1 + p) * BS_TILE_BYTES,
                              rows.scales[p] + (long long)(kb_begin + i) * BS_TILE_BYTES, BS_TILE_BYTES, &full[s]);
                }
            };
            const int first = my_kb < stages ? my_kb : stages;
            for (int i = 0; i < first; ++i) load_weights(i, i);      // written by no kernel: before the wait for the one before
            pdl_wait();
            for (int i = 0; i < first; ++i) load_rows(i, i);
            int issued = first;
            for (int i = first; i < my_kb; ++i) {
                const int s = i % stages;
                ok = mbar_wait(&empty[s], (uint32_t)((i / stages - 1) & 1));
                if (!ok) break;
                load_weights(i, s);
                load_rows(i, s);
                issued = i + 1;
            }
            if (!ok) {
                atomicExch(status, 1);
                for (int j = issued > stages ? issued - stages : 0; j < issued; ++j)      // copies under way land first
                    mbar_wait(&full[j % stages], (uint32_t)((j / stages) & 1));
            }
        }
    } else if (warp == 1) {
        const bool one = elect_one();
        constexpr uint32_t idesc = idesc_block_scaled(BM_E2M1, BM_E4M3, QF_BN, NB);
        for (int i = 0; i < my_kb; ++i) {
            const int s = i % stages;
            ok = mbar_wait(&full[s], (uint32_t)((i / stages) & 1));
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            if (!one) continue;
            const uint32_t w_addr = smem_u32(base + (size_t)s * STAGE), s_addr = smem_u32(scale_smem + (size_t)s * SCALE_STAGE);
            const uint32_t tmem_s = tmem_acc + ACC_COLS + (i & 1) * SCALE_COLS;      // two sets, in turn
#pragma unroll
            for (int p = 0; p <= PIECES; ++p) copy_scales(tmem_s + 4 * p, s_addr + p * BS_TILE_BYTES);
#pragma unroll
            for (int j = 0; j < QF_BK / 32; ++j)
#pragma unroll
                for (int p = 0; p < PIECES; ++p)
                    umma_block_scaled(tmem_acc, smem_desc_sw128(w_addr + j * 32), smem_desc_sw128(w_addr + QF_W_BYTES + p * X_BYTES + j * 32),
                                      idesc | idesc_scale_byte(j), tmem_s, tmem_s + 4 + 4 * p, (i > 0 || j > 0 || p > 0) ? 1u : 0u);
            umma_commit(&empty[s]);
        }
        if (ok && one) umma_commit(&acc_full);
        if (!ok && one) atomicExch(status, 2);
    } else {
        const int quad = warp & 3, col = quad * 32 + lane;        // a lane is an output column: n0 + col
        const bool to_bf16 = sizeof(TC) == 2;
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
                    if (n < N) {
                        float res[CHUNK];                         // all asked for before anything is stored: it may be C itself
#pragma unroll
                        for (int e = 0; e < CHUNK; ++e) res[e] = (residual && c0 + e < M) ? residual[(long long)(c0 + e) * ldr + n] : 0.0f;
#pragma unroll
                        for (int e = 0; e < CHUNK; ++e)
                            if (c0 + e < M)
                                C[(long long)(c0 + e) * ldc + n] = from_float<TC>(qf_act(__uint_as_float(r[e]) + bias_s[col], act, to_bf16) + res[e]);
                    }
                    __syncwarp();                                 // the lanes are together for the next load
                }
            }
        } else {
            const int cols_per = QF_BN / splits;                  // output columns each block of the cluster finishes
            const int groups = (M + 3) / 4;                       // batch rows travel four at a time
            const int pitch = 4 * groups + 4;
            const uint32_t slice_bytes = (uint32_t)(cols_per * pitch) * 4u;
            {
                float* mine = outbox + (size_t)col * pitch;
#pragma unroll
                for (int c0 = 0; c0 < NB; c0 += CHUNK) {
                    if (c0 >= M) break;
                    uint32_t r[CHUNK];
                    qf_load_columns<CHUNK>(acc_addr + c0, r);
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
            qf_cluster_wait();                                    // (the arrive was at the top) everyone is running
            if (threadIdx.x == 64) {
                mbar_expect_tx(&parts_in, (uint32_t)(splits - 1) * slice_bytes);
                for (int step = 1; step < splits; ++step) {
                    const int owner = (rank + step) % splits;
                    uint32_t dst, bar;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                                 : "=r"(dst) : "r"(smem_u32(part + (size_t)rank * cols_per * pitch)), "r"(owner));
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(bar) : "r"(smem_u32(&parts_in)), "r"(owner));
                    asm volatile("cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                                 ::"r"(dst), "r"(smem_u32(outbox + (size_t)owner * cols_per * pitch)), "r"(slice_bytes), "r"(bar)
                                 : "memory");
                }
            }
            const bool arrived = mbar_wait(&parts_in, 0);
            if (!arrived && lane == 0) atomicExch(status, 3);
            __syncwarp();
            qf_cluster_arrive();
            pdl_wait();
            const int who = (int)threadIdx.x - 64, total = groups * cols_per;
            for (int idx = who; idx < total && arrived; idx += 128) {
                const int g = idx / cols_per, i = idx - g * cols_per;
                const int c = rank * cols_per + i, n = n0 + c;
                if (n >= N) continue;
                float res[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    res[e] = (residual && 4 * g + e < M) ? residual[(long long)(4 * g + e) * ldr + n] : 0.0f;
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                for (int r = 0; r < splits; ++r) {                // in rank order, whoever sent when
                    const float* src = r == rank ? outbox + (size_t)c * pitch : part + ((size_t)r * cols_per + i) * pitch;
                    const float4 p = *reinterpret_cast<const float4*>(src + 4 * g);
                    v.x += p.x; v.y += p.y; v.z += p.z; v.w += p.w;
                }
                const float out4[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (4 * g + e < M)
                        C[(long long)(4 * g + e) * ldc + n] = from_float<TC>(qf_act(out4[e] + bias_s[c], act, to_bf16) + res[e]);
            }
            __syncwarp();
            qf_cluster_wait();                                    // nobody leaves while a copy may still read its outbox
        }
    }
    if (splits > 1 && warp < 2) {                                 // the same two cluster barriers as the epilogue warps
        __syncwarp();
        qf_cluster_wait();
        qf_cluster_arrive();
        qf_cluster_wait();
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_acc), "r"(TMEM_COLS) : "memory");
}

template <int NB, int PIECES, typename TC>
static int launch_few(const CUtensorMap& map_w, const CUtensorMap& map_x0, const CUtensorMap& map_x1, const unsigned char* w_scales,
                      const QfRows& rows, const float* bias, const float* residual, TC* C, int M, int N, int kb_all, long long ldc,
                      long long ldr, int act, int* status, int splits, int stages, size_t smem, cudaStream_t s) {
    auto kernel = q4_few_rows_kernel<NB, PIECES, TC>;
    static bool raised = false;
    if (!raised) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 224 * 1024) != cudaSuccess) return MU_ERR_LAUNCH;
        cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        cudaGetLastError();
        raised = true;
    }
    const int tiles = (N + QF_BN - 1) / QF_BN;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * splits));
    cfg.blockDim = dim3(QF_THREADS);
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
    return cudaLaunchKernelEx(&cfg, kernel, map_w, map_x0, map_x1, w_scales, rows, bias, residual, C, M, N, kb_all, ldc, ldr, act,
                              status, splits, stages) == cudaSuccess ? MU_OK : MU_ERR_LAUNCH;
}

// Whether clusters of 16 blocks of this kernel can be scheduled here (asked once).
static int few_max_cluster() {
    static int limit = 0;
    if (limit == 0) {
        int found = 8;
        auto kernel = q4_few_rows_kernel<64, 2, float>;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 224 * 1024) == cudaSuccess &&
            cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(16);
            cfg.blockDim = dim3(QF_THREADS);
            cfg.dynamicSmemBytes = 108 * 1024;
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = 16;
            attr[0].val.clusterDim.y = 1;
            attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            int clusters = 0;
            if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) == cudaSuccess && clusters > 0) found = 16;
        }
        cudaGetLastError();
        limit = found;
    }
    return limit;
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
bool tensor_map_q4(CUtensorMap* map, const void* base, long long rows, int kp, int box_rows) {
    return tensor_map_codes(map, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, base, rows, kp, kp / 2, box_rows);
}
bool tensor_map_q8(CUtensorMap* map, const void* base, long long rows, int kp, int box_rows) {
    return tensor_map_codes(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, rows, kp, kp, box_rows);
}

}  // namespace mu

// X: codes [M, kp] and exponents of one piece, or of two (x1 and its exponents not null); W: codes [N, kp / 2], exponents.
// kp a multiple of 128, codes 32-byte (W) and 16-byte (X) aligned, exponents 16-byte aligned.  C bfloat16 or float32 (ldc);
// residual float32 (ldr), may be C itself.  splits: blocks that share a tile and cut K (a power of two up to 16; 0: chosen
// here).  `status` as mu_gemm_tc.
MU_EXPORT int mu_q4_few_rows(const void* x0, const void* x0_scales, const void* x1, const void* x1_scales, const void* w,
                             const void* w_scales, const float* bias, const float* residual, void* C, int M, int N, int kp,
                             long long ldc, long long ldr, int act, int out_bf16, int splits, int* status, void* stream) {
    if (M <= 0 || N <= 0) return MU_OK;
    if (M > 128) return MU_ERR_UNSUPPORTED_SIZE;
    if (kp <= 0 || kp % 128 || !x0 || !x0_scales || !w || !w_scales || !C || !status || (x1 != nullptr) != (x1_scales != nullptr))
        return MU_ERR_BAD_ARGUMENT;
    if (((uintptr_t)w & 31) || (((uintptr_t)x0 | (uintptr_t)x1 | (uintptr_t)x0_scales | (uintptr_t)x1_scales | (uintptr_t)w_scales) & 15))
        return MU_ERR_ALIGNMENT;
    if ((M > 1 && ldc < N) || (residual && M > 1 && ldr < N)) return MU_ERR_BAD_ARGUMENT;
    if (splits < 0 || splits > mu::QF_MAX_SPLIT || (splits & (splits - 1))) return MU_ERR_BAD_ARGUMENT;
    const int sms = mu::sm_count();
    if (sms <= 0) return MU_ERR_LAUNCH;
    const long long tiles = ((long long)N + 127) / 128;
    const int kb_all = kp / 128, pieces = x1 ? 2 : 1;
    if (tiles * mu::QF_MAX_SPLIT > 2147483647ll) return MU_ERR_UNSUPPORTED_SIZE;
    const int limit = mu::few_max_cluster();
    if (splits == 0) {
        splits = 1;
        while (splits * 2 <= limit && tiles * splits * 2 <= sms + sms / 3 && splits * 2 <= kb_all) splits *= 2;
    }
    while (splits > limit || splits > kb_all) splits /= 2;
    const int nb = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
    const size_t stage_bytes = mu::QF_W_BYTES + (size_t)pieces * nb * 128 + (1 + pieces) * 512;
    const size_t tile_bytes = splits > 1 ? (size_t)((M + 3) / 4 * 4 + 4) * 128 * 4 : 0;
    const int per_block = (kb_all + splits - 1) / splits;
    size_t room = 108 * 1024;                                     // two blocks an SM where that leaves a ring of three or so
    if (1024 + tile_bytes + 3 * stage_bytes > room) room = 220 * 1024;
    int stages = (int)((room - 1024 - tile_bytes) / stage_bytes);
    const int least = (int)((tile_bytes + mu::QF_W_BYTES + (size_t)pieces * nb * 128 - 1) / (mu::QF_W_BYTES + (size_t)pieces * nb * 128));
    if (stages > per_block) stages = per_block;
    if (stages < least) stages = least;                           // the partial tile lies on the stages
    if (stages > 16) stages = 16;
    if (stages < 1) stages = 1;
    const size_t smem = 1024 + (size_t)stages * stage_bytes + tile_bytes;
    if (smem > 224 * 1024) return MU_ERR_UNSUPPORTED_SIZE;
    CUtensorMap map_w, map_x0, map_x1;
    if (!mu::tensor_map_q4(&map_w, w, N, kp, 128) || !mu::tensor_map_q8(&map_x0, x0, M, kp, nb) ||
        !mu::tensor_map_q8(&map_x1, x1 ? x1 : x0, M, kp, nb))
        return MU_ERR_LAUNCH;
    const mu::QfRows rows = {{(const unsigned char*)x0_scales, (const unsigned char*)x1_scales}};
    cudaStream_t s = (cudaStream_t)stream;
#define MU_FEW(NB, PIECES)                                                                                                          \
    (out_bf16 ? mu::launch_few<NB, PIECES, __nv_bfloat16>(map_w, map_x0, map_x1, (const unsigned char*)w_scales, rows, bias, residual, \
                                                          (__nv_bfloat16*)C, M, N, kb_all, ldc, ldr, act, status, splits, stages, smem, s) \
              : mu::launch_few<NB, PIECES, float>(map_w, map_x0, map_x1, (const unsigned char*)w_scales, rows, bias, residual, (float*)C, \
                                                  M, N, kb_all, ldc, ldr, act, status, splits, stages, smem, s))
#define MU_FEW_BOTH(NB) (pieces == 2 ? MU_FEW(NB, 2) : MU_FEW(NB, 1))
    if (nb == 16) return MU_FEW_BOTH(16);
    if (nb == 32) return MU_FEW_BOTH(32);
    if (nb == 64) return MU_FEW_BOTH(64);
    return MU_FEW_BOTH(128);
#undef MU_FEW_BOTH
#undef MU_FEW
}

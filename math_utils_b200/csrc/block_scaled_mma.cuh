// The tensor-core side of the block-scaled products: tcgen05.mma kind::mxf8f6f4 with e4m3 rows and e2m1 weights, their
// exponent bytes copied from shared to tensor memory, and the TMA maps of both.
#pragma once
#include "block_scaled.cuh"
#include "tcgen05.cuh"

namespace mu {

// The LayerNorm that a product makes of its rows: float32 gamma and beta (or null) [K], the rows picked (or null: the first ones).
struct RowNorm { const float *gamma, *beta; const int* pick; float eps; };

constexpr int BM_E4M3 = 0, BM_E2M1 = 5;         // operand types of the instruction

// Instruction descriptor of kind::mxf8f6f4: type of A at bit 7, of B at bit 10, both K-major, N >> 3 at bit 17, exponent
// bytes (ue8m0) bit 23, M >> 7 at bit 27.  Which of a word's four exponent bytes a product of 32 along k takes: bits 4 (B)
// and 29 (A).
__host__ __device__ constexpr uint32_t idesc_block_scaled(int a_type, int b_type, int m, int n) {
    return ((uint32_t)a_type << 7) | ((uint32_t)b_type << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) | ((uint32_t)(m >> 7) << 27);
}
__host__ __device__ constexpr uint32_t idesc_scale_byte(int j) { return ((uint32_t)j << 4) | ((uint32_t)j << 29); }

__device__ __forceinline__ void umma_block_scaled(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc,
                                                  uint32_t tmem_scale_a, uint32_t tmem_scale_b, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(tmem_scale_a), "r"(tmem_scale_b), "r"(accumulate) : "memory");
}

// A tile of exponent bytes (512 bytes: 32 rows of 16) from shared memory to four columns of tensor memory, the same in
// each quarter of its lanes.  In order with the products issued after it by the same thread.
__device__ __forceinline__ uint64_t scales_desc(uint32_t smem_addr) {
    uint64_t d = 0;                                     // no swizzle: 8 rows of 16 bytes one after another, groups 128 bytes apart
    d |= (uint64_t)((smem_addr & 0x3FFFF) >> 4);
    d |= (uint64_t)1 << 16;
    d |= (uint64_t)(128 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    return d;
}
__device__ __forceinline__ void copy_scales(uint32_t tmem_dst, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem_dst), "l"(desc) : "memory");
}

// `bytes` (a multiple of 16) from global to shared memory, both 16-byte aligned.
__device__ __forceinline__ void bulk_load(void* smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(smem_dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

// Codes of weights [n, kp / 2 bytes] in boxes of box_rows x 128: four-bit codes that the copy spreads to 16 codes per 16
// bytes of shared memory, as the instruction reads them beside eight-bit ones (a box takes 128 bytes a row).
bool tensor_map_q4(CUtensorMap* map, const void* base, long long rows, int kp, int box_rows);
// Codes of rows [m, kp bytes] in boxes of box_rows x 128.
bool tensor_map_q8(CUtensorMap* map, const void* base, long long rows, int kp, int box_rows);
// As tensor_map_out, made anew.
bool tensor_map_boxes(CUtensorMap* map, const void* base, long long rows, int cols, long long ld, int is_bf16);

}  // namespace mu

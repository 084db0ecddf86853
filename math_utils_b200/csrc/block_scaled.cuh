// Numbers in 8 and 4 bits with a power-of-two scale for every 32 along a row.
//
// A group of 32 entries v is kept as codes c and one exponent byte b (0..254): v = c * 2^(b - 127).  Rows take the
// codes e4m3 (a sign, four exponent and three mantissa bits, up to 448), weights e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a
// sign).  The exponent of a row's group is the smallest at which its largest entry is no larger than 448.
//
// Exponent bytes lie as the tensor cores read them: tiles of 128 rows by 128 columns, 512 bytes each, the tiles of a row
// of tiles one after another; within a tile row r has its four bytes at (r % 32) * 16 + (r / 32) * 4.
#pragma once
#include "common.cuh"

#include <cuda_fp16.h>
#include <cuda_fp4.h>
#include <cuda_fp8.h>

namespace mu {

constexpr int BS_GROUP = 32;               // entries that share a scale
constexpr int BS_TILE = 128;               // rows and columns of a tile of scales
constexpr int BS_TILE_BYTES = 512;

// Where the exponent byte of (row, group) lies; kb: tiles along a row.
__host__ __device__ __forceinline__ long long scale_at(long long row, int group, int kb) {
    return ((row / BS_TILE) * kb + group / 4) * BS_TILE_BYTES + (row % 32) * 16 + (row % BS_TILE) / 32 * 4 + group % 4;
}

// Magnitudes are compared as bit patterns without the sign: they order as the numbers do, an infinity and NaN above every one.
__device__ __forceinline__ unsigned int magnitude_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
__device__ __forceinline__ bool is_number(unsigned int top) { return top < 0x7F800000u; }

// The exponent byte for a group whose largest magnitude's pattern is `top` (a number's): the smallest b with top <= 448 * 2^(b - 127).
// 448 = 1.75 * 2^8, so b is the exponent field of top less 8, and one more where top's mantissa is above 1.75.
__device__ __forceinline__ int exponent_e4m3(unsigned int top) {
    const int b = (int)(top >> 23) - 8 + ((top & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return b > 0 ? b : 0;
}
// The same for e2m1, whose largest value is 6 = 1.5 * 2^2.
__device__ __forceinline__ int exponent_e2m1(unsigned int top) {
    const int b = (int)(top >> 23) - 2 + ((top & 0x7FFFFFu) > 0x400000u ? 1 : 0);
    return b > 0 ? (b < 254 ? b : 254) : 0;
}
// 2^(127 - b), by which a group's entries are multiplied on the way to their codes (exact: a power of two).
__device__ __forceinline__ float inverse_scale(int b) { return __uint_as_float((unsigned int)(254 - b) << 23); }
__device__ __forceinline__ float scale_value(int b) { return b > 0 ? __uint_as_float((unsigned int)b << 23) : __uint_as_float(0x00400000u); }

__device__ __forceinline__ unsigned int e4m3_pair(float lo, float hi) {
    return (unsigned int)__nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float2 of_e4m3_pair(unsigned int pair) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)pair, __NV_E4M3);
    return __half22float2(__half2(h));
}

constexpr unsigned int E4M3_NAN4 = 0x7F7F7F7Fu;

// Eight entries of a group of exponent byte b, as codes.
__device__ __forceinline__ uint2 e4m3_of_eight(const float (&v)[8], int b) {
    const float f = inverse_scale(b);
    uint2 c;
    c.x = e4m3_pair(v[0] * f, v[1] * f) | e4m3_pair(v[2] * f, v[3] * f) << 16;
    c.y = e4m3_pair(v[4] * f, v[5] * f) | e4m3_pair(v[6] * f, v[7] * f) << 16;
    return c;
}

// Eight bfloat16 entries of a group as TWO codes each: hi = e4m3(v / 2^e), lo = e4m3((v - hi 2^e) / 2^(e - 4)), so that
// v = hi 2^e + lo 2^(e - 4).  A bfloat16 has 8 significant bits, hi takes the upper 4 and leaves a remainder of at most
// 2^-4 of v that is a multiple of 2^-7 of v's leading bit: 4 bits, which lo holds exactly while they are multiples of its least
// step, 2^-13 2^e.  The group's largest entry lies above 224 2^e, so entries down to 2^-13 of it are held exactly and smaller ones
// within 2^-14 2^e, which is less than 2^-21 of it.  Beside that entry's own product a float32 sum keeps no more; where its
// weight is 0 the sum could, and does not here: a third piece would hold it, for half as much time again.  The exponent byte of lo is b - 4; where
// b < 4 (a group below 2^-115) its scale stays at 2^-127 and lo is made for that scale.
//
// words: the entries as they lie in memory, two a word.
__device__ __forceinline__ int low_exponent(int b) { return b > 4 ? b - 4 : 0; }
__device__ __forceinline__ void e4m3_pieces_of_eight(const unsigned int (&words)[4], int b, uint2& hi, uint2& lo) {
    const float f = inverse_scale(b);
    const float up = b > 4 ? 16.0f : __uint_as_float((unsigned int)(127 + b) << 23);      // 2^(scale of hi - scale of lo)
    unsigned int h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float v0 = __uint_as_float(words[i] << 16) * f, v1 = __uint_as_float(words[i] & 0xFFFF0000u) * f;
        h[i] = e4m3_pair(v0, v1);
        const float2 back = of_e4m3_pair(h[i]);
        l[i] = e4m3_pair((v0 - back.x) * up, (v1 - back.y) * up);
    }
    hi = make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
    lo = make_uint2(l[0] | l[1] << 16, l[2] | l[3] << 16);
}

// The largest magnitude of the group that four neighbouring lanes hold, eight bfloat16 each (two a word), as its bit pattern
// without the sign: patterns order as magnitudes do, an infinity and NaN above every number.
__device__ __forceinline__ unsigned int group_top_bf16(const unsigned int (&words)[4]) {
    unsigned int top = __vmaxu2(__vmaxu2(words[0] & 0x7FFF7FFFu, words[1] & 0x7FFF7FFFu), __vmaxu2(words[2] & 0x7FFF7FFFu, words[3] & 0x7FFF7FFFu));
    top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = __vmaxu2(top, __shfl_xor_sync(0xffffffffu, top, 2));
    return max(top & 0xFFFFu, top >> 16);
}
// exponent_e4m3 of a bfloat16's pattern, and whether it is a number's.
__device__ __forceinline__ int exponent_e4m3_bf16(unsigned int top) {
    const int b = (int)(top >> 7) - 8 + ((top & 0x7Fu) > 0x60u ? 1 : 0);
    return b > 0 ? b : 0;
}

}  // namespace mu

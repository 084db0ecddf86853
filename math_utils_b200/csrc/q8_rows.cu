// Rows and weights in 8 and 4 bits with a power-of-two scale for every 32 entries (block_scaled.cuh).
//
// mu_quantize_q4          a weight matrix to e2m1 codes and exponent bytes.
// mu_quantize_q8          rows to e4m3 codes and exponent bytes; with two pieces, bfloat16 rows to codes that together hold
//                         them (block_scaled.cuh says how exactly).
// mu_residual_add_norm_q8 x += (mult * y + mult2 * y2) * scale on the float32 stream, then h = x / sqrt(mean(x^2) + eps) *
//                         weight, written in 8 bits.
//
// What bounds them is bytes: the norm reads 8 and writes 4 + 1 + 1/32 for an entry: 4,096 x 8,192 in 82-87 us, 5.0-5.3 TB/s, four
// fifths of what a copy reaches (two turns a thread in blocks of 512 took 87: fewer blocks to fill one another's gaps); 8 x 2,048 in 2.6.
// The two pieces of 2,048 x 1,024 rows 4 us before a product.  A weight of 6,400 x 1,600 to 4 bits, once at load: 25 us; of 16,384 x 8,192:
// 253 (a thread reads its 32 entries one by one).
#include "addend.cuh"
#include "block_scaled.cuh"

namespace mu {

__device__ __forceinline__ unsigned int group_max(unsigned int top) {      // over the four lanes that hold a group, eight entries each
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    return max(top, __shfl_xor_sync(0xffffffffu, top, 2));
}
__device__ __forceinline__ unsigned int max_of_eight(const float (&v)[8]) {
    unsigned int top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, magnitude_bits(v[i]));
    return top;
}

// Two bfloat16 that were widened, as they lay in memory.
__device__ __forceinline__ unsigned int bf16_words(float lo, float hi) { return __float_as_uint(lo) >> 16 | (__float_as_uint(hi) & 0xFFFF0000u); }

// Eight entries of a row from column c on; columns from k on are zeros.
template <bool VEC, typename TE>
__device__ __forceinline__ void load_eight(const TE* row, int c, int k, float (&v)[8]) {
    if (VEC) {
        if (c >= k) {                                              // (k is a multiple of eight then)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.0f;
        } else if (sizeof(TE) == 2) {
            const uint4 raw = *reinterpret_cast<const uint4*>(row + c);
            const unsigned int w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            }
        } else {
            const float4 a = *reinterpret_cast<const float4*>(row + c), b = *reinterpret_cast<const float4*>(row + c + 4);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c + i < k ? to_float(row[c + i]) : 0.0f;
    }
}

// ------------------------------------------------------------------------------------------------- weights
// A thread a group.  The exponent is the smallest at which no entry is cut off at 6, or the one below it where that leaves
// the smaller sum of squared errors (most entries gain a bit, the largest is cut).
__device__ __forceinline__ float e2m1_error(const float (&v)[32], int b) {
    const float f = inverse_scale(b), s = scale_value(b);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const __nv_fp4x2_storage_t c = __nv_cvt_float2_to_fp4x2(make_float2(v[2 * i] * f, v[2 * i + 1] * f), __NV_E2M1, cudaRoundNearest);
        const float2 back = __half22float2(__half2(__nv_cvt_fp4x2_to_halfraw2(c, __NV_E2M1)));
        const float d0 = (back.x - v[2 * i] * f), d1 = (back.y - v[2 * i + 1] * f);
        sum = fmaf(d0, d0, fmaf(d1, d1, sum));
    }
    return sum * s * s;
}

template <typename TE>
__global__ void __launch_bounds__(128)
quantize_q4_kernel(const TE* __restrict__ w, long long ldw, int n, int k, int kp, unsigned char* __restrict__ codes,
                   unsigned char* __restrict__ scales) {
    const int groups = kp / BS_GROUP;
    const long long item = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const long long row = item / groups;
    const int g = (int)(item % groups);
    const long long rows = ((long long)n + BS_TILE - 1) / BS_TILE * BS_TILE;
    if (row >= rows) return;
    unsigned char* at = scales + scale_at(row, g, kp / BS_TILE);
    if (row >= n) {                                                // the tile's rows past the matrix: a scale, no codes
        *at = 0;
        return;
    }
    float v[32];
    unsigned int top = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        const int c = g * BS_GROUP + i;
        v[i] = c < k ? to_float(w[row * ldw + c]) : 0.0f;
        top = max(top, magnitude_bits(v[i]));
    }
    uint4 packed = make_uint4(0, 0, 0, 0);
    int b = 255;                                                   // a group holding an infinity or NaN is NaN
    if (is_number(top)) {
        b = exponent_e2m1(top);
        if (b > 0 && e2m1_error(v, b - 1) < e2m1_error(v, b)) --b;
        const float f = inverse_scale(b);
        unsigned int word[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 16; ++i)
            word[i / 4] |= (unsigned int)__nv_cvt_float2_to_fp4x2(make_float2(v[2 * i] * f, v[2 * i + 1] * f), __NV_E2M1, cudaRoundNearest) << (8 * (i % 4));
        packed = make_uint4(word[0], word[1], word[2], word[3]);
    }
    *reinterpret_cast<uint4*>(codes + row * (kp / 2) + (long long)g * 16) = packed;
    *at = (unsigned char)b;
    // a product launched next may fetch its weights before it waits for this kernel's end: what is written is in memory by
    // the time this block has gone
    __threadfence();
    asm volatile("fence.proxy.async.global;" ::: "memory");
}

// ------------------------------------------------------------------------------------------------- rows
// Eight entries a thread, four neighbouring lanes a group, ROWS rows a thread, all asked for before any is worked on: one where
// that makes no more blocks than the SMs hold at a time, four for more.
// PIECES = 2: the second piece's rows lie `behind` rows behind the first's, in one matrix with one set of exponents.
template <typename TE, int PIECES, bool VEC, int ROWS>
__global__ void __launch_bounds__(256)
quantize_q8_kernel(const TE* __restrict__ x, long long ldx, int m, int k, int kp, int behind, unsigned char* __restrict__ codes,
                   unsigned char* __restrict__ scales) {
    pdl_trigger();
    pdl_wait();
    const int row0 = blockIdx.x * blockDim.y * ROWS + threadIdx.y, c = (blockIdx.y * blockDim.x + threadIdx.x) * 8;
    const int rows = (m + BS_TILE - 1) / BS_TILE * BS_TILE;
    float v[ROWS][8];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
        const int row = row0 + j * blockDim.y;
        if (row < m && c < kp) load_eight<VEC>(x + (long long)row * ldx, c, k, v[j]);
        else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[j][i] = 0.0f;
        }
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
        const int row = row0 + j * blockDim.y;
        const unsigned int top = group_max(max_of_eight(v[j]));    // (every lane of the warp takes part)
        const bool fine = is_number(top);
        const int b = fine ? exponent_e4m3(top) : 127;
        if (row < m && c < kp) {
            uint2 hi, lo;
            if (PIECES == 2) {
                const unsigned int words[4] = {bf16_words(v[j][0], v[j][1]), bf16_words(v[j][2], v[j][3]), bf16_words(v[j][4], v[j][5]),
                                               bf16_words(v[j][6], v[j][7])};
                e4m3_pieces_of_eight(words, b, hi, lo);
            } else {
                hi = e4m3_of_eight(v[j], b);
            }
            if (!fine) hi = lo = make_uint2(E4M3_NAN4, E4M3_NAN4);
            *reinterpret_cast<uint2*>(codes + (long long)row * kp + c) = hi;
            if (PIECES == 2) *reinterpret_cast<uint2*>(codes + ((long long)behind + row) * kp + c) = lo;
        }
        // sixteen lanes hold 128 columns, a word of exponents
        unsigned int word = (unsigned int)b << (8 * (c / BS_GROUP % 4));
        word |= __shfl_xor_sync(0xffffffffu, word, 4);
        word |= __shfl_xor_sync(0xffffffffu, word, 8);
        if (row < (PIECES == 2 ? m : rows) && c < kp && c % BS_TILE == 0) {
            unsigned int low = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) low |= (unsigned int)low_exponent(word >> (8 * i) & 255u) << (8 * i);
            *reinterpret_cast<unsigned int*>(scales + scale_at(row, c / BS_GROUP, kp / BS_TILE)) = word;
            if (PIECES == 2) *reinterpret_cast<unsigned int*>(scales + scale_at(row + behind, c / BS_GROUP, kp / BS_TILE)) = low;
        }
    }
}

// ------------------------------------------------------------------------------------------------- the norm
// The sum of every thread's v, the same in all of them.
template <int THREADS>
__device__ __forceinline__ double sum_of_block(double v, double* scratch) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    double all = 0.0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) all += scratch[w];
    return all;
}

__device__ __forceinline__ double squares_of_eight(const float (&v)[8]) {
    const float a = fmaf(v[0], v[0], v[1] * v[1]), b = fmaf(v[2], v[2], v[3] * v[3]);
    const float c = fmaf(v[4], v[4], v[5] * v[5]), d = fmaf(v[6], v[6], v[7] * v[7]);
    return (double)((a + b) + (c + d));
}

// A block a row, eight entries a thread and turn; up to KEEP turns stay in registers between the sum and the codes, wider
// rows are read again from the stream (each entry by the thread that wrote it).  Eight squares are added pairwise in 32 bits (the
// row's factor is off by 2^-23 of itself at most), the eights in 64, and an entry times its row's factor and its weight is
// rounded once: an entry that is off by a bit of its 24 gets its neighbour's code wherever it lies that near the middle of two.
// With a thread's 32 squares on one 32-bit sum a row with a few large entries lost the small ones, and twice as many codes of
// ordinary rows went to the neighbour.
template <int THREADS, int KEEP, bool VEC>
__global__ void __launch_bounds__(THREADS)
residual_add_norm_q8_kernel(float* __restrict__ x, long long ldx, const Addend add, const float* __restrict__ weight, float eps,
                            int m, int width, int kp, unsigned char* __restrict__ codes, unsigned char* __restrict__ scales) {
    __shared__ double scratch[THREADS / 32];
    pdl_trigger();
    pdl_wait();
    const long long t = blockIdx.x;
    float* xs = x + t * ldx;
    float kept[KEEP][8];
    double sq = 0.0;
    auto take = [&](int c, float (&v)[8]) {                        // the stream's entries with the addition made
        load_eight<VEC>(xs, c, width, v);
        if (!add.y || c >= width) return;
        if (VEC) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float4 s = ra_added4(make_float4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]), add, t, c + 4 * h);
                *reinterpret_cast<float4*>(xs + c + 4 * h) = s;
                v[4 * h] = s.x; v[4 * h + 1] = s.y; v[4 * h + 2] = s.z; v[4 * h + 3] = s.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < width) { v[i] = ra_added(v[i], add, t, c + i); xs[c + i] = v[i]; }
        }
    };
#pragma unroll
    for (int j = 0; j < KEEP; ++j) {
        const int c = 8 * (threadIdx.x + j * THREADS);
        take(c, kept[j]);
        sq += squares_of_eight(kept[j]);
    }
    for (int c = 8 * (threadIdx.x + KEEP * THREADS); c < width; c += 8 * THREADS) {
        float v[8];
        take(c, v);
        sq += squares_of_eight(v);
    }
    const double exact = rsqrt(sum_of_block<THREADS>(sq, scratch) / (double)width + (double)eps);
    const float inv = (float)exact, inv_rest = (float)(exact - (double)inv);
    auto put = [&](int c, float (&v)[8]) {                         // all four lanes of a group are here together
        float g[8];
        load_eight<VEC>(weight, c, width, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float near = v[i] * inv;                         // and what its rounding and inv's left out, then one rounding
            v[i] = fmaf(near, g[i], fmaf(v[i], inv_rest, fmaf(v[i], inv, -near)) * g[i]);
        }
        const unsigned int top = group_max(max_of_eight(v));
        const bool fine = is_number(top);
        const int b = fine ? exponent_e4m3(top) : 127;
        const uint2 code = fine ? e4m3_of_eight(v, b) : make_uint2(E4M3_NAN4, E4M3_NAN4);
        // sixteen lanes hold 128 columns, a word of exponents
        unsigned int word = (unsigned int)b << (8 * (c / BS_GROUP % 4));
        word |= __shfl_xor_sync(0xffffffffu, word, 4);
        word |= __shfl_xor_sync(0xffffffffu, word, 8);
        if (c < kp) {
            *reinterpret_cast<uint2*>(codes + t * kp + c) = code;
            if (c % BS_TILE == 0) *reinterpret_cast<unsigned int*>(scales + scale_at(t, c / BS_GROUP, kp / BS_TILE)) = word;
        }
    };
#pragma unroll
    for (int j = 0; j < KEEP; ++j) put(8 * (threadIdx.x + j * THREADS), kept[j]);
    for (int c = 8 * (threadIdx.x + KEEP * THREADS); c - 8 * (threadIdx.x & 31) < kp; c += 8 * THREADS) {
        float v[8];
        load_eight<VEC>(xs, c, width, v);                          // written above by this very thread
        put(c, v);
    }
    // the rows behind the last one in its tile get (unused) exponents, every block's share of them
    const int words = kp / BS_TILE, behind = (m + BS_TILE - 1) / BS_TILE * BS_TILE - m;
    const unsigned int mine = (int)t < behind ? (unsigned int)((behind - (int)t + m - 1) / m * words) : 0u;
    for (unsigned int i = threadIdx.x; i < mine; i += THREADS)
        *reinterpret_cast<unsigned int*>(scales + scale_at(m + t + (long long)(i / words) * m, 4 * (int)(i % words), words)) = 0u;
}

}  // namespace mu

// w [n, k] (ldw) bfloat16 or float32 -> codes [n, kp / 2], scales [ceil(n / 128), kp / 128, 512]; kp: k rounded up to 128.
MU_EXPORT int mu_quantize_q4(const void* w, long long ldw, int is_bf16, int n, int k, int kp, void* codes, void* scales,
                             void* stream) {
    if (n <= 0) return MU_OK;
    if (!w || !codes || !scales || k <= 0 || kp % 128 || kp < k || kp - k >= 128 || ldw < k) return MU_ERR_BAD_ARGUMENT;
    if (((uintptr_t)codes | (uintptr_t)scales) & 15) return MU_ERR_ALIGNMENT;
    const long long rows = ((long long)n + 127) / 128 * 128, items = rows * (kp / 32);
    const long long blocks = (items + 127) / 128;
    if (blocks > 2147483647ll) return MU_ERR_UNSUPPORTED_SIZE;
    cudaStream_t s = (cudaStream_t)stream;
    if (is_bf16)
        mu::quantize_q4_kernel<__nv_bfloat16><<<(unsigned)blocks, 128, 0, s>>>((const __nv_bfloat16*)w, ldw, n, k, kp, (unsigned char*)codes, (unsigned char*)scales);
    else
        mu::quantize_q4_kernel<float><<<(unsigned)blocks, 128, 0, s>>>((const float*)w, ldw, n, k, kp, (unsigned char*)codes, (unsigned char*)scales);
    MU_CHECK_LAUNCH();
    return MU_OK;
}

namespace mu {

// x [m, k] (ldx) bfloat16 or float32 -> codes [m, kp], scales [ceil(m / 128), kp / 128, 512]; behind > 0: two pieces of bfloat16 rows, the
// second one's rows that many behind the first's (m at least, and both in the same tiles or a multiple of 128).
int launch_quantize_q8(const void* x, long long ldx, int is_bf16, int m, int k, int kp, int behind, void* codes, void* scales, void* stream) {
    const int rows = (m + 127) / 128 * 128, eights = kp / 8;
    // a block's threads along a row and its rows: whole warps of a row where it has as many eights
    const int along = eights >= 256 ? 256 : eights >= 128 ? 128 : eights >= 64 ? 64 : eights >= 32 ? 32 : 16;
    const int deep = 256 / along;
    const int sms = sm_count();
    if (sms <= 0) return MU_ERR_LAUNCH;
    const bool many = rows * (long long)eights >= 2ll * sms * 2048;
    const int each = many ? 4 : 1;
    const dim3 block(along, deep), grid((unsigned)((rows + deep * each - 1) / (deep * each)), (eights + along - 1) / along);
    if (grid.y > 65535) return MU_ERR_UNSUPPORTED_SIZE;
    const bool vec = k % 8 == 0 && ((uintptr_t)x & 15) == 0 && (m == 1 || ldx % (is_bf16 ? 8 : 4) == 0);
    cudaStream_t s = (cudaStream_t)stream;
#define MU_Q8_ROWS(TE, PIECES, VEC, ROWS) \
    return launch_pdl(quantize_q8_kernel<TE, PIECES, VEC, ROWS>, grid, block, 0, s, 1, (const TE*)x, ldx, m, k, kp, behind, (unsigned char*)codes, (unsigned char*)scales)
#define MU_Q8(TE, PIECES, VEC) { if (many) MU_Q8_ROWS(TE, PIECES, VEC, 4); MU_Q8_ROWS(TE, PIECES, VEC, 1); }
    if (behind > 0) { if (vec) MU_Q8(__nv_bfloat16, 2, true) MU_Q8(__nv_bfloat16, 2, false) }
    if (is_bf16) { if (vec) MU_Q8(__nv_bfloat16, 1, true) MU_Q8(__nv_bfloat16, 1, false) }
    if (vec) MU_Q8(float, 1, true)
    MU_Q8(float, 1, false)
#undef MU_Q8_ROWS
#undef MU_Q8
}

}  // namespace mu

MU_EXPORT int mu_quantize_q8(const void* x, long long ldx, int is_bf16, int m, int k, int kp, void* codes, void* scales, void* stream) {
    if (m <= 0) return MU_OK;
    if (!x || !codes || !scales || k <= 0 || kp % 128 || kp < k || kp - k >= 128 || (m > 1 && ldx < k)) return MU_ERR_BAD_ARGUMENT;
    if (((uintptr_t)codes | (uintptr_t)scales) & 15) return MU_ERR_ALIGNMENT;
    return mu::launch_quantize_q8(x, m > 1 ? ldx : k, is_bf16, m, k, kp, 0, codes, scales, stream);
}

// As mu_residual_add_norm with one group, the normed rows in 8 bits: codes [m, kp], scales [ceil(m / 128), kp / 128, 512].  The
// arguments come as one packed record (q4_linear.cu says why).
struct NormQ8Args {
    float* x;
    const float *y, *y2, *scale, *weight;
    void *codes, *scales, *stream;
    long long ldx, ldy, ldy2;
    float mult, mult2, eps;
    int m, width, kp;
};
MU_EXPORT int mu_norm_q8_args_size() { return (int)sizeof(NormQ8Args); }

MU_EXPORT int mu_residual_add_norm_q8(const NormQ8Args* p) {
    const NormQ8Args a = *p;
    float* x = a.x;
    const float *y = a.y, *y2 = a.y2, *scale = a.scale, *weight = a.weight;
    const long long ldx = a.ldx, ldy = a.ldy, ldy2 = a.ldy2;
    const float mult = a.mult, mult2 = a.mult2, eps = a.eps;
    const int m = a.m, width = a.width, kp = a.kp;
    void *codes = a.codes, *scales = a.scales, *stream = a.stream;
    if (m <= 0) return MU_OK;
    if (!x || !weight || !codes || !scales || width <= 0 || kp % 128 || kp < width || kp - width >= 128 || (y2 && !y) || (scale && !y))
        return MU_ERR_BAD_ARGUMENT;
    if (((uintptr_t)codes | (uintptr_t)scales) & 15) return MU_ERR_ALIGNMENT;
    const mu::Addend add = {y, ldy, mult, y2, ldy2, mult2, scale};
    const bool vec = width % 8 == 0 && (m == 1 || (ldx % 4 == 0 && ldy % 4 == 0 && ldy2 % 4 == 0)) &&
                     (((uintptr_t)x | (uintptr_t)y | (uintptr_t)y2 | (uintptr_t)scale | (uintptr_t)weight) & 15) == 0;
    cudaStream_t s = (cudaStream_t)stream;
#define MU_NORM8(THREADS, KEEP, VEC)                                                                                            \
    return mu::launch_pdl(mu::residual_add_norm_q8_kernel<THREADS, KEEP, VEC>, dim3((unsigned)m), dim3(THREADS), 0, s, 1, x, ldx, add, \
                          weight, eps, m, width, kp, (unsigned char*)codes, (unsigned char*)scales)
    if (vec) {
        if (kp <= 1024) MU_NORM8(128, 1, true);
        if (kp <= 2048) MU_NORM8(256, 1, true);
        if (kp <= 4096) MU_NORM8(256, 2, true);
        MU_NORM8(256, 4, true);
    }
    if (kp <= 1024) MU_NORM8(128, 1, false);
    if (kp <= 2048) MU_NORM8(256, 1, false);
    MU_NORM8(256, 4, false);
#undef MU_NORM8
}

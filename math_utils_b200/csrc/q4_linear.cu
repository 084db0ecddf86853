// The product with 4-bit weights as the library offers it: which of its kernels runs.
#include "block_scaled_mma.cuh"

namespace mu {

int q4_few_rows_tile(int M, bool cut_here);
int launch_q4_few_rows(const void* x, const void* x_scales, bool two_pieces, long long ldx, int K, const void* w, const void* w_scales,
                       const float* bias, const float* residual, void* C, int M, int N, int kp, long long ldc, long long ldr, int act,
                       int out_bf16, int splits, const RowNorm* norm, int fixed, int* status, void* stream);
int launch_q4_prompt(const void* x0, const void* x0_scales, const void* x1, const void* x1_scales, const void* w, const void* w_scales,
                     const float* bias, const float* residual, void* C, int M, int N, int kp, long long ldc, long long ldr, int act,
                     int out_bf16, int bn, int fixed, int* status, void* stream);
int launch_quantize_q8(const void* x, long long ldx, int is_bf16, int m, int k, int kp, int behind, void* codes, void* scales, void* stream);

// Up to 32 rows go to the kernel with the weights as the wide operand; up to 64 where that kernel can cut a long k and the other
// would leave most SMs idle.  Microseconds, 8-bit rows, that kernel and the other: 8 x 6,400 x 1,600 4.1 and 6.0; 32 x 11,264 x
// 2,048 6.9 and 9.3; 32 x 6,400 x 1,600 5.8 and 5.7; 48 x 1,600 x 6,400 7.2 and 12.0; 64 x 4,096 x 2,048 9.0 and 5.9.
static bool few_rows(int m, int n, int kp, int sms) {
    return m <= 32 || (m <= 64 && kp >= 32 * 128 && ((long long)n + 127) / 128 * 4 <= sms);
}

}  // namespace mu

// The arguments come as one packed record: a call with twenty of them costs the caller's side more than the launch.
struct LinearQ4Args {
    const void *x, *x_scales;            // 8-bit rows: codes [m, kp] and exponents; bfloat16 rows [m, k] (ldx): exponents null
    const void *w, *w_scales;            // codes [n, kp / 2], exponents
    const float *bias, *residual;        // null or [n]; null or [m, n] (ldr), may be out
    void *out, *room;                    // out [m, n] (ldo); room for the pieces of more than 8 bfloat16 rows: twice m
                                         // rounded up to 128 rows of kp codes and kp / 32 exponents
    int* status;
    void* stream;
    const float *gamma, *beta;           // gamma not null: x is float32, the rows are its LayerNorms (m <= 8), ...
    const int* pick;                     // ... of the rows picked, or of the first m
    long long ldx, ldo, ldr;
    int m, n, k, kp, act, out_bf16, way; // way 0: the kernel is chosen here; tests: 1 + blocks a tile, or -(columns of a tile)
    float eps;
    int fixed;                           // weights, exponents, bias, gamma and beta are written by no work that may still be under way on any
                                         // stream: they are fetched before the launches in front of this one have ended
};

constexpr int Q4_CUT_INSIDE = 8;         // bfloat16 rows that the few-rows kernel cuts itself

MU_EXPORT int mu_linear_q4_args_size() { return (int)sizeof(LinearQ4Args); }

MU_EXPORT int mu_linear_q4(const LinearQ4Args* p) {
    const LinearQ4Args a = *p;
    if (a.m <= 0 || a.n <= 0) return MU_OK;
    const bool sixteen = !a.x_scales;
    if (a.kp <= 0 || a.kp % 128 || a.k <= a.kp - 128 || a.k > a.kp || !a.x || !a.w || !a.w_scales || !a.out || !a.status) return MU_ERR_BAD_ARGUMENT;
    // (one row's stride is never used)
    if (a.m > 1 && (a.ldo < a.n || (a.residual && a.ldr < a.n) || (sixteen && a.ldx < a.k))) return MU_ERR_BAD_ARGUMENT;
    if (a.gamma && (!sixteen || a.m > Q4_CUT_INSIDE)) return MU_ERR_BAD_ARGUMENT;
    if (a.gamma && (a.k % 8 != 0 || a.ldx % 4 != 0 || (((uintptr_t)a.x | (uintptr_t)a.gamma | (uintptr_t)a.beta) & 15))) return MU_ERR_ALIGNMENT;
    if (((uintptr_t)a.w & 31) || (((uintptr_t)a.w_scales | (uintptr_t)a.x_scales | (uintptr_t)a.room) & 15) || ((uintptr_t)a.x & (sixteen ? 1 : 15)) ||
        ((uintptr_t)a.out & (a.out_bf16 ? 1 : 3)))
        return MU_ERR_ALIGNMENT;
    const int sms = mu::sm_count();
    if (sms <= 0) return MU_ERR_LAUNCH;
    const long long ldo = a.m > 1 ? a.ldo : a.n, ldr = a.m > 1 ? a.ldr : a.n, ldx = a.m > 1 || a.gamma ? a.ldx : a.k;
    const mu::RowNorm norm = {a.gamma, a.beta, a.pick, a.eps};
    const bool few = a.way > 0 || a.gamma || (a.way == 0 && mu::few_rows(a.m, a.n, a.kp, sms));
    const unsigned char *x = (const unsigned char*)a.x, *scales = (const unsigned char*)a.x_scales, *x1 = nullptr, *scales1 = nullptr;
    const bool cut = sixteen && (a.m > Q4_CUT_INSIDE || !few);
    if (cut) {
        if (!a.room) return MU_ERR_BAD_ARGUMENT;
        const long long rows = ((long long)a.m + 127) / 128 * 128;
        const int behind = few ? mu::q4_few_rows_tile(a.m, false) : (int)rows;
        unsigned char* codes = (unsigned char*)a.room;
        const int code = mu::launch_quantize_q8(a.x, ldx, 1, a.m, a.k, a.kp, behind, codes, codes + 2 * rows * a.kp, a.stream);
        if (code != MU_OK) return code;
        x = codes;
        scales = codes + 2 * rows * a.kp;
        x1 = x + rows * a.kp;                             // (of many rows: whole tiles behind the first)
        scales1 = scales + rows * (a.kp / 32);
    }
    if (few)
        return mu::launch_q4_few_rows(x, scales, cut, ldx, a.k, a.w, a.w_scales, a.bias, a.residual, a.out, a.m, a.n, a.kp, ldo, ldr, a.act,
                                      a.out_bf16, a.way > 0 ? a.way - 1 : 0, a.gamma ? &norm : nullptr, a.fixed, a.status, a.stream);
    return mu::launch_q4_prompt(x, scales, x1, scales1, a.w, a.w_scales, a.bias, a.residual, a.out, a.m, a.n, a.kp, ldo, ldr, a.act, a.out_bf16,
                                -a.way, a.fixed, a.status, a.stream);
}

/* Launchers of the microscaled 4-bit kernels (mx4_quantize.hip, gemm_mx4.hip,
 * gemm_mx4_weights.hip) and of the mixture-of-experts layer (moe.hip). Plain
 * C ABI: the host C++ calls them without HIP headers. No counterpart in the
 * reference, whose lowest type is fp16 (src/cuda/matmul_tensor_core.cu:96-297).
 *
 * A quantised operand of `rows` rows of k numbers: k padded with zeros to
 * kp = mchip_mx4_k(k), a multiple of 128; codes [rows, kp / 2], two e2m1 codes
 * per byte, the first in the low half; scales [rows, kp / 32], one byte s per
 * 32 elements, worth 2^(s - 127), 255 for a block that holds no number. As the
 * weights of unquantised rows and of experts, its numbers are fp32's: codes
 * from 4 up at byte 253 and from 2 up at 254 (quantising gives at most 252)
 * pass its range, and no product with them is finite.
 *
 * Each launcher returns 0 or a hipError_t value; for hipErrorInvalidValue (1)
 * *why names the argument at fault. Types are MCHIP_DTYPE_* (matmul.h). */
#pragma once

#include "matmul.h"

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

enum { MCHIP_DTYPE_MX4 = 4 };

long long mchip_mx4_k(int k);

/* x [rows, k], rows ld elements apart, to codes and scales; values (or null):
 * what the codes stand for, [rows, k] in x's type. */
int mchip_quantize_mx4(int dtype, const void* x, long long ld, void* codes, void* scales, int rows, int k,
                       void* values, void* stream, const char** why);
/* w [k, n] (ld elements between rows of n), blocks down its columns, to an
 * operand of n rows of k; values (or null): [k, n]. */
int mchip_quantize_mx4_columns(int dtype, const void* w, long long ld, void* codes, void* scales, int k, int n,
                               void* values, void* stream, const char** why);

/* C[m, n] = A B^T, A of m and B of n quantised rows; fp32 sums, C in c_dtype. */
int mchip_launch_matmul_mx4(const void* a_codes, const void* a_scales, const void* b_codes, const void* b_scales,
                            int c_dtype, void* c, int m, int n, int k, void* stream, const char** why);

/* C[m, n] = A B^T with A [m, k] of a_dtype, rows lda elements apart, as it is
 * (fp32: numbers below 2^-110 cut to multiples of 2^-133), and B of n
 * quantised rows. */
long long mchip_matmul_mx4_weights_workspace_bytes(int a_dtype, int m, int n, int k);
int mchip_launch_matmul_mx4_weights(int a_dtype, const void* a, long long lda, const void* b_codes,
                                    const void* b_scales, int c_dtype, void* c, int m, int n, int k, void* stream,
                                    void* workspace, const char** why);

enum { MCHIP_MOE_RELU = 0, MCHIP_MOE_GELU = 1, MCHIP_MOE_SWIGLU = 2 };
enum { MCHIP_MOE_MAX_TOKENS = 64, MCHIP_MOE_MAX_EXPERTS = 512, MCHIP_MOE_MAX_TOP_K = 16 };

typedef struct mchip_moe_args {
    int dtype; /* of x and y */
    const void* x;
    long long ldx;
    const float* router; /* [experts, d] */
    int weights;         /* MCHIP_DTYPE_BF16, _F16 or _MX4 */
    const void* w1;      /* [experts, h (swiglu: 2 h, gates first), d] */
    const void* w1_scales;
    const float* b1;
    const void* w2; /* [experts, d, h] */
    const void* w2_scales;
    const float* b2;
    void* y;      /* [tokens, d] */
    int* chosen;  /* [tokens, top_k] or null */
    float* gates; /* [tokens, top_k] or null */
    int tokens, d, h, experts, top_k, activation, normalize;
    void* workspace;
} mchip_moe_args;

long long mchip_moe_workspace_bytes(int dtype, int tokens, int d, int h, int experts, int top_k);
int mchip_launch_moe(const mchip_moe_args* args, void* stream, const char** why);

#ifdef __cplusplus
}
#endif

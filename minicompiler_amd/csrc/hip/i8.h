/* Launchers of the 8-bit integer kernels (i8_quantize.hip, gemm_i8.hip) and of
 * the router (route.hip). Plain C ABI: the host C++ calls them without HIP
 * headers. No counterpart in the reference, whose lowest type is fp16
 * (src/cuda/matmul_tensor_core.cu:96-297).
 *
 * An i8 operand of `rows` rows of k numbers: k padded with zeros to
 * kp = mchip_i8_k(k), a multiple of 128; codes [rows, kp], one signed byte
 * each, -127..127 as quantised; scales [rows], fp32. A code stands for
 * code x scale.
 *
 * Each launcher returns 0 or a hipError_t value; for hipErrorInvalidValue (1)
 * *why names the argument at fault. Types are MCHIP_DTYPE_* (matmul.h). */
#pragma once

#include "matmul.h"

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

long long mchip_i8_k(int k);

/* x [rows, k], rows ld elements apart, to codes and scales; values (or null):
 * what the codes stand for, [rows, k] in x's type. */
int mchip_quantize_i8(int dtype, const void* x, long long ld, void* codes, float* scales, int rows, int k, void* values,
                      void* stream, const char** why);
/* w [k, n] (ld elements between rows of n) to an operand of its n columns;
 * values (or null): [k, n]. */
int mchip_quantize_i8_columns(int dtype, const void* w, long long ld, void* codes, float* scales, int k, int n,
                              void* values, void* stream, const char** why);

enum { MCHIP_ACT_RELU = 0, MCHIP_ACT_GELU = 1, MCHIP_ACT_SWIGLU = 2, MCHIP_ACT_NONE = 3 };
/* 32-bit sums of products of bytes: 128^2 k < 2^31. */
enum { MCHIP_I8_MAX_K = 131071 };

/* C[m, n] = act(A B^T scaled by row and column + bias), in c_dtype. SwiGLU:
 * B and bias have 2 n rows, gates first. */
int mchip_launch_matmul_i8(const void* a_codes, const float* a_scales, const void* b_codes, const float* b_scales,
                           const float* bias, int activation, int c_dtype, void* c, int m, int n, int k, void* stream,
                           const char** why);

enum { MCHIP_ROUTE_SOFTMAX = 0, MCHIP_ROUTE_SIGMOID = 1 };
enum { MCHIP_ROUTE_MAX_EXPERTS = 512, MCHIP_ROUTE_MAX_TOP_K = 16, MCHIP_ROUTE_MAX_GROUPS = 64 };

typedef struct mchip_route_args {
    int dtype; /* of logits */
    const void* logits;
    long long ld;
    const float* bias; /* [experts] or null */
    int tokens, experts, top_k, score, groups, top_groups, group_best, normalize;
    float scale;
    int* chosen;  /* [tokens, top_k] */
    float* gates; /* [tokens, top_k] */
    int* order;   /* [tokens * top_k] or null */
    int* offsets; /* [experts + 1] or null */
    void* workspace;
} mchip_route_args;

long long mchip_route_workspace_bytes(int tokens, int experts, int top_k);
int mchip_launch_route(const mchip_route_args* args, void* stream, const char** why);

/* The experts' products on a plan (order, offsets as mchip_launch_route
 * writes them). Up: C[slot, n] = act(x[order[slot] / top_k] W_e^T + b_e).
 * Down: y[token, n] = sum over its pairs of gate (h[slot] W_e^T + b_e). */
typedef struct mchip_experts_args {
    const void* a_codes; /* up: [tokens, kp]; down: [tokens * top_k, kp] */
    const float* a_scales;
    const void* w_codes; /* [experts, n (up with SwiGLU: 2 n), kp] */
    const float* w_scales;
    const float* bias; /* [experts, n (2 n)] or null */
    int activation, c_dtype;
    void* c;
    const int* order;
    const int* offsets;
    const float* gates; /* down */
    int tokens, top_k, experts, n, k;
    void* workspace; /* down */
} mchip_experts_args;

int mchip_launch_experts_up_i8(const mchip_experts_args* args, void* stream, const char** why);

/* The kernel that a product of these sizes runs on a chip of cu_count CUs, for the
 * tests: blocks or tiles of rows x columns; -1: none, one launch is too small. *halves: how many of the last 256x256
 * tiles run as two of 128 rows. */
enum {
    MCHIP_I8_BLOCKS_16X32 = 0,
    MCHIP_I8_BLOCKS_32X32 = 1,
    MCHIP_I8_BLOCKS_32X64 = 2,
    MCHIP_I8_TILES_128 = 3,
    MCHIP_I8_TILES_256 = 4,
    MCHIP_I8_TILES_FAR = 5 /* as 256x256, gathered from 2 GiB of A or more */
};
int mchip_matmul_i8_plan(int activation, int m, int n, int k, int cu_count, int* halves);
int mchip_experts_i8_plan(int down, int activation, int tokens, int top_k, int experts, int n, int k, int cu_count);
long long mchip_experts_down_i8_workspace_bytes(int c_dtype, int tokens, int top_k, int n, int k);
int mchip_launch_experts_down_i8(const mchip_experts_args* args, void* stream, const char** why);

#ifdef __cplusplus
}
#endif

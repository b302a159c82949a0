// What the 8-bit integer kernels share.
//
// v_mfma_i32_16x16x64_i8: lane l supplies row (A) or column (B) l % 16, bytes
// 16 (l / 16) .. + 15 of the 64-wide step in four registers; products and sums
// are exact 32-bit integers. Value v of lane l of the result is row
// 4 (l / 16) + v, column l % 16: issued with the C column's operand first, a lane
// has four consecutive columns of one row of C.
#pragma once

#include "i8.h"
#include "mx4_device.h"

namespace i8 {

using namespace mx4;

constexpr int kLine = 128;  // a row's codes are padded to a multiple of it

__host__ __device__ inline int padded_k(int k) { return (k + kLine - 1) / kLine * kLine; }

__device__ __forceinline__ i32x4 mfma(i32x4 a, i32x4 b, i32x4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// x sigmoid(x), and GELU in its tanh form, u (1 + tanh(z)) / 2 = u sigmoid(2 z).
__device__ __forceinline__ float sigmoid(float u) { return 1.0f / (1.0f + __expf(-u)); }
__device__ __forceinline__ float gelu(float u) {
    return u * sigmoid(1.5957691216057308f * (u + 0.044715f * u * u * u));
}
__device__ __forceinline__ float activate(float u, int act) {
    if (act == MCHIP_ACT_RELU) return u < 0.0f ? 0.0f : u;  // a NaN stays one
    if (act == MCHIP_ACT_GELU) return gelu(u);
    return u;
}

// As store_four, the type known at run time.
__device__ __forceinline__ void store_four_as(int dtype, void* c, long long at, f32x4 v, int left) {
    if (dtype == kF32) store_four<kF32>(c, at, v, left);
    else if (dtype == kBf16) store_four<kBf16>(c, at, v, left);
    else store_four<kF16>(c, at, v, left);
}

}  // namespace i8

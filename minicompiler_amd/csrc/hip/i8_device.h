// What the 8-bit integer kernels share.
//
// v_mfma_i32_16x16x64_i8: lane l supplies row (A) or column (B) l % 16, bytes
// 16 (l / 16) .. + 15 of the 64-wide step in four registers; products and sums
// are exact 32-bit integers. Value v of lane l of the result is row
// 4 (l / 16) + v, column l % 16: issued with the C column's operand first, a lane
// has four consecutive columns of one row of C. v_mfma_i32_32x32x32_i8: row or
// column l % 32, bytes 16 (l / 32) .. + 15 of the 32-wide step; value v of the result
// is row 8 (v / 4) + 4 (l / 32) + v % 4, column l % 32.
#pragma once

#include "i8.h"
#include "mx4_device.h"

namespace i8 {

using namespace mx4;

typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int kLine = 128;  // a row's codes are padded to a multiple of it

__host__ __device__ inline int padded_k(int k) { return (k + kLine - 1) / kLine * kLine; }

__device__ __forceinline__ i32x4 mfma(i32x4 a, i32x4 b, i32x4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// A row's scale for sum x s x (a column's scale) x back, of which no part leaves fp32's range unless the
// whole does: rows of numbers past 2^97 have scales with which a sum of up to 2^31 alone would. What
// is taken times 2^-64 stays above 2^26, so that no column's scale (2^-149 at least) makes it subnormal.
struct RowScale {
    float s, back;
};
__device__ __forceinline__ RowScale row_scale(float s) {
    const bool far = __builtin_fabsf(s) >= 0x1p90f;
    return {far ? s * 0x1p-64f : s, far ? 0x1p64f : 1.0f};
}

// Between one lane's writes to LDS and another's reads of the same wave, or back. The hardware
// keeps a wave's LDS accesses in order; the compiler, which sees one lane, is held to it here.
__device__ __forceinline__ void wave_lds_order() {
    __builtin_amdgcn_wave_barrier();
    asm volatile("" ::: "memory");
}

// GELU in its tanh form is u (1 + tanh(z)) / 2 = u sigmoid(2 z). The reciprocal is good
// to a unit in the last place; a division would be ten instructions.
__device__ __forceinline__ float sigmoid(float u) { return __builtin_amdgcn_rcpf(1.0f + __expf(-u)); }
__device__ __forceinline__ float gelu(float u) {
    return u * sigmoid(1.5957691216057308f * (u + 0.044715f * u * u * u));
}
__device__ __forceinline__ float activate(float u, int act) {
    if (act == MCHIP_ACT_RELU) return u < 0.0f ? 0.0f : u;  // a NaN stays one
    if (act == MCHIP_ACT_GELU) return gelu(u);
    return u;
}

// Eight consecutive elements of which the first `left` are there; kPast: past the caches
// (a large result: 4096x4096 bf16 sums of one step in 14.6 us, 16.8 with plain stores).
template <int kType, bool kPast = true>
__device__ __forceinline__ void store_eight(void* c, long long at, const float (&v)[8], int left) {
    if (left >= 8) {
        if constexpr (kType == kF32) {
            f32x4_loose* d = reinterpret_cast<f32x4_loose*>(static_cast<float*>(c) + at);
            const f32x4 lo = {v[0], v[1], v[2], v[3]}, hi = {v[4], v[5], v[6], v[7]};
            if constexpr (kPast) {
                __builtin_nontemporal_store(lo, d);
                __builtin_nontemporal_store(hi, d + 1);
            } else {
                d[0] = lo, d[1] = hi;
            }
        } else {
            u16x8 h;
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] = to_16<kType>(v[e]);
            u16x8_loose* d = reinterpret_cast<u16x8_loose*>(static_cast<unsigned short*>(c) + at);
            if constexpr (kPast) __builtin_nontemporal_store(h, d);
            else *d = h;
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < left) store_one<kType>(c, at + e, v[e]);
}

// As store_four, the type known at run time.
__device__ __forceinline__ void store_four_as(int dtype, void* c, long long at, f32x4 v, int left) {
    if (dtype == kF32) store_four<kF32>(c, at, v, left);
    else if (dtype == kBf16) store_four<kBf16>(c, at, v, left);
    else store_four<kF16>(c, at, v, left);
}

}  // namespace i8

// What the microscaled 4-bit kernels share: types, the matrix instruction on
// two quantised operands, exact conversions, loads and stores with edges.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 on e2m1 operands: lane l supplies row (A)
// or column (B) l % 16, elements 32 (l / 16) .. + 31 of the 128-wide step in
// its first four registers (16 bytes, as they lie in the codes), and that
// block's scale in the low byte of a register of its own. Products and scales
// are exact, sums fp32, scale 255 gives NaN. Value v of lane l of the result is
// row 4 (l / 16) + v, column l % 16: issued with the C column's operand first,
// a lane has four consecutive columns of one row of C.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstddef>
#include <cstdint>
#include <tuple>

#include "mx4.h"

namespace mx4 {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kStep = 128;  // elements of k per matrix instruction
constexpr int kF32 = MCHIP_DTYPE_F32, kBf16 = MCHIP_DTYPE_BF16, kF16 = MCHIP_DTYPE_F16, kMx4 = MCHIP_DTYPE_MX4;

template <int kType>
constexpr int kSize = kType == kF32 ? 4 : 2;

// kByte: which byte of the scale registers.
template <int kByte = 0>
__device__ __forceinline__ f32x4 mfma(i32x4 a, int sa, i32x4 b, int sb, f32x4 c) {
    const i32x8 a8 = {a[0], a[1], a[2], a[3], 0, 0, 0, 0};
    const i32x8 b8 = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a8, b8, c, 4, 4, kByte, sa, kByte, sb);
}

__device__ __forceinline__ f32x4 mfma_bf16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
}

__device__ __forceinline__ f32x4 mfma_f16(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
}

// A 16-bit value, or an fp32 one, as fp32 (exact).
template <int kType>
__device__ __forceinline__ float to_f32(unsigned bits) {
    if constexpr (kType == kF32) return __builtin_bit_cast(float, bits);
    if constexpr (kType == kBf16) return __builtin_bit_cast(float, bits << 16);
    return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<unsigned short>(bits)));
}

// fp32 rounded once (to nearest even) to the stored type.
template <int kType>
__device__ __forceinline__ unsigned short to_16(float v) {
    if constexpr (kType == kBf16) return __builtin_bit_cast(unsigned short, static_cast<__bf16>(v));
    return __builtin_bit_cast(unsigned short, static_cast<_Float16>(v));
}

template <int kType>
__device__ __forceinline__ float load_one(const void* p, long long i) {
    if constexpr (kType == kF32) return static_cast<const float*>(p)[i];
    return to_f32<kType>(static_cast<const unsigned short*>(p)[i]);
}

template <int kType>
__device__ __forceinline__ void store_one(void* p, long long i, float v) {
    if constexpr (kType == kF32)
        static_cast<float*>(p)[i] = v;
    else
        static_cast<unsigned short*>(p)[i] = to_16<kType>(v);
}

// Vectors at any address of their elements (one load all the same).
typedef f32x4 f32x4_loose __attribute__((aligned(4)));
typedef u16x8 u16x8_loose __attribute__((aligned(2)));
typedef u32x4 u32x4_loose __attribute__((aligned(2)));
typedef u32x4 u32x4_dwords __attribute__((aligned(4)));
typedef u16x4 u16x4_loose __attribute__((aligned(2)));
typedef unsigned u32_loose __attribute__((aligned(2)));

// The first `left` of four consecutive elements of a row of C at element `at`.
template <int kType>
__device__ __forceinline__ void store_four(void* c, long long at, f32x4 v, int left) {
    if (left >= 4) {
        if constexpr (kType == kF32) {
            *reinterpret_cast<f32x4_loose*>(static_cast<float*>(c) + at) = v;
        } else {
            u16x4 h;
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = to_16<kType>(v[e]);
            *reinterpret_cast<u16x4_loose*>(static_cast<unsigned short*>(c) + at) = h;
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (e < left) store_one<kType>(c, at + e, v[e]);
}

// Eight consecutive elements from element `at` as fp32, zeros from `left` on.
template <int kType>
__device__ __forceinline__ void load_eight(const void* p, long long at, int left, float (&v)[8]) {
    if (left >= 8) {
        if constexpr (kType == kF32) {
            const f32x4_loose* s = reinterpret_cast<const f32x4_loose*>(static_cast<const float*>(p) + at);
            const f32x4 lo = s[0], hi = s[1];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[e] = lo[e];
                v[4 + e] = hi[e];
            }
        } else {
            const u16x8 s = *reinterpret_cast<const u16x8_loose*>(static_cast<const unsigned short*>(p) + at);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = to_f32<kType>(s[e]);
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < left ? load_one<kType>(p, at + e) : 0.0f;
}

// Four.
template <int kType>
__device__ __forceinline__ f32x4 load_four(const void* p, long long at, int left) {
    f32x4 v;
    if (left >= 4) {
        if constexpr (kType == kF32) return *reinterpret_cast<const f32x4_loose*>(static_cast<const float*>(p) + at);
        const u16x4 s = *reinterpret_cast<const u16x4_loose*>(static_cast<const unsigned short*>(p) + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = to_f32<kType>(s[e]);
        return v;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = e < left ? load_one<kType>(p, at + e) : 0.0f;
    return v;
}

// Reductions over the 64 lanes, the result in every lane (as a scalar).
__device__ __forceinline__ unsigned wave_max(unsigned v) {
#define MX4_STEP(ctrl, rows)                                                                                     \
    {                                                                                                            \
        const unsigned o =                                                                                       \
            static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), ctrl, rows, 0xf, false)); \
        v = v > o ? v : o;                                                                                       \
    }
    MX4_STEP(0x111, 0xf) MX4_STEP(0x112, 0xf) MX4_STEP(0x114, 0xf) MX4_STEP(0x118, 0xf)
    MX4_STEP(0x142, 0xa) MX4_STEP(0x143, 0xc)
#undef MX4_STEP
    return static_cast<unsigned>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
}
__device__ __forceinline__ unsigned wave_min(unsigned v) { return ~wave_max(~v); }
__device__ __forceinline__ float wave_sum(float v) {
#define MX4_STEP(ctrl, rows) \
    v += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl, rows, 0xf, false));
    MX4_STEP(0x111, 0xf) MX4_STEP(0x112, 0xf) MX4_STEP(0x114, 0xf) MX4_STEP(0x118, 0xf)
    MX4_STEP(0x142, 0xa) MX4_STEP(0x143, 0xc)
#undef MX4_STEP
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// The high halves of two registers in one (a: low half).
__device__ __forceinline__ unsigned high_halves(float a, float b) {
    return __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, b), __builtin_bit_cast(unsigned, a), 0x07060302u);
}

// An fp32 value as a sum of bf16 pieces, each the leading 8 bits of what is
// left: one piece holds a bf16 exactly, two an fp16, three an fp32 (24 bits) from
// 2^-110 up, below that its multiple of 2^-133, the smallest bf16. Cutting,
// unlike rounding, never overflows; an infinity is its first piece, the others
// zeros (which an infinite other operand turns into NaN).
template <int kPieces>
__device__ __forceinline__ void cut(float v, float (&piece)[kPieces]) {
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
        piece[p] = v;
        if (p + 1 == kPieces) break;
        const float head = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, v) & 0xffff0000u);
        v = __builtin_fabsf(v) == __builtin_inff() ? 0.0f : v - head;
    }
}

// Eight fp32 values as kPieces operands of the bf16 matrix instruction.
template <int kPieces>
__device__ __forceinline__ void cut_eight(const float (&v)[8], u32x4 (&out)[kPieces]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float a[kPieces], b[kPieces];
        cut<kPieces>(v[2 * j], a);
        cut<kPieces>(v[2 * j + 1], b);
#pragma unroll
        for (int p = 0; p < kPieces; ++p) out[p][j] = high_halves(a[p], b[p]);
    }
}

template <int kType>
constexpr int kPieces = kType == kBf16 ? 1 : kType == kF16 ? 2 : 3;

// Eight codes (a dword) with their block's scale as the bf16 matrix
// instruction's operand: exact, two significant bits, subnormal ones too; an
// infinity past fp32's range (codes from 4 up at byte 253, from 2 up at 254).
__device__ __forceinline__ u32x4 decode_eight(unsigned codes, float scale) {
    u32x4 r;
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
    r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
    r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
    return r;
}

// Without it, as the fp16 one's.
__device__ __forceinline__ u32x4 decode_eight_f16(unsigned codes) {
    u32x4 r;
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.0f, 0));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.0f, 1));
    r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.0f, 2));
    r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.0f, 3));
    return r;
}

// The scale as the conversions take it: an fp32 whose exponent field is the
// scale byte (they read no more of it; field 0 counts as 2^-127, 255 as NaN).
__device__ __forceinline__ float scale_operand(unsigned byte) { return __builtin_bit_cast(float, byte << 23); }

#define MX4_LDS __attribute__((address_space(3)))

// 16 bytes per lane from memory to LDS without registers, lane l at dst + 16 l.
__device__ __forceinline__ void buffer_to_lds(__amdgpu_buffer_rsrc_t rsrc, MX4_LDS unsigned char* dst, int voffset,
                                              int soffset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, reinterpret_cast<MX4_LDS void*>(dst), 16, voffset, soffset, 0, 0);
}

// A workgroup barrier without a memory fence (which would wait for fetches in
// flight), which nothing is moved across.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// The partial sums of a block's waves (each kCount vectors per lane) added up in
// wave order, vector i by wave i % kWaves, which hands it to take(i, sum): short
// code, and all waves store. `space`: kWaves * kCount * 64 vectors.
template <int kWaves, int kCount, typename Take>
__device__ __forceinline__ void sum_waves(const f32x4 (&acc)[kCount], f32x4* space, int wave, int lane, Take take) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) space[(wave * kCount + i) * 64 + lane] = acc[i];
    __syncthreads();
#pragma unroll 1
    for (int i = wave; i < kCount; i += kWaves) {
        f32x4 sum = space[i * 64 + lane];
#pragma unroll
        for (int v = 1; v < kWaves; ++v) sum += space[(v * kCount + i) * 64 + lane];
        take(i, sum);
    }
}

inline bool aligned(const void* p, std::size_t to) { return reinterpret_cast<std::uintptr_t>(p) % to == 0; }
inline std::size_t size_of(int dtype) { return dtype == MCHIP_DTYPE_F32 ? 4 : 2; }
inline bool is_float_type(int dtype) {
    return dtype == MCHIP_DTYPE_F32 || dtype == MCHIP_DTYPE_BF16 || dtype == MCHIP_DTYPE_F16;
}

// A launch takes fewer than 2^32 threads along a dimension of its grid.
inline bool fits_launch(long long blocks, int threads) { return blocks < (1LL << 32) / threads; }

// A launch's own status (hipGetLastError() would report, and take away, what an
// earlier call of the program left behind).
template <typename... Params, typename... Args>
inline int launch_kernel(void (*kernel)(Params...), dim3 grid, unsigned threads, std::size_t lds, hipStream_t stream,
                         Args... args) {
    std::tuple<Params...> values(static_cast<Params>(args)...);
    return std::apply(
        [&](auto&... value) {
            void* list[] = {const_cast<void*>(static_cast<const volatile void*>(&value))...};
            return hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, dim3(threads), list, lds, stream);
        },
        values);
}

// CUs of the current device, asked once per device.
inline int device_cus() {
    static std::atomic<int> cache[64];
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
    int cus = cache[dev].load(std::memory_order_relaxed);
    if (cus > 0) return cus;
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || cus < 1) return 256;
    cache[dev].store(cus, std::memory_order_relaxed);
    return cus;
}

}  // namespace mx4

// Quantisation to microscaled 4-bit floats (the format: mx4.h).
//
// A block of 32 with largest magnitude a: s = max(0, floor(log2 a) - 2 + 127),
// which puts a in [4, 8) of the codes' units (6 is the largest code); each
// element is then x 2^(127 - s), rounded to the nearest code, ties to the even
// code, 6 beyond it. floor(log2 a) is read from the exponent field, so fields
// 0 to 2 (where 2^(s - 127) would pass below the smallest scale) take s = 0.
// A block with an infinity or a NaN has no scale: 255, codes 0, NaN as a whole.
// v_cvt_scalef32_pk_fp4_f32 divides, rounds and saturates so in one step.
//
// Bound by memory: 2 or 4 bytes read and 17/32 written per element (and 2 or 4
// written for `values`, past the caches: the codes are what is read next). By
// rows 8192x2048 fp32 with values in 24.8 us (5.8 TB/s; 28.6 with plain stores),
// codes and scales alone 12.0 (6.3); 4096x14336 bf16 44 us (6.0) and 30.0 (4.9); one
// row of 4096 1.5 us: a launch.

#include <type_traits>

#include "mx4_device.h"

namespace {

using namespace mx4;

// The scale byte of a block from the bits of its largest magnitude (as
// unsigned numbers, infinities and NaNs are above all others).
__device__ __forceinline__ unsigned scale_byte(unsigned top) {
    if (top >= 0x7f800000u) return 255u;
    const int s = static_cast<int>(top >> 23) - 2;
    return static_cast<unsigned>(s > 0 ? s : 0);
}

__device__ __forceinline__ unsigned magnitude(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }

// Eight codes of one block, four bytes.
__device__ __forceinline__ unsigned encode_eight(const float (&v)[8], unsigned scale) {
    if (scale == 255u) return 0u;
    const float f = scale_operand(scale);
    unsigned c = 0;
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], f, 0);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], f, 1);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], f, 2);
    c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], f, 3);
    return c;
}

__device__ __forceinline__ void decode_eight_f32(unsigned codes, unsigned scale, float (&v)[8]) {
    const float f = scale_operand(scale);
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, f, 0);
    const f32x2 b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, f, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, f, 2);
    const f32x2 d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, f, 3);
    v[0] = a[0], v[1] = a[1], v[2] = b[0], v[3] = b[1];
    v[4] = c[0], v[5] = c[1], v[6] = d[0], v[7] = d[1];
}

// Eight values of row `row` from element `at` on (exact in x's type: a code is
// never finer than the numbers it was rounded from).
template <int kType>
__device__ __forceinline__ void store_eight(void* p, long long at, const float (&v)[8], int left) {
    if (left >= 8) {
        if constexpr (kType == kF32) {
            f32x4_loose* d = reinterpret_cast<f32x4_loose*>(static_cast<float*>(p) + at);
            const f32x4 lo = {v[0], v[1], v[2], v[3]}, hi = {v[4], v[5], v[6], v[7]};
            __builtin_nontemporal_store(lo, d);
            __builtin_nontemporal_store(hi, d + 1);
        } else {
            u16x8 h;
#pragma unroll
            for (int e = 0; e < 8; ++e) h[e] = to_16<kType>(v[e]);
            __builtin_nontemporal_store(h, reinterpret_cast<u16x8_loose*>(static_cast<unsigned short*>(p) + at));
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (e < left) store_one<kType>(p, at + e, v[e]);
}

constexpr int kThreads = 256;

// The largest over the four lanes of a block (lanes 4 i .. 4 i + 3).
__device__ __forceinline__ unsigned max_of_four(unsigned v) {
    unsigned o = static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0xb1, 0xf, 0xf, false));
    v = v > o ? v : o;
    o = static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x4e, 0xf, 0xf, false));
    return v > o ? v : o;
}

// A lane takes eight consecutive elements of a row, four neighbouring lanes a
// block. `per_row` = kp / 8 such chunks (a multiple of 16, so a block's lanes
// are never in two rows), chunks counted over all rows.
template <int kType>
__global__ __launch_bounds__(kThreads) void quantize_rows(const void* __restrict__ x, long long ld,
                                                          unsigned* __restrict__ codes,
                                                          unsigned char* __restrict__ scales,
                                                          void* __restrict__ values, long long rows, int k,
                                                          unsigned per_row) {
    const long long first = static_cast<long long>(blockIdx.x) * kThreads;
    const long long row0 = first / per_row;
    const unsigned in_row = static_cast<unsigned>(first - row0 * per_row) + threadIdx.x;
    const long long row = row0 + in_row / per_row;
    const unsigned chunk = in_row % per_row;
    if (row >= rows) return;  // whole blocks of lanes: a row has a multiple of 16 chunks
    const int left = k - static_cast<int>(chunk) * 8;
    float v[8];
    load_eight<kType>(x, row * ld + chunk * 8, left, v);
    unsigned top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const unsigned m = magnitude(v[e]);
        top = m > top ? m : top;
    }
    const unsigned s = scale_byte(max_of_four(top));
    const unsigned c = encode_eight(v, s);
    codes[row * per_row + chunk] = c;
    if (chunk % 4 == 0) scales[row * (per_row / 4) + chunk / 4] = static_cast<unsigned char>(s);
    if (values != nullptr && left > 0) {
        decode_eight_f32(c, s, v);
        store_eight<kType>(values, row * k + chunk * 8, v, left);
    }
}

// A lane takes eight elements down kPer neighbouring columns, the lanes 16 q + r,
// q = 0..3, a block of them; a wave 16 kPer columns, a thread block 64 kPer
// (whole lines of 16-bit rows) of four blocks of k (a step, 64 bytes of codes per
// column). Rows past k are read as the last one and count as zeros. Code is
// short, since a launch meets a cold instruction cache (32 elements per lane,
// 5.5 KB of code: 1001x2047 fp16 in 6.9 us, so in 4.4). With values 4096x4096
// fp32 25 us (5.8 TB/s; 37 with plain stores), 4096x14336 bf16 74 us (3.6 TB/s:
// codes come in pieces of 4 bytes, 64 to a column and block); codes and scales
// alone 13.6 and 46. Loads past the caches took 92: a line of x is read by several
// lanes' loads.
constexpr int kColumnThreads = 1024;

template <int kType, int kPer>
__global__ __launch_bounds__(kColumnThreads) void quantize_columns(const void* __restrict__ w, long long ld,
                                                                   unsigned* __restrict__ codes,
                                                                   unsigned char* __restrict__ scales,
                                                                   void* __restrict__ values, int k, int n,
                                                                   int k_blocks) {
    typedef std::conditional_t<kType == kF32, float, unsigned short> Element;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, q = lane / 16;
    // Blocks go to the XCDs in turn; consecutive steps of one, so that its L2 joins
    // their pieces of a line of codes or scales.
    const unsigned block = blockIdx.y * gridDim.x + blockIdx.x, all = gridDim.x * gridDim.y;
    const unsigned mine = block % 8 * (all / 8) + block / 8, at_block = block < all / 8 * 8 ? mine : block;
    const int col = static_cast<int>(at_block / gridDim.x) * 64 * kPer + (wave % 4 * 16 + lane % 16) * kPer;
    const int kb = static_cast<int>(at_block % gridDim.x) * 4 + wave / 4;
    const int k0 = kb * 32 + q * 8, last = k - 1;
    const bool has = col < n;
    const Element* at = static_cast<const Element*>(w) + (has ? col : n - kPer);
    float v[kPer][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const Element* row = at + (k0 + e < last ? k0 + e : last) * ld;
        if constexpr (kPer == 1) {
            v[0][e] = load_one<kType>(row, 0);
        } else {
            const unsigned two = *reinterpret_cast<const u32_loose*>(row);
            v[0][e] = to_f32<kType>(two & 0xffffu);
            v[1][e] = to_f32<kType>(two >> 16);
        }
    }
    unsigned c[kPer], s[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        unsigned top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            v[j][e] = k0 + e < k ? v[j][e] : 0.0f;
            const unsigned m = magnitude(v[j][e]);
            top = m > top ? m : top;
        }
        u32x2 other = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(top, top, false, false));
        top = other[0] > other[1] ? other[0] : other[1];
        other = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(top, top, false, false));
        s[j] = scale_byte(other[0] > other[1] ? other[0] : other[1]);
        c[j] = encode_eight(v[j], s[j]);
    }
    if (!has) return;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        codes[(static_cast<long long>(col + j) * k_blocks + kb) * 4 + q] = c[j];
        if (q == 0) scales[static_cast<long long>(col + j) * k_blocks + kb] = static_cast<unsigned char>(s[j]);
    }
    if (values == nullptr) return;
    Element* to = static_cast<Element*>(values) + col;
#pragma unroll
    for (int j = 0; j < kPer; ++j) decode_eight_f32(c[j], s[j], v[j]);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if (k0 + e >= k) continue;
        Element* row = to + static_cast<long long>(k0 + e) * n;
        if constexpr (kType == kF32)
            __builtin_nontemporal_store(v[0][e], row);
        else if constexpr (kPer == 1)
            __builtin_nontemporal_store(to_16<kType>(v[0][e]), row);
        else
            __builtin_nontemporal_store(to_16<kType>(v[0][e]) | static_cast<unsigned>(to_16<kType>(v[1][e])) << 16,
                                        reinterpret_cast<u32_loose*>(row));
    }
}

const char* refusal(int dtype, const void* x, long long ld, const void* codes, const void* scales, int outer, int inner,
                    int k, const void* values) {
    if (!is_float_type(dtype)) return "the type is none of fp32 (0), bf16 (1), fp16 (2)";
    if (outer < 1 || inner < 1) return "a size below 1";
    if (k > 0x7fffff80) return "k above 2^31 - 128";
    if (ld < inner) return "rows closer together than they are long";
    if (x == nullptr || codes == nullptr || scales == nullptr) return "a null input or output";
    const std::size_t size = size_of(dtype);
    if (!aligned(x, size) || !aligned(values, size)) return "an address that is no multiple of its element's size";
    if (!aligned(codes, 16) || !aligned(scales, 4)) return "codes not 16-byte or scales not 4-byte aligned";
    return nullptr;
}

// `elements` of x's type from p on (or null).
template <int kType>
const void* offset(const void* p, long long elements) {
    return p == nullptr ? nullptr : static_cast<const unsigned char*>(p) + elements * kSize<kType>;
}
template <int kType>
void* offset(void* p, long long elements) {
    return const_cast<void*>(offset<kType>(static_cast<const void*>(p), elements));
}

// As many rows at a time as a launch takes.
template <int kType>
int launch_rows(const void* x, long long ld, void* codes, void* scales, int rows, int k, void* values,
                hipStream_t stream) {
    const unsigned per_row = static_cast<unsigned>(mchip_mx4_k(k) / 8);
    const long long most = ((1LL << 32) - kThreads) / per_row;
    for (long long from = 0; from < rows; from += most) {
        const long long count = std::min(most, rows - from);
        const unsigned blocks = static_cast<unsigned>((count * per_row + kThreads - 1) / kThreads);
        const int rc = launch_kernel(quantize_rows<kType>, blocks, kThreads, 0, stream, offset<kType>(x, from * ld), ld,
                                     static_cast<unsigned*>(codes) + from * per_row,
                                     static_cast<unsigned char*>(scales) + from * (per_row / 4),
                                     offset<kType>(values, from * k), count, k, per_row);
        if (rc != hipSuccess) return rc;
    }
    return hipSuccess;
}

// As much of k at a time as a launch takes.
template <int kType>
int launch_columns(const void* w, long long ld, void* codes, void* scales, int k, int n, void* values,
                   hipStream_t stream, const char** why) {
    const int k_blocks = static_cast<int>(mchip_mx4_k(k) / 32), most = (1 << 22) - 1;  // steps
    const auto go = [&](auto kernel, int per) {
        const unsigned cols = static_cast<unsigned>((static_cast<long long>(n) + 64 * per - 1) / (64 * per));
        if (cols > 65535u) {
            *why = per == 2 ? "more columns than one launch takes in pairs (8388480)"
                            : "more columns than one launch takes (4194240)";
            return static_cast<int>(hipErrorInvalidValue);
        }
        for (int step = 0; step < k_blocks / 4; step += most) {
            const int steps = std::min(most, k_blocks / 4 - step), from = step * kStep;
            const int rc = launch_kernel(kernel, dim3(static_cast<unsigned>(steps), cols), kColumnThreads, 0, stream,
                                         offset<kType>(w, from * ld), ld, static_cast<unsigned*>(codes) + step * 16LL,
                                         static_cast<unsigned char*>(scales) + step * 4LL,
                                         offset<kType>(values, static_cast<long long>(from) * n), k - from, n, k_blocks);
            if (rc != hipSuccess) return rc;
        }
        return static_cast<int>(hipSuccess);
    };
    if constexpr (kType != kF32) {
        // Two columns to a lane load dwords (4096x14336 bf16 with values: 74 us, 80 by one).
        if (n % 2 == 0) return go(quantize_columns<kType, 2>, 2);
    }
    return go(quantize_columns<kType, 1>, 1);
}

}  // namespace

extern "C" {

long long mchip_mx4_k(int k) { return (static_cast<long long>(k) + mx4::kStep - 1) / mx4::kStep * mx4::kStep; }

int mchip_quantize_mx4(int dtype, const void* x, long long ld, void* codes, void* scales, int rows, int k, void* values,
                       void* stream, const char** why) {
    *why = refusal(dtype, x, ld, codes, scales, rows, k, k, values);
    if (*why != nullptr) return hipErrorInvalidValue;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == kF32) return launch_rows<kF32>(x, ld, codes, scales, rows, k, values, s);
    if (dtype == kBf16) return launch_rows<kBf16>(x, ld, codes, scales, rows, k, values, s);
    return launch_rows<kF16>(x, ld, codes, scales, rows, k, values, s);
}

int mchip_quantize_mx4_columns(int dtype, const void* w, long long ld, void* codes, void* scales, int k, int n,
                               void* values, void* stream, const char** why) {
    *why = refusal(dtype, w, ld, codes, scales, k, n, k, values);
    if (*why != nullptr) return hipErrorInvalidValue;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == kF32) return launch_columns<kF32>(w, ld, codes, scales, k, n, values, s, why);
    if (dtype == kBf16) return launch_columns<kBf16>(w, ld, codes, scales, k, n, values, s, why);
    return launch_columns<kF16>(w, ld, codes, scales, k, n, values, s, why);
}

}  // extern "C"

// Quantisation to 8-bit integers with a scale per row (the format: i8.h).
//
// A row with largest magnitude a has the scale s = a / 127, rounded to fp32, and
// each code is the exact quotient x / s rounded to the nearest integer, ties to
// the even one: n = rint(x (1 / s)) is off by one at most, and next to a half
// only; r = x - n s is exact in one fma (a multiple of the finer of two ulps that
// is at most s), so comparing 2 r with s decides. Rows whose scale would be near
// or below the smallest normal number are first taken times 2^64, exactly. A row
// with an infinity or a NaN has the scale NaN and codes 0.

#include "i8_device.h"

namespace {

using namespace i8;

constexpr int kThreads = 256;

struct Scale {
    float s;       // as stored
    float up;      // a power of two that keeps what follows normal
    float big;     // s x up
    float inverse; // 1 / big, 0 where codes are 0
};

// top: the bits of the row's largest magnitude (infinities and NaNs are above all others).
__device__ __forceinline__ Scale scale_of(unsigned top) {
    Scale r;
    const float a = __builtin_bit_cast(float, top);
    r.s = top >= 0x7f800000u ? __builtin_nanf("") : a / 127.0f;
    r.up = r.s < 0x1p-100f ? 0x1p64f : 1.0f;
    r.big = r.s * r.up;
    r.inverse = r.s > 0.0f ? 1.0f / r.big : 0.0f;
    return r;
}

__device__ __forceinline__ int code_of(float x, const Scale& c) {
    // No number, or no scale: 0 (and an infinity times 0 would be no number).
    if (c.inverse == 0.0f || !(c.s == c.s)) return 0;
    x *= c.up;
    float n = __builtin_rintf(x * c.inverse);
    const float r = __builtin_fmaf(-n, c.big, x), twice = __builtin_fabsf(r) * 2.0f;
    const bool odd = (static_cast<int>(n) & 1) != 0;
    if (twice > c.big || (twice == c.big && odd)) n += r < 0.0f ? -1.0f : 1.0f;
    n = n > 127.0f ? 127.0f : n < -127.0f ? -127.0f : n;
    return static_cast<int>(n);
}

__device__ __forceinline__ unsigned magnitude(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }

__device__ __forceinline__ unsigned pack(int a, int b, int c, int d) {
    return static_cast<unsigned>(a & 255) | static_cast<unsigned>(b & 255) << 8 | static_cast<unsigned>(c & 255) << 16 |
           static_cast<unsigned>(d) << 24;
}

// What a code stands for. Both factors are exact; of a row without a scale, NaN.
__device__ __forceinline__ float value_of(int code, const Scale& c) { return static_cast<float>(code) * c.s; }

// A block takes a row, twice over.
template <int kType>
__global__ __launch_bounds__(kThreads) void quantize_rows(const void* __restrict__ x, long long ld,
                                                          unsigned* __restrict__ codes, float* __restrict__ scales,
                                                          void* __restrict__ values, int rows, int k, int dwords) {
    __shared__ unsigned tops[kThreads / 64];
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        unsigned top = 0;
        for (int i = threadIdx.x; i < dwords; i += kThreads) {
            const f32x4 v = load_four<kType>(x, row * ld + i * 4LL, k - i * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, magnitude(v[e]));
        }
        top = wave_max(top);
        if (threadIdx.x % 64 == 0) tops[threadIdx.x / 64] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kThreads / 64; ++w) top = max(top, tops[w]);
        const Scale c = scale_of(top);
        if (threadIdx.x == 0) scales[row] = c.s;
        for (int i = threadIdx.x; i < dwords; i += kThreads) {
            const f32x4 v = load_four<kType>(x, row * ld + i * 4LL, k - i * 4);
            int n[4];
            f32x4 back;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                n[e] = code_of(v[e], c);
                back[e] = value_of(n[e], c);
            }
            codes[row * dwords + i] = pack(n[0], n[1], n[2], n[3]);
            if (values != nullptr && i * 4 < k) store_four<kType>(values, row * k + i * 4LL, back, k - i * 4);
        }
        __syncthreads();
    }
}

// A block takes 64 columns, twice over, its waves every fourth dword of codes.
template <int kType>
__global__ __launch_bounds__(kThreads) void quantize_columns(const void* __restrict__ w, long long ld,
                                                             unsigned* __restrict__ codes, float* __restrict__ scales,
                                                             void* __restrict__ values, int k, int n, int dwords) {
    __shared__ unsigned tops[kThreads / 64][64];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const long long col = static_cast<long long>(blockIdx.x) * 64 + lane;
    const bool has = col < n;
    unsigned top = 0;
    for (int i = wave; has && i < k; i += kThreads / 64) top = max(top, magnitude(load_one<kType>(w, i * ld + col)));
    tops[wave][lane] = top;
    __syncthreads();
    if (!has) return;
#pragma unroll
    for (int v = 0; v < kThreads / 64; ++v) top = max(top, tops[v][lane]);
    const Scale c = scale_of(top);
    if (wave == 0) scales[col] = c.s;
    for (int i = wave; i < dwords; i += kThreads / 64) {
        int code[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            code[e] = 0;
            if (i * 4 + e < k) {
                code[e] = code_of(load_one<kType>(w, (i * 4LL + e) * ld + col), c);
                if (values != nullptr) store_one<kType>(values, (i * 4LL + e) * n + col, value_of(code[e], c));
            }
        }
        codes[col * dwords + i] = pack(code[0], code[1], code[2], code[3]);
    }
}

const char* refusal(int dtype, const void* x, long long ld, const void* codes, const float* scales, int outer, int inner,
                    int k, const void* values) {
    if (!is_float_type(dtype)) return "the type is none of fp32 (0), bf16 (1), fp16 (2)";
    if (outer < 1 || inner < 1) return "a size below 1";
    if (k > (1 << 28)) return "k above 2^28";
    if (ld < inner) return "rows closer together than they are long";
    if (x == nullptr || codes == nullptr || scales == nullptr) return "a null input or output";
    const std::size_t size = size_of(dtype);
    if (!aligned(x, size) || !aligned(values, size)) return "an address that is no multiple of its element's size";
    if (!aligned(codes, 16) || !aligned(scales, 4)) return "codes not 16-byte or scales not 4-byte aligned";
    return nullptr;
}

template <int kType>
int launch_rows(const void* x, long long ld, void* codes, float* scales, int rows, int k, void* values,
                hipStream_t stream) {
    const unsigned blocks = static_cast<unsigned>(std::min(rows, 1 << 20));
    return launch_kernel(quantize_rows<kType>, blocks, kThreads, 0, stream, x, ld, static_cast<unsigned*>(codes), scales,
                         values, rows, k, padded_k(k) / 4);
}

template <int kType>
int launch_columns(const void* w, long long ld, void* codes, float* scales, int k, int n, void* values,
                   hipStream_t stream, const char** why) {
    const long long blocks = (static_cast<long long>(n) + 63) / 64;
    if (!fits_launch(blocks, kThreads)) {
        *why = "more columns than one launch takes";
        return hipErrorInvalidValue;
    }
    return launch_kernel(quantize_columns<kType>, static_cast<unsigned>(blocks), kThreads, 0, stream, w, ld,
                         static_cast<unsigned*>(codes), scales, values, k, n, padded_k(k) / 4);
}

}  // namespace

extern "C" {

long long mchip_i8_k(int k) { return (static_cast<long long>(k) + i8::kLine - 1) / i8::kLine * i8::kLine; }

int mchip_quantize_i8(int dtype, const void* x, long long ld, void* codes, float* scales, int rows, int k, void* values,
                      void* stream, const char** why) {
    *why = refusal(dtype, x, ld, codes, scales, rows, k, k, values);
    if (*why != nullptr) return hipErrorInvalidValue;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == kF32) return launch_rows<kF32>(x, ld, codes, scales, rows, k, values, s);
    if (dtype == kBf16) return launch_rows<kBf16>(x, ld, codes, scales, rows, k, values, s);
    return launch_rows<kF16>(x, ld, codes, scales, rows, k, values, s);
}

int mchip_quantize_i8_columns(int dtype, const void* w, long long ld, void* codes, float* scales, int k, int n,
                              void* values, void* stream, const char** why) {
    *why = refusal(dtype, w, ld, codes, scales, k, n, k, values);
    if (*why != nullptr) return hipErrorInvalidValue;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == kF32) return launch_columns<kF32>(w, ld, codes, scales, k, n, values, s, why);
    if (dtype == kBf16) return launch_columns<kBf16>(w, ld, codes, scales, k, n, values, s, why);
    return launch_columns<kF16>(w, ld, codes, scales, k, n, values, s, why);
}

}  // extern "C"

// Quantisation to 8-bit integers with a scale per row (the format: i8.h).
//
// A row with largest magnitude a has the scale s = a / 127, rounded to fp32, and
// each code is the exact quotient x / s rounded to the nearest integer, ties to
// the even one: n = rint(x (1 / s)) is off by one at most, and next to a half
// only; r = x - n s is exact in one fma (a multiple of the finer of two ulps that
// is at most s), so comparing it with s / 2 decides. Rows whose scale would be near
// or below the smallest normal number are first taken times 2^64, exactly. A row
// with an infinity or a NaN has the scale NaN and codes 0.
//
// Bound by HBM, and for little by the launch. Numbers are read once and stay in registers
// between the largest magnitude and the codes: 8192x2048 fp32 with its values 28-29 us (151
// MB at 5.3 TB/s; 32.7 where a second pass reads again), 4096x14336 bf16 52 (5.65 TB/s),
// one row of 4096 4.3 (2.1 in the kernel). By columns too where a block holds them
// (1001x2047 fp16 7.6 us); taller ones are read twice, mostly from the last-level cache
// (k = 14336 by 1000 fp16 35 us; k = 4096 by 14336 bf16 101).

#include "i8_device.h"

namespace {

using namespace i8;

struct Scale {
    float s;        // as stored
    float up;       // a power of two that keeps what follows normal
    float big;      // s x up
    float inverse;  // 1 / big, 0 where codes are 0
    float past;     // the least number above big / 2
    bool none;      // no number
};

__device__ __forceinline__ Scale of_scale(float s) {
    Scale r;
    r.s = s;
    r.none = !(s == s);
    r.up = s < 0x1p-100f ? 0x1p64f : 1.0f;
    r.big = s * r.up;
    r.inverse = s > 0.0f ? 1.0f / r.big : 0.0f;
    r.past = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, 0.5f * r.big) + 1u);
    return r;
}

// top: the bits of the row's largest magnitude (infinities and NaNs are above all others).
__device__ __forceinline__ float scale_of(unsigned top) {
    return top >= 0x7f800000u ? __builtin_nanf("") : __builtin_bit_cast(float, top) / 127.0f;
}

// Of a row without a scale (0 or NaN) the caller passes zeros.
__device__ __forceinline__ int code_of(float x, const Scale& c) {
    x *= c.up;
    const float n = __builtin_rintf(x * c.inverse);
    const float r = __builtin_fmaf(-n, c.big, x);
    int code = static_cast<int>(n);
    // At a half exactly the even one is right, past it the next.
    const float most = __builtin_bit_cast(float, __builtin_bit_cast(unsigned, c.past) - (code & 1));
    if (__builtin_fabsf(r) >= most) code += r < 0.0f ? -1 : 1;
    // Past 127 only where the scale is no normal number and so rounded by much.
    return code > 127 ? 127 : code < -127 ? -127 : code;
}

__device__ __forceinline__ unsigned magnitude(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }

// The low bytes of four codes.
__device__ __forceinline__ unsigned pack(int a, int b, int c, int d) {
    const unsigned low = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), high = __builtin_amdgcn_perm(d, c, 0x0c0c0400u);
    return low | high << 16;
}

// Eight numbers to two dwords of codes; back: what they stand for (of a row without a scale, NaN).
__device__ __forceinline__ u32x2 codes_of(float (&v)[8], const Scale& c) {
    int n[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        n[e] = c.none || c.inverse == 0.0f ? 0 : code_of(v[e], c);
        v[e] = static_cast<float>(n[e]) * c.s;
    }
    return u32x2{pack(n[0], n[1], n[2], n[3]), pack(n[4], n[5], n[6], n[7])};
}

// The largest of a row over its kLanes lanes (a wave, or a block of waves).
template <int kLanes>
__device__ __forceinline__ unsigned row_max(unsigned top, unsigned* space) {
    top = wave_max(top);
    if constexpr (kLanes > 64) {
        if (threadIdx.x % 64 == 0) space[threadIdx.x / 64] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kLanes / 64; ++w) top = max(top, space[w]);
    }
    return top;
}

// Values go past the caches: the codes are what is read next.
// kLanes lanes take a row, each kPer chunks of eight elements, which stay in registers
// between the row's largest magnitude and the codes; a block of 256 lanes takes four
// rows of one wave each.
template <int kType, int kLanes, int kPer>
__global__ __launch_bounds__(kLanes < 256 ? 256 : kLanes) void quantize_rows(const void* __restrict__ x, long long ld,
                                                                            u32x2* __restrict__ codes,
                                                                            float* __restrict__ scales,
                                                                            void* __restrict__ values, int rows, int k,
                                                                            int chunks) {
    __shared__ unsigned space[kLanes / 64];
    constexpr int kRows = kLanes < 256 ? 256 / kLanes : 1;
    const long long row = static_cast<long long>(blockIdx.x) * kRows + threadIdx.x / kLanes;
    if (kRows > 1 && row >= rows) return;
    const int lane = threadIdx.x % kLanes;
    float v[kPer][8];
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) load_eight<kType>(x, row * ld + (lane + i * kLanes) * 8, k - (lane + i * kLanes) * 8, v[i]);
#pragma unroll
    for (int i = 0; i < kPer; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, magnitude(v[i][e]));
    const Scale c = of_scale(scale_of(row_max<kLanes>(top, space)));
    if (lane == 0) scales[row] = c.s;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int at = lane + i * kLanes;
        if (at >= chunks) break;
        codes[row * chunks + at] = codes_of(v[i], c);
        if (values != nullptr && at * 8 < k) store_eight<kType>(values, row * k + at * 8, v[i], k - at * 8);
    }
}

// Longer rows: a block a row, twice over.
constexpr int kLong = 1024;
template <int kType>
__global__ __launch_bounds__(kLong) void quantize_long_rows(const void* __restrict__ x, long long ld,
                                                            u32x2* __restrict__ codes, float* __restrict__ scales,
                                                            void* __restrict__ values, int k, int chunks) {
    __shared__ unsigned space[kLong / 64];
    const long long row = blockIdx.x;
    unsigned top = 0;
    float v[8];
    for (int at = threadIdx.x; at < chunks; at += kLong) {
        load_eight<kType>(x, row * ld + at * 8LL, k - at * 8, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, magnitude(v[e]));
    }
    const Scale c = of_scale(scale_of(row_max<kLong>(top, space)));
    if (threadIdx.x == 0) scales[row] = c.s;
    for (int at = threadIdx.x; at < chunks; at += kLong) {
        load_eight<kType>(x, row * ld + at * 8LL, k - at * 8, v);
        codes[row * chunks + at] = codes_of(v, c);
        if (values != nullptr && at * 8 < k) store_eight<kType>(values, row * k + at * 8LL, v, k - at * 8);
    }
}

// Two neighbouring elements of a row (one where the row ends) as fp32.
template <int kType>
__device__ __forceinline__ f32x2 load_two(const void* p, long long at, int left) {
    typedef f32x2 f32x2_loose __attribute__((aligned(4)));
    if (left >= 2) {
        if constexpr (kType == kF32) return *reinterpret_cast<const f32x2_loose*>(static_cast<const float*>(p) + at);
        const unsigned two = *reinterpret_cast<const u32_loose*>(static_cast<const unsigned short*>(p) + at);
        return f32x2{to_f32<kType>(two & 0xffffu), to_f32<kType>(two >> 16)};
    }
    return f32x2{left == 1 ? load_one<kType>(p, at) : 0.0f, 0.0f};
}

template <int kType>
__device__ __forceinline__ void store_two(void* p, long long at, float a, float b, int left) {
    typedef f32x2 f32x2_loose __attribute__((aligned(4)));
    if (left >= 2) {
        if constexpr (kType == kF32)
            __builtin_nontemporal_store(f32x2{a, b}, reinterpret_cast<f32x2_loose*>(static_cast<float*>(p) + at));
        else
            __builtin_nontemporal_store(to_16<kType>(a) | static_cast<unsigned>(to_16<kType>(b)) << 16,
                                        reinterpret_cast<u32_loose*>(static_cast<unsigned short*>(p) + at));
    } else if (left == 1) {
        store_one<kType>(p, at, a);
    }
}

// A block takes 2 kAcross columns whole: kAcross lanes a row of them, two columns each,
// and eight rows down, which stay in registers between the columns' largest magnitudes
// and the codes. For up to 8 x 1024 / kAcross rows.
constexpr int kColumnThreads = 1024;

template <int kType, int kAcross>
__global__ __launch_bounds__(kColumnThreads) void quantize_columns(const void* __restrict__ w, long long ld,
                                                                   u32x2* __restrict__ codes,
                                                                   float* __restrict__ scales,
                                                                   void* __restrict__ values, int k, int n,
                                                                   int chunks) {
    __shared__ unsigned tops[kColumnThreads / 64][2 * kAcross];
    __shared__ float found[2 * kAcross];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int across = threadIdx.x % kAcross, chunk = threadIdx.x / kAcross;
    // Blocks go to the XCDs in turn; neighbouring columns to one, whose L2 has the lines that they share.
    const unsigned all = gridDim.x, mine = blockIdx.x % 8 * (all / 8) + blockIdx.x / 8;
    const unsigned block = blockIdx.x < all / 8 * 8 ? mine : blockIdx.x;
    const long long col = static_cast<long long>(block) * 2 * kAcross + 2 * across;
    const int left = static_cast<int>(min(static_cast<long long>(n) - col, 2LL));
    float v[2][8];
    unsigned top[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const f32x2 two = load_two<kType>(w, (chunk * 8 + e) * ld + col, chunk * 8 + e < k ? left : 0);
        v[0][e] = two[0], v[1][e] = two[1];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        top[0] = max(top[0], magnitude(v[0][e]));
        top[1] = max(top[1], magnitude(v[1][e]));
    }
#pragma unroll
    for (int d = kAcross; d < 64; d *= 2) {
        top[0] = max(top[0], static_cast<unsigned>(__shfl_xor(static_cast<int>(top[0]), d)));
        top[1] = max(top[1], static_cast<unsigned>(__shfl_xor(static_cast<int>(top[1]), d)));
    }
    if (lane < kAcross) tops[wave][2 * lane] = top[0], tops[wave][2 * lane + 1] = top[1];
    __syncthreads();
    if (threadIdx.x < 2 * kAcross) {
        unsigned most = 0;
#pragma unroll
        for (int u = 0; u < kColumnThreads / 64; ++u) most = max(most, tops[u][threadIdx.x]);
        const float s = scale_of(most);
        found[threadIdx.x] = s;
        if (static_cast<long long>(block) * 2 * kAcross + threadIdx.x < n)
            scales[static_cast<long long>(block) * 2 * kAcross + threadIdx.x] = s;
    }
    __syncthreads();
    if (chunk >= chunks) return;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const u32x2 packed = codes_of(v[j], of_scale(found[2 * across + j]));
        if (j < left) codes[(col + j) * chunks + chunk] = packed;
    }
    if (values == nullptr) return;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (chunk * 8 + e < k) store_two<kType>(values, (chunk * 8LL + e) * n + col, v[0][e], v[1][e], left);
}

// More rows, in three launches: scales cleared, found (the largest of the scales of parts
// of a column is the column's: rounding keeps the order), and the codes. A block of the
// last two takes 128 columns, a wave whole lines of a row, two columns a lane.
constexpr int kAcrossAll = 128, kPartRows = 512;

__global__ __launch_bounds__(256) void clear_scales(float* __restrict__ scales, int n) {
    const unsigned i = blockIdx.x * 256u + threadIdx.x;
    if (i < static_cast<unsigned>(n)) scales[i] = 0.0f;
}

template <int kType>
__global__ __launch_bounds__(kColumnThreads) void column_scales(const void* __restrict__ w, long long ld,
                                                                unsigned* __restrict__ scales, int k, int n) {
    constexpr int kWaves = kColumnThreads / 64;
    __shared__ unsigned tops[kWaves][kAcrossAll];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const long long col = static_cast<long long>(blockIdx.x) * kAcrossAll + 2 * lane;
    const int left = static_cast<int>(min(static_cast<long long>(n) - col, 2LL));
    unsigned top[2] = {0, 0};
#pragma unroll 8
    for (int i = 0; i < kPartRows / kWaves; ++i) {
        const long long row = static_cast<long long>(blockIdx.y) * kPartRows + i * kWaves + wave;
        const f32x2 two = load_two<kType>(w, row * ld + col, row < k ? left : 0);
        top[0] = max(top[0], magnitude(two[0]));
        top[1] = max(top[1], magnitude(two[1]));
    }
    tops[wave][2 * lane] = top[0], tops[wave][2 * lane + 1] = top[1];
    __syncthreads();
    if (threadIdx.x >= kAcrossAll) return;
    unsigned most = 0;
#pragma unroll
    for (int u = 0; u < kWaves; ++u) most = max(most, tops[u][threadIdx.x]);
    const long long at = static_cast<long long>(blockIdx.x) * kAcrossAll + threadIdx.x;
    if (at < n && most != 0) atomicMax(scales + at, __builtin_bit_cast(unsigned, scale_of(most)));
}

// A wave eight rows, the block 128: a line of codes for each column, by way of LDS.
template <int kType>
__global__ __launch_bounds__(kColumnThreads) void column_codes(const void* __restrict__ w, long long ld,
                                                               unsigned char* __restrict__ codes,
                                                               const float* __restrict__ scales,
                                                               void* __restrict__ values, int k, int n, int row_bytes) {
    constexpr int kStride = kLine + 16;
    __shared__ __attribute__((aligned(16))) unsigned char lines[kAcrossAll * kStride];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const long long col0 = static_cast<long long>(blockIdx.x) * kAcrossAll, col = col0 + 2 * lane;
    const long long row = static_cast<long long>(blockIdx.y) * kLine + wave * 8;
    const int left = static_cast<int>(min(static_cast<long long>(n) - col, 2LL));
    float v[2][8], s[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) s[j] = j < left ? scales[col + j] : 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const f32x2 two = load_two<kType>(w, (row + e) * ld + col, row + e < k ? left : 0);
        v[0][e] = two[0], v[1][e] = two[1];
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
        *reinterpret_cast<u32x2*>(lines + (2 * lane + j) * kStride + wave * 8) = codes_of(v[j], of_scale(s[j]));
    if (values != nullptr) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (row + e < k) store_two<kType>(values, (row + e) * n + col, v[0][e], v[1][e], left);
    }
    __syncthreads();
    const int c = threadIdx.x / 8, part = threadIdx.x % 8 * 16;
    if (col0 + c < n)
        *reinterpret_cast<u32x4*>(codes + (col0 + c) * row_bytes + static_cast<long long>(blockIdx.y) * kLine + part) =
            *reinterpret_cast<const u32x4*>(lines + c * kStride + part);
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
int launch_rows(const void* x, long long ld, void* codes, float* scales, int rows, int k, void* values,
                hipStream_t stream) {
    const int chunks = padded_k(k) / 8, cus = device_cus();
    constexpr int kMost = 1 << 21;
    for (long long from = 0; from < rows; from += kMost) {
        const int count = static_cast<int>(std::min<long long>(kMost, rows - from));
        const void* at = offset<kType>(x, from * ld);
        u32x2* to = static_cast<u32x2*>(codes) + from * chunks;
        void* back = offset<kType>(values, from * k);
        const auto go = [&](auto kernel, int lanes) {
            const unsigned blocks = static_cast<unsigned>(lanes < 256 ? (count + 256 / lanes - 1) / (256 / lanes) : count);
            return launch_kernel(kernel, blocks, lanes < 256 ? 256 : lanes, 0, stream, at, ld, to, scales + from, back, count,
                                 k, chunks);
        };
        // Few rows: as many lanes to a row as have something to do. Many: as few as hold it,
        // so that no wave waits for another.
        const bool few = count < 4 * cus;
        int rc;
        if (chunks <= 64) rc = go(quantize_rows<kType, 64, 1>, 64);
        else if (!few && chunks <= 128) rc = go(quantize_rows<kType, 64, 2>, 64);
        else if (!few && chunks <= 256) rc = go(quantize_rows<kType, 64, 4>, 64);
        else if (chunks <= 256) rc = go(quantize_rows<kType, 256, 1>, 256);
        else if (!few && chunks <= 512) rc = go(quantize_rows<kType, 256, 2>, 256);
        else if (!few && chunks <= 1024) rc = go(quantize_rows<kType, 256, 4>, 256);
        else if (chunks <= 1024) rc = go(quantize_rows<kType, 1024, 1>, 1024);
        else if (chunks <= 2048) rc = go(quantize_rows<kType, 1024, 2>, 1024);
        else rc = launch_kernel(quantize_long_rows<kType>, static_cast<unsigned>(count), kLong, 0, stream, at, ld, to,
                                scales + from, back, k, chunks);
        if (rc != hipSuccess) return rc;
    }
    return hipSuccess;
}

template <int kType>
int launch_columns(const void* w, long long ld, void* codes, float* scales, int k, int n, void* values,
                   hipStream_t stream, const char** why) {
    const auto whole = [&](auto kernel, int across) {
        const long long blocks = (static_cast<long long>(n) + 2 * across - 1) / (2 * across);
        return launch_kernel(kernel, static_cast<unsigned>(blocks), kColumnThreads, 0, stream, w, ld,
                             static_cast<u32x2*>(codes), scales, values, k, n, padded_k(k) / 8);
    };
    // Few enough rows for one launch, and not so many columns that their narrow strips take
    // longer than the two launches more (2048 rows by 8192 columns of fp32 103 us).
    if (k <= 1024 && n <= (1 << 22)) return whole(quantize_columns<kType, 8>, 8);
    if (k <= 2048 && static_cast<long long>(k) * n <= (1 << 22)) return whole(quantize_columns<kType, 4>, 4);
    const unsigned across = static_cast<unsigned>((static_cast<long long>(n) + kAcrossAll - 1) / kAcrossAll);
    if (!fits_launch(across, kColumnThreads)) {
        *why = "more columns than one launch takes (536870784)";
        return hipErrorInvalidValue;
    }
    int rc = launch_kernel(clear_scales, static_cast<unsigned>((static_cast<long long>(n) + 255) / 256), 256, 0, stream, scales, n);
    // As much of k at a time as a launch takes.
    constexpr int kParts = 65535;
    for (long long from = 0; rc == hipSuccess && from < k; from += static_cast<long long>(kParts) * kPartRows) {
        const int rows = static_cast<int>(std::min<long long>(k - from, static_cast<long long>(kParts) * kPartRows));
        rc = launch_kernel(column_scales<kType>, dim3(across, static_cast<unsigned>((rows + kPartRows - 1) / kPartRows)),
                           kColumnThreads, 0, stream, offset<kType>(w, from * ld), ld, reinterpret_cast<unsigned*>(scales),
                           rows, n);
    }
    for (long long from = 0; rc == hipSuccess && from < k; from += static_cast<long long>(kParts) * kLine) {
        const int rows = static_cast<int>(std::min<long long>(k - from, static_cast<long long>(kParts) * kLine));
        rc = launch_kernel(column_codes<kType>, dim3(across, static_cast<unsigned>((rows + kLine - 1) / kLine)),
                           kColumnThreads, 0, stream, offset<kType>(w, from * ld), ld,
                           static_cast<unsigned char*>(codes) + from, scales, offset<kType>(values, from * n), rows, n,
                           padded_k(k));
    }
    return rc;
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

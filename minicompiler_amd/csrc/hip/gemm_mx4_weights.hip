// C = A B^T with A in fp32, bf16 or fp16 as it is and B quantised to microscaled
// 4-bit floats (mx4.h): a layer whose weights alone are in 4 bits.
//
// The matrix instruction on bf16 multiplies exactly, and every operand is
// exact in bf16: a weight (two significant bits and a power of two), and A cut
// into one, two or three bf16 pieces (8, 11 or 24 significant bits), each
// multiplied by the same weights into the same fp32 sum.

#include "mx4_device.h"

namespace {

using namespace mx4;

// A block computes 16 kM rows by 16 kN columns of C; its kWaves waves take the
// steps of 128 k in turn and their sums are added at the end. Lane (r, q) of a
// wave holds block q of weight row r: dword s of its codes, decoded, is the
// operand of instruction s, so group q supplies elements 32 q + 8 s .. + 7.
template <int kIn, int kM, int kN, int kWaves, int kOut>
__global__ __launch_bounds__(kWaves * 64) void weights_direct(const void* __restrict__ a, long long lda,
                                                              const unsigned char* __restrict__ b_codes,
                                                              const unsigned char* __restrict__ b_scales,
                                                              void* __restrict__ c, int m, int n, int k, int steps,
                                                              unsigned tiles_n) {
    constexpr int kP = kPieces<kIn>;
    __shared__ f32x4 space[kWaves / 2 * kM * kN * 64];
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int r = lane % 16, q = lane / 16;
    const long long row0 = static_cast<long long>(blockIdx.x / tiles_n) * 16 * kM;
    const long long col0 = static_cast<long long>(blockIdx.x % tiles_n) * 16 * kN;

    const unsigned char *bc[kN], *bs[kN];
#pragma unroll
    for (int j = 0; j < kN; ++j) {
        const long long col = col0 + 16 * j + r < n ? col0 + 16 * j + r : n - 1;
        bc[j] = b_codes + col * steps * 64 + q * 16;
        bs[j] = b_scales + col * steps * 4 + q;
    }
    f32x4 acc[kM * kN];
#pragma unroll
    for (int i = 0; i < kM * kN; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    for (int t = wave; t < steps; t += kWaves) {
        u32x4 codes[kN];
        float scale[kN];
#pragma unroll
        for (int j = 0; j < kN; ++j) {
            codes[j] = *reinterpret_cast<const u32x4*>(bc[j] + static_cast<long long>(t) * 64);
            scale[j] = scale_operand(bs[j][t * 4]);
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int k0 = t * kStep + 32 * q + 8 * s;
            u32x4 x[kM][kP];
#pragma unroll
            for (int i = 0; i < kM; ++i) {
                const long long row = row0 + 16 * i + r;
                float v[8];
                load_eight<kIn>(a, row * lda + k0, row < m ? k - k0 : 0, v);
                cut_eight<kP>(v, x[i]);
            }
#pragma unroll
            for (int j = 0; j < kN; ++j) {
                const u32x4 w = decode_eight(codes[j][s], scale[j]);
#pragma unroll
                for (int i = 0; i < kM; ++i)
#pragma unroll
                    for (int p = 0; p < kP; ++p) acc[i * kN + j] = mfma_bf16(w, x[i][p], acc[i * kN + j]);
            }
        }
    }
    add_waves<kWaves, kM * kN>(acc, space, wave, lane);
    if (wave != 0) return;
#pragma unroll
    for (int i = 0; i < kM; ++i) {
        const long long row = row0 + 16 * i + r;
        if (row >= m) continue;
#pragma unroll
        for (int j = 0; j < kN; ++j) {
            const long long col = col0 + 16 * j + 4 * q;
            if (col < n)
                store_four<kOut>(c, row * n + col, acc[i * kN + j], static_cast<int>(n - col < 4 ? n - col : 4));
        }
    }
}

struct Product {
    const void* a;
    long long lda;
    const unsigned char *b_codes, *b_scales;
    void* c;
    int m, n, k, steps;
    hipStream_t stream;
};

long long tiles(int size, int tile) { return (static_cast<long long>(size) + tile - 1) / tile; }

template <int kIn, int kM, int kN, int kOut>
int launch_direct(const Product& p) {
    constexpr int kWaves = 8;
    const long long tn = tiles(p.n, 16 * kN), blocks = tiles(p.m, 16 * kM) * tn;
    if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    hipLaunchKernelGGL((weights_direct<kIn, kM, kN, kWaves, kOut>), dim3(static_cast<unsigned>(blocks)),
                       dim3(kWaves * 64), 0, p.stream, p.a, p.lda, p.b_codes, p.b_scales, p.c, p.m, p.n, p.k, p.steps,
                       static_cast<unsigned>(tn));
    return hipGetLastError();
}

template <int kIn, int kOut>
int launch_shape(const Product& p) {
    if (p.m <= 16) return launch_direct<kIn, 1, 2, kOut>(p);
    return launch_direct<kIn, 2, 2, kOut>(p);
}

template <int kIn>
int launch(int c_dtype, const Product& p) {
    if (c_dtype == kF32) return launch_shape<kIn, kF32>(p);
    if (c_dtype == kBf16) return launch_shape<kIn, kBf16>(p);
    return launch_shape<kIn, kF16>(p);
}

}  // namespace

extern "C" {

long long mchip_matmul_mx4_weights_workspace_bytes(int a_dtype, int m, int n, int k) { return 0; }

int mchip_launch_matmul_mx4_weights(int a_dtype, const void* a, long long lda, const void* b_codes,
                                    const void* b_scales, int c_dtype, void* c, int m, int n, int k, void* stream,
                                    void* workspace, const char** why) {
    *why = nullptr;
    if (!is_float_type(a_dtype) || !is_float_type(c_dtype)) *why = "a type that is none of fp32 (0), bf16 (1), fp16 (2)";
    else if (m < 1 || n < 1 || k < 1) *why = "a size below 1";
    else if (k > (1 << 24)) *why = "k above 2^24";
    else if (lda < k) *why = "rows of A closer together than they are long";
    else if (!a || !b_codes || !b_scales || !c) *why = "a null operand";
    else if (!aligned(b_codes, 16)) *why = "codes not 16-byte aligned";
    else if (!aligned(b_scales, 4)) *why = "scales not 4-byte aligned";
    else if (!aligned(a, size_of(a_dtype)) || !aligned(c, size_of(c_dtype)))
        *why = "an address that is no multiple of its element's size";
    if (*why != nullptr) return hipErrorInvalidValue;
    Product p{a, lda, static_cast<const unsigned char*>(b_codes), static_cast<const unsigned char*>(b_scales),
              c, m, n, k, static_cast<int>(mchip_mx4_k(k) / kStep),
              static_cast<hipStream_t>(stream)};
    const int rc = a_dtype == kF32   ? launch<kF32>(c_dtype, p)
                   : a_dtype == kBf16 ? launch<kBf16>(c_dtype, p)
                                      : launch<kF16>(c_dtype, p);
    if (rc == hipErrorInvalidValue) *why = "more tiles of C than one launch takes";
    return rc;
}

}  // extern "C"

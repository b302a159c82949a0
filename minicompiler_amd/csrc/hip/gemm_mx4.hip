// The product of two operands quantised to microscaled 4-bit floats (mx4.h):
// C = A B^T, on v_mfma_scale_f32_16x16x128_f8f6f4, which multiplies codes and
// scales exactly and adds in fp32.

#include "gemm_mx4_tiles.h"
#include "mx4_rows.h"

namespace {

using namespace mx4;

// A block computes 16 kM rows by 16 kN columns of C; its kWaves waves take the
// steps of 128 k in turn and their sums are added at the end. Fragments come
// straight from memory, the next step's while one is multiplied. Bound by
// latency: a launch, two trips to memory, and code read into a cold instruction
// cache (1000x1001x1023 with 4x4 fragments: 8.5 KB of it in 7.9 us, 4.1 KB in 6.3,
// and 5.9 with four neighbouring lanes' loads from one row; 16x4096x4096 4.7 us and
// so 3.6).
template <int kM, int kN, int kWaves, int kOut>
__global__ __launch_bounds__(kWaves * 64) void product_direct(const unsigned char* __restrict__ a_codes,
                                                              const unsigned char* __restrict__ a_scales,
                                                              const unsigned char* __restrict__ b_codes,
                                                              const unsigned char* __restrict__ b_scales,
                                                              void* __restrict__ c, int m, int n, int steps,
                                                              unsigned tiles_n) {
    __shared__ f32x4 space[kWaves * kM * kN * 64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int r = lane % 16, q = lane / 16;
    const long long row0 = static_cast<long long>(blockIdx.x / tiles_n) * 16 * kM;
    const long long col0 = static_cast<long long>(blockIdx.x % tiles_n) * 16 * kN;
    Rows<kMx4, kM> a;
    Rows<kMx4, kN> b;
    a.open(a_codes, a_scales, steps * kStep, m, [&](int i) { return row0 + 16 * i < m ? row0 + 16 * i : 0; });
    b.open(b_codes, b_scales, steps * kStep, n, [&](int j) { return col0 + 16 * j < n ? col0 + 16 * j : 0; });
    f32x4 acc[kM * kN];
#pragma unroll
    for (int i = 0; i < kM * kN; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    typename Rows<kMx4, kM>::Step a_now, a_next;
    typename Rows<kMx4, kN>::Step b_now, b_next;
    if (wave < steps) {
        a.load(wave, a_next);
        b.load(wave, b_next);
    }
    for (int t = wave; t < steps; t += kWaves) {
        a_now = a_next;
        b_now = b_next;
        if (t + kWaves < steps) {
            a.load(t + kWaves, a_next);
            b.load(t + kWaves, b_next);
        }
        int sa[kM], sb[kN];
#pragma unroll
        for (int i = 0; i < kM; ++i) sa[i] = static_cast<int>(a.scale(a_now, i));
#pragma unroll
        for (int j = 0; j < kN; ++j) sb[j] = static_cast<int>(b.scale(b_now, j));
        i32x4 av[kM], bv[kN];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
#pragma unroll
            for (int i = 0; i < kM; ++i) av[i][e] = static_cast<int>(a.pass(a_now.w[i][0][e]));
#pragma unroll
            for (int j = 0; j < kN; ++j) bv[j][e] = static_cast<int>(b.pass(b_now.w[j][0][e]));
        }
#pragma unroll
        for (int i = 0; i < kM; ++i)
#pragma unroll
            for (int j = 0; j < kN; ++j) acc[i * kN + j] = mfma(bv[j], sb[j], av[i], sa[i], acc[i * kN + j]);
    }
    sum_waves<kWaves>(acc, space, wave, lane, [&](int i, f32x4 sum) {
        const long long row = row0 + 16 * (i / kN) + r, col = col0 + 16 * (i % kN) + 4 * q;
        if (row < m && col < n)
            store_four<kOut>(c, row * n + col, sum, static_cast<int>(n - col < 4 ? n - col : 4));
    });
}

// Tiles in row-major order, as gemm_mfma16_fast.h has them: the grid has one
// block per 256x256 tile plus `halves` more, for which that many of the last
// tiles run as two blocks of 128x256.
template <int kOut>
__global__ __launch_bounds__(kTileThreads, 1) void product_tiles(const unsigned char* __restrict__ a_codes,
                                                                 const unsigned char* __restrict__ a_scales,
                                                                 const unsigned char* __restrict__ b_codes,
                                                                 const unsigned char* __restrict__ b_scales,
                                                                 void* __restrict__ c, int m, int n, int steps,
                                                                 int tiles_n, int full, bool eights) {
    __shared__ __attribute__((aligned(1024))) unsigned char smem[kRingBytes];
    MX4_LDS unsigned char* lds = (MX4_LDS unsigned char*)(smem);  // generic -> LDS address space
    const int block = static_cast<int>(blockIdx.x);
    if (block < full) {
        product_tile<256, kOut>(lds, a_codes, a_scales, b_codes, b_scales, c, m, n, steps, block / tiles_n * 256,
                                block % tiles_n * 256, eights);
    } else {
        const int t = full + (block - full) / 2;
        const int row0 = t / tiles_n * 256 + (block - full) % 2 * 128;
        if (row0 >= m) return;  // the last tile row has no second half
        product_tile<128, kOut>(lds, a_codes, a_scales, b_codes, b_scales, c, m, n, steps, row0, t % tiles_n * 256,
                                eights);
    }
}

struct Product {
    const unsigned char *a_codes, *a_scales, *b_codes, *b_scales;
    void* c;
    int m, n, steps;
    hipStream_t stream;
    const char** why;
};

long long tiles(int size, int tile) { return (static_cast<long long>(size) + tile - 1) / tile; }

template <int kM, int kN, int kOut>
int launch_direct(const Product& p) {
    constexpr int kWaves = 8;
    const long long tn = tiles(p.n, 16 * kN), blocks = tiles(p.m, 16 * kM) * tn;
    if (!fits_launch(blocks, kWaves * 64)) {
        *p.why = "more tiles of C than one launch takes";
        return hipErrorInvalidValue;
    }
    return launch_kernel(product_direct<kM, kN, kWaves, kOut>, static_cast<unsigned>(blocks), kWaves * 64, 0, p.stream,
                         p.a_codes, p.a_scales, p.b_codes, p.b_scales, p.c, p.m, p.n, p.steps, static_cast<unsigned>(tn));
}

template <int kOut>
int launch_tiles(const Product& p) {
    const int tn = static_cast<int>(tiles(p.n, kTileCols)), all = static_cast<int>(tiles(p.m, kTileRows)) * tn;
    const int cus = device_cus(), rest = all % cus;
    const int halves = rest <= cus / 2 ? rest : 0;
    return launch_kernel(product_tiles<kOut>, static_cast<unsigned>(all + halves), kTileThreads, 0, p.stream, p.a_codes,
                         p.a_scales, p.b_codes, p.b_scales, p.c, p.m, p.n, p.steps, tn, all - halves, p.n % 8 == 0);
}

// Four steps at least (a slot of scales), and 32-bit offsets from a tile's origin.
bool tiles_fit(const Product& p) {
    return p.steps >= 4 && p.steps <= (1 << 16) && fits_launch(tiles(p.m, kTileRows) * tiles(p.n, kTileCols) * 2, kTileThreads);
}

template <int kOut>
int launch(const Product& p) {
    const int cus = device_cus();
    const auto blocks = [&](int bm, int bn) { return tiles(p.m, 16 * bm) * tiles(p.n, 16 * bn); };
    if (p.m <= 16) {
        if (blocks(1, 4) >= cus) return launch_direct<1, 4, kOut>(p);
        if (blocks(1, 2) >= cus) return launch_direct<1, 2, kOut>(p);
        return launch_direct<1, 1, kOut>(p);
    }
    if (p.m <= 32) {
        if (blocks(2, 4) >= cus) return launch_direct<2, 4, kOut>(p);
        if (blocks(2, 2) >= cus) return launch_direct<2, 2, kOut>(p);
        return launch_direct<1, 1, kOut>(p);
    }
    // A round of 256x256 tiles takes as long as 2.25 rounds of 64x64 (24 and 10.4 us each at
    // k = 4096), however few of the CUs have one: 2048x3840x4096, 120 tiles, in 26 us, by 64x64
    // in 77; 1024x2560x600 in 10.9 and 16.0.
    const long long large = blocks(4, 4), rounds = (large + cus - 1) / cus;
    const long long tile_rounds = (tiles(p.m, kTileRows) * tiles(p.n, kTileCols) + cus - 1) / cus;
    if (tiles_fit(p) && 4 * large >= 9 * cus * tile_rounds) return launch_tiles<kOut>(p);
    // 64x64 per block read the least, one block to a CU at a time: where that leaves no
    // round a fifth empty (1000x1001x8000 in 19.3 us, 22.4 by 32x64; 1400x1001x4096,
    // 352 blocks on 256 CUs, in 20.4, 17.0 by 32x64).
    if (large >= cus && 5 * large >= 4 * rounds * cus) return launch_direct<4, 4, kOut>(p);
    if (blocks(2, 4) >= cus) return launch_direct<2, 4, kOut>(p);
    if (blocks(2, 2) >= cus) return launch_direct<2, 2, kOut>(p);
    return launch_direct<1, 1, kOut>(p);
}

}  // namespace

extern "C" int mchip_launch_matmul_mx4(const void* a_codes, const void* a_scales, const void* b_codes,
                                       const void* b_scales, int c_dtype, void* c, int m, int n, int k, void* stream,
                                       const char** why) {
    *why = nullptr;
    if (!is_float_type(c_dtype)) *why = "the result's type is none of fp32 (0), bf16 (1), fp16 (2)";
    else if (m < 1 || n < 1 || k < 1) *why = "a size below 1";
    else if (k > (1 << 24)) *why = "k above 2^24";
    else if (!a_codes || !a_scales || !b_codes || !b_scales || !c) *why = "a null operand";
    else if (!aligned(a_codes, 16) || !aligned(b_codes, 16)) *why = "codes not 16-byte aligned";
    else if (!aligned(a_scales, 4) || !aligned(b_scales, 4)) *why = "scales not 4-byte aligned";
    else if (!aligned(c, size_of(c_dtype))) *why = "a result that is not aligned to its elements";
    if (*why != nullptr) return hipErrorInvalidValue;
    Product p{static_cast<const unsigned char*>(a_codes), static_cast<const unsigned char*>(a_scales),
              static_cast<const unsigned char*>(b_codes), static_cast<const unsigned char*>(b_scales),
              c, m, n, static_cast<int>(mchip_mx4_k(k) / kStep),
              static_cast<hipStream_t>(stream), why};
    return c_dtype == kF32 ? launch<kF32>(p) : c_dtype == kBf16 ? launch<kBf16>(p) : launch<kF16>(p);
}

// C = A B^T with A in fp32, bf16 or fp16 as it is and B quantised to microscaled
// 4-bit floats (mx4.h): a layer whose weights alone are in 4 bits.
//
// The matrix instruction on bf16 multiplies exactly, and every operand is
// exact in bf16: a weight (two significant bits and a power of two), and A cut
// into one, two or three bf16 pieces (8, 11 or 24 significant bits; of fp32 below
// 2^-110 those from 2^-133 up), each multiplied by the same weights into the same
// fp32 sum.
//
//   weights_few     up to 16 rows: A cut by every wave as it reads it;
//   weights_whole   up to 64 rows of 16 bits, not cut: fp16 ones by the fp16
//                   instruction, scales applied to its sums;
//   cut_rows        A's pieces into the workspace, for the two below:
//   weights_direct  few tiles: a block's waves share out k, fragments come
//                   straight from memory;
//   weights_tiles   many: 128x128 tiles, k in stages through LDS.
// The pieces are kept as [pieces][kp / 8][rows][8], a row's eight elements beside
// its neighbours', so that a fragment of 16 rows is read in whole lines.

#include "mx4_rows.h"

namespace {

using namespace mx4;

constexpr int kFew = 16;
constexpr int kWholeRows = 64;
constexpr int kFewWaves = 16;

// ---------------------------------------------------------------- few rows

// These kernels' code is kept short: a launch meets a cold instruction cache, and
// on an MI355X every 128 bytes of straight code cost about 0.2 us (31 MB through
// 8.5 KB of code with four steps of each wave unrolled in 12.4 us, through 3.2 KB
// in 11.4; 9 MB and fp32 rows 9.6 and 7.2), so the loop has one copy of its body,
// and 16 waves two steps each where 8 had four.

// Eight elements of a row as they lie in memory.
template <int kIn>
struct Eight {
    u32x4 v[kIn == kF32 ? 2 : 1];

    // From byte `at` of the rows on; what lies past them reads as zeros.
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t rows, int at, int step_at) {
        v[0] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rows, at, step_at, 0));
        if constexpr (kIn == kF32)
            v[1] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rows, at + 16, step_at, 0));
    }
    // At any address and any distance.
    __device__ __forceinline__ void load_loose(const void* a, long long at, int left) {
        if (left >= 8) {
            if constexpr (kIn == kF32) {
                const u32x4_dwords* p = reinterpret_cast<const u32x4_dwords*>(static_cast<const float*>(a) + at);
                v[0] = p[0];
                v[1] = p[1];
            } else {
                v[0] = *reinterpret_cast<const u32x4_loose*>(static_cast<const unsigned short*>(a) + at);
            }
            return;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (kIn == kF32) {
                v[e / 4][e % 4] = e < left ? static_cast<const unsigned*>(a)[at + e] : 0u;
            } else {
                const unsigned h = e < left ? static_cast<const unsigned short*>(a)[at + e] : 0u;
                v[0][e / 2] = e % 2 ? v[0][e / 2] | h << 16 : h;
            }
        }
    }
    // Zeros from element `left` on.
    __device__ __forceinline__ void cut_off(int left) {
#pragma unroll
        for (int e = 0; e < 8; e += kIn == kF32 ? 1 : 2) {
            unsigned keep = e < left ? 0xffffu : 0u;
            keep |= (kIn == kF32 ? e : e + 1) < left ? 0xffff0000u : 0u;
            v[kIn == kF32 ? e / 4 : 0][kIn == kF32 ? e % 4 : e / 2 % 4] &= keep;
        }
    }

    __device__ __forceinline__ void pieces(u32x4 (&out)[kPieces<kIn>]) const {
        if constexpr (kIn == kBf16) {
            out[0] = v[0];
        } else {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const unsigned word = kIn == kF32 ? v[kIn == kF32 ? e / 4 : 0][e % 4] : v[0][e / 2 % 4];
                f[e] = to_f32<kIn>(kIn == kF32 ? word : e % 2 ? word >> 16 : word & 0xffffu);
            }
            cut_eight<kPieces<kIn>>(f, out);
        }
    }
};

// 16 kN columns of C for all rows (at most 16); the waves take the steps of 128 k
// in turn, the next one under way while one is multiplied. Bound by the weights
// and a launch's latency: one row by 14336x4096 in 7.6 us (31 MB at 4.1 TB/s),
// two by 4096x4096 in 3.7. 16 bf16 rows by 14336x4096 take 10.4 us a call where
// a launch that cuts them and one that multiplies took 12.0; 12 fp32 rows by
// 4096x4096 9.8 and 9.7, three pieces of every number cut in each of 256 blocks.
// kLoose: rows that do not all start at dwords, or more than 2 GiB of them.
template <int kIn, int kN, int kOut, bool kLoose>
__global__ __launch_bounds__(kFewWaves * 64) void weights_few(const void* __restrict__ a, long long lda,
                                                              const unsigned char* __restrict__ b_codes,
                                                              const unsigned char* __restrict__ b_scales,
                                                              void* __restrict__ c, int m, int n, int k) {
    constexpr int kP = kPieces<kIn>, kSizeIn = kSize<kIn>;
    __shared__ f32x4 space[kFewWaves * kN * 64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int r = lane % 16, q = lane / 16, steps = padded(k) / kStep;
    const long long col0 = static_cast<long long>(blockIdx.x) * 16 * kN;
    Rows<kMx4, kN> b;
    b.open(b_codes, b_scales, k, n, [&](int j) { return col0 + 16 * j < n ? col0 + 16 * j : 0; });
    const bool has = r < m;
    const int bytes = kLoose ? 0 : static_cast<int>(((m - 1) * lda + k) * kSizeIn + 3) & ~3;
    const __amdgpu_buffer_rsrc_t rows = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(a), 0, bytes, 0x00020000);
    const int at = kLoose ? 0 : static_cast<int>((has ? r : 0) * lda + 32 * q) * kSizeIn;
    f32x4 acc[kN];
#pragma unroll
    for (int j = 0; j < kN; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    struct Step {
        Eight<kIn> x[4];
        typename Rows<kMx4, kN>::Step w;
    } now, next;
    const auto load = [&](int t) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (kLoose) {
                const int e = t * kStep + 32 * q + 8 * i;
                next.x[i].load_loose(a, has ? r * lda + e : 0, has ? k - e : 0);
            } else {
                if (has) next.x[i].load(rows, at + 8 * i * kSizeIn, t * kStep * kSizeIn);  // the others stay zeros
            }
        }
        b.load(t, next.w);
    };
    next.x[0] = next.x[1] = next.x[2] = next.x[3] = Eight<kIn>{};
    int t = wave;
    if (t < steps) load(t);
    while (t < steps) {
        now = next;
        const int then = t + kFewWaves;
        if (then < steps) load(then);
        if (!kLoose && (t + 1) * kStep > k) {
#pragma unroll
            for (int i = 0; i < 4; ++i) now.x[i].cut_off(k - (t * kStep + 32 * q + 8 * i));
        }
        float scale[kN];
#pragma unroll
        for (int j = 0; j < kN; ++j) scale[j] = scale_operand(b.scale(now.w, j));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            u32x4 piece[kP];
            now.x[i].pieces(piece);
#pragma unroll
            for (int j = 0; j < kN; ++j) {
                const u32x4 w = decode_eight(b.pass(now.w.w[j][0][i]), scale[j]);
#pragma unroll
                for (int p = 0; p < kP; ++p) acc[j] = mfma_bf16(w, piece[p], acc[j]);
            }
        }
        t = then;
    }
    sum_waves<kFewWaves>(acc, space, wave, lane, [&](int j, f32x4 sum) {
        const long long col = col0 + 16 * j + 4 * q;
        if (has && col < n)
            store_four<kOut>(c, r * static_cast<long long>(n) + col, sum, static_cast<int>(n - col < 4 ? n - col : 4));
    });
}

// ---------------------------------------------------------------- 16-bit rows as they are

// 16 kM rows by 16 kN columns of C per block, 16-bit rows that start at dwords,
// straight from memory: no pieces and no workspace. The waves take the steps of
// 128 k in turn. Instruction s of a step multiplies its block s (lane (r, q)
// elements 8 q .. + 7 of it), so that one scale holds for all that it adds up:
// fp16 rows meet the bare codes (exact in fp16) in a sum from zero, which the
// scale multiplies as it joins the others (a power of two: one rounding, the
// sum's); bf16 ones the scaled weights.
//
// A wave's steps of A go to LDS without registers, one multiplied while the next
// is under way; lanes 4 g .. 4 g + 3 fetch 64 bytes of row g, chunk c of it to
// slot c ^ (g / 4), so that 16 lanes read 16 rows' chunks from all banks. Bound by
// A, which every block reads from its L2 (256 KiB for 32 rows of 4096), and the
// scales' work. A call on 32 fp16 rows by 4096x4096 takes 7.4 us (9.4 with A in
// registers, passed on between lanes; 10.4 in two launches, cutting and
// weights_direct), by 6144x2048 6.9 (11.0), by 14336x4096 16.5 (17.9); bf16 6.6
// (7.9), 5.6 (8.3) and 13.7 (15.0); 16 fp16 rows by 4096x4096 5.8 (7.2 by
// weights_few), bf16 5.3 (6.5).
// 16 waves of 16 rows, 8 of 32, 4 of 64: two steps of A each are 128 KiB of LDS.
template <int kM>
constexpr int kWhole = 16 / kM;

template <int kIn, int kM, int kN, int kOut>
__global__ __launch_bounds__(kWhole<kM> * 64) void weights_whole(const void* __restrict__ a, int lda,
                                                                const unsigned char* __restrict__ b_codes,
                                                                const unsigned char* __restrict__ b_scales,
                                                                void* __restrict__ c, int m, int n, int k) {
    constexpr int kTileBytes = 4096, kStepBytes = kM * kTileBytes;  // of A: 16 rows by 128
    __shared__ __attribute__((aligned(1024))) unsigned char smem[kWhole<kM> * 2 * kStepBytes];
    static_assert(sizeof smem >= sizeof(f32x4) * kWhole<kM> * kM * kN * 64);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int r = lane % 16, q = lane / 16, steps = padded(k) / kStep, row_bytes = padded(k) / 2;
    const long long col0 = static_cast<long long>(blockIdx.x) * 16 * kN;
    MX4_LDS unsigned char* const mine = (MX4_LDS unsigned char*)(smem) + wave * 2 * kStepBytes;
    // To the last row's last dword; rows past it read as zeros.
    const __amdgpu_buffer_rsrc_t rows = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<void*>(a), 0, (2 * ((m - 1) * lda + k) + 3) & ~3, 0x00020000);
    const int a_at = 2 * (lane / 4 * lda + 8 * (lane % 4 ^ lane / 16)), a_from = 64 * r + 16 * (q ^ r / 4);
    const int from = (4 * r + q) * 4;  // where a column's dword q was loaded
    __amdgpu_buffer_rsrc_t codes[kN];
    const unsigned char* scale_row = b_scales;
    const int at = lane / 4 * row_bytes + lane % 4 * 4;
#pragma unroll
    for (int j = 0; j < kN; ++j) {
        const long long col = col0 + 16 * j < n ? col0 + 16 * j : 0, left = n - col;
        codes[j] = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(b_codes + col * row_bytes), 0,
                                                     (left < 16 ? static_cast<int>(left) : 16) * row_bytes, 0x00020000);
        if (q == j) scale_row = b_scales + (col + (r < left ? r : 0)) * (padded(k) / 32);
    }
    f32x4 acc[kM * kN];
#pragma unroll
    for (int i = 0; i < kM * kN; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    struct Step {
        unsigned w[kN][4], scales;  // lane 16 j + r: of column r of tile j
    } now, next;
    const auto load = [&](int t, int half) {
#pragma unroll
        for (int i = 0; i < kM; ++i)
#pragma unroll
            for (int s = 0; s < 4; ++s)
                buffer_to_lds(rows, mine + half * kStepBytes + i * kTileBytes + s * 1024, a_at + 32 * lda * i + 64 * s, t * 256);
#pragma unroll
        for (int j = 0; j < kN; ++j)
#pragma unroll
            for (int s = 0; s < 4; ++s)
                next.w[j][s] = __builtin_amdgcn_raw_buffer_load_b32(codes[j], at + 16 * s, t * 64, 0);
        next.scales = q < kN ? *reinterpret_cast<const unsigned*>(scale_row + t * 4) : 0u;
    };
    const auto of_column = [&](int j, int column, unsigned v) {
        return static_cast<unsigned>(__builtin_amdgcn_ds_bpermute((16 * j + column) * 4, static_cast<int>(v)));
    };
    // A scale of 255 in lane's column (high bits of bytes); the tiles in whose column r the lane met a weight past
    // fp32's largest number (its products might fit the sums, but are not finite in the other kernels).
    unsigned nans = 0, past = 0;
    int t = wave, half = 0;
    if (t < steps) load(t, 0);
    while (t < steps) {
        const int then = t + kWhole<kM>;
        // This step has landed; the reads of the other half are over.
        __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0), lgkmcnt(0)
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        now = next;
        if (then < steps) load(then, half ^ 1);
        if ((t + 1) * kStep > k) {  // the next row's elements, or a gap's, to zeros
#pragma unroll 1
            for (int i = 0; i < 4 * kM; ++i) {
                MX4_LDS u32x4* const of_row = reinterpret_cast<MX4_LDS u32x4*>(mine + half * kStepBytes + i * 1024 + a_from);
                u32x4 x = *of_row;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int at_k = t * kStep + i % 4 * 32 + 8 * q + 2 * e;
                    x[e] &= (at_k < k ? 0xffffu : 0u) | (at_k + 1 < k ? 0xffff0000u : 0u);
                }
                *of_row = x;
            }
        }
        // Scales from 253 up: of no number, or past the type with some codes.
        if constexpr (kIn == kF16) {
            if (__ballot(((now.scales & 0x7f7f7f7fu) + 0x03030303u) & now.scales & 0x80808080u) != 0) {
                nans |= (~now.scales - 0x01010101u) & now.scales & 0x80808080u;
#pragma unroll
                for (int j = 0; j < kN; ++j) {
                    const unsigned of_row = of_column(j, r, now.scales);
#pragma unroll
                    for (int s = 0; s < 4; ++s) {
                        const unsigned w = static_cast<unsigned>(__builtin_amdgcn_ds_bpermute(from, static_cast<int>(now.w[j][s])));
                        const unsigned byte = of_row >> 8 * s & 255u, four = w & 0x44444444u;  // 2, 3, 4 and 6
                        if (byte == 254u ? four != 0 : byte == 253u && (four & w << 1) != 0) past |= 1u << j;
                    }
                }
            }
        }
        unsigned scales[kN][kIn == kF16 ? 4 : 1];
#pragma unroll
        for (int j = 0; j < kN; ++j) {
            if constexpr (kIn == kF16) {
#pragma unroll
                for (int v = 0; v < 4; ++v) scales[j][v] = of_column(j, 4 * q + v, now.scales);
            } else {
                scales[j][0] = of_column(j, r, now.scales);
            }
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            u32x4 x[kM];
#pragma unroll
            for (int i = 0; i < kM; ++i)
                x[i] = *reinterpret_cast<const MX4_LDS u32x4*>(mine + half * kStepBytes + i * kTileBytes + s * 1024 + a_from);
#pragma unroll
            for (int j = 0; j < kN; ++j) {
                const unsigned w = static_cast<unsigned>(__builtin_amdgcn_ds_bpermute(from, static_cast<int>(now.w[j][s])));
                if constexpr (kIn == kF16) {
                    const u32x4 of_codes = decode_eight_f16(w);
                    f32x4 scale;
#pragma unroll
                    for (int v = 0; v < 4; ++v) {
                        // 2^(byte - 127), of byte 0 too.
                        const unsigned bits = (s < 3 ? scales[j][v] << (23 - 8 * s) : scales[j][v] >> 1) & 0x7f800000u;
                        scale[v] = __builtin_bit_cast(float, bits > 0x00400000u ? bits : 0x00400000u);
                    }
#pragma unroll
                    for (int i = 0; i < kM; ++i) {
                        const f32x4 sum = mfma_f16(of_codes, x[i], f32x4{0.0f, 0.0f, 0.0f, 0.0f});
#pragma unroll
                        for (int v = 0; v < 4; ++v)
                            acc[i * kN + j][v] = __builtin_fmaf(sum[v], scale[v], acc[i * kN + j][v]);
                    }
                } else {
                    const u32x4 scaled = decode_eight(w, scale_operand(scales[j][0] >> 8 * s & 255u));
#pragma unroll
                    for (int i = 0; i < kM; ++i) acc[i * kN + j] = mfma_bf16(scaled, x[i], acc[i * kN + j]);
                }
            }
        }
        t = then;
        half ^= 1;
    }
    if constexpr (kIn == kF16) {
        if (__ballot(past != 0) != 0) {
            past |= static_cast<unsigned>(__shfl_xor(static_cast<int>(past), 16));
            past |= static_cast<unsigned>(__shfl_xor(static_cast<int>(past), 32));
            nans |= past >> q & 1u;
        }
#pragma unroll
        for (int j = 0; j < kN; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const bool nan = of_column(j, 4 * q + v, nans) != 0;
#pragma unroll
                for (int i = 0; i < kM; ++i)
                    acc[i * kN + j][v] = nan ? __builtin_nanf("") : acc[i * kN + j][v];
            }
    }
    __syncthreads();  // all have read their A
    sum_waves<kWhole<kM>>(acc, reinterpret_cast<f32x4*>(smem), wave, lane, [&](int i, f32x4 sum) {
        const int row = 16 * (i / kN) + r;
        const long long col = col0 + 16 * (i % kN) + 4 * q;
        if (row < m && col < n)
            store_four<kOut>(c, static_cast<long long>(row) * n + col, sum, static_cast<int>(n - col < 4 ? n - col : 4));
    });
}

// ---------------------------------------------------------------- pieces

// A lane a row's eight elements; neighbouring lanes neighbouring rows, so that
// the pieces are written in whole lines.
template <int kIn>
__global__ __launch_bounds__(256) void cut_rows(const void* __restrict__ a, long long lda, unsigned short* __restrict__ out,
                                                int m, int rows, int k, int chunks) {
    constexpr int kP = kPieces<kIn>;
    const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x, all = static_cast<long long>(rows) * chunks;
    if (i >= all) return;
    const int row = static_cast<int>(i % rows), e = static_cast<int>(i / rows) * 8;
    float v[8];
    load_eight<kIn>(a, row < m ? row * lda + e : 0, row < m ? k - e : 0, v);
    u32x4 x[kP];
    cut_eight<kP>(v, x);
#pragma unroll
    for (int p = 0; p < kP; ++p) *reinterpret_cast<u32x4*>(out + (p * all + i) * 8) = x[p];
}

// 16 kM rows by 16 kN columns of C per block, A in pieces (`rows` of them, a
// multiple of 16). A step's pieces are loaded before the next step's weights,
// because loads arrive in order; where they would take too many registers, by
// instruction. Bound by A's pieces, which every block reads from its L2 (at most
// 64 bytes a cycle): 300x1001x1023 fp32 in 7.1 us after 3.7 of cutting.
template <int kPieceRows, int kN>
struct Direct {
    static constexpr bool kPiecesFirst = kPieceRows <= 4;
    static constexpr int kWaves = kPieceRows <= 2 || (kPieceRows <= 4 && kN == 1) ? 16 : 8;  // as the registers allow
};

template <typename Shape, int kP, int kM, int kN, int kOut>
__global__ __launch_bounds__(64 * Shape::kWaves) void weights_direct(const unsigned short* __restrict__ a,
                                                              const unsigned char* __restrict__ b_codes,
                                                              const unsigned char* __restrict__ b_scales,
                                                              void* __restrict__ c, int m, int rows, int n, int k,
                                                              unsigned tiles_n) {
    constexpr int kW = Shape::kWaves;
    __shared__ f32x4 space[kW * kM * kN * 64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int r = lane % 16, q = lane / 16, steps = padded(k) / kStep;
    const int row0 = static_cast<int>(blockIdx.x / tiles_n) * 16 * kM;
    const long long col0 = static_cast<long long>(blockIdx.x % tiles_n) * 16 * kN;
    Rows<kMx4, kN> b;
    b.open(b_codes, b_scales, k, n, [&](int j) { return col0 + 16 * j < n ? col0 + 16 * j : 0; });
    const unsigned short* x[kM];
#pragma unroll
    for (int i = 0; i < kM; ++i) {
        const int row = row0 + 16 * i < rows ? row0 + 16 * i + r : r;
        x[i] = a + (static_cast<long long>(4 * q) * rows + row) * 8;
    }
    const long long plane = static_cast<long long>(rows) * padded(k), chunk = 8LL * rows;
    f32x4 acc[kM * kN];
#pragma unroll
    for (int i = 0; i < kM * kN; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    typename Rows<kMx4, kN>::Step now, next;
    if (wave < steps) b.load(wave, next);
    for (int t = wave; t < steps; t += kW) {
        now = next;
        u32x4 xs[4][kM][kP];
        const auto load = [&](int e) {
#pragma unroll
            for (int i = 0; i < kM; ++i)
#pragma unroll
                for (int p = 0; p < kP; ++p)
                    xs[e][i][p] = *reinterpret_cast<const u32x4*>(x[i] + p * plane + (t * 16 + e) * chunk);
        };
        if constexpr (Shape::kPiecesFirst) {
#pragma unroll
            for (int e = 0; e < 4; ++e) load(e);
        }
        if (t + kW < steps) b.load(t + kW, next);
        float scale[kN];
#pragma unroll
        for (int j = 0; j < kN; ++j) scale[j] = scale_operand(b.scale(now, j));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if constexpr (!Shape::kPiecesFirst) load(e);
#pragma unroll
            for (int j = 0; j < kN; ++j) {
                const u32x4 w = decode_eight(b.pass(now.w[j][0][e]), scale[j]);
#pragma unroll
                for (int i = 0; i < kM; ++i)
#pragma unroll
                    for (int p = 0; p < kP; ++p) acc[i * kN + j] = mfma_bf16(w, xs[e][i][p], acc[i * kN + j]);
            }
        }
    }
    sum_waves<kW>(acc, space, wave, lane, [&](int i, f32x4 sum) {
        const int row = row0 + 16 * (i / kN) + r;
        const long long col = col0 + 16 * (i % kN) + 4 * q;
        if (row < m && col < n)
            store_four<kOut>(c, static_cast<long long>(row) * n + col, sum, static_cast<int>(n - col < 4 ? n - col : 4));
    });
}

// ---------------------------------------------------------------- large tiles

constexpr int kTile = 128, kTileThreads = 256;
constexpr int kStageA = 16 * 1024, kStagesA = 3;
constexpr int kStageB = 8 * 1024 + 512;  // codes, then a dword of scales per row
constexpr int kLdsBytes = kStagesA * kStageA + 2 * kStageB;

// 128x128 tiles by 4 waves in a 2x2 grid, each a 64x64 quadrant as 4x4
// accumulators; two blocks per CU, so that one multiplies while the other
// waits. A step of 128 k brings one stage of B (codes and scales), decoded once
// into registers, and 2 kP stages of A, each a piece's half of the chunks (those
// of instructions 0 and 1, then 2 and 3: chunks 4 q + 2 h and 4 q + 2 h + 1).
//
// LDS: A as [8 chunks][128 rows][16 bytes], as it lies in memory, a fetch
// instruction 64 rows of a chunk, a fragment read 16 rows of four chunks, no bank
// twice per 16 lanes; B's rows of 64 bytes, block c at c ^ (r / 2 % 4). One
// barrier per stage: stage i has landed and stage i - 1 has been read, so i + 2
// is fetched over it. 4096x14336x4096 bf16 in 420 us (1.15 PFLOP/s), 768x4096x4096
// bf16 in 42.
template <int kP, int kOut>
__global__ __launch_bounds__(kTileThreads, 2) void weights_tiles(const unsigned short* __restrict__ a,
                                                                 const unsigned char* __restrict__ b_codes,
                                                                 const unsigned char* __restrict__ b_scales,
                                                                 void* __restrict__ c, int m, int rows, int n, int k,
                                                                 int tiles_n) {
    __shared__ __attribute__((aligned(1024))) unsigned char smem[kLdsBytes];
    MX4_LDS unsigned char* lds = (MX4_LDS unsigned char*)(smem);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int r = lane % 16, q = lane / 16;
    const int kp = padded(k), steps = kp / kStep, stages = steps * 2 * kP;
    const int row0 = static_cast<int>(blockIdx.x) / tiles_n * kTile, col0 = static_cast<int>(blockIdx.x) % tiles_n * kTile;

    // What lies past the operands reads as zeros.
    const int a_left = rows - row0 < kTile ? rows - row0 : kTile, b_left = n - col0 < kTile ? n - col0 : kTile;
    const long long plane = static_cast<long long>(rows) * kp;
    const unsigned char* b_tile = b_codes + static_cast<long long>(col0) * (kp / 2);
    const __amdgpu_buffer_rsrc_t b_rsrc =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(b_tile), 0, b_left * (kp / 2), 0x00020000);
    const __amdgpu_buffer_rsrc_t s_rsrc = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<unsigned char*>(b_scales + static_cast<long long>(col0) * (kp / 32)), 0, b_left * (kp / 32), 0x00020000);
    // Waves 2 i and 2 i + 1 fetch rows 0-63 and 64-127 of chunks 4 j + 2 h + i, j = 0..3.
    const int a_row = wave % 2 * 64 + lane;
    const int b_src = (wave * 32 + lane / 4) * (kp / 2) + (lane % 4 ^ lane / 8 % 4) * 16;

    const auto fetch_a = [&](int i) {
        const int t = i / (2 * kP), p = i % (2 * kP) / 2, h = i % 2;
        MX4_LDS unsigned char* to = lds + i % kStagesA * kStageA;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int chunk = 4 * j + 2 * h + wave / 2;
            const unsigned short* from = a + p * plane + (static_cast<long long>(t * 16 + chunk) * rows + row0) * 8;
            const __amdgpu_buffer_rsrc_t rsrc =
                __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned short*>(from), 0, a_left * 16, 0x00020000);
            buffer_to_lds(rsrc, to + (2 * j + wave / 2) * 2048 + wave % 2 * 1024, a_row * 16, 0);
        }
    };
    const auto fetch_b = [&](int t) {
        MX4_LDS unsigned char* to = lds + kStagesA * kStageA + (t & 1) * kStageB;
#pragma unroll
        for (int j = 0; j < 2; ++j) buffer_to_lds(b_rsrc, to + (wave * 2 + j) * 1024, b_src + j * 16 * (kp / 2), t * 64);
        if (wave < 2)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(s_rsrc, reinterpret_cast<MX4_LDS void*>(to + 8192 + wave * 256), 4,
                                                     (wave * 64 + lane) * (kp / 32), t * 4, 0, 0);
    };

    f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const int wave_row = wave / 2 * 64, wave_col = wave % 2 * 64;
    fetch_b(0);
    fetch_a(0);
    fetch_a(1);
    int i = 0;
    for (int t = 0; t < steps; ++t) {
        u32x4 w[4][4];
#pragma unroll
        for (int part = 0; part < 2 * kP; ++part, ++i) {
            // Stage i (and this step's B, fetched before) has landed once the four fetches of i + 1 are left;
            // this wave's reads of stage i - 1 are over.
            __builtin_amdgcn_s_waitcnt(0x0074);  // vmcnt(4), lgkmcnt(0)
            lds_barrier();
            if (part == 0 && t + 1 < steps) fetch_b(t + 1);
            fetch_a(i + 2 < stages ? i + 2 : stages - 1);
            const MX4_LDS unsigned char* from = lds + i % kStagesA * kStageA;
            if (part == 0) {
                const MX4_LDS unsigned char* b = lds + kStagesA * kStageA + (t & 1) * kStageB;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int row = wave_col + 16 * j + r;
                    const u32x4 codes = *reinterpret_cast<const MX4_LDS u32x4*>(b + row * 64 + (q ^ r / 2 % 4) * 16);
                    const float scale = scale_operand(b[8192 + row * 4 + q]);
#pragma unroll
                    for (int s = 0; s < 4; ++s) w[j][s] = decode_eight(codes[s], scale);
                }
            }
            u32x4 x[4][2];
#pragma unroll
            for (int f = 0; f < 4; ++f)
#pragma unroll
                for (int s = 0; s < 2; ++s)
                    x[f][s] = *reinterpret_cast<const MX4_LDS u32x4*>(from + (2 * q + s) * 2048 + (wave_row + 16 * f + r) * 16);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int f = 0; f < 4; ++f)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[f][j] = mfma_bf16(w[j][part % 2 * 2 + s], x[f][s], acc[f][j]);
        }
    }
    __builtin_amdgcn_s_waitcnt(0);  // no fetch may land in LDS that is another block's
#pragma unroll
    for (int f = 0; f < 4; ++f) {
        const int row = row0 + wave_row + 16 * f + r;
        if (row >= m) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int col = col0 + wave_col + 16 * j + 4 * q;
            if (col < n) store_four<kOut>(c, static_cast<long long>(row) * n + col, acc[f][j], n - col);
        }
    }
}

// ---------------------------------------------------------------- launches

struct Product {
    const void* a;
    long long lda;
    const unsigned char *b_codes, *b_scales;
    void* c;
    int m, n, k;
    unsigned short* pieces;
    hipStream_t stream;
    const char** why;
};

int too_many(const Product& p) {
    *p.why = "more tiles of C than one launch takes";
    return hipErrorInvalidValue;
}

long long tiles(long long size, int tile) { return (size + tile - 1) / tile; }
int piece_rows(int m) { return (m + 15) / 16 * 16; }

template <int kIn, int kN, int kOut>
int launch_few(const Product& p) {
    const long long size = kSize<kIn>;
    const bool loose = !aligned(p.a, 4) || p.lda * size % 4 != 0 || ((p.m - 1) * p.lda + p.k) * size > 0x7fffff00LL;
    const long long blocks = tiles(p.n, 16 * kN);
    if (!fits_launch(blocks, kFewWaves * 64)) return too_many(p);
    const auto go = [&](auto kernel) {
        return launch_kernel(kernel, static_cast<unsigned>(blocks), kFewWaves * 64, 0, p.stream, p.a, p.lda, p.b_codes,
                             p.b_scales, p.c, p.m, p.n, p.k);
    };
    if (loose) return go(weights_few<kIn, kN, kOut, true>);
    return go(weights_few<kIn, kN, kOut, false>);
}

template <int kIn, int kM, int kN, int kOut>
int launch_whole(const Product& p) {
    const long long blocks = tiles(p.n, 16 * kN);
    if (!fits_launch(blocks, kWhole<kM> * 64)) return too_many(p);
    return launch_kernel(weights_whole<kIn, kM, kN, kOut>, static_cast<unsigned>(blocks), kWhole<kM> * 64, 0, p.stream, p.a,
                         static_cast<int>(p.lda), p.b_codes, p.b_scales, p.c, p.m, p.n, p.k);
}

// A's pieces, once the launch that multiplies them is known to fit.
template <int kP>
int cut_a(const Product& p) {
    constexpr int kIn = kP == 1 ? kBf16 : kP == 2 ? kF16 : kF32;
    const int rows = piece_rows(p.m), chunks = padded(p.k) / 8;
    const long long blocks = tiles(static_cast<long long>(rows) * chunks, 256);
    if (!fits_launch(blocks, 256)) {
        *p.why = "more of A than one launch cuts into pieces";
        return hipErrorInvalidValue;
    }
    return launch_kernel(cut_rows<kIn>, static_cast<unsigned>(blocks), 256, 0, p.stream, p.a, p.lda, p.pieces, p.m, rows, p.k,
                         chunks);
}

template <int kP, int kM, int kN, int kOut>
int launch_direct(const Product& p) {
    typedef Direct<kP * kM, kN> Shape;
    const long long tn = tiles(p.n, 16 * kN), blocks = tiles(p.m, 16 * kM) * tn;
    if (!fits_launch(blocks, 64 * Shape::kWaves)) return too_many(p);
    if (const int rc = cut_a<kP>(p); rc != hipSuccess) return rc;
    return launch_kernel(weights_direct<Shape, kP, kM, kN, kOut>, static_cast<unsigned>(blocks), 64 * Shape::kWaves, 0,
                         p.stream, p.pieces, p.b_codes, p.b_scales, p.c, p.m, piece_rows(p.m), p.n, p.k,
                         static_cast<unsigned>(tn));
}

template <int kP, int kOut>
int launch_pieces(const Product& p) {
    const int cus = device_cus();
    const auto blocks = [&](int bm, int bn) { return tiles(p.m, 16 * bm) * tiles(p.n, 16 * bn); };
    // 128x128 tiles: where three quarters of the CUs have one (512x4096x4096 bf16, 128 of them, in
    // 42 us, by the direct kernel in 33; fp16 64 in 76 and 27, which grows with their number).
    // (32-bit offsets from a tile's origin.)
    if (4 * blocks(8, 8) >= 3 * cus && p.k <= (1 << 22) && fits_launch(blocks(8, 8), kTileThreads)) {
        if (const int rc = cut_a<kP>(p); rc != hipSuccess) return rc;
        return launch_kernel(weights_tiles<kP, kOut>, static_cast<unsigned>(blocks(8, 8)), kTileThreads, 0, p.stream, p.pieces,
                             p.b_codes, p.b_scales, p.c, p.m, piece_rows(p.m), p.n, p.k,
                             static_cast<int>(tiles(p.n, kTile)));
    }
    if constexpr (kP < 3) {  // three pieces of 64 rows do not fit the registers
        if (p.m > 32 && blocks(4, 2) >= cus) return launch_direct<kP, 4, 2, kOut>(p);
    }
    if (blocks(2, 2) >= cus) return launch_direct<kP, 2, 2, kOut>(p);
    return launch_direct<kP, 2, 1, kOut>(p);
}

template <int kIn, int kOut>
int launch(const Product& p) {
    // One block of these runs on a CU at a time. Rounds of blocks, each as
    // long as its columns and a fixed part take: one row by 14336 columns of
    // k = 4096, 64 per block, in 8.9 us, 32 (two rounds) in 11.4.
    const auto cost = [&](int wide) { return tiles(tiles(p.n, 16 * wide), device_cus()) * (2 * wide + 3); };
    if constexpr (kIn != kF32) {
        // (32-bit offsets over all rows.)
        if (p.m <= kWholeRows && aligned(p.a, 4) && p.lda % 2 == 0 && p.lda < (p.m <= 32 ? 1 << 25 : 1 << 23)) {
            const bool by_16 = cost(1) <= cost(2) && cost(1) <= cost(4);
            if (p.m > 32) {
                // One round, four steps per wave: 64 fp16 rows by 6144x2048 in 10.7 us (11.5 in two launches), bf16
                // 7.7 (9.8), 33 by 1024x1024 4.8 (7.1). By 4096x4096, eight steps for each of the four
                // waves, 13.3 (11.4).
                if (p.k <= 2048 && tiles(p.n, 32) <= device_cus())
                    return by_16 ? launch_whole<kIn, 4, 1, kOut>(p) : launch_whole<kIn, 4, 2, kOut>(p);
            } else if (p.m > 16) {
                if (by_16) return launch_whole<kIn, 2, 1, kOut>(p);
                if (cost(4) < cost(2)) return launch_whole<kIn, 2, 4, kOut>(p);
                return launch_whole<kIn, 2, 2, kOut>(p);
            }
            if (p.m <= 16 && by_16 && p.k > kWhole<1> * kStep && (kIn == kF16 || p.m >= 8)) {
                // From a wave's second step on; weights_few's short code is faster below (12 rows by 1000x1000
                // in 4.1 us, 4.6 here), for wide blocks (16 fp16 rows by 14336x4096: 11.3 and 13.9), and for bf16
                // rows that are too few to crowd its loads (2 by 4096x4096: 4.3 and 5.1; 8: 5.4 and 5.0).
                return launch_whole<kIn, 1, 1, kOut>(p);
            }
        }
    }
    if (p.m <= kFew) {
        if constexpr (kIn != kF32) {  // fp32 rows by 64 columns do not fit the registers
            if (cost(4) < cost(2) && cost(4) < cost(1)) return launch_few<kIn, 4, kOut>(p);
        }
        if (cost(2) < cost(1)) return launch_few<kIn, 2, kOut>(p);
        return launch_few<kIn, 1, kOut>(p);
    }
    return launch_pieces<kPieces<kIn>, kOut>(p);
}

template <int kIn>
int launch_out(int c_dtype, const Product& p) {
    if (c_dtype == kF32) return launch<kIn, kF32>(p);
    if (c_dtype == kBf16) return launch<kIn, kBf16>(p);
    return launch<kIn, kF16>(p);
}

}  // namespace

extern "C" {

long long mchip_matmul_mx4_weights_workspace_bytes(int a_dtype, int m, int n, int k) {
    if (!is_float_type(a_dtype) || m <= kFew || n < 1 || k < 1 || k > (1 << 24)) return 0;
    const int pieces = a_dtype == kF32 ? kPieces<kF32> : a_dtype == kBf16 ? kPieces<kBf16> : kPieces<kF16>;
    return 2LL * pieces * ((static_cast<long long>(m) + 15) / 16 * 16) * padded(k);
}

int mchip_launch_matmul_mx4_weights(int a_dtype, const void* a, long long lda, const void* b_codes,
                                    const void* b_scales, int c_dtype, void* c, int m, int n, int k, void* stream,
                                    void* workspace, const char** why) {
    *why = nullptr;
    if (!is_float_type(a_dtype) || !is_float_type(c_dtype)) *why = "a type that is none of fp32 (0), bf16 (1), fp16 (2)";
    else if (m < 1 || n < 1 || k < 1) *why = "a size below 1";
    else if (m > (1 << 30)) *why = "m above 2^30";
    else if (k > (1 << 24)) *why = "k above 2^24";
    else if (lda < k) *why = "rows of A closer together than they are long";
    else if (!a || !b_codes || !b_scales || !c) *why = "a null operand";
    else if (!aligned(b_codes, 16)) *why = "codes not 16-byte aligned";
    else if (!aligned(b_scales, 4)) *why = "scales not 4-byte aligned";
    else if (!aligned(a, size_of(a_dtype)) || !aligned(c, size_of(c_dtype)))
        *why = "an address that is no multiple of its element's size";
    else if (m > kFew && (workspace == nullptr || !aligned(workspace, 256)))
        *why = "no workspace, or one that is not 256-byte aligned";
    if (*why != nullptr) return hipErrorInvalidValue;
    Product p{a, lda, static_cast<const unsigned char*>(b_codes), static_cast<const unsigned char*>(b_scales),
              c, m, n, k, static_cast<unsigned short*>(workspace), static_cast<hipStream_t>(stream), why};
    return a_dtype == kF32    ? launch_out<kF32>(c_dtype, p)
           : a_dtype == kBf16 ? launch_out<kBf16>(c_dtype, p)
                              : launch_out<kF16>(c_dtype, p);
}

}  // extern "C"

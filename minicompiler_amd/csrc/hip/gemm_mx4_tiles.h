// The large-tile body of the product of two mx4 operands (gemm_mx4.hip).
//
// Block tile 256x256 (or 128x256) by 4 waves in a 2x2 grid, one per SIMD, each
// a 128x128 quadrant as 8x8 accumulators (256 registers). One block per CU. The
// 16x16x128 instruction takes 16 cycles for two 1 KiB fragments, so LDS and the
// caches have to feed it four times as fast per element as bf16: the quadrant
// is as large as the registers allow (a third fewer LDS reads than the 128x64
// quadrants of 8 waves), and a fetch takes whole 128-byte lines (64-byte pieces,
// 128 k per row, were twice the requests to L2: 8192^3 in 286 us with both).
//
// K goes in stages of 256 through two 64 KiB LDS buffers, each stage as two
// steps of 128, each step as 8 rows of 8 products. While a step's products
// issue, the next step's fragments are read from LDS: B's into registers of
// their own, A's row i into row i's once its products have issued. In the second
// step of stage s, after two rows, one barrier: every wave has read all of
// stage s and its own share of stage s + 1 has landed, so after it stage s + 2 is
// fetched over stage s, and stage s + 1 is read.
//
// LDS layout of a stage: rows of 128 bytes, A's 256 at 0 and B's at 32 KiB; block
// c of row r lies at 128 r + 16 (c ^ (r / 2 % 8)). A fetch instruction fills 8
// rows, eight neighbouring lanes one row (the address unit takes neighbours'
// 16 bytes together; a lane per row made an access of each lane). A fragment
// read, lane (r, q) block q of row r, touches every bank once per 16 lanes
// that the LDS serves together (lanes 0-3, 12-15 and 20-27 the first).
//
// Scales: a row has 4 bytes per step. A lane takes 16 bytes of a row, four
// steps' worth, two lanes 8 steps (a window), and turns them (four steps of four
// blocks) into four blocks' dwords of four steps each, in one of two 16 KiB
// slots of LDS. A lane then reads one dword per fragment for four steps and the
// instruction picks the step's byte. (Read from LDS a byte per fragment and
// step, the scales took 50 of 332 us at 8192^3.) A row's last 16 bytes are
// loaded whole where its end falls inside a window, so nothing is read outside
// the operand (K >= 512).
//
// Measured, bf16 out: 4096x14336x4096 137-142 us (3.4-3.5 PFLOP/s), 8192^3
// 250-265 us (4.1-4.4). A loop of the instruction alone, on random data in
// registers, runs at 7.4 PFLOP/s: the chip lowers its clock (1.9 GHz here). With
// the fetch left out the loop's matrix units are busy 64% instead of 57%, with
// the scales' work left out as well 70%, and 72% without LDS reads; the rest is
// a tile's start and its store, which all blocks do at one time (13 of 250 us,
// four tiles to a CU). In a tile's last two stages the fetches repeat its last
// stage, where a next tile's first two could come.
// 8 waves with quadrants of 128x64 took 261 us where 4 took 254.
#pragma once

#include "mx4_device.h"

namespace mx4 {

template <int kValue>
struct Constant {
    static constexpr int value = kValue;
};

constexpr int kTileRows = 256, kTileCols = 256, kTileThreads = 256;
constexpr int kStageBytes = 64 * 1024, kStageB = 32 * 1024;
constexpr int kSlotBytes = 16 * 1024, kSlotHalf = 8 * 1024, kSlotB = 4 * 1024;
constexpr int kRingBytes = 2 * kStageBytes + 2 * kSlotBytes;
constexpr int kColFrags = 8;

// `rows` rows of `row_bytes` from p on; what lies past them reads as zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_of(const unsigned char* p, int rows, int row_bytes) {
    const int most = rows < kTileRows ? rows : kTileRows;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p), 0, most * row_bytes, 0x00020000);
}

template <int kRows>
struct TileLane {
    static constexpr int kRowFrags = kRows / 32;  // of a wave
    static constexpr int kFetchA = kRows / 32;    // instructions per wave and stage
    static constexpr int kFetchB = 8;
    __amdgpu_buffer_rsrc_t a, b, scales;  // codes at the tile's origin; this wave's operand's scales
    int src[2];                           // the lane's offset in a fetch of rows 16 j .. + 7 and 16 j + 8 .. + 15
    int scale_src;                        // ... in a load of 32 rows' scales
    int a_off[2], b_off[2];               // LDS offsets of the wave's first fragments in each step
    int a_scale, b_scale;                 // ... and of their scales
    int row_bytes, scale_row;             // bytes of codes and of scales in a row
    int wave, lane;
};

// Instruction i of this wave's share of stage s (A's first). Where K ends in the
// middle of the last stage, lanes past the end take the half before.
template <int kRows>
__device__ __forceinline__ void fetch_one(MX4_LDS unsigned char* wr, const TileLane<kRows>& L, int s, int i) {
    constexpr int kA = TileLane<kRows>::kFetchA, kB = TileLane<kRows>::kFetchB;
    const bool of_a = i < kA;
    const int k = of_a ? i : i - kA;
    const int at = s * 128;
    const int back = at + 128 > L.row_bytes ? ((L.lane % 8 ^ (4 * (k & 1) + L.lane / 16)) & 4) * 16 : 0;
    const int part = L.wave * (of_a ? kA : kB) + k;  // eight rows
    buffer_to_lds(of_a ? L.a : L.b, wr + (of_a ? 0 : kStageB) + part * 1024, L.src[k & 1] - back,
                  part * 8 * L.row_bytes + at);
}

// Instructions `from` to `to` of them.
template <int kRows>
__device__ __forceinline__ void fetch_range(MX4_LDS unsigned char* wr, const TileLane<kRows>& L, int s, int from, int to) {
    constexpr int kAll = TileLane<kRows>::kFetchA + TileLane<kRows>::kFetchB;
#pragma unroll
    for (int i = 0; i < kAll; ++i)
        if (i >= from && i < to) fetch_one<kRows>(wr, L, s, i);
}

// Part n % 4 of window n / 4: 32 rows' scales of 8 steps, a lane 16 bytes as
// they lie in the row, moved back where the row ends inside.
template <int kRows>
__device__ __forceinline__ int scale_at(const TileLane<kRows>& L, int n) {
    return n / 4 * 32 + L.lane % 2 * 16;
}
template <int kRows>
__device__ __forceinline__ u32x4 load_scales(const TileLane<kRows>& L, int n) {
    const int at = scale_at<kRows>(L, n), last = L.scale_row - 16;
    return __builtin_bit_cast(
        u32x4, __builtin_amdgcn_raw_buffer_load_b128(L.scales, L.scale_src + (at < last ? at : last),
                                                     (L.wave % 2 * 128 + n % 4 * 32) * L.scale_row, 0));
}

// A window's slot: [steps 0-3, steps 4-7][256 rows of A, 256 of B][16 bytes].
// Bytes of steps past the end are zeros, a scale of 2^-127 on both sides, which
// makes nothing of whatever codes they meet: an odd last step needs no branch.
// (Without branches: a product's loop is one block, or the compiler moves
// products from before a branch behind it.) In six pieces, to go between products.
template <int kRows, int kPiece>
__device__ __forceinline__ void store_scales_piece(MX4_LDS unsigned char* slots, const TileLane<kRows>& L, u32x4& v, int n) {
    const int late = (scale_at<kRows>(L, n) - (L.scale_row - 16)) / 4;  // dwords moved back, if above 0
    if constexpr (kPiece == 0) {
        const bool one = late > 0 && (late & 1);
        v = u32x4{one ? v[1] : v[0], one ? v[2] : v[1], one ? v[3] : v[2], one ? 0u : v[3]};
    } else if constexpr (kPiece == 1) {
        const bool two = late > 0 && (late & 2);
        v = u32x4{two ? v[2] : v[0], two ? v[3] : v[1], two ? 0u : v[2], two ? 0u : v[3]};
    } else if constexpr (kPiece == 2) {
        const bool past = late > 3;
        v = u32x4{past ? 0u : v[0], past ? 0u : v[1], past ? 0u : v[2], past ? 0u : v[3]};
    } else if constexpr (kPiece == 3) {
        // Pairs of steps: blocks 0 and 1 of steps 0 and 1, of 2 and 3; blocks 2 and 3.
        v = u32x4{__builtin_amdgcn_perm(v[1], v[0], 0x05010400u), __builtin_amdgcn_perm(v[3], v[2], 0x05010400u),
                  __builtin_amdgcn_perm(v[1], v[0], 0x07030602u), __builtin_amdgcn_perm(v[3], v[2], 0x07030602u)};
    } else if constexpr (kPiece == 4) {
        // Dword q: block q's bytes of the four steps.
        v = u32x4{__builtin_amdgcn_perm(v[1], v[0], 0x05040100u), __builtin_amdgcn_perm(v[1], v[0], 0x07060302u),
                  __builtin_amdgcn_perm(v[3], v[2], 0x05040100u), __builtin_amdgcn_perm(v[3], v[2], 0x07060302u)};
    } else {
        const int row = (L.wave / 2 * 256) + (L.wave % 2 * 128) + n % 4 * 32 + L.lane / 2;
        *reinterpret_cast<MX4_LDS u32x4*>(slots + (n / 4 & 1) * kSlotBytes + L.lane % 2 * kSlotHalf + row * 16) = v;
    }
}

template <int kRows>
__device__ __forceinline__ void store_scales(MX4_LDS unsigned char* slots, const TileLane<kRows>& L, u32x4 v, int n) {
    store_scales_piece<kRows, 0>(slots, L, v, n);
    store_scales_piece<kRows, 1>(slots, L, v, n);
    store_scales_piece<kRows, 2>(slots, L, v, n);
    store_scales_piece<kRows, 3>(slots, L, v, n);
    store_scales_piece<kRows, 4>(slots, L, v, n);
    store_scales_piece<kRows, 5>(slots, L, v, n);
}

// One fragment of step u of the stage at `rd`, and a fragment's scales of four
// steps. The regions read are not being written; __restrict__ says so, or the
// compiler would wait for the fetches in flight.
template <int kRows>
__device__ __forceinline__ i32x4 read_a(const MX4_LDS unsigned char* __restrict__ rd, const TileLane<kRows>& L, int u,
                                        int f) {
    return *reinterpret_cast<const MX4_LDS i32x4*>(rd + L.a_off[u] + f * 2048);
}
template <int kRows>
__device__ __forceinline__ i32x4 read_b(const MX4_LDS unsigned char* __restrict__ rd, const TileLane<kRows>& L, int u,
                                        int f) {
    return *reinterpret_cast<const MX4_LDS i32x4*>(rd + kStageB + L.b_off[u] + f * 2048);
}
template <int kRows>
__device__ __forceinline__ int read_scale_a(const MX4_LDS unsigned char* __restrict__ rd, const TileLane<kRows>& L,
                                            int f) {
    return *reinterpret_cast<const MX4_LDS int*>(rd + L.a_scale + f * 256);
}
template <int kRows>
__device__ __forceinline__ int read_scale_b(const MX4_LDS unsigned char* __restrict__ rd, const TileLane<kRows>& L,
                                            int f) {
    return *reinterpret_cast<const MX4_LDS int*>(rd + kSlotB + L.b_scale + f * 256);
}

// acc += a b in acc's own registers. Written out, because the compiler, with the
// products held in their places, gives them other registers and copies (8192^3
// in 311 us); it also keeps asm statements in their order. What it no longer
// knows: a value is there only after the instruction's passes (settle()).
template <int kByte>
__device__ __forceinline__ void mfma_in_place(f32x4& acc, i32x4 a, int sa, i32x4 b, int sb) {
    if constexpr (kByte == 0)
        asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0] cbsz:4 blgp:4"
                     : "+a"(acc)
                     : "v"(a), "v"(b), "v"(sa), "v"(sb));
    else if constexpr (kByte == 1)
        asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[0,0,0] cbsz:4 blgp:4"
                     : "+a"(acc)
                     : "v"(a), "v"(b), "v"(sa), "v"(sb));
    else if constexpr (kByte == 2)
        asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[1,1,0] cbsz:4 blgp:4"
                     : "+a"(acc)
                     : "v"(a), "v"(b), "v"(sa), "v"(sb));
    else
        asm volatile("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[1,1,0] op_sel_hi:[1,1,0] cbsz:4 blgp:4"
                     : "+a"(acc)
                     : "v"(a), "v"(b), "v"(sa), "v"(sb));
}

// Between the last product and the first use of its value: its passes are over.
__device__ __forceinline__ void settle() {
    asm volatile("s_nop 15\n s_nop 15" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// A wave's accumulators, first row and column (row, col): lane (r, q) holds
// C[row + 16 i + r][col + 16 j + 4 q + v]. eights: N is a multiple of 8.
template <int kRowFrags, int kOut>
__device__ __forceinline__ void store_tile(const f32x4 (&acc)[kRowFrags][kColFrags], void* c, int row, int col, int m,
                                           int n, int lane, bool eights) {
    const int r = lane % 16, q = lane / 16;
    if constexpr (kOut != kF32) {
        // Eight columns per lane, so that no lane straddles the edge: odd rows of 16
        // lanes of one fragment change places with even rows of its neighbour.
        if (eights) {
#pragma unroll
            for (int i = 0; i < kRowFrags; ++i)
#pragma unroll
                for (int j = 0; j < kColFrags; j += 2) {
                    u32x4 out;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const unsigned x = to_16<kOut>(acc[i][j][2 * e]) | to_16<kOut>(acc[i][j][2 * e + 1]) << 16;
                        const unsigned y =
                            to_16<kOut>(acc[i][j + 1][2 * e]) | to_16<kOut>(acc[i][j + 1][2 * e + 1]) << 16;
                        const u32x2 s = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(x, y, false, false));
                        out[e] = s[0];
                        out[2 + e] = s[1];
                    }
                    const int at_row = row + 16 * i + r, at_col = col + 16 * (j + (q & 1)) + 8 * (q >> 1);
                    if (at_row < m && at_col < n)
                        *reinterpret_cast<u32x4_loose*>(static_cast<unsigned short*>(c) +
                                                  static_cast<long long>(at_row) * n + at_col) = out;
                }
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < kRowFrags; ++i) {
        const int at_row = row + 16 * i + r;
        if (at_row >= m) continue;
#pragma unroll
        for (int j = 0; j < kColFrags; ++j) {
            const int at_col = col + 16 * j + 4 * q;
            if (at_col < n)
                store_four<kOut>(c, static_cast<long long>(at_row) * n + at_col, acc[i][j], n - at_col);
        }
    }
}

// One kRows x 256 tile of C at (row0, col0). steps >= 4.
template <int kRows, int kOut>
__device__ __forceinline__ void product_tile(MX4_LDS unsigned char* lds, const unsigned char* a_codes,
                                             const unsigned char* a_scales, const unsigned char* b_codes,
                                             const unsigned char* b_scales, void* c, int m, int n, int steps, int row0,
                                             int col0, bool eights) {
    typedef TileLane<kRows> Lane;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int r = lane % 16, q = lane / 16;
    Lane L;
    L.wave = wave;
    L.lane = lane;
    L.row_bytes = steps * 64;
    L.scale_row = steps * 4;
    L.a = rsrc_of(a_codes + static_cast<long long>(row0) * L.row_bytes, m - row0, L.row_bytes);
    L.b = rsrc_of(b_codes + static_cast<long long>(col0) * L.row_bytes, n - col0, L.row_bytes);
    // The block that the lane's place in LDS takes, of row lane / 8 of a fetch.
#pragma unroll
    for (int i = 0; i < 2; ++i) L.src[i] = lane / 8 * L.row_bytes + (lane % 8 ^ (4 * i + lane / 16)) * 16;
    // Waves 0 and 1 see to A's scales, 2 and 3 to B's, 128 rows each.
    const bool for_a = wave < 2;
    L.scales = for_a ? rsrc_of(a_scales + static_cast<long long>(row0) * L.scale_row, m - row0, L.scale_row)
                     : rsrc_of(b_scales + static_cast<long long>(col0) * L.scale_row, n - col0, L.scale_row);
    L.scale_src = lane / 2 * L.scale_row;
    const int wave_row = wave / 2 * (kRows / 2), wave_col = wave % 2 * 128;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        L.a_off[u] = (wave_row + r) * 128 + ((4 * u + q) ^ r / 2) * 16;
        L.b_off[u] = (wave_col + r) * 128 + ((4 * u + q) ^ r / 2) * 16;
    }
    L.a_scale = (wave_row + r) * 16 + q * 4;
    L.b_scale = (wave_col + r) * 16 + q * 4;

    f32x4 acc[Lane::kRowFrags][kColFrags];
    const auto stage = [&](int s) { return lds + (s & 1) * kStageBytes; };
    MX4_LDS unsigned char* slots = lds + 2 * kStageBytes;
    const auto scales_of = [&](int s) { return slots + (s / 4 & 1) * kSlotBytes + (s / 2 & 1) * kSlotHalf; };
    const int stages = (steps + 1) / 2;

    // The scales' parts 0 to 5 and stages 0 and 1, all on their way at once; the
    // first five parts go to LDS.
    u32x4 first[5];
#pragma unroll
    for (int i = 0; i < 5; ++i) first[i] = load_scales<kRows>(L, i);
    u32x4 scales = load_scales<kRows>(L, 5);
    // The fetch of a stage is spread over the rows between two barriers and a
    // few behind the second: the address unit takes 16 cycles for an
    // instruction, and a wave that waits for it multiplies nothing.
    constexpr int kI = Lane::kRowFrags, kAll = Lane::kFetchA + Lane::kFetchB, kEarly = kAll * 5 / 8;
    fetch_range<kRows>(stage(0), L, 0, 0, kAll);
    fetch_range<kRows>(stage(1), L, 1, 0, kEarly);
#pragma unroll
    for (int i = 0; i < Lane::kRowFrags; ++i)
#pragma unroll
        for (int j = 0; j < kColFrags; ++j) {
            acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            asm volatile("" : "+a"(acc[i][j]));  // cleared here, while the fetch is under way
        }
#pragma unroll
    for (int i = 0; i < 5; ++i) store_scales<kRows>(slots, L, first[i], i);
    __builtin_amdgcn_s_waitcnt(0);
    lds_barrier();

    constexpr int kB = kColFrags / kI;
    i32x4 av[kI], bv[2][kColFrags];
    int sa[kI], sb[kColFrags], sb_next[kColFrags];
#pragma unroll
    for (int f = 0; f + 1 < kI; ++f) {
        av[f] = read_a<kRows>(lds, L, 0, f);
        sa[f] = read_scale_a<kRows>(scales_of(0), L, f);
    }
#pragma unroll
    for (int f = 0; f < kColFrags; ++f) {
        bv[0][f] = read_b<kRows>(lds, L, 0, f);
        sb[f] = read_scale_b<kRows>(scales_of(0), L, f);
    }

    // Stage s, `which` = s % 2. The part of scales stored at stage s is s + 5
    // (the fourth of a window two stages before its first use), loaded a stage
    // before. Every product is held in its place, with one piece of the other
    // work behind it: the matrix unit is busy meanwhile, and a product leaves
    // room for a few instructions; gathered between the rows they left it idle.
    const auto run = [&](int s, auto which) {
        constexpr int w = decltype(which)::value;
        const MX4_LDS unsigned char *here = stage(s), *there = stage(s + 1);
        const int rest = s + 1 < stages ? s + 1 : stages - 1, next = s + 2 < stages ? s + 2 : stages - 1;
#pragma unroll
        for (int i = 0; i < kI; ++i) {
#pragma unroll
            for (int f = 0; f < kColFrags; ++f) {
                mfma_in_place<w * 2>(acc[i][f], bv[0][f], sb[f], av[i], sa[i]);
                if (f == 0 && i == 0) {
                    av[kI - 1] = read_a<kRows>(here, L, 0, kI - 1);
                    if constexpr (w == 0) sa[kI - 1] = read_scale_a<kRows>(scales_of(s), L, kI - 1);
                }
                if (f == 0 && i > 0) av[i - 1] = read_a<kRows>(here, L, 1, i - 1);
                if (f > 0 && f <= kB) bv[1][i * kB + f - 1] = read_b<kRows>(here, L, 1, i * kB + f - 1);
                // The rest of stage s + 1.
                if (i < kI / 2 && f >= 4) {
                    const int from = kEarly + i * (kAll - kEarly) / (kI / 2), to = kEarly + (i + 1) * (kAll - kEarly) / (kI / 2);
                    if (from + f - 4 < to) fetch_one<kRows>(stage(s + 1), L, rest, from + f - 4);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int i = 0; i < kI; ++i) {
            if (i == 2) {
                __builtin_amdgcn_s_waitcnt(0);
                lds_barrier();
            }
#pragma unroll
            for (int f = 0; f < kColFrags; ++f) {
                mfma_in_place<w * 2 + 1>(acc[i][f], bv[1][f], sb[f], av[i], sa[i]);
                if (f == 0 && i == 0) av[kI - 1] = read_a<kRows>(here, L, 1, kI - 1);
                if (i >= 2) {
                    // What is left after two rows, over the other rows.
                    constexpr int kLeft = kI - 2;
                    if (f == 0) {
                        av[i - 1] = read_a<kRows>(there, L, 0, i - 1);
                        if constexpr (w == 1) sa[i - 1] = read_scale_a<kRows>(scales_of(s + 1), L, i - 1);
                        if (i == 2) {
                            av[0] = read_a<kRows>(there, L, 0, 0);
                            if constexpr (w == 1) sa[0] = read_scale_a<kRows>(scales_of(s + 1), L, 0);
                        }
                    }
                    const int from = (i - 2) * kEarly / kLeft, to = (i - 1) * kEarly / kLeft;
                    if (f >= 4 && from + f - 4 < to) fetch_one<kRows>(stage(s), L, next, from + f - 4);
                    const int b0 = (i - 2) * kColFrags / kLeft, b1 = (i - 1) * kColFrags / kLeft;
                    if (f > 0 && b0 + f - 1 < b1) {
                        bv[0][b0 + f - 1] = read_b<kRows>(there, L, 0, b0 + f - 1);
                        if constexpr (w == 1) sb_next[b0 + f - 1] = read_scale_b<kRows>(scales_of(s + 1), L, b0 + f - 1);
                    }
                }
                if (i == 3) {
                    if (f == 0) store_scales_piece<kRows, 0>(slots, L, scales, s + 5);
                    if (f == 1) store_scales_piece<kRows, 1>(slots, L, scales, s + 5);
                    if (f == 2) store_scales_piece<kRows, 2>(slots, L, scales, s + 5);
                    if (f == 3) store_scales_piece<kRows, 3>(slots, L, scales, s + 5);
                    if (f == 4) store_scales_piece<kRows, 4>(slots, L, scales, s + 5);
                    if (f == 5) store_scales_piece<kRows, 5>(slots, L, scales, s + 5);
                    if (f == 6) scales = load_scales<kRows>(L, s + 6);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    // Two stages at a time, the four steps of a scale dword; what is past the
    // end has zero scales.
    for (int s = 0; s < stages; s += 2) {
        run(s, Constant<0>{});
        run(s + 1, Constant<1>{});
#pragma unroll
        for (int f = 0; f < kColFrags; ++f) sb[f] = sb_next[f];
        // A product's operand may have been written two instructions before it at the latest.
        asm volatile("s_nop 1" ::: "memory");
    }
    __builtin_amdgcn_s_waitcnt(0);
    settle();
#pragma unroll
    for (int i = 0; i < Lane::kRowFrags; ++i)
#pragma unroll
        for (int j = 0; j < kColFrags; ++j) asm volatile("" : "+a"(acc[i][j]));  // read behind it only
    store_tile<Lane::kRowFrags, kOut>(acc, c, row0 + wave_row, col0 + wave_col, m, n, lane, eights);
}

}  // namespace mx4

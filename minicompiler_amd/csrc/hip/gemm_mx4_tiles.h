// The large-tile body of the product of two mx4 operands (gemm_mx4.hip).
//
// Block tile 256x256 (or 128x256), 512 lanes = 8 waves in a 2x4 grid (two
// waves per SIMD), each a 128x64 quadrant as 8x4 accumulators. One block per
// CU. The schedule is that of gemm_mfma16_fast.h: K in steps of 128 through a
// ring of four 32 KiB LDS stages, the two waves of each SIMD one phase apart,
// one reading its operands from LDS while the other multiplies.
//
// LDS layout of a stage: A [16 blocks of 16 rows][4 blocks of 32 k][16 rows] of
// 16 bytes, at 0, and B likewise at 16 KiB: a fragment (16 rows, 128 k) is
// 1 KiB read linearly, lane l at 16 l, and one fetch instruction fills one
// fragment from 64 bytes of each of 16 rows.
//
// Scales: a row has four bytes per step. Fetched a step at a time, a fetch
// instruction would touch 64 rows, 64 lines, for 256 bytes; instead 16 bytes
// of each row, four steps' worth, go to one of two 8 KiB slots ([256 rows][16]
// of A, then of B) every fourth step. A row's last 16 bytes are fetched whole
// where its end falls inside a slot, so nothing is read outside the operand
// (K >= 512). A lane reads its fragment row's byte for its block.
#pragma once

#include "mx4_device.h"

namespace mx4 {

#define MX4_LDS __attribute__((address_space(3)))

constexpr int kTileRows = 256, kTileCols = 256, kTileThreads = 512;
constexpr int kStages = 4, kStageBytes = 32 * 1024, kStageB = 16 * 1024;
constexpr int kSlotBytes = 8 * 1024, kSlotB = 4 * 1024;
constexpr int kRingBytes = kStages * kStageBytes + 2 * kSlotBytes;
constexpr int kColFrags = 4;

__device__ __forceinline__ void buffer_to_lds(__amdgpu_buffer_rsrc_t rsrc, MX4_LDS unsigned char* dst, int voffset,
                                              int soffset) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, reinterpret_cast<MX4_LDS void*>(dst), 16, voffset, soffset, 0, 0);
}

// A workgroup barrier without a memory fence, which nothing is moved across.
__device__ __forceinline__ void phase_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_at(const unsigned char* p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p), 0, 0x7fffffff, 0x00020000);
}

template <int kRows>
struct TileLane {
    static constexpr int kRowFrags = kRows / 32;  // of a wave
    static constexpr int kFetchA = kRows / 128;   // instructions per wave and step
    __amdgpu_buffer_rsrc_t a, b, scales;          // codes at the tile's origin; this wave's rows' scales
    int a_src[kFetchA], b_src[2], scale_src;
    int a_off, b_off, a_scale, b_scale;  // LDS offsets of the wave's first fragments and their scales
    int scale_row;                       // bytes of scales in a row
    int wave;
};

template <int kRows>
__device__ __forceinline__ void fetch_a(MX4_LDS unsigned char* wr, const TileLane<kRows>& L, int t) {
#pragma unroll
    for (int i = 0; i < TileLane<kRows>::kFetchA; ++i)
        buffer_to_lds(L.a, wr + (L.wave * TileLane<kRows>::kFetchA + i) * 1024, L.a_src[i], t * 64);
}

template <int kRows>
__device__ __forceinline__ void fetch_b(MX4_LDS unsigned char* wr, const TileLane<kRows>& L, int t) {
#pragma unroll
    for (int i = 0; i < 2; ++i) buffer_to_lds(L.b, wr + kStageB + (L.wave * 2 + i) * 1024, L.b_src[i], t * 64);
}

// Where a slot's bytes start in a row: 16 per slot, moved back where the row ends inside.
__device__ __forceinline__ int slot_start(int slot, int scale_row) {
    const int last = scale_row - 16;
    return slot * 16 < last ? slot * 16 : last;
}

// Scales of steps 4 slot .. 4 slot + 3: waves 0-3 fetch 64 rows of A each, waves 4-7 of B.
template <int kRows>
__device__ __forceinline__ void fetch_scales(MX4_LDS unsigned char* wr, const TileLane<kRows>& L, int slot) {
    buffer_to_lds(L.scales, wr + L.wave * 1024, L.scale_src, slot_start(slot, L.scale_row));
}

// A memory phase: the fetch of A of step `next` (and of the scales of slot
// `next_slot`, if it is one), and step t's operands from LDS into registers.
// The regions written and read are distinct; __restrict__ says so, or the
// compiler would wait for the fetch before the reads.
template <int kRows>
__device__ __forceinline__ void memory_phase(const MX4_LDS unsigned char* __restrict__ rd,
                                             MX4_LDS unsigned char* __restrict__ wr,
                                             const MX4_LDS unsigned char* __restrict__ scale_rd,
                                             MX4_LDS unsigned char* __restrict__ scale_wr, const TileLane<kRows>& L,
                                             int next, int next_slot, int scale_at,
                                             i32x4 (&av)[TileLane<kRows>::kRowFrags], i32x4 (&bv)[kColFrags],
                                             int (&sa)[TileLane<kRows>::kRowFrags], int (&sb)[kColFrags]) {
    if (next_slot >= 0) fetch_scales<kRows>(scale_wr, L, next_slot);
    fetch_a<kRows>(wr, L, next);
#pragma unroll
    for (int f = 0; f < TileLane<kRows>::kRowFrags; ++f) {
        av[f] = *reinterpret_cast<const MX4_LDS i32x4*>(rd + L.a_off + f * 1024);
        sa[f] = scale_rd[L.a_scale + f * 256 + scale_at];
    }
#pragma unroll
    for (int f = 0; f < kColFrags; ++f) {
        bv[f] = *reinterpret_cast<const MX4_LDS i32x4*>(rd + kStageB + L.b_off + f * 1024);
        sb[f] = scale_rd[kSlotB + L.b_scale + f * 256 + scale_at];
    }
}

// A wave's accumulators, first row and column (row, col): lane (r, q) holds
// C[row + 16 i + r][col + 16 j + 4 q + v]. vec: how many columns N and C's
// alignment let a lane store at once (1, 4, 8).
template <int kRowFrags, int kOut>
__device__ __forceinline__ void store_tile(const f32x4 (&acc)[kRowFrags][kColFrags], void* c, int row, int col, int m,
                                           int n, int lane, int vec) {
    const int r = lane % 16, q = lane / 16;
    if constexpr (kOut != kF32) {
        // Eight columns per lane where N allows 16-byte stores: odd rows of 16
        // lanes of one fragment change places with even rows of its neighbour.
        if (vec == 8) {
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
                        *reinterpret_cast<u32x4*>(static_cast<unsigned short*>(c) +
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
                store_four<kOut>(c, static_cast<long long>(at_row) * n + at_col, acc[i][j], n - at_col,
                                 vec >= 4 && at_col + 4 <= n);
        }
    }
}

// One kRows x 256 tile of C at (row0, col0). steps >= 4.
template <int kRows, int kOut>
__device__ __forceinline__ void product_tile(MX4_LDS unsigned char* lds, const unsigned char* a_codes,
                                             const unsigned char* a_scales, const unsigned char* b_codes,
                                             const unsigned char* b_scales, void* c, int m, int n, int steps, int row0,
                                             int col0, int vec) {
    typedef TileLane<kRows> Lane;
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int r = lane % 16, q = lane / 16;
    const int row_bytes = steps * 64;
    Lane L;
    L.wave = wave;
    L.scale_row = steps * 4;
    L.a = rsrc_at(a_codes + static_cast<long long>(row0) * row_bytes);
    L.b = rsrc_at(b_codes + static_cast<long long>(col0) * row_bytes);
    // Rows past the edge read the last one.
    const auto row_of = [](int first, int i, int size) { return first + i < size ? i : size - 1 - first; };
#pragma unroll
    for (int i = 0; i < Lane::kFetchA; ++i)
        L.a_src[i] = row_of(row0, (wave * Lane::kFetchA + i) * 16 + r, m) * row_bytes + q * 16;
#pragma unroll
    for (int i = 0; i < 2; ++i) L.b_src[i] = row_of(col0, (wave * 2 + i) * 16 + r, n) * row_bytes + q * 16;
    const bool for_a = wave < 4;
    L.scales = rsrc_at(for_a ? a_scales + static_cast<long long>(row0) * L.scale_row
                             : b_scales + static_cast<long long>(col0) * L.scale_row);
    L.scale_src = row_of(for_a ? row0 : col0, (wave % 4) * 64 + lane, for_a ? m : n) * L.scale_row;
    const int wave_row = wave / 4 * (kRows / 2), wave_col = wave % 4 * 64;
    L.a_off = wave_row * 64 + lane * 16;
    L.b_off = wave_col * 64 + lane * 16;
    L.a_scale = (wave_row + r) * 16 + q;
    L.b_scale = (wave_col + r) * 16 + q;

    f32x4 acc[Lane::kRowFrags][kColFrags];
#pragma unroll
    for (int i = 0; i < Lane::kRowFrags; ++i)
#pragma unroll
        for (int j = 0; j < kColFrags; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    const auto stage = [&](int t) { return lds + (t & (kStages - 1)) * kStageBytes; };
    MX4_LDS unsigned char* slots = lds + kStages * kStageBytes;
    const auto slot = [&](int s) { return slots + (s & 1) * kSlotBytes; };

    fetch_scales<kRows>(slot(0), L, 0);
#pragma unroll
    for (int t = 0; t < kStages - 1; ++t) {
        fetch_a<kRows>(stage(t), L, t);
        fetch_b<kRows>(stage(t), L, t);
    }
    __builtin_amdgcn_s_waitcnt(0);
    phase_barrier();
    const bool late = wave >= 4;
    if (late) phase_barrier();

    i32x4 av[Lane::kRowFrags], bv[kColFrags];
    int sa[Lane::kRowFrags], sb[kColFrags];
    const int last_slot = (steps - 1) / 4;
    for (int t = 0; t < steps; ++t) {
        // Step t + 3 goes to the stage of step t - 1, the next slot's scales to
        // the slot of steps up to t - 1, which no wave reads any more (past the
        // end the last step is fetched again).
        const int next = t + 3 < steps ? t + 3 : steps - 1;
        const int s = t / 4;
        const int next_slot = t % 4 == 0 && s < last_slot ? s + 1 : -1;
        const int scale_at = t * 4 - slot_start(s, L.scale_row);
        memory_phase<kRows>(stage(t), stage(t + 3), slot(s), slot(s + 1), L, next, next_slot, scale_at, av, bv, sa, sb);
        // The fetch of step t + 1 has landed once at most those of A and B of
        // t + 2 and of A of t + 3 are left (loads into LDS land in order; a
        // slot's scales, issued before A of t + 3, are then two steps early).
        __builtin_amdgcn_s_waitcnt(0x0070 | (2 * Lane::kFetchA + 2));  // vmcnt, lgkmcnt(0)
        phase_barrier();
#pragma unroll
        for (int i = 0; i < Lane::kRowFrags / 2; ++i)
#pragma unroll
            for (int j = 0; j < kColFrags; ++j) acc[i][j] = mfma(bv[j], sb[j], av[i], sa[i], acc[i][j]);
        __builtin_amdgcn_sched_barrier(0);
        fetch_b<kRows>(stage(t + 3), L, next);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = Lane::kRowFrags / 2; i < Lane::kRowFrags; ++i)
#pragma unroll
            for (int j = 0; j < kColFrags; ++j) acc[i][j] = mfma(bv[j], sb[j], av[i], sa[i], acc[i][j]);
        phase_barrier();
    }
    if (!late) phase_barrier();
    __builtin_amdgcn_s_waitcnt(0);
    store_tile<Lane::kRowFrags, kOut>(acc, c, row0 + wave_row, col0 + wave_col, m, n, lane, vec);
}

}  // namespace mx4

// The large-tile body of the product of two mx4 operands (gemm_mx4.hip).
//
// Block tile 256x256 (or 128x256), 512 lanes = 8 waves in a 2x4 grid (two
// waves per SIMD), each a 128x64 quadrant as 8x4 accumulators. One block per
// CU. The schedule is that of gemm_mfma16_fast.h: K in steps of 128 through a
// ring of four 32 KiB LDS stages, the two waves of each SIMD one phase apart,
// one reading its operands from LDS while the other multiplies.
//
// LDS layout of a stage: rows of 64 bytes, A's 256 at 0 and B's at 16 KiB; block
// c of row r lies at 64 r + 16 (c ^ (r / 2 % 4)). A fetch instruction fills 16
// rows, four neighbouring lanes one row: the address unit takes four lanes'
// adjacent 16 bytes in one access (with a lane per row it made 64 accesses of
// an instruction and bound the kernel: 2400 a step, 8192^3 in 342 us).
// A fragment read (lane (r, q) block q of row r) goes over every bank once per
// 16 lanes that the LDS serves together (lanes 0-3, 12-15 and 20-27 the first);
// of the swizzles tried, this one and one other had no conflicts.
//
// Scales: a row has four bytes per step. Fetched a step at a time, a load would
// touch 64 rows, 64 lines, for 256 bytes; instead a lane takes 16 bytes of its
// row, four steps' worth, once in four steps, and turns them (four steps of
// four blocks) into four blocks' dwords of four steps each, in one of two 8 KiB
// slots of LDS. A lane then reads one dword per fragment for four steps and the
// instruction picks the step's byte. (Read from LDS a byte per fragment and
// step, the scales took 50 of 332 us at 8192^3.) A row's last 16 bytes are
// loaded whole where its end falls inside a slot, so nothing is read outside
// the operand (K >= 512).
#pragma once

#include "mx4_device.h"

namespace mx4 {

template <int kValue>
struct Constant {
    static constexpr int value = kValue;
};

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

// Scales of steps 4 slot .. 4 slot + 3 of 64 rows (waves 0-3 of A, waves 4-7 of
// B), as they lie in the row: 16 bytes per slot, moved back where it ends inside.
__device__ __forceinline__ int slot_start(int slot, int scale_row) {
    const int last = scale_row - 16;
    return slot * 16 < last ? slot * 16 : last;
}

template <int kRows>
__device__ __forceinline__ u32x4 load_scales(const TileLane<kRows>& L, int slot) {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(L.scales, L.scale_src,
                                                                           slot_start(slot, L.scale_row), 0));
}

// Dword q of the result: block q's bytes of the four steps.
__device__ __forceinline__ u32x4 by_block(u32x4 v) {
    const unsigned lo01 = __builtin_amdgcn_perm(v[1], v[0], 0x05010400u), lo23 = __builtin_amdgcn_perm(v[3], v[2], 0x05010400u);
    const unsigned hi01 = __builtin_amdgcn_perm(v[1], v[0], 0x07030602u), hi23 = __builtin_amdgcn_perm(v[3], v[2], 0x07030602u);
    return u32x4{__builtin_amdgcn_perm(lo23, lo01, 0x05040100u), __builtin_amdgcn_perm(lo23, lo01, 0x07060302u),
                 __builtin_amdgcn_perm(hi23, hi01, 0x05040100u), __builtin_amdgcn_perm(hi23, hi01, 0x07060302u)};
}

template <int kRows>
__device__ __forceinline__ void store_scales(MX4_LDS unsigned char* wr, const TileLane<kRows>& L, u32x4 v, int slot) {
    for (int late = slot * 16 - slot_start(slot, L.scale_row); late > 0; late -= 4) v = u32x4{v[1], v[2], v[3], 0};
    *reinterpret_cast<MX4_LDS u32x4*>(wr + threadIdx.x * 16) = by_block(v);
}

// A memory phase: the fetch of A of step `next`, and step t's operands from LDS
// into registers. The regions written and read are distinct; __restrict__ says
// so, or the compiler would wait for the fetch before the reads.
template <int kRows>
__device__ __forceinline__ void memory_phase(const MX4_LDS unsigned char* __restrict__ rd,
                                             MX4_LDS unsigned char* __restrict__ wr, const TileLane<kRows>& L,
                                             int next, i32x4 (&av)[TileLane<kRows>::kRowFrags],
                                             i32x4 (&bv)[kColFrags]) {
    fetch_a<kRows>(wr, L, next);
#pragma unroll
    for (int f = 0; f < TileLane<kRows>::kRowFrags; ++f)
        av[f] = *reinterpret_cast<const MX4_LDS i32x4*>(rd + L.a_off + f * 1024);
#pragma unroll
    for (int f = 0; f < kColFrags; ++f)
        bv[f] = *reinterpret_cast<const MX4_LDS i32x4*>(rd + kStageB + L.b_off + f * 1024);
}

// The fragments' scales of a slot's four steps.
template <int kRows>
__device__ __forceinline__ void read_scales(const MX4_LDS unsigned char* __restrict__ rd, const TileLane<kRows>& L,
                                            int (&sa)[TileLane<kRows>::kRowFrags], int (&sb)[kColFrags]) {
#pragma unroll
    for (int f = 0; f < TileLane<kRows>::kRowFrags; ++f)
        sa[f] = *reinterpret_cast<const MX4_LDS int*>(rd + L.a_scale + f * 256);
#pragma unroll
    for (int f = 0; f < kColFrags; ++f)
        sb[f] = *reinterpret_cast<const MX4_LDS int*>(rd + kSlotB + L.b_scale + f * 256);
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
    const int from = (lane % 4 ^ lane / 8 % 4) * 16;  // the block that lane's place in LDS takes
    // Rows past the edge read the last one.
    const auto row_of = [](int first, int i, int size) { return first + i < size ? i : size - 1 - first; };
#pragma unroll
    for (int i = 0; i < Lane::kFetchA; ++i)
        L.a_src[i] = row_of(row0, (wave * Lane::kFetchA + i) * 16 + lane / 4, m) * row_bytes + from;
#pragma unroll
    for (int i = 0; i < 2; ++i) L.b_src[i] = row_of(col0, (wave * 2 + i) * 16 + lane / 4, n) * row_bytes + from;
    const bool for_a = wave < 4;
    L.scales = rsrc_at(for_a ? a_scales + static_cast<long long>(row0) * L.scale_row
                             : b_scales + static_cast<long long>(col0) * L.scale_row);
    L.scale_src = row_of(for_a ? row0 : col0, (wave % 4) * 64 + lane, for_a ? m : n) * L.scale_row;
    const int wave_row = wave / 4 * (kRows / 2), wave_col = wave % 4 * 64;
    L.a_off = (wave_row + r) * 64 + (q ^ r / 2 % 4) * 16;
    L.b_off = (wave_col + r) * 64 + (q ^ r / 2 % 4) * 16;
    L.a_scale = (wave_row + r) * 16 + q * 4;
    L.b_scale = (wave_col + r) * 16 + q * 4;

    f32x4 acc[Lane::kRowFrags][kColFrags];
#pragma unroll
    for (int i = 0; i < Lane::kRowFrags; ++i)
#pragma unroll
        for (int j = 0; j < kColFrags; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    const auto stage = [&](int t) { return lds + (t & (kStages - 1)) * kStageBytes; };
    MX4_LDS unsigned char* slots = lds + kStages * kStageBytes;
    const auto slot = [&](int s) { return slots + (s & 1) * kSlotBytes; };

    u32x4 scales = load_scales<kRows>(L, 0);
#pragma unroll
    for (int t = 0; t < kStages - 1; ++t) {
        fetch_a<kRows>(stage(t), L, t);
        fetch_b<kRows>(stage(t), L, t);
    }
    store_scales<kRows>(slot(0), L, scales, 0);
    __builtin_amdgcn_s_waitcnt(0);
    phase_barrier();
    const bool late = wave >= 4;
    if (late) phase_barrier();

    i32x4 av[Lane::kRowFrags], bv[kColFrags];
    int sa[Lane::kRowFrags], sb[kColFrags];
    const int last_slot = (steps - 1) / 4;
    // Step t = 4 s + j. Step t + 3 goes to the stage of step t - 1, the next
    // slot's scales to the slot of steps up to 4 s - 1, which no wave reads any
    // more (past the end the last step and slot are taken again).
    const auto step = [&](int t, auto which) {
        constexpr int j = decltype(which)::value;
        const int next = t + 3 < steps ? t + 3 : steps - 1;
        const int s = t / 4, next_slot = s < last_slot ? s + 1 : last_slot;
        if constexpr (j == 0) {
            read_scales<kRows>(slot(s), L, sa, sb);
            scales = load_scales<kRows>(L, next_slot);
        }
        memory_phase<kRows>(stage(t), stage(t + 3), L, next, av, bv);
        if constexpr (j == 3) store_scales<kRows>(slot(s + 1), L, scales, next_slot);
        // The fetch of step t + 1 has landed once at most those of A and B of
        // t + 2 and of A of t + 3 are left, and the scales loaded at the
        // slot's first step between them (loads land in order).
        __builtin_amdgcn_s_waitcnt(0x0070 | (2 * Lane::kFetchA + (j < 2 ? 3 : 2)));  // vmcnt, lgkmcnt(0)
        phase_barrier();
#pragma unroll
        for (int i = 0; i < Lane::kRowFrags / 2; ++i)
#pragma unroll
            for (int f = 0; f < kColFrags; ++f) acc[i][f] = mfma<j>(bv[f], sb[f], av[i], sa[i], acc[i][f]);
        __builtin_amdgcn_sched_barrier(0);
        fetch_b<kRows>(stage(t + 3), L, next);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = Lane::kRowFrags / 2; i < Lane::kRowFrags; ++i)
#pragma unroll
            for (int f = 0; f < kColFrags; ++f) acc[i][f] = mfma<j>(bv[f], sb[f], av[i], sa[i], acc[i][f]);
        phase_barrier();
    };
    for (int t = 0;;) {
        step(t, Constant<0>{});
        if (++t == steps) break;
        step(t, Constant<1>{});
        if (++t == steps) break;
        step(t, Constant<2>{});
        if (++t == steps) break;
        step(t, Constant<3>{});
        if (++t == steps) break;
    }
    if (!late) phase_barrier();
    __builtin_amdgcn_s_waitcnt(0);
    store_tile<Lane::kRowFrags, kOut>(acc, c, row0 + wave_row, col0 + wave_col, m, n, lane, vec);
}

}  // namespace mx4

// The large-tile body of the products of 8-bit integers (gemm_i8.hip).
//
// Block tile 256x256 (or 128x256) by 4 waves in a 2x2 grid, one per SIMD, each a
// 128x128 quadrant as 8x8 accumulators (256 registers); one block per CU. The
// 16x16x64 instruction takes 16 cycles for two 1 KiB fragments; quadrants this
// large keep LDS reads at half of what LDS gives, and a fetch takes whole lines.
//
// K goes in stages of 128 through two 64 KiB LDS buffers, each stage as two steps
// of 64, each step as 8 rows of 8 products. While a step's products issue, the next
// step's fragments are read from LDS: B's into registers of their own, A's row i
// into row i's once its products have issued. In the second step of stage s, after
// two rows, one barrier: every wave has read all of stage s and its own share of
// stage s + 1 has landed, so after it stage s + 2 is fetched over stage s, and stage
// s + 1 is read. In the last two stages the fetches repeat the last stage.
//
// LDS layout of a stage: rows of 128 bytes, A's 256 at 0 and B's at 32 KiB; block c
// of 16 bytes of row r lies at 128 r + 16 (c ^ (r / 2 % 8)). A fetch instruction
// fills 8 rows, eight neighbouring lanes one row. A fragment read, lane (r, q) block
// q of row r, touches every bank once per 16 lanes that the LDS serves together.
//
// SwiGLU: a wave's column fragments 0-3 are gate columns and 4-7 the up columns of
// the same results, so the two meet in one lane.
#pragma once

#include "i8_device.h"

namespace i8 {

constexpr int kTileRows = 256, kTileCols = 256, kTileThreads = 256;
constexpr int kStageBytes = 64 * 1024, kStageB = 32 * 1024;
constexpr int kRingBytes = 2 * kStageBytes;
constexpr int kColFrags = 8;

// `rows` rows (up to kTileRows) of `row_bytes` from p on; what lies past them reads as zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_of(const unsigned char* p, long long rows, int row_bytes) {
    const int most = rows < 0 ? 0 : rows < kTileRows ? static_cast<int>(rows) : kTileRows;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p), 0, most * row_bytes, 0x00020000);
}

template <int kRows>
struct TileLane {
    static constexpr int kRowFrags = kRows / 32;  // of a wave
    static constexpr int kFetchA = kRows / 32;    // instructions per wave and stage
    static constexpr int kFetchB = 8;
    __amdgpu_buffer_rsrc_t a, b;  // A's rows (this wave's share of the tile, or all of A), this wave's share of B's
    int a_src[kFetchA];           // the lane's offset in each fetch of A
    int b_src[2];                 // ... in a fetch of B's rows 16 j .. + 7 and 16 j + 8 .. + 15
    int a_off[2], b_off[2];       // LDS offsets of the wave's first fragments in each step
    int row_bytes, wave, lane;
};

// Instruction i of this wave's share of stage s (A's first).
template <int kRows>
__device__ __forceinline__ void fetch_one(MX4_LDS unsigned char* wr, const TileLane<kRows>& L, int s, int i) {
    constexpr int kA = TileLane<kRows>::kFetchA, kB = TileLane<kRows>::kFetchB;
    if (i < kA)
        buffer_to_lds(L.a, wr + (L.wave * kA + i) * 1024, L.a_src[i < kA ? i : 0], s * kLine);
    else
        buffer_to_lds(L.b, wr + kStageB + (L.wave * kB + i - kA) * 1024, L.b_src[(i - kA) & 1],
                      (i - kA) * 8 * L.row_bytes + s * kLine);
}

template <int kRows>
__device__ __forceinline__ void fetch_range(MX4_LDS unsigned char* wr, const TileLane<kRows>& L, int s, int from, int to) {
    constexpr int kAll = TileLane<kRows>::kFetchA + TileLane<kRows>::kFetchB;
#pragma unroll
    for (int i = 0; i < kAll; ++i)
        if (i >= from && i < to) fetch_one<kRows>(wr, L, s, i);
}

// One fragment of step u of the stage at `rd`. What is read is not being written;
// __restrict__ says so, or the compiler would wait for the fetches in flight.
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

// acc += a b in acc's own registers, written out because the compiler, with the
// products held in their places, gives them other registers and copies. It does not
// know that a value is there only after the instruction's passes (settle()).
__device__ __forceinline__ void mfma_in_place(i32x4& acc, i32x4 a, i32x4 b) {
    asm volatile("v_mfma_i32_16x16x64_i8 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}

// Between the last product and the first use of its value: its passes are over.
__device__ __forceinline__ void settle() {
    asm volatile("s_nop 15\n s_nop 15" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// acc[i][f] = the sums of rows wave_row + 16 i + r and B's rows 16 f + 4 q .. + 3 of the
// wave's 128. a_row(i): where the lane's row of the wave's fetch i of A begins, in bytes
// from A's resource on.
template <int kRows, typename RowOf>
__device__ __forceinline__ void tile_sums(MX4_LDS unsigned char* lds, __amdgpu_buffer_rsrc_t a, RowOf a_row,
                                          __amdgpu_buffer_rsrc_t b, int row_bytes, int wave, int lane,
                                          i32x4 (&acc)[kRows / 32][kColFrags]) {
    typedef TileLane<kRows> Lane;
    const int r = lane % 16, q = lane / 16;
    Lane L;
    L.a = a, L.b = b;
    L.wave = wave, L.lane = lane, L.row_bytes = row_bytes;
    // The block that the lane's place in LDS takes, of row lane / 8 of a fetch.
#pragma unroll
    for (int i = 0; i < Lane::kFetchA; ++i) L.a_src[i] = a_row(i) + (lane % 8 ^ (4 * (i & 1) + lane / 16)) * 16;
#pragma unroll
    for (int i = 0; i < 2; ++i) L.b_src[i] = lane / 8 * row_bytes + (lane % 8 ^ (4 * i + lane / 16)) * 16;
    const int wave_row = wave / 2 * (kRows / 2), wave_col = wave % 2 * 128;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        L.a_off[u] = (wave_row + r) * 128 + ((4 * u + q) ^ r / 2) * 16;
        L.b_off[u] = (wave_col + r) * 128 + ((4 * u + q) ^ r / 2) * 16;
    }
    const auto stage = [&](int s) { return lds + (s & 1) * kStageBytes; };
    const int stages = row_bytes / kLine;

    // The fetch of a stage is spread over the rows between two barriers and a few
    // behind the second: the address unit takes 16 cycles for an instruction, and a
    // wave that waits for it multiplies nothing.
    constexpr int kI = Lane::kRowFrags, kAll = Lane::kFetchA + Lane::kFetchB, kEarly = kAll * 5 / 8;
    fetch_range<kRows>(stage(0), L, 0, 0, kAll);
    fetch_range<kRows>(stage(1), L, stages > 1 ? 1 : 0, 0, kEarly);
#pragma unroll
    for (int i = 0; i < kI; ++i)
#pragma unroll
        for (int f = 0; f < kColFrags; ++f) {
            acc[i][f] = i32x4{0, 0, 0, 0};
            asm volatile("" : "+a"(acc[i][f]));  // cleared here, while the fetch is under way
        }
    __builtin_amdgcn_s_waitcnt(0);
    lds_barrier();

    constexpr int kB = kColFrags / kI;
    i32x4 av[kI], bv[2][kColFrags];
#pragma unroll
    for (int f = 0; f + 1 < kI; ++f) av[f] = read_a<kRows>(lds, L, 0, f);
#pragma unroll
    for (int f = 0; f < kColFrags; ++f) bv[0][f] = read_b<kRows>(lds, L, 0, f);

    // Every product is held in its place, with one piece of the other work behind it:
    // the matrix unit is busy meanwhile, and a product leaves room for a few instructions.
    for (int s = 0; s < stages; ++s) {
        const MX4_LDS unsigned char *here = stage(s), *there = stage(s + 1);
        const int rest = s + 1 < stages ? s + 1 : stages - 1, next = s + 2 < stages ? s + 2 : stages - 1;
#pragma unroll
        for (int i = 0; i < kI; ++i) {
#pragma unroll
            for (int f = 0; f < kColFrags; ++f) {
                mfma_in_place(acc[i][f], bv[0][f], av[i]);
                if (f == 0 && i == 0) av[kI - 1] = read_a<kRows>(here, L, 0, kI - 1);
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
                mfma_in_place(acc[i][f], bv[1][f], av[i]);
                if (f == 0 && i == 0) av[kI - 1] = read_a<kRows>(here, L, 1, kI - 1);
                if (i >= 2) {
                    // What is left after two rows, over the other rows.
                    constexpr int kLeft = kI - 2;
                    if (f == 0) {
                        av[i - 1] = read_a<kRows>(there, L, 0, i - 1);
                        if (i == 2) av[0] = read_a<kRows>(there, L, 0, 0);
                    }
                    const int from = (i - 2) * kEarly / kLeft, to = (i - 1) * kEarly / kLeft;
                    if (f >= 4 && from + f - 4 < to) fetch_one<kRows>(stage(s), L, next, from + f - 4);
                    const int b0 = (i - 2) * kColFrags / kLeft, b1 = (i - 1) * kColFrags / kLeft;
                    if (f > 0 && b0 + f - 1 < b1) bv[0][b0 + f - 1] = read_b<kRows>(there, L, 0, b0 + f - 1);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        // A product's operand may have been written two instructions before it at the latest.
        asm volatile("s_nop 1" ::: "memory");
    }
    __builtin_amdgcn_s_waitcnt(0);
    settle();
#pragma unroll
    for (int i = 0; i < kI; ++i)
#pragma unroll
        for (int f = 0; f < kColFrags; ++f) asm volatile("" : "+a"(acc[i][f]));  // read behind it only
}

}  // namespace i8

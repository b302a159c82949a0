// The large-tile body of the products of 8-bit integers (gemm_i8.hip).
//
// Block tile 256x256 (or 128x256) by 4 waves in a 2x2 grid, one per SIMD, each a
// 128x128 quadrant as 4x4 accumulators of 32x32 (256 registers); one block per CU.
// The 32x32x32 instruction takes 32 cycles for two 1 KiB fragments; quadrants this
// large keep LDS reads at half of what LDS gives, and a fetch takes whole lines. (A
// loop of the instruction alone runs at 4.95 POP/s on zeros and 3.40 on random bytes,
// where the chip lowers its clock; the 16x16x64 instruction at 2.91 and 2.71.)
//
// K goes in stages of 128 through two 64 KiB LDS buffers, each stage as four steps
// of 32 and 16 products. While a step's products issue, the next step's fragments
// are read from LDS into the other of two sets of registers. Before a stage's last
// step a barrier: every wave has read all of stage s and its own share of stage
// s + 1 has landed, so after it stage s + 2 is fetched over stage s, and stage s + 1
// is read. In the last two stages the fetches repeat the last stage.
//
// LDS layout of a stage: rows of 128 bytes, A's 256 at 0 and B's at 32 KiB; block c
// of 16 bytes of row r lies at 128 r + 16 (c ^ (r / 2 % 8)). A fetch instruction
// fills 8 rows, eight neighbouring lanes one row. A fragment read, lane (r, h) of 32
// rows and two blocks, touches every bank once per 16 lanes that the LDS serves
// together (lanes 0-3, 12-15 and 20-27 the first).
//
// SwiGLU: a wave's column fragments 0 and 1 are gate columns, 2 and 3 the up columns
// of the same results.
#pragma once

#include "i8_device.h"

namespace i8 {

constexpr int kTileRows = 256, kTileCols = 256, kTileThreads = 256;
constexpr int kStageBytes = 64 * 1024, kStageB = 32 * 1024;
constexpr int kRingBytes = 2 * kStageBytes;
constexpr int kColFrags = 4;

// `bytes` bytes from p on, the same in every lane, which the compiler has to be told
// (or it tries each lane's resource in turn: 40 of 230 us at 4096x4096x16384); what
// lies past them reads as zeros.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t resource(const unsigned char* p, int bytes) {
    const unsigned long long at = reinterpret_cast<unsigned long long>(p);
    const unsigned lo = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(at));
    const unsigned hi = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(at >> 32));
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(static_cast<unsigned long long>(hi) << 32 | lo), 0,
                                             __builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}

// `rows` rows (up to kTileRows) of `row_bytes` from p on.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_from(const unsigned char* p, long long rows, int row_bytes) {
    const int most = rows < 0 ? 0 : rows < kTileRows ? static_cast<int>(rows) : kTileRows;
    return resource(p, most * row_bytes);
}

template <int kRows>
struct TileLane {
    static constexpr int kRowFrags = kRows / 64;  // of a wave
    static constexpr int kFetchA = kRows / 32;    // instructions per wave and stage
    static constexpr int kFetchB = 8;
    __amdgpu_buffer_rsrc_t a, b;  // A's rows (this wave's share of the tile, or all of A), this wave's share of B's
    int a_src[kFetchA];           // the lane's offset in each fetch of A
    int b_src[kFetchB];           // ... of B
    int a_off[4], b_off[4];       // LDS offsets of the wave's first fragments in each step
    int wave;
};

// Instruction i of this wave's share of stage s (A's first). Rows are in the lane's
// offset, which is held against the resource's end; the scalar one stays within a row.
template <int kRows>
__device__ __forceinline__ void fetch_one(MX4_LDS unsigned char* wr, const TileLane<kRows>& L, int s, int i) {
    constexpr int kA = TileLane<kRows>::kFetchA, kB = TileLane<kRows>::kFetchB;
    if (i < kA)
        buffer_to_lds(L.a, wr + (L.wave * kA + i) * 1024, L.a_src[i < kA ? i : 0], s * kLine);
    else
        buffer_to_lds(L.b, wr + kStageB + (L.wave * kB + i - kA) * 1024, L.b_src[i < kA ? 0 : i - kA], s * kLine);
}

// One fragment of step u of the stage at `rd`. What is read is not being written;
// __restrict__ says so, or the compiler would wait for the fetches in flight.
template <int kRows>
__device__ __forceinline__ i32x4 read_a(const MX4_LDS unsigned char* __restrict__ rd, const TileLane<kRows>& L, int u,
                                        int f) {
    return *reinterpret_cast<const MX4_LDS i32x4*>(rd + L.a_off[u] + f * 4096);
}
template <int kRows>
__device__ __forceinline__ i32x4 read_b(const MX4_LDS unsigned char* __restrict__ rd, const TileLane<kRows>& L, int u,
                                        int f) {
    return *reinterpret_cast<const MX4_LDS i32x4*>(rd + kStageB + L.b_off[u] + f * 4096);
}

// acc += a b in acc's own registers, written out because the compiler, with the
// products held in their places, gives them other registers and copies. It does not
// know that a value is there only after the instruction's passes (settle()).
__device__ __forceinline__ void mfma_in_place(i32x16& acc, i32x4 a, i32x4 b) {
    asm volatile("v_mfma_i32_32x32x32_i8 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}

// Between the last product and the first use of its value: its passes are over.
__device__ __forceinline__ void settle() {
    asm volatile("s_nop 15\n s_nop 15" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// acc[i][f][v] = the sum of row wave_row + 32 i + lane % 32 and of the wave's column
// 32 f + 8 (v / 4) + 4 (lane / 32) + v % 4. a_row(i): where the lane's row of the wave's
// fetch i of A begins, in bytes from A's resource on.
template <int kRows, typename RowOf>
__device__ __forceinline__ void tile_sums(MX4_LDS unsigned char* lds, __amdgpu_buffer_rsrc_t a, RowOf a_row,
                                          __amdgpu_buffer_rsrc_t b, int row_bytes, int wave, int lane,
                                          i32x16 (&acc)[kRows / 64][kColFrags]) {
    typedef TileLane<kRows> Lane;
    const int r = lane % 32, h = lane / 32;
    Lane L;
    L.a = a, L.b = b;
    L.wave = wave;
    // The block that the lane's place in LDS takes, of row lane / 8 of a fetch.
#pragma unroll
    for (int i = 0; i < Lane::kFetchA; ++i) L.a_src[i] = a_row(i) + (lane % 8 ^ (4 * (i & 1) + lane / 16)) * 16;
#pragma unroll
    for (int i = 0; i < Lane::kFetchB; ++i)
        L.b_src[i] = (8 * i + lane / 8) * row_bytes + (lane % 8 ^ (4 * (i & 1) + lane / 16)) * 16;
    const int wave_row = wave / 2 * (kRows / 2), wave_col = wave % 2 * 128;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        L.a_off[t] = (wave_row + r) * 128 + ((2 * t + h) ^ r / 2 % 8) * 16;
        L.b_off[t] = (wave_col + r) * 128 + ((2 * t + h) ^ r / 2 % 8) * 16;
    }
    const auto stage = [&](int s) { return lds + (s & 1) * kStageBytes; };
    const int stages = row_bytes / kLine;

    constexpr int kI = Lane::kRowFrags, kAll = Lane::kFetchA + Lane::kFetchB, kEarly = kAll / 2;
    constexpr int kSlots = kI * kColFrags;
#pragma unroll
    for (int i = 0; i < kAll; ++i) fetch_one<kRows>(stage(0), L, 0, i);
#pragma unroll
    for (int i = 0; i < kEarly; ++i) fetch_one<kRows>(stage(1), L, stages > 1 ? 1 : 0, i);
#pragma unroll
    for (int i = 0; i < kI; ++i)
#pragma unroll
        for (int f = 0; f < kColFrags; ++f) {
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][f][e] = 0;
            asm volatile("" : "+a"(acc[i][f]));  // cleared here, while the fetch is under way
        }
    __builtin_amdgcn_s_waitcnt(0);
    lds_barrier();

    i32x4 av[2][kI], bv[2][kColFrags];
#pragma unroll
    for (int f = 0; f < kColFrags; ++f) bv[0][f] = read_b<kRows>(lds, L, 0, f);
#pragma unroll
    for (int i = 0; i < kI; ++i) av[0][i] = read_a<kRows>(lds, L, 0, i);

    // Every product is held in its place, with at most a fragment's read and a fetch
    // behind it: the matrix unit is busy meanwhile. The fetch of a stage is spread over
    // two steps: the address unit takes 16 cycles for an instruction, and a wave that
    // waits for it multiplies nothing.
    for (int s = 0; s < stages; ++s) {
        const int rest = s + 1 < stages ? s + 1 : stages - 1, next = s + 2 < stages ? s + 2 : stages - 1;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const MX4_LDS unsigned char* from = t < 3 ? stage(s) : stage(s + 1);
            if (t == 3) {
                __builtin_amdgcn_s_waitcnt(0);
                lds_barrier();
            }
#pragma unroll
            for (int m = 0; m < kSlots; ++m) {
                const int i = m / kColFrags, f = m % kColFrags;
                mfma_in_place(acc[i][f], bv[t & 1][f], av[t & 1][i]);
                if (m < kColFrags)
                    bv[(t + 1) & 1][m < kColFrags ? m : 0] = read_b<kRows>(from, L, (t + 1) % 4, m);
                else if (m < kColFrags + kI)
                    av[(t + 1) & 1][m < kColFrags + kI ? m - kColFrags : 0] = read_a<kRows>(from, L, (t + 1) % 4, m - kColFrags);
                // Fetch j of a step's lies behind product (j + 1) kSlots / kEarly - 1.
#pragma unroll
                for (int j = 0; j < kEarly; ++j)
                    if (m == (j + 1) * kSlots / kEarly - 1) {
                        if (t == 0) fetch_one<kRows>(stage(s + 1), L, rest, kEarly + j);  // what is left of it
                        if (t == 3) fetch_one<kRows>(stage(s), L, next, j);
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

// The large-tile body of the products of 8-bit integers (gemm_i8.hip).
//
// Block tile 256x256 (or 128x256, 128x128) by 4 waves in a 2x2 grid, one per SIMD, each
// a 128x128 quadrant as 4x4 accumulators of 32x32 (256 registers); one block per CU (of
// 128x128 two, in 80 KiB of LDS each, so that one stores while the other multiplies).
// The 32x32x32 instruction takes 32 cycles for two 1 KiB fragments; quadrants this
// large keep LDS reads at half of what LDS gives, and a fetch takes whole lines. (A
// loop of the instruction alone runs at 4.95 POP/s on zeros and 3.40 on random bytes,
// where the chip lowers its clock; the 16x16x64 instruction at 2.91 and 2.71.)
//
// 8192^3 413-432 us (by the chip; 2.65 POP/s), 4096x14336x4096 204-222 (the library's 32-bit
// sums alone 231). Matrix units are busy 76% of the time, at 1.65 GHz, in
// 4096x4096x16384 (204 us); without any fetch 79%, at 1.83: power bounds the loop. A tile's
// results take 16 thousand cycles, the loop over k = 4096 72 thousand; two blocks of 128x128
// on a CU overlap the two, and read twice as much LDS for a product.
//
// K goes in stages of 128 through two buffers of LDS for A and three for B (of 32 KiB each:
// all of LDS), each stage as four steps of 32 and 16 products. While a step's products
// issue, the next step's fragments are read from LDS into the other of two sets of
// registers. Before a stage's last step a barrier: every wave has read all of stage s
// and its own share of stage s + 1 has landed, so after it A's stage s + 2 and B's
// stage s + 3 are fetched over stage s, and stage s + 1 is read. (B, the weights, comes
// from further away than A, whose rows all columns' tiles share.) In the last stages the
// fetches repeat the last stage.
//
// LDS layout of a stage: rows of 128 bytes; block c of 16 bytes of row r lies at
// 128 r + 16 (c ^ (r / 2 % 8)). A fetch instruction
// fills 8 rows, eight neighbouring lanes one row. A fragment read, lane (r, h) of 32
// rows and two blocks, touches every bank once per 16 lanes that the LDS serves
// together (lanes 0-3, 12-15 and 20-27 the first).
//
// SwiGLU: the first half of a wave's column fragments are gate columns, the second the
// up columns of the same results.
#pragma once

#include "i8_device.h"

namespace i8 {

constexpr int kTileThreads = 256;
constexpr int kRingA = 2, kRingB = 3;  // buffers

// A tile of kRows by kCols, whose buffers hold kSlotRows rows of either operand.
template <int kRows, int kCols, int kSlotRows>
struct Tile {
    static constexpr int kRowFrags = kRows / 64, kColFrags = kCols / 64;  // of a wave
    static constexpr int kFetchA = kRows / 32, kFetchB = kCols / 32;      // instructions per wave and stage
    static constexpr int kSlotBytes = kSlotRows * kLine, kFirstB = kRingA * kSlotBytes;
    static constexpr int kRingBytes = (kRingA + kRingB) * kSlotBytes;
    typedef i32x16 Sums[kRowFrags][kColFrags];
};

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

// `rows` rows (up to 256) of `row_bytes` from p on.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_from(const unsigned char* p, long long rows, int row_bytes) {
    const int most = rows < 0 ? 0 : rows < 256 ? static_cast<int>(rows) : 256;
    return resource(p, most * row_bytes);
}

typedef const __attribute__((address_space(1))) unsigned char* global_bytes;

// kFar: A's rows have addresses of their own, for gathered rows further apart than a resource reaches.
template <typename T, bool kFar>
struct TileLane {
    __amdgpu_buffer_rsrc_t a, b;             // A's rows (this wave's share of the tile, or all of A), this wave's of B's
    int a_src[T::kFetchA], b_src[T::kFetchB];  // the lane's offset in each fetch
    global_bytes a_far[kFar ? T::kFetchA : 1];   // kFar: where it begins
    int a_off[4], b_off[4];                  // LDS offsets of the wave's first fragments in each step
    int wave;
};

// Instruction i of this wave's share of a stage of A to `wr`, `at` bytes into the rows.
// Rows are in the lane's offset, which is held against the resource's end; the scalar
// one stays within a row.
template <typename T, bool kFar>
__device__ __forceinline__ void fetch_a(MX4_LDS unsigned char* wr, const TileLane<T, kFar>& L, int at, int i) {
    MX4_LDS unsigned char* const to = wr + (L.wave * T::kFetchA + i) * 1024;
    if constexpr (kFar)
        __builtin_amdgcn_global_load_lds(reinterpret_cast<const __attribute__((address_space(1))) void*>(L.a_far[i] + at),
                                         reinterpret_cast<MX4_LDS void*>(to), 16, 0, 0);
    else
        buffer_to_lds(L.a, to, L.a_src[i], at);
}
template <typename T, bool kFar>
__device__ __forceinline__ void fetch_b(MX4_LDS unsigned char* wr, const TileLane<T, kFar>& L, int at, int i) {
    buffer_to_lds(L.b, wr + (L.wave * T::kFetchB + i) * 1024, L.b_src[i], at);
}

// One fragment of step u of the stage at `rd`. What is read is not being written;
// __restrict__ says so, or the compiler would wait for the fetches in flight.
template <typename T, bool kFar>
__device__ __forceinline__ i32x4 read_a(const MX4_LDS unsigned char* __restrict__ rd, const TileLane<T, kFar>& L, int u, int f) {
    return *reinterpret_cast<const MX4_LDS i32x4*>(rd + L.a_off[u] + f * 4096);
}
template <typename T, bool kFar>
__device__ __forceinline__ i32x4 read_b(const MX4_LDS unsigned char* __restrict__ rd, const TileLane<T, kFar>& L, int u, int f) {
    return *reinterpret_cast<const MX4_LDS i32x4*>(rd + L.b_off[u] + f * 4096);
}

// acc += a b in acc's own registers, written out because the compiler, with the
// products held in their places, gives them other registers and copies. It does not
// know that a value is there only after the instruction's passes (settle()).
__device__ __forceinline__ void mfma_in_place(i32x16& acc, i32x4 a, i32x4 b) {
    asm volatile("v_mfma_i32_32x32x32_i8 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}

// Until all but the last kCount loads have landed, and all reads of LDS.
template <int kCount>
__device__ __forceinline__ void wait_for_all_but() {
    static_assert(kCount < 64);
    __builtin_amdgcn_s_waitcnt((kCount & 15) | (kCount >> 4) << 14 | 7 << 4);
}

// Between the last product and the first use of its value: its passes are over.
__device__ __forceinline__ void settle() {
    asm volatile("s_nop 15\n s_nop 15" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// acc[i][f][v] = the sum of row wave_row + 32 i + lane % 32 and of the wave's column
// 32 f + 8 (v / 4) + 4 (lane / 32) + v % 4. a_row(i): where the lane's row of the wave's
// fetch i of A begins, in bytes from A's resource on (kFar: its address).
template <typename T, bool kFar, typename RowOf>
__device__ __forceinline__ void tile_sums(MX4_LDS unsigned char* lds, __amdgpu_buffer_rsrc_t a, RowOf a_row,
                                          __amdgpu_buffer_rsrc_t b, int row_bytes, int wave, int lane,
                                          typename T::Sums& acc) {
    constexpr int kColFrags = T::kColFrags;
    const int r = lane % 32, h = lane / 32;
    TileLane<T, kFar> L;
    L.a = a, L.b = b;
    L.wave = wave;
    // The block that the lane's place in LDS takes, of row lane / 8 of a fetch.
#pragma unroll
    for (int i = 0; i < T::kFetchA; ++i) {
        const int block = (lane % 8 ^ (4 * (i & 1) + lane / 16)) * 16;
        if constexpr (kFar) L.a_far[i] = (global_bytes)(a_row(i)) + block;  // generic -> global address space
        else L.a_src[i] = a_row(i) + block;
    }
#pragma unroll
    for (int i = 0; i < T::kFetchB; ++i)
        L.b_src[i] = (8 * i + lane / 8) * row_bytes + (lane % 8 ^ (4 * (i & 1) + lane / 16)) * 16;
    const int wave_row = wave / 2 * (T::kRowFrags * 32), wave_col = wave % 2 * (T::kColFrags * 32);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        L.a_off[t] = (wave_row + r) * 128 + ((2 * t + h) ^ r / 2 % 8) * 16;
        L.b_off[t] = (wave_col + r) * 128 + ((2 * t + h) ^ r / 2 % 8) * 16;
    }
    const int stages = row_bytes / kLine, end = row_bytes - kLine;
    const auto slot_a = [&](int s) { return lds + (s & 1) * T::kSlotBytes; };
    // B's buffers in turn: of stage s, s + 1 and s + 2.
    MX4_LDS unsigned char *b_here = lds + T::kFirstB, *b_next = b_here + T::kSlotBytes, *b_last = b_next + T::kSlotBytes;
    const auto offset_of = [&](int s) { return s < stages ? s * kLine : end; };

    // What is fetched in a stage's time, A's before B's, half of it after the barrier and
    // half in the next stage's first step.
    constexpr int kI = T::kRowFrags, kA = T::kFetchA, kAll = kA + T::kFetchB, kEarly = kAll / 2;
    constexpr int kSlots = kI * kColFrags;
#pragma unroll
    for (int i = 0; i < kA; ++i) fetch_a<T, kFar>(slot_a(0), L, 0, i);
#pragma unroll
    for (int i = 0; i < T::kFetchB; ++i) fetch_b<T, kFar>(b_here, L, 0, i);
#pragma unroll
    for (int i = 0; i < T::kFetchB; ++i) fetch_b<T, kFar>(b_next, L, offset_of(1), i);
#pragma unroll
    for (int i = 0; i < kEarly; ++i) {
        if (i < kA) fetch_a<T, kFar>(slot_a(1), L, offset_of(1), i < kA ? i : 0);
        else fetch_b<T, kFar>(b_last, L, offset_of(2), i - kA);
    }
#pragma unroll
    for (int i = 0; i < kI; ++i)
#pragma unroll
        for (int f = 0; f < kColFrags; ++f) {
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][f][e] = 0;
            asm volatile("" : "+a"(acc[i][f]));  // cleared here, while the fetch is under way
        }
    wait_for_all_but<T::kFetchB + kEarly>();
    lds_barrier();

    i32x4 av[2][kI], bv[2][kColFrags];
#pragma unroll
    for (int f = 0; f < kColFrags; ++f) bv[0][f] = read_b<T, kFar>(b_here, L, 0, f);
#pragma unroll
    for (int i = 0; i < kI; ++i) av[0][i] = read_a<T, kFar>(lds, L, 0, i);

    // Every product is held in its place, with at most a fragment's read and a fetch
    // behind it: the matrix unit is busy meanwhile. The fetch of a stage is spread over
    // two steps: the address unit takes 16 cycles for an instruction, and a wave that
    // waits for it multiplies nothing.
    for (int s = 0; s < stages; ++s) {
        const int a_next = offset_of(s + 1), a_after = offset_of(s + 2), b_after = offset_of(s + 3);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const MX4_LDS unsigned char *a_from = t < 3 ? slot_a(s) : slot_a(s + 1), *b_from = t < 3 ? b_here : b_next;
            if (t == 3) {
                // All of stage s + 1; what may be missing is B's stage s + 2.
                wait_for_all_but<T::kFetchB>();
                lds_barrier();
            }
#pragma unroll
            for (int m = 0; m < kSlots; ++m) {
                const int i = m / kColFrags, f = m % kColFrags;
                mfma_in_place(acc[i][f], bv[t & 1][f], av[t & 1][i]);
                if (m < kColFrags)
                    bv[(t + 1) & 1][m < kColFrags ? m : 0] = read_b<T, kFar>(b_from, L, (t + 1) % 4, m);
                else if (m < kColFrags + kI)
                    av[(t + 1) & 1][m < kColFrags + kI ? m - kColFrags : 0] = read_a<T, kFar>(a_from, L, (t + 1) % 4, m - kColFrags);
                // Fetch j of a step's lies behind product (j + 1) kSlots / kEarly - 1.
#pragma unroll
                for (int j = 0; j < kEarly; ++j)
                    if (m == (j + 1) * kSlots / kEarly - 1) {
                        const int i0 = kEarly + j;
                        if (t == 0) {
                            if (i0 < kA) fetch_a<T, kFar>(slot_a(s + 1), L, a_next, i0 < kA ? i0 : 0);
                            else fetch_b<T, kFar>(b_last, L, a_after, i0 - kA);
                        }
                        if (t == 3) {
                            if (j < kA) fetch_a<T, kFar>(slot_a(s), L, a_after, j < kA ? j : 0);
                            else fetch_b<T, kFar>(b_here, L, b_after, j - kA);
                        }
                    }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        MX4_LDS unsigned char* const free = b_here;
        b_here = b_next, b_next = b_last, b_last = free;
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

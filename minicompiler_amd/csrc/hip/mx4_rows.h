// Tiles of 16 rows of a weight matrix as operands of the bf16 (fp16) matrix
// instruction, straight from memory, for products of few rows (moe.hip,
// gemm_mx4_weights.hip) and of two quantised operands (gemm_mx4.hip).
#pragma once

#include "mx4_device.h"

namespace mx4 {

__host__ __device__ inline int padded(int k) { return (k + kStep - 1) / kStep * kStep; }

// kTiles tiles of 16 rows in steps of 128 elements. Lane (r, q) supplies row r in
// four instructions s: of 16-bit rows elements 32 s + 8 q .. + 7 of the step, of
// mx4 ones 32 q + 8 s .. + 7 (block q of the step is its 16 bytes).
// Loaded by lane 4 r + q, and given to lane (r, q) afterwards: the address unit
// takes the 16 bytes of four neighbouring lanes together where they follow each
// other, and a lane of each row by itself.
// kOdd: 16-bit rows that start at odd elements, or some of them. Loads at odd
// elements halved the rate (101 MB in 61 us, 30 with even rows): a lane takes the
// four dwords from the one with its first element on, gets the fifth, with its
// last, from the lane behind, and shifts.
// kHalf: fp16 rows, for the fp16 instruction (else cut into two bf16 pieces).
template <int kType, int kTiles, bool kOdd = false, bool kHalf = false>
struct Rows {
    static constexpr bool kQuant = kType == kMx4;
    static constexpr int kPiecesW = kType == kF16 && !kHalf ? 2 : 1;
    static constexpr int kRaw = kQuant ? 1 : 4;

    struct Step {
        u32x4 w[kTiles][kRaw];
        unsigned behind[kTiles];  // odd rows, lanes of part 0: the dword behind the step
        int shift[kTiles];
        unsigned scales;  // lane 16 i + r: of row r of tile i
    };

    __amdgpu_buffer_rsrc_t rows[kTiles];  // from each tile's first row on, to the weights' end
    int at[kTiles];                       // lane's row and chunk as loaded: row lane / 4, chunk lane % 4
    const unsigned char* scale_row;
    int shift[kTiles];
    int k, r, q, part, from;  // part: the chunk that the lane loads; from: where its own was loaded, in bytes

    __device__ __forceinline__ static int offset(int q, int s) { return kQuant ? 32 * q + 8 * s : 32 * s + 8 * q; }

    // first(i): tile i's first row of `all`, the same in every lane.
    template <typename First>
    __device__ __forceinline__ void open(const void* base, const unsigned char* scales, int k_, long long all, First first) {
        const int lane = threadIdx.x % 64;
        r = lane % 16, q = lane / 16, part = lane % 4, from = (4 * r + q) * 4, k = k_;
        const int row_bytes = kQuant ? padded(k) / 2 : 2 * k;
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
            const long long row = first(i), left = all - row;
            const unsigned char* p = static_cast<const unsigned char*>(base) + row * row_bytes;
            const int odd = kOdd ? static_cast<int>(reinterpret_cast<std::uintptr_t>(p) & 2) : 0;
            // Whole dwords, to the one with the last element: what lies past it reads as zeros.
            const int bytes = (odd + (left < 16 ? static_cast<int>(left) : 16) * row_bytes + 3) & ~3;
            rows[i] = __builtin_amdgcn_make_buffer_rsrc(const_cast<unsigned char*>(p - odd), 0, bytes, 0x00020000);
            const int start = odd + lane / 4 * row_bytes;
            shift[i] = kOdd ? start & 2 : 0;
            at[i] = start - shift[i] + 16 * part;
            if constexpr (kQuant) {
                if (q == i) scale_row = scales + (row + (r < left ? r : 0)) * (padded(k) / 32);
            }
        }
    }

    __device__ __forceinline__ void load(int t, Step& st) const {
        if constexpr (kQuant) {
            static_assert(kTiles <= 4);
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
                st.w[i][0] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rows[i], at[i], t * 64, 0));
            // A dword per row from one lane each, shared out later: a byte per
            // lane would be as many accesses as the codes.
            if (q < kTiles) st.scales = *reinterpret_cast<const unsigned*>(scale_row + t * 4);
        } else {
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
#pragma unroll
                for (int s = 0; s < 4; ++s)
                    st.w[i][s] = __builtin_bit_cast(
                        u32x4, __builtin_amdgcn_raw_buffer_load_b128(rows[i], at[i] + 64 * s, t * 256, 0));
                if constexpr (kOdd) {
                    st.shift[i] = shift[i];
                    if (part == 0)
                        st.behind[i] = __builtin_amdgcn_raw_buffer_load_b32(rows[i], at[i] + 256, t * 256, 0);
                }
            }
        }
    }

    // Whether step t reaches past the end of 16-bit rows, into the next one's elements;
    // those to zeros (they meet zeros, but may be no numbers).
    __device__ __forceinline__ bool past_end(int t) const { return !kQuant && (t + 1) * kStep > k; }
    __device__ __forceinline__ void cut_off(int t, Step& st) const {
        if constexpr (!kQuant) {
#pragma unroll
            for (int i = 0; i < kTiles; ++i) {
#pragma unroll
                for (int s = 0; s < 4; ++s)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int low = t * kStep + offset(part, s) + 2 * j - (kOdd && st.shift[i] != 0 ? 1 : 0);
                        st.w[i][s][j] &= (low < k ? 0xffffu : 0u) | (low + 1 < k ? 0xffff0000u : 0u);
                    }
                if constexpr (kOdd) st.behind[i] = 0;
            }
        }
    }

    // Tile i's scale byte of lane's block.
    __device__ __forceinline__ unsigned scale(const Step& st, int i) const {
        const int of_row = __builtin_amdgcn_ds_bpermute((16 * i + r) * 4, static_cast<int>(st.scales));
        return static_cast<unsigned>(of_row) >> (8 * q) & 255u;
    }

    __device__ __forceinline__ unsigned pass(unsigned loaded) const {
        return static_cast<unsigned>(__builtin_amdgcn_ds_bpermute(from, static_cast<int>(loaded)));
    }

    // Tile i's operand of instruction s (mx4: with lane's scale).
    __device__ __forceinline__ void operand(const Step& st, int i, int s, float scale, u32x4 (&w)[kPiecesW]) const {
        if constexpr (kQuant) {
            w[0] = decode_eight(pass(st.w[i][0][s]), scale);
        } else {
            u32x4 raw = st.w[i][s];
            if constexpr (kOdd) {
                // A chunk's fifth dword is the first of the next, in the next lane or the next load's first lane.
                const unsigned give = part != 0 ? raw[0] : s < 3 ? st.w[i][s < 3 ? s + 1 : 3][0] : st.behind[i];
                const unsigned fifth =
                    static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(give), 0x39, 0xf, 0xf, false));
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    raw[j] = __builtin_amdgcn_alignbyte(j < 3 ? st.w[i][s][j + 1] : fifth, raw[j], st.shift[i]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) raw[j] = pass(raw[j]);
            if constexpr (kType == kBf16 || kHalf) {
                w[0] = raw;
            } else {
                float v[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[2 * j] = to_f32<kF16>(raw[j] & 0xffffu);
                    v[2 * j + 1] = to_f32<kF16>(raw[j] >> 16);
                }
                cut_eight<2>(v, w);
            }
        }
    }
};

}  // namespace mx4

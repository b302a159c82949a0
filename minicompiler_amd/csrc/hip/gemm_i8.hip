// Products of two operands quantised to 8-bit integers (i8.h): C = A B^T in exact
// 32-bit sums, scaled by row and column, with bias and activation; and the
// experts' products on a plan, the same for each expert's slots.
//
// Scales belong to whole rows of A and B, so that sums over all of k stay integers and
// the scales, the bias and the activation are one step at the end, in fp32.
//
// Few rows: B is what has to be read (one row by 14336x4096 10.5 us, 5.6 TB/s; one token's 8
// experts, 2048 by 2 x 1024, 8.9). Blocks of 16x32 to 32x64 take all of k, without LDS
// before the end: a wave's loads are in flight at once (1000x1001x1023 7.0 us, 4096 of k and
// columns by 32 rows 5.5). Many rows: tiles of 128x128 or 256x256 (gemm_i8_tiles.h; on the
// plan of 2048 tokens, 8 of 64 experts, up 105-126 us by the chip, down 111-115).
//
// Down keeps each pair's product in fp32 until the token's pairs are summed in their order:
// 16-bit ones would save half of 268 MB there (2048 tokens, 21 of 111 us in the sum) and
// round each term, atomic sums would depend on the order. So its plan has every pair; a part of a
// plan's experts is Up's alone.

#include <cmath>
#include <type_traits>

#include "gemm_i8_tiles.h"

namespace {

using namespace i8;

// What the rows of C are. Dense: row i of A makes row i of C. Up: slot i takes row
// order[i] / top_k of A and makes row i of C. Down: slot i takes row i of A and makes
// row order[i] of the workspace, fp32 and times its gate.
constexpr int kDense = 0, kUp = 1, kDown = 2;

struct Product {
    const unsigned char *a, *b;
    const float *a_scales, *b_scales, *bias;
    void* c;
    const int *order, *offsets;
    const float* gates;
    int m, n;  // rows of C (slots), columns of C
    int row_bytes, a_rows, top_k, experts, activation, c_dtype;
    unsigned tiles_n;
};

// Where a block works: rows `first` to `end` of C, on expert `expert`.
struct Place {
    int expert, first, end;
};

// Entry `want` of what count(slots of an expert) adds up to over the experts in order: the
// expert and the entry's number there, or no expert, `want` less the sum of all. A wave
// looks at 64 experts at a time.
struct Entry {
    int expert, from, to;  // the expert's slots
    unsigned number;
};
template <typename Count>
__device__ __forceinline__ bool find_entry(const Product& p, unsigned& want, Entry& found, Count count) {
    const int lane = threadIdx.x % 64;
    for (int base = 0; base < p.experts; base += 64) {
        const int e = base + lane;
        int from = 0, to = 0;
        if (e < p.experts) from = p.offsets[e], to = p.offsets[e + 1];
        from = max(from, 0), to = max(min(to, p.m), from);
        const unsigned mine = count(static_cast<unsigned>(to - from));
        unsigned up_to = mine;  // of the lanes up to this one
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const unsigned o = __shfl_up(up_to, d);
            if (lane >= d) up_to += o;
        }
        const unsigned long long here = __ballot(up_to > want);
        if (here != 0) {
            const int at = __builtin_ctzll(here);
            found = {base + at, static_cast<int>(__builtin_amdgcn_readlane(from, at)),
                     static_cast<int>(__builtin_amdgcn_readlane(to, at)),
                     want - __builtin_amdgcn_readlane(up_to - mine, at)};
            return true;
        }
        want -= __builtin_amdgcn_readlane(up_to, 63);
    }
    return false;
}

// What all experts' slots add up to.
template <typename Count>
__device__ __forceinline__ unsigned sum_of_entries(const Product& p, Count count) {
    unsigned all = 0;
    for (int base = 0; base < p.experts; base += 64) {
        const int e = base + static_cast<int>(threadIdx.x % 64);
        int from = 0, to = 0;
        if (e < p.experts) from = p.offsets[e], to = p.offsets[e + 1];
        from = max(from, 0), to = max(min(to, p.m), from);
        all += count(static_cast<unsigned>(to - from));
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) all += __shfl_xor(all, d);
    return __builtin_amdgcn_readfirstlane(all);
}

// Job `want` of the experts' slots, up to kRows of one expert's each; end = first: none.
template <int kRows>
__device__ __forceinline__ Place find_job(const Product& p, unsigned want) {
    Entry e;
    if (!find_entry(p, want, e, [](unsigned n) { return (n + kRows - 1) / kRows; })) return {0, 0, 0};
    return {e.expert, e.from + static_cast<int>(e.number * kRows), e.to};
}

// The same in tiles of kRows, an expert's last of half as many rows where that holds it.
// Those come after all others, so that the launch ends on short work.
template <int kRows>
__device__ __forceinline__ Place find_tile(const Product& p, unsigned want) {
    Entry e;
    if (find_entry(p, want, e, [](unsigned n) { return (n + kRows / 2 - 1) / kRows; })) {
        const int first = e.from + static_cast<int>(e.number * kRows);
        return {e.expert, first, min(first + kRows, e.to)};
    }
    if (find_entry(p, want, e, [](unsigned n) { return (n + kRows / 2 - 1) / kRows * kRows < n ? 1u : 0u; }))
        return {e.expert, e.to - (e.to - e.from) % kRows, e.to};
    return {0, 0, 0};
}

constexpr int kDirectWaves = 8;

// A block computes 16 kM rows by 16 kN columns of C (SwiGLU: the second half of the
// column tiles are the up rows of the first half's columns); its kWaves waves take
// the steps of 128 k in turn and their sums are added at the end. Four neighbouring
// lanes load 64 bytes of a row, which are then passed to the lanes that multiply them.
template <int kMode, bool kGated, int kM, int kN, int kWaves>
__global__ __launch_bounds__(kWaves * 64) void i8_direct(const Product p) {
    __shared__ i32x4 space[kWaves * kM * kN * 64];
    constexpr int kCols = kGated ? kN / 2 : kN;  // column tiles of C
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int r = lane % 16, q = lane / 16, part = lane % 4, pass = (4 * r + q) * 4;
    unsigned chunk = blockIdx.x / p.tiles_n, tile = blockIdx.x % p.tiles_n;
    if constexpr (kMode == kDense) {
        // A column tile's rows one after the other on one XCD, whose L2 has its weights.
        const unsigned all = gridDim.x, t = blockIdx.x < all / 8 * 8 ? blockIdx.x % 8 * (all / 8) + blockIdx.x / 8 : blockIdx.x;
        const unsigned chunks = all / p.tiles_n;
        chunk = t % chunks, tile = t / chunks;
    }
    const int col0 = static_cast<int>(tile) * 16 * kCols;
    Place place{0, 0, p.m};
    long long row0 = static_cast<long long>(chunk) * 16 * kM;
    if constexpr (kMode != kDense) {
        place = find_job<16 * kM>(p, chunk);
        if (place.first >= place.end) return;
        row0 = place.first;
    }
    const int end = place.end;
    const long long b_rows = kGated ? 2LL * p.n : p.n;
    const unsigned char* b0 = p.b + place.expert * b_rows * p.row_bytes;
    const unsigned char *a[kM], *b[kN];
#pragma unroll
    for (int i = 0; i < kM; ++i) {
        long long row = row0 + 16 * i + lane / 4;
        row = row < end ? row : end - 1;
        if constexpr (kMode == kUp) {
            row = p.order[row] / p.top_k;
            row = row < 0 ? 0 : row < p.a_rows ? row : p.a_rows - 1;
        }
        a[i] = p.a + row * p.row_bytes + part * 16;
    }
#pragma unroll
    for (int j = 0; j < kN; ++j) {
        const int col = col0 + 16 * (j % kCols) + lane / 4;
        const long long row = (col < p.n ? col : p.n - 1) + (j >= kCols ? p.n : 0LL);
        b[j] = b0 + row * p.row_bytes + part * 16;
    }
    i32x4 acc[kM * kN];
#pragma unroll
    for (int i = 0; i < kM * kN; ++i) acc[i] = i32x4{0, 0, 0, 0};
    // Of small dense blocks the next line is on its way while one is multiplied (one row by
    // 14336x4096 10.5 us, 10.9 without); larger ones lose a block per CU to it (1000x1001x1023
    // 8.0 and 6.3), and on a plan it gains nothing.
    constexpr bool kAhead = kMode == kDense && kM * kN <= 4;
    i32x4 a_next[2][kM], b_next[2][kN];
    const auto load = [&](int at) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < kM; ++i) a_next[h][i] = *reinterpret_cast<const i32x4*>(a[i] + at + 64 * h);
#pragma unroll
            for (int j = 0; j < kN; ++j) b_next[h][j] = *reinterpret_cast<const i32x4*>(b[j] + at + 64 * h);
        }
    };
    if (kAhead && wave * kLine < p.row_bytes) load(wave * kLine);
    for (int at = wave * kLine; at < p.row_bytes; at += kWaves * kLine) {
        if (!kAhead) load(at);
        i32x4 av[2][kM], bv[2][kN];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < kM; ++i) av[h][i] = a_next[h][i];
#pragma unroll
            for (int j = 0; j < kN; ++j) bv[h][j] = b_next[h][j];
        }
        if (kAhead && at + kWaves * kLine < p.row_bytes) load(at + kWaves * kLine);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
#pragma unroll
                for (int i = 0; i < kM; ++i) av[h][i][e] = __builtin_amdgcn_ds_bpermute(pass, av[h][i][e]);
#pragma unroll
                for (int j = 0; j < kN; ++j) bv[h][j][e] = __builtin_amdgcn_ds_bpermute(pass, bv[h][j][e]);
            }
#pragma unroll
            for (int i = 0; i < kM; ++i)
#pragma unroll
                for (int j = 0; j < kN; ++j) acc[i * kN + j] = mfma(bv[h][j], av[h][i], acc[i * kN + j]);
        }
    }
#pragma unroll
    for (int i = 0; i < kM * kN; ++i) space[(wave * kM * kN + i) * 64 + lane] = acc[i];
    __syncthreads();
    const auto sum_of = [&](int tile) {
        i32x4 sum = space[tile * 64 + lane];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) sum += space[(w * kM * kN + tile) * 64 + lane];
        return sum;
    };
#pragma unroll 1
    for (int t = wave; t < kM * kCols; t += kWaves) {
        const int i = t / kCols, j = t % kCols;
        const long long row = row0 + 16 * i + r;
        const int col = col0 + 16 * j + 4 * q;
        if (row >= end || col >= p.n) continue;
        const int left = p.n - col;
        long long a_row = row, c_row = row;
        if constexpr (kMode == kUp) {
            a_row = p.order[row] / p.top_k;
            a_row = a_row < 0 ? 0 : a_row < p.a_rows ? a_row : p.a_rows - 1;
        }
        if constexpr (kMode == kDown) {
            c_row = p.order[row];
            if (c_row < 0 || c_row >= p.m) continue;
        }
        const RowScale sa = row_scale(p.a_scales[a_row]);
        const long long b_row = place.expert * b_rows + col;
        // One half's four columns, scaled, with the bias.
        const auto scaled = [&](i32x4 sum, long long at) {
            f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (e < left) v[e] = static_cast<float>(sum[e]) * sa.s * p.b_scales[at + e];
            if (sa.back != 1.0f) v *= sa.back;
            if (p.bias != nullptr) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (e < left) v[e] += p.bias[at + e];
            }
            return v;
        };
        f32x4 v = scaled(sum_of(i * kN + j), b_row);
        if constexpr (kGated) {
            const f32x4 up = scaled(sum_of(i * kN + kCols + j), b_row + p.n);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = v[e] * sigmoid(v[e]) * up[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = activate(v[e], p.activation);
        }
        if constexpr (kMode == kDown) {
            const float gate = p.gates[c_row];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] *= gate;
            store_four<kF32>(p.c, c_row * p.n + col, v, left);
        } else {
            store_four_as(p.c_dtype, p.c, c_row * p.n + col, v, left);
        }
    }
}

// The row of A that row `row` of C takes.
template <int kMode>
__device__ __forceinline__ long long a_row_of(const Product& p, long long row) {
    if constexpr (kMode != kUp) return row;
    const int token = p.order[row] / p.top_k;
    return token < 0 ? 0 : token < p.a_rows ? token : p.a_rows - 1;
}

// A wave's sums (tile_sums) scaled, with bias and activation, to C: rows row0 .. up to
// `end`, columns col0 on, by way of the wave's share of LDS (`lds`), so that a short loop
// (a launch meets a cold instruction cache) stores whole lines. In passes: 64 columns of
// all rows, or (kGated) 64 rows with both halves of their columns. Block c of 16 bytes of
// row r lies at c ^ (r % 16). What goes with a row lies in `side`, 16 bytes each: in
// registers it would be held through everything, and the large tiles have none to spare.
template <int kMode, bool kGated, int kOut, typename T>
__device__ __forceinline__ void store_tile(MX4_LDS unsigned char* lds, MX4_LDS unsigned char* side, const Product& p,
                                           const typename T::Sums& acc, int expert, long long row0, long long end, int col0,
                                           int lane) {
    constexpr int kRowFrags = T::kRowFrags, kColFrags = T::kColFrags;
    constexpr int kHalves = kRowFrags / 2;  // of 64 rows
    constexpr int kPasses = kGated ? kHalves : kColFrags / 2, kPassFrags = kGated ? kColFrags : 2;
    constexpr int kRowBytes = kPassFrags * 128, kPassRows = kGated ? 64 : 64 * kHalves;
    constexpr int kAcross = (kGated ? kColFrags / 2 : 2) * 4, kBatch = 64 / kAcross;  // lanes along a row, rows at a time
    static_assert(kPasses <= 2 && kPassRows / kBatch % 4 == 0);
    const long long b_row = expert * (kGated ? 2LL * p.n : p.n);
    const int line = lane % 32, half = lane / 32;
    // Rows lane and lane + 64: on their way while sums go to LDS.
    float sa[kHalves], gate[kHalves];
    int c_row[kHalves];  // Down: of the workspace, -1: not stored
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
        const long long row = row0 + lane + 64 * h;
        sa[h] = 0.0f, gate[h] = 0.0f, c_row[h] = -1;
        if (row < end) {
            sa[h] = p.a_scales[a_row_of<kMode>(p, row)];
            if constexpr (kMode == kDown) {
                c_row[h] = p.order[row];
                if (c_row[h] >= p.m) c_row[h] = -1;
                if (c_row[h] >= 0) gate[h] = p.gates[c_row[h]];
            }
        }
    }
    const auto rows_to_lds = [&] {
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
            const RowScale r = row_scale(sa[h]);
            MX4_LDS unsigned char* at = side + (lane + 64 * h) * 16;
            if constexpr (kMode == kDown)
                *reinterpret_cast<MX4_LDS f32x4*>(at) = f32x4{r.s, r.back, gate[h], __builtin_bit_cast(float, c_row[h])};
            else
                *reinterpret_cast<MX4_LDS f32x2*>(at) = f32x2{r.s, r.back};
        }
    };
    const auto to_lds = [&](auto pass) {
        constexpr int h = decltype(pass)::value;
#pragma unroll
        for (int i = 0; i < (kGated ? 2 : kRowFrags); ++i)
#pragma unroll
            for (int f = 0; f < kPassFrags; ++f) {
                const i32x16& sums = kGated ? acc[2 * h % kRowFrags + i][f] : acc[i][2 * h % kColFrags + f];
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *reinterpret_cast<MX4_LDS i32x4*>(lds + (32 * i + line) * kRowBytes +
                                                      ((8 * f + 2 * g + half) ^ line % 16) * 16) =
                        i32x4{sums[4 * g], sums[4 * g + 1], sums[4 * g + 2], sums[4 * g + 3]};
            }
    };
    // Columns 8 c .. + 7 of the wave's row: blocks 2 c and 2 c + 1 (the up ones behind all gate ones).
    const auto sums_of = [&](int row, int block, int (&sum)[8]) {
        const MX4_LDS unsigned char* at = lds + row * kRowBytes;
        const i32x4 lo = *reinterpret_cast<const MX4_LDS i32x4*>(at + ((block + lane % kAcross * 2) ^ row % 16) * 16);
        const i32x4 hi = *reinterpret_cast<const MX4_LDS i32x4*>(at + ((block + lane % kAcross * 2 + 1) ^ row % 16) * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = lo[e], sum[4 + e] = hi[e];
    };
#pragma unroll 1
    for (int h = 0; h < kPasses; ++h) {
        if (h == 0) {
            to_lds(std::integral_constant<int, 0>{});
            rows_to_lds();
        } else {
            wave_lds_order();  // behind the first pass's reads
            to_lds(std::integral_constant<int, 1>{});
        }
        wave_lds_order();
        // Eight columns of a row per lane, kBatch rows at a time, four times that under way.
        const int col = col0 + (kGated ? 0 : 64 * h) + lane % kAcross * 8, left = p.n - col;
        float scale[8], bias[8], up_scale[8], up_bias[8];
        load_eight<kF32>(p.b_scales, b_row + col, left, scale);
        load_eight<kF32>(p.bias, b_row + col, p.bias != nullptr ? left : 0, bias);
        if constexpr (kGated) {
            load_eight<kF32>(p.b_scales, b_row + p.n + col, left, up_scale);
            load_eight<kF32>(p.bias, b_row + p.n + col, p.bias != nullptr ? left : 0, up_bias);
        }
        const auto rows = [&](auto act, auto store) {
#pragma unroll 1
            for (int it = 0; it < kPassRows / kBatch; it += 4) {
                int sum[4][8], up[4][8];
                f32x2 scale_of[4];
                float g[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int row = kBatch * (it + u) + lane / kAcross;
                    const MX4_LDS unsigned char* with = side + (row + (kGated ? 64 * h : 0)) * 16;
                    scale_of[u] = *reinterpret_cast<const MX4_LDS f32x2*>(with);
                    if constexpr (kMode == kDown) g[u] = *reinterpret_cast<const MX4_LDS float*>(with + 8);
                    sums_of(row, 0, sum[u]);
                    if constexpr (kGated) sums_of(row, 2 * kAcross, up[u]);
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float s = scale_of[u][0], back = scale_of[u][1];
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        v[e] = static_cast<float>(sum[u][e]) * s * scale[e] * back + bias[e];
                        if constexpr (kGated)
                            v[e] *= sigmoid(v[e]) * (static_cast<float>(up[u][e]) * s * up_scale[e] * back + up_bias[e]);
                        else if constexpr (kMode == kDown)
                            v[e] *= g[u];
                        else
                            v[e] = act(v[e]);
                    }
                    store(it + u, v);
                }
            }
        };
        const auto with_act = [&](auto store) {
            if (kGated || kMode == kDown || p.activation == MCHIP_ACT_NONE) rows([](float u) { return u; }, store);
            else if (p.activation == MCHIP_ACT_RELU) rows([](float u) { return activate(u, MCHIP_ACT_RELU); }, store);
            else rows([](float u) { return gelu(u); }, store);
        };
        // Rows of whole eights go out through a resource of the wave's rows of C: no
        // addresses to work out, and what lies past the last row or column is dropped.
        constexpr int kOne = kSize<kOut>;
        const long long row_size = static_cast<long long>(p.n) * kOne;
        if (kMode != kDown && p.n % 8 == 0 && row_size * 16 * 16 < (1LL << 31)) {
            const __amdgpu_buffer_rsrc_t c = rows_from(static_cast<unsigned char*>(p.c) + row0 * row_size, end - row0,
                                                       static_cast<int>(row_size));
            const int step = __builtin_amdgcn_readfirstlane(kBatch * static_cast<int>(row_size));
            const unsigned at = left > 0 ? static_cast<unsigned>(lane / kAcross * static_cast<int>(row_size) + col * kOne) : 1u << 31;
            with_act([&](int it, const float(&v)[8]) {
                const int from = static_cast<int>(at + static_cast<unsigned>((it + (kGated ? h * (64 / kBatch) : 0)) * step));
                if constexpr (kOut == kF32) {
                    const f32x4 lo = {v[0], v[1], v[2], v[3]}, hi = {v[4], v[5], v[6], v[7]};
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, lo), c, from, 0, 2);
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, hi), c, from + 16, 0, 2);
                } else {
                    u16x8 out;
#pragma unroll
                    for (int e = 0; e < 8; ++e) out[e] = to_16<kOut>(v[e]);
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, out), c, from, 0, 2);
                }
            });
        } else {
            with_act([&](int it, const float(&v)[8]) {
                const int row = kBatch * it + lane / kAcross;
                if constexpr (kMode == kDown) {
                    const int c_row = *reinterpret_cast<const MX4_LDS int*>(side + row * 16 + 12);
                    if (c_row >= 0 && left > 0) store_eight<kOut, false>(p.c, static_cast<long long>(c_row) * p.n + col, v, left);
                } else {
                    const long long c_row = row0 + (kGated ? 64 * h : 0) + row;
                    if (c_row < end && left > 0) store_eight<kOut>(p.c, c_row * p.n + col, v, left);
                }
            });
        }
    }
}

// Rows row0 .. of C up to `end` (at most kRows) by kCols (kGated: half of it) columns from
// col0 on. kFar: gathered rows of an A past what a resource reaches.
template <int kMode, bool kGated, int kOut, int kRows, int kCols, int kSlotRows, bool kFar = false>
__device__ __forceinline__ void product_tile(MX4_LDS unsigned char* lds, const Product& p, int expert, long long row0,
                                             long long end, int col0) {
    typedef Tile<kRows, kCols, kSlotRows> T;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    constexpr int kShareA = kRows / 4, kShareB = kCols / 4;  // rows, a wave's to fetch
    // A's rows, from the wave's share of the tile on, or (gathered) all.
    const long long a0 = kMode == kUp ? 0 : row0 + wave * kShareA;
    const __amdgpu_buffer_rsrc_t a = kFar            ? resource(p.a, 0)
                                     : kMode == kUp ? resource(p.a, p.a_rows * p.row_bytes)
                                                    : rows_from(p.a + a0 * p.row_bytes, end - a0, p.row_bytes);
    const auto a_row = [&](int i) {
        const int in_share = i * 8 + lane / 8;
        if constexpr (kMode != kUp) return in_share * p.row_bytes;
        const long long row = row0 + wave * kShareA + in_share;
        const long long token = a_row_of<kMode>(p, row < end ? row : end - 1);
        if constexpr (kFar) return p.a + token * p.row_bytes;
        else return static_cast<int>(token) * p.row_bytes;
    };
    // B's rows that the wave fetches: of columns, of gate or of up ones.
    const int b_col = col0 + (kGated ? wave / 2 : wave) * kShareB;
    const long long b0 = expert * (kGated ? 2LL * p.n : p.n) + (kGated ? wave % 2 * static_cast<long long>(p.n) : 0) + b_col;
    const __amdgpu_buffer_rsrc_t b = rows_from(p.b + b0 * p.row_bytes, p.n - b_col, p.row_bytes);
    typename T::Sums acc;
    tile_sums<T, kFar>(lds, a, a_row, b, p.row_bytes, wave, lane, acc);
    lds_barrier();  // every wave is past its reads of the ring
    static_assert(kRingA + kRingB > 4);  // behind the waves' shares
    store_tile<kMode, kGated, kOut, T>(lds + wave * T::kSlotBytes, lds + 4 * T::kSlotBytes + wave * 2048, p, acc, expert, row0 + wave / 2 * (kRows / 2), end,
                                       col0 + wave % 2 * (kGated ? kCols / 4 : kCols / 2), lane);
}

// Block t's tile on a plan: an XCD takes an eighth of the tiles that the plan has, consecutive
// ones, so that an expert's weights and a chunk's rows come through one L2.
template <int kTile>
__device__ __forceinline__ bool tile_on_plan(const Product& p, unsigned& t) {
    const unsigned long long have =
        static_cast<unsigned long long>(sum_of_entries(p, [](unsigned n) { return (n + kTile - 1) / kTile; })) * p.tiles_n;
    const unsigned first = static_cast<unsigned>(have * (t % 8) / 8), last = static_cast<unsigned>(have * (t % 8 + 1) / 8);
    t = first + t / 8;
    return t < last;
}

// kTile 256: dense tiles are 256 rows high; the grid has one block per tile plus `halves`
// more, for which that many of the last tiles run as two blocks of 128 rows; on a plan an
// expert's last tile is of 128 rows where that holds it. kTile 128: tiles of 128x128.
// Dense tiles go in panels of kPanel rows of them, column after column. An XCD takes
// consecutive ones, so that those which it works on at a time read few rows through its
// L2 (4 + 8 tiles' rows of 256).
template <int kMode, bool kGated, int kOut, int kTile>
__global__ __launch_bounds__(kTileThreads, kTile == 256 ? 1 : 2) void i8_tiles(const Product p, unsigned full) {
    __shared__ __attribute__((aligned(1024))) unsigned char smem[Tile<kTile, kTile, kTile>::kRingBytes];
    MX4_LDS unsigned char* lds = (MX4_LDS unsigned char*)(smem);  // generic -> LDS address space
    constexpr int kPanel = kTile == 256 ? 4 : 8;
    unsigned t = blockIdx.x, chunk, tile;
    int half = 0;
    if constexpr (kMode == kDense) {
        // Blocks go to the XCDs in turn.
        const auto in_turn = [](unsigned i, unsigned all) { return i < all / 8 * 8 ? i % 8 * (all / 8) + i / 8 : i; };
        if (t >= full) {
            const unsigned part = in_turn(t - full, gridDim.x - full);
            half = 1 + static_cast<int>(part % 2), t = full + part / 2;
        } else {
            t = in_turn(t, full);
        }
        const unsigned all = (static_cast<unsigned>(p.m) + kTile - 1) / kTile;
        const unsigned panel = t / (kPanel * p.tiles_n), in = t % (kPanel * p.tiles_n);
        const unsigned high = min(static_cast<unsigned>(kPanel), all - panel * kPanel);
        chunk = panel * kPanel + in % high, tile = in / high;
    } else {
        if (!tile_on_plan<kTile>(p, t)) return;
        chunk = t / p.tiles_n, tile = t % p.tiles_n;
    }
    const int col0 = static_cast<int>(tile) * (kGated ? kTile / 2 : kTile);
    long long row0 = static_cast<long long>(chunk) * kTile, end = p.m;
    int expert = 0;
    if constexpr (kMode == kDense) {
        if (half == 2) row0 += kTile / 2;
        if (half == 1 && row0 + kTile / 2 < end) end = row0 + kTile / 2;
    } else {
        const Place place = kTile == 256 ? find_tile<256>(p, chunk) : find_job<kTile>(p, chunk);
        expert = place.expert, row0 = place.first, end = place.end;
    }
    if (row0 >= end) return;
    if constexpr (kTile == 256) {
        if (end - row0 > 128)
            product_tile<kMode, kGated, kOut, 256, 256, 256>(lds, p, expert, row0, end, col0);
        else
            product_tile<kMode, kGated, kOut, 128, 256, 256>(lds, p, expert, row0, end, col0);
    } else {
        product_tile<kMode, kGated, kOut, 128, 128, 128>(lds, p, expert, row0, end, col0);
    }
}

// Up by 256x256 tiles where A has 2 GiB or more: 524288 tokens of 4096 on 8 experts, 2 x 1024
// columns, 4.1 ms, as long as 64 tokens less take through a resource (by 32x64 blocks 12.4).
template <bool kGated, int kOut>
__global__ __launch_bounds__(kTileThreads, 1) void i8_far_rows(const Product p, unsigned) {
    __shared__ __attribute__((aligned(1024))) unsigned char smem[Tile<256, 256, 256>::kRingBytes];
    MX4_LDS unsigned char* lds = (MX4_LDS unsigned char*)(smem);  // generic -> LDS address space
    unsigned t = blockIdx.x;
    if (!tile_on_plan<256>(p, t)) return;
    const Place place = find_tile<256>(p, t / p.tiles_n);
    const int col0 = static_cast<int>(t % p.tiles_n) * (kGated ? 128 : 256);
    if (place.first >= place.end) return;
    if (place.end - place.first > 128)
        product_tile<kUp, kGated, kOut, 256, 256, 256, true>(lds, p, place.expert, place.first, place.end, col0);
    else
        product_tile<kUp, kGated, kOut, 128, 256, 256, true>(lds, p, place.expert, place.first, place.end, col0);
}

// y[token] = the sum of its top_k rows of the workspace, in order: 134 MB in 21.7 us, 6.5
// TB/s (most of it still in the last-level cache, past which the tiles do not store).
template <int kOut>
__global__ __launch_bounds__(256) void sum_pairs(const float* __restrict__ pairs, void* __restrict__ y, int tokens,
                                                 int top_k, int n) {
    const unsigned per_row = (static_cast<unsigned>(n) + 3) / 4;
    for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < static_cast<long long>(tokens) * per_row;
         i += static_cast<long long>(gridDim.x) * 256) {
        const long long t = i / per_row;
        const int col = static_cast<int>(i % per_row) * 4;
        f32x4 sum = load_four<kF32>(pairs, t * top_k * n + col, n - col);
        for (int j = 1; j < top_k; ++j) sum += load_four<kF32>(pairs, (t * top_k + j) * n + col, n - col);
        store_four<kOut>(y, t * n + col, sum, n - col);
    }
}

long long tiles(long long size, int tile) { return (size + tile - 1) / tile; }

// Jobs of up to `rows` slots that the plan may have, at most.
long long most_jobs(long long slots, int experts, int rows) {
    return std::min(slots, (slots + std::min<long long>(experts, slots) * (rows - 1)) / rows);
}

// Blocks of a launch in blocks or tiles of rows by columns of B. On a plan of tiles eight XCDs
// have the same number each.
template <int kMode, bool kGated>
long long grid_of(const Product& p, int rows, int cols) {
    const long long chunks = kMode == kDense ? tiles(p.m, rows) : most_jobs(p.m, p.experts, rows);
    const long long all = chunks * tiles(p.n, kGated ? cols / 2 : cols);
    return kMode != kDense && rows >= 128 ? (all + 7) / 8 * 8 : all;
}

template <int kMode, bool kGated, int kM, int kN>
int launch_direct(Product p, hipStream_t stream) {
    constexpr int kCols = kGated ? kN / 2 : kN;
    p.tiles_n = static_cast<unsigned>(tiles(p.n, 16 * kCols));
    return launch_kernel(i8_direct<kMode, kGated, kM, kN, kDirectWaves>,
                         static_cast<unsigned>(grid_of<kMode, kGated>(p, 16 * kM, 16 * kN)), kDirectWaves * 64, 0, stream, p);
}

// How many of `all` dense tiles of 256x256 run as two of 128 rows: those that would leave half
// of a last round or more empty.
int halves_of(long long all, int cus) {
    const int rest = static_cast<int>(all % cus);
    return rest <= cus / 2 ? rest : 0;
}

template <int kMode, bool kGated, int kTile, bool kFar = false>
int launch_tiles(Product p, hipStream_t stream) {
    p.tiles_n = static_cast<unsigned>(tiles(p.n, kGated ? kTile / 2 : kTile));
    const long long all = grid_of<kMode, kGated>(p, kTile, kTile);
    const int halves = kMode == kDense && kTile == 256 ? halves_of(all, device_cus()) : 0;
    const auto go = [&](auto kernel) {
        return launch_kernel(kernel, static_cast<unsigned>(all + halves), kTileThreads, 0, stream, p,
                             static_cast<unsigned>(all - halves));
    };
    if constexpr (kMode == kDown) {
        return go(i8_tiles<kMode, kGated, kF32, kTile>);
    } else if constexpr (kFar) {
        static_assert(kMode == kUp && kTile == 256);
        return p.c_dtype == kF32    ? go(i8_far_rows<kGated, kF32>)
               : p.c_dtype == kBf16 ? go(i8_far_rows<kGated, kBf16>)
                                    : go(i8_far_rows<kGated, kF16>);
    } else {
        return p.c_dtype == kF32    ? go(i8_tiles<kMode, kGated, kF32, kTile>)
               : p.c_dtype == kBf16 ? go(i8_tiles<kMode, kGated, kBf16, kTile>)
                                    : go(i8_tiles<kMode, kGated, kF16, kTile>);
    }
}

// Offsets within A have 32 bits where its rows are gathered through a resource.
template <int kMode>
bool one_resource(const Product& p) {
    return kMode != kUp || static_cast<long long>(p.a_rows) * p.row_bytes < (1LL << 31);
}

// What a variant takes, in microseconds, by its rounds of blocks and k (in units of 4096).
// Measured, 4096 wide and deep unless said: 16x32 blocks 5.5 (16 rows, 128 of them), 5.8 (32
// rows, 256), 8.3 (64, 512), 12.0 (128), 20.6 (256); 32x32 6.5 (32 rows), 7.0 (64), 10.1
// (128), 15.9 (256); 32x64 9.1, 8.9, 8.6, 13.6 and 23.2 (512); 128x128 tiles 17.3 (64 rows),
// 18.4 (512), 20.8 (1024), 35.3 (2048), 68.8 (4096), 103 (6144), 237 (4096 by 14336), 251 (4096, k
// 16384), 516 (8192^3); 256x256 39.5 (1024), 50.7 (2048), 58.9, 108, 222, 204, 432. 4096x4096 of k =
// 128 and 1024: 57 and 113, 61 and 109, 40 and 74, 12.0 and 24.6, 12.2 and 22.9; 4096x14336 of
// 1024: 78.0 and 78.5 by tiles. 64x64 blocks were nowhere a fifth faster than the next. (Half of
// a large tile takes 0.87 of it: fetches bound it.)
// On a plan all take longer (rows gathered, weights from memory). Tokens x 8 of 64 experts, 2048
// deep, 1024 gated columns, by 128x128 and 256x256: 128 tokens 56.1 and 61.3, 512 58 and 62,
// 1024 84 and 79, 2048 121 and 123, 4096 200 and 186; by 16x32 blocks, 128 tokens 60.1, 64 tokens
// 48.3 (55.5, 60.6). Down, 1024 deep, 2048 columns: 512 tokens 45 and 49, 2048 110 and 121.
// (Fitted to that one plan. Where two kernels are near each other it may take the slower: 1024
// tokens' up product runs by 128x128.)
struct Cost {
    double k, cus;
    bool plan;
    double few(double blocks, double one, double fixed, double each) const {
        return 2.5 + (plan ? 1.8 : 1.0) * (blocks <= cus ? 0.5 + one * k : (fixed + each * k) * std::max(1.0, blocks / (2.0 * cus)));
    }
    double small_tiles(double tiles) const {
        if (plan) return 5.0 + 50.0 * k * std::ceil(tiles / (2.0 * cus));
        if (tiles <= cus) return 5.0 + k * (2.0 * tiles <= cus ? 13.0 : 17.0);
        return 3.0 + (3.0 + 30.5 * k) * std::ceil(tiles / cus) / 2.0;
    }
    double large_tiles(double rounds) const { return plan ? 4.0 + rounds * (8.0 + 66.0 * k) : 3.5 + rounds * (6.5 + 49.5 * k); }
};

// The kernel of least cost (MCHIP_I8_*) of those that one launch takes, -1: none.
template <int kMode, bool kGated>
int choose(const Product& p, int cu_count) {
    constexpr bool kPlan = kMode != kDense;
    const double cus = cu_count, experts = static_cast<double>(std::min(p.experts, p.m));
    const Cost cost{p.row_bytes / 4096.0, cus, kPlan};
    const double columns = kGated ? 2.0 * p.n : p.n;
    // Blocks, of rows by columns of B; on a plan every second expert's last is half full.
    const auto blocks = [&](int rows, int cols) {
        const double down = kPlan ? std::max(experts, p.m / static_cast<double>(rows) + experts / 2)
                                  : static_cast<double>(tiles(p.m, rows));
        return down * std::ceil(columns / cols);
    };
    // None where a launch has no room for it.
    const auto or_none = [&](double microseconds, int rows, int cols, int threads) {
        return fits_launch(grid_of<kMode, kGated>(p, rows, cols), threads) ? microseconds : 1e30;
    };
    constexpr int kDirectThreads = kDirectWaves * 64;
    const double b16 = or_none(cost.few(blocks(16, 32), 3.0, 0.8, 4.1), 16, 32, kDirectThreads),
                 b32 = or_none(cost.few(blocks(32, 32), 4.2, 1.6, 7.0), 32, 32, kDirectThreads),
                 b64 = or_none(cost.few(blocks(32, 64), 6.0, 2.1, 9.5), 32, 64, kDirectThreads);
    double rounds;
    if (kPlan) {
        // In rounds and halves of them; a third of the experts' last tiles are halves, which
        // take 0.7 of a tile.
        const double all = std::max(experts * 0.7, p.m / 256.0 + experts * 0.35) * std::ceil(columns / 256.0) / cus;
        rounds = std::max(1.0, std::ceil(2.0 * all) / 2.0);
    } else {
        // Tiles that leave half a round or more empty run as halves.
        const double all = blocks(256, 256), rest = std::fmod(all, cus);
        rounds = std::floor(all / cus) + (rest == 0.0 ? 0.0 : rest <= cus / 2 ? 0.87 : 1.0);
    }
    const bool near = one_resource<kMode>(p);
    const double t128 = near ? or_none(cost.small_tiles(blocks(128, 128)), 128, 128, kTileThreads) : 1e30;
    const double t256 = or_none(cost.large_tiles(rounds), 256, 256, kTileThreads);
    const double best = std::min({b16, b32, b64, t128, t256});
    return best == 1e30 ? -1
           : best == t256 ? (near ? MCHIP_I8_TILES_256 : MCHIP_I8_TILES_FAR)
           : best == t128 ? MCHIP_I8_TILES_128
           : best == b64  ? MCHIP_I8_BLOCKS_32X64
           : best == b32  ? MCHIP_I8_BLOCKS_32X32
                          : MCHIP_I8_BLOCKS_16X32;
}

template <int kMode, bool kGated>
int launch(const Product& p, hipStream_t stream, const char** why) {
    switch (choose<kMode, kGated>(p, device_cus())) {
        case MCHIP_I8_TILES_256: return launch_tiles<kMode, kGated, 256>(p, stream);
        case MCHIP_I8_TILES_128: return launch_tiles<kMode, kGated, 128>(p, stream);
        case MCHIP_I8_BLOCKS_32X64: return launch_direct<kMode, kGated, 2, 4>(p, stream);
        case MCHIP_I8_BLOCKS_32X32: return launch_direct<kMode, kGated, 2, 2>(p, stream);
        case MCHIP_I8_BLOCKS_16X32: return launch_direct<kMode, kGated, 1, 2>(p, stream);
        case MCHIP_I8_TILES_FAR:
            if constexpr (kMode == kUp) return launch_tiles<kMode, kGated, 256, true>(p, stream);
    }
    *why = "more tiles of C than one launch takes";
    return hipErrorInvalidValue;
}

const char* refusal(const void* a, const float* a_scales, const void* b, const float* b_scales, const float* bias,
                    int activation, int c_dtype, const void* c, int rows, int n, int k) {
    if (!is_float_type(c_dtype)) return "the result's type is none of fp32 (0), bf16 (1), fp16 (2)";
    if (activation < MCHIP_ACT_RELU || activation > MCHIP_ACT_NONE)
        return "the activation is none of ReLU (0), GELU (1), SwiGLU (2), none (3)";
    if (rows < 1 || n < 1 || k < 1) return "a size below 1";
    if (k > MCHIP_I8_MAX_K) return "k above 131071, whose sums may pass 32 bits";
    if (n > (1 << 30)) return "n above 2^30";
    if (a == nullptr || a_scales == nullptr || b == nullptr || b_scales == nullptr || c == nullptr)
        return "a null operand";
    if (!aligned(a, 16) || !aligned(b, 16)) return "codes not 16-byte aligned";
    if (!aligned(a_scales, 4) || !aligned(b_scales, 4) || !aligned(bias, 4)) return "scales or a bias not 4-byte aligned";
    if (!aligned(c, size_of(c_dtype))) return "a result that is not aligned to its elements";
    return nullptr;
}

const char* plan_refusal(const mchip_experts_args& x) {
    if (x.tokens < 1 || x.top_k < 1 || x.experts < 1) return "a size below 1";
    if (x.experts > MCHIP_ROUTE_MAX_EXPERTS) return "more than 512 experts";
    if (x.top_k > MCHIP_ROUTE_MAX_TOP_K) return "more than 16 experts for a token";
    if (static_cast<long long>(x.tokens) * x.top_k > (1 << 30)) return "more than 2^30 pairs of a token and an expert";
    if (x.order == nullptr || x.offsets == nullptr) return "a null plan";
    if (!aligned(x.order, 4) || !aligned(x.offsets, 4)) return "a plan that is not 4-byte aligned";
    return nullptr;
}

Product product_of(const mchip_experts_args& x) {
    return {static_cast<const unsigned char*>(x.a_codes), static_cast<const unsigned char*>(x.w_codes), x.a_scales,
            x.w_scales, x.bias, x.c, x.order, x.offsets, x.gates, x.tokens * x.top_k, x.n, padded_k(x.k), x.tokens,
            x.top_k, x.experts, x.activation, x.c_dtype, 0};
}

}  // namespace

extern "C" {

int mchip_launch_matmul_i8(const void* a_codes, const float* a_scales, const void* b_codes, const float* b_scales,
                           const float* bias, int activation, int c_dtype, void* c, int m, int n, int k, void* stream,
                           const char** why) {
    *why = refusal(a_codes, a_scales, b_codes, b_scales, bias, activation, c_dtype, c, m, n, k);
    if (*why != nullptr) return hipErrorInvalidValue;
    const Product p{static_cast<const unsigned char*>(a_codes), static_cast<const unsigned char*>(b_codes), a_scales,
                    b_scales, bias, c, nullptr, nullptr, nullptr, m, n, padded_k(k), m, 1, 1, activation, c_dtype, 0};
    hipStream_t s = static_cast<hipStream_t>(stream);
    return activation == MCHIP_ACT_SWIGLU ? launch<kDense, true>(p, s, why) : launch<kDense, false>(p, s, why);
}

int mchip_matmul_i8_plan(int activation, int m, int n, int k, int cu_count, int* halves) {
    Product p{};
    p.m = p.a_rows = m, p.n = n, p.row_bytes = padded_k(k), p.experts = 1;
    const bool gated = activation == MCHIP_ACT_SWIGLU;
    const int kernel = gated ? choose<kDense, true>(p, cu_count) : choose<kDense, false>(p, cu_count);
    *halves = kernel == MCHIP_I8_TILES_256 ? halves_of(tiles(m, 256) * tiles(n, gated ? 128 : 256), cu_count) : 0;
    return kernel;
}

int mchip_experts_i8_plan(int down, int activation, int tokens, int top_k, int experts, int n, int k, int cu_count) {
    Product p{};
    p.m = tokens * top_k, p.a_rows = tokens, p.n = n, p.row_bytes = padded_k(k), p.top_k = top_k, p.experts = experts;
    if (down != 0) return choose<kDown, false>(p, cu_count);
    return activation == MCHIP_ACT_SWIGLU ? choose<kUp, true>(p, cu_count) : choose<kUp, false>(p, cu_count);
}

int mchip_launch_experts_up_i8(const mchip_experts_args* args, void* stream, const char** why) {
    const mchip_experts_args& x = *args;
    *why = refusal(x.a_codes, x.a_scales, x.w_codes, x.w_scales, x.bias, x.activation, x.c_dtype, x.c, x.tokens, x.n, x.k);
    if (*why == nullptr) *why = plan_refusal(x);
    if (*why != nullptr) return hipErrorInvalidValue;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return x.activation == MCHIP_ACT_SWIGLU ? launch<kUp, true>(product_of(x), s, why)
                                            : launch<kUp, false>(product_of(x), s, why);
}

long long mchip_experts_down_i8_workspace_bytes(int c_dtype, int tokens, int top_k, int n, int k) {
    if (!is_float_type(c_dtype) || tokens < 1 || top_k < 1 || n < 1 || k < 1) return 0;
    return static_cast<long long>(tokens) * top_k * n * 4;
}

int mchip_launch_experts_down_i8(const mchip_experts_args* args, void* stream, const char** why) {
    const mchip_experts_args& x = *args;
    *why = refusal(x.a_codes, x.a_scales, x.w_codes, x.w_scales, x.bias, MCHIP_ACT_NONE, x.c_dtype, x.c, x.tokens, x.n, x.k);
    if (*why == nullptr) *why = plan_refusal(x);
    if (*why == nullptr && x.top_k > x.experts) *why = "more experts for a token than there are";
    if (*why == nullptr && (x.gates == nullptr || x.workspace == nullptr)) *why = "null gates, or a null workspace";
    if (*why == nullptr && (!aligned(x.gates, 4) || !aligned(x.workspace, 256)))
        *why = "gates not 4-byte, or a workspace not 256-byte aligned";
    if (*why != nullptr) return hipErrorInvalidValue;
    hipStream_t s = static_cast<hipStream_t>(stream);
    Product p = product_of(x);
    p.activation = MCHIP_ACT_NONE;
    p.c = x.workspace;
    const int rc = launch<kDown, false>(p, s, why);
    if (rc != hipSuccess) return rc;
    const auto sum = [&](auto kernel) {
        const long long blocks = tiles(static_cast<long long>(x.tokens) * ((x.n + 3) / 4), 256);
        return launch_kernel(kernel, static_cast<unsigned>(std::min<long long>(blocks, 1 << 20)), 256, 0, s,
                             static_cast<const float*>(x.workspace), x.c, x.tokens, x.top_k, x.n);
    };
    return x.c_dtype == kF32 ? sum(sum_pairs<kF32>) : x.c_dtype == kBf16 ? sum(sum_pairs<kBf16>) : sum(sum_pairs<kF16>);
}

}  // extern "C"

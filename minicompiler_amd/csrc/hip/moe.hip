// A mixture-of-experts MLP for the few tokens of a decoding step (mx4.h):
//   p = softmax(x R^T); the top_k largest experts e of each token, ties to the
//   lower index, with gates g_e = p_e, or p_e / sum of the chosen p;
//   y = sum over the chosen e of g_e (act(x W1_e^T + b1_e) W2_e^T + b2_e).
//
// Three launches, in stream order:
//   moe_router  x R^T on the FP32 matrix instruction, d shared out over blocks; x
//               cut into bf16 pieces; the last block to arrive adds the parts
//               of the logits in order, picks the experts and lists the jobs
//               (one per chosen expert and 16 of its tokens);
//   moe_up      per job and 32 (swiglu: 16) columns of h: act(x W1^T + b1), cut
//               into bf16 pieces;
//   moe_down    per 32 columns of y and share of the jobs' steps: h W2^T weighed
//               by the gates; the last block of a column tile adds the shares
//               in order.
// Bound by the chosen experts' weights, each read once per job. Weights are the
// matrix instruction's first operand, 16 rows of them, and a job's 16 tokens
// the second. Products are exact (bf16 pieces of x, h and the weights), sums fp32.

#include "mx4_device.h"

#include "gemm_split_arrival.h"

namespace {

using namespace mx4;

constexpr int kMaxTokens = MCHIP_MOE_MAX_TOKENS, kMaxExperts = MCHIP_MOE_MAX_EXPERTS, kMaxTopK = MCHIP_MOE_MAX_TOP_K;
constexpr int kMaxWidth = 1 << 20;  // of d and h
constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kNone = -1;  // the token of a job's empty place

// A job's tokens and what they weigh.
struct Job {
    int expert;
    int token[16];
    float gate[16];
};

// The workspace: counters (zero between calls), the jobs, then the arrays.
struct Workspace {
    unsigned* arrived;  // [1 + column tiles of y]
    int* jobs;          // how many
    Job* job;           // [max_jobs]
    float* logits;      // [parts][tokens, experts]
    unsigned short* x;  // [pieces][tokens][dp]
    unsigned short* h;  // [pieces][max_jobs * 16][hp]
    float* y;           // [shares][tokens][column tiles * 32]
};

struct Sizes {
    int tokens, d, h, experts, top_k;
    int dp, hp;  // padded to 128
    int max_jobs;
};

__host__ __device__ inline int padded(int k) { return (k + kStep - 1) / kStep * kStep; }

Sizes sizes_of(int tokens, int d, int h, int experts, int top_k) {
    // Every chosen pair a job of its own, or every expert's full tiles and one more.
    const int pairs = tokens * top_k, tiled = experts + pairs / 16;
    return {tokens, d, h, experts, top_k, padded(d), padded(h), pairs < tiled ? pairs : tiled};
}

constexpr int kCols = 32;  // of y per block

// The parts that d is cut into for the logits: 64 elements for each wave.
int router_parts(int d) { return std::min((d + 64 * kWaves - 1) / (64 * kWaves), 16); }

int column_tiles(int d) { return (d + kCols - 1) / kCols; }

// The shares that a column tile of y is cut into: two blocks per CU in all, as
// long as a wave has a step to do.
int down_shares(const Sizes& s) {
    const int want = 2 * device_cus() / column_tiles(s.d);
    const int most = (s.max_jobs * (s.hp / kStep) + kWaves - 1) / kWaves;
    return std::max(1, std::min({want, most, 64}));
}

int pieces_of(int dtype) { return dtype == kF32 ? 3 : dtype == kF16 ? 2 : 1; }
// h is an fp32 sum: 24 bits of it for an fp32 result, 16 otherwise.
int h_pieces_of(int dtype) { return dtype == kF32 ? 3 : 2; }

std::size_t round_up(std::size_t v) { return (v + 255) / 256 * 256; }

std::size_t lay_out(const Sizes& s, int dtype, unsigned char* base, Workspace* w) {
    std::size_t at = 0;
    const auto take = [&](std::size_t bytes) {
        unsigned char* p = base + at;
        at += round_up(bytes);
        return p;
    };
    w->arrived = reinterpret_cast<unsigned*>(take(sizeof(unsigned) * (1 + column_tiles(kMaxWidth))));
    w->jobs = reinterpret_cast<int*>(take(sizeof(int)));
    w->job = reinterpret_cast<Job*>(take(sizeof(Job) * static_cast<std::size_t>(s.max_jobs)));
    w->logits = reinterpret_cast<float*>(take(sizeof(float) * static_cast<std::size_t>(router_parts(s.d)) * s.tokens * s.experts));
    w->x = reinterpret_cast<unsigned short*>(
        take(2 * static_cast<std::size_t>(pieces_of(dtype)) * s.tokens * s.dp));
    w->h = reinterpret_cast<unsigned short*>(
        take(2 * static_cast<std::size_t>(h_pieces_of(dtype)) * s.max_jobs * 16 * s.hp));
    w->y = reinterpret_cast<float*>(
        take(sizeof(float) * static_cast<std::size_t>(down_shares(s)) * s.tokens * column_tiles(s.d) * kCols));
    return at;
}

// ---------------------------------------------------------------- router

// One token's experts and gates, by one wave, from its logits in LDS. Logits are
// compared as unsigned numbers in the order of the floats, from 2 up; a NaN
// counts as 1, smaller than all, and a chosen one as 0. A NaN makes every gate
// NaN, as softmax does.
__device__ void choose(const float* logits, int experts, int top_k, bool normalize, int lane, int* chosen, float* gate) {
    constexpr int kEach = kMaxExperts / 64;
    unsigned key[kEach];
    unsigned best = 0;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        key[j] = 0;
        if (64 * j >= experts) continue;
        const int e = lane + 64 * j;
        if (e < experts) {
            const float l = logits[e] + 0.0f;  // -0 to 0
            const unsigned u = __builtin_bit_cast(unsigned, l);
            key[j] = l != l ? 1u : u >> 31 ? ~u : u | 0x80000000u;
        }
        best = key[j] > best ? key[j] : best;
    }
    const unsigned first = wave_max(best);
    const float top = __builtin_bit_cast(float, first >> 31 ? first & 0x7fffffffu : ~first);
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kEach; ++j)
        if (64 * j < experts && lane + 64 * j < experts) sum += expf(logits[lane + 64 * j] - top);
    sum = wave_sum(sum);
    float kept = 0.0f, mine = 0.0f;
    for (int i = 0; i < top_k; ++i) {
        unsigned most = 0, at = 0xffffffffu;
#pragma unroll
        for (int j = 0; j < kEach; ++j)
            if (64 * j < experts && key[j] > most) {
                most = key[j];
                at = static_cast<unsigned>(lane + 64 * j);
            }
        const unsigned winner = wave_max(most);
        const unsigned e = wave_min(most == winner ? at : 0xffffffffu);
#pragma unroll
        for (int j = 0; j < kEach; ++j)
            if (e == static_cast<unsigned>(lane + 64 * j)) key[j] = 0;
        const float p = expf(logits[e] - top) / sum;
        kept += p;
        if (lane == i) {
            mine = p;
            chosen[i] = static_cast<int>(e);
        }
    }
    if (lane < top_k) gate[lane] = normalize ? mine / kept : mine;
}

// The jobs from the chosen experts in LDS, by the whole block: a thread per
// expert for their places, then one per chosen pair.
__device__ void list_jobs(const Workspace& w, const Sizes& s, const int (*chosen)[kMaxTopK],
                          const float (*gate)[kMaxTopK], unsigned long long* mask, int* place) {
    static_assert(kThreads == kMaxExperts);
    const int e = threadIdx.x, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    mask[e] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < s.tokens * s.top_k; i += kThreads)
        atomicOr(mask + chosen[i / s.top_k][i % s.top_k], 1ull << (i / s.top_k));
    __syncthreads();
    const int count = __builtin_popcountll(mask[e]), mine = (count + 15) / 16;
    int before = mine;
    for (int o = 1; o < 64; o *= 2) {
        const int add = __shfl_up(before, o);
        if (lane >= o) before += add;
    }
    if (lane == 63) place[kMaxExperts + wave] = before;
    __syncthreads();
    for (int v = 0; v < wave; ++v) before += place[kMaxExperts + v];
    if (e == kMaxExperts - 1) *w.jobs = before;
    place[e] = before - mine;
    for (int n = 0; n < mine; ++n) w.job[before - mine + n].expert = e;
    for (int i = count; i < 16 * mine; ++i) {
        Job& job = w.job[before - mine + i / 16];
        job.token[i % 16] = kNone;
        job.gate[i % 16] = 0.0f;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < s.tokens * s.top_k; i += kThreads) {
        const int t = i / s.top_k, j = i % s.top_k, to = chosen[t][j];
        const int rank = __builtin_popcountll(mask[to] & ((1ull << t) - 1));
        Job& job = w.job[place[to] + rank / 16];
        job.token[rank % 16] = t;
        job.gate[rank % 16] = gate[t][j];
    }
}

// 16 experts by 16 tokens of the logits over one part of d, 64 elements at a time
// for each wave. v_mfma_f32_16x16x4_f32: lane (r, q) supplies row or column r,
// element q; here a lane's four elements go to four instructions.
template <int kIn>
__global__ __launch_bounds__(kThreads) void moe_router(const void* __restrict__ x, long long ldx,
                                                       const float* __restrict__ router, Workspace w, Sizes s,
                                                       bool normalize, int* __restrict__ chosen_out,
                                                       float* __restrict__ gates_out) {
    constexpr int kP = kPieces<kIn>;
    extern __shared__ float logits[];  // [tokens, experts], in the last block
    __shared__ f32x4 space[kWaves / 2 * 64];
    __shared__ int chosen[kMaxTokens][kMaxTopK];
    __shared__ float gate[kMaxTokens][kMaxTopK];
    __shared__ unsigned long long mask[kMaxExperts];
    __shared__ int place[kMaxExperts + kWaves];
    __shared__ int flag;
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int r = lane % 16, q = lane / 16;
    const int e0 = blockIdx.x * 16, t0 = blockIdx.y * 16, parts = gridDim.z;
    const int blocks = gridDim.x * gridDim.y * parts;
    const int block = (blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
    const long long all_logits = static_cast<long long>(s.tokens) * s.experts;

    const long long expert = e0 + r < s.experts ? e0 + r : s.experts - 1;
    const long long token = t0 + r < s.tokens ? t0 + r : s.tokens - 1;
    f32x4 acc[1] = {{0.0f, 0.0f, 0.0f, 0.0f}};
    for (int k0 = (blockIdx.z * kWaves + wave) * 64; k0 < s.d; k0 += parts * kWaves * 64) {
        f32x4 a[4], b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = k0 + 16 * i + 4 * q;
            a[i] = load_four<kF32>(router, expert * s.d + k, s.d - k);
            b[i] = load_four<kIn>(x, token * ldx + k, s.d - k);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i][j], b[i][j], acc[0], 0, 0, 0);
    }
    add_waves<kWaves, 1>(acc, space, wave, lane);
    if (wave == 0 && t0 + r < s.tokens) {
        float* out = w.logits + blockIdx.z * all_logits + static_cast<long long>(t0 + r) * s.experts + e0 + 4 * q;
#pragma unroll
        for (int v = 0; v < 4; ++v)
            if (e0 + 4 * q + v < s.experts) mc_split_store(out + v, acc[0][v]);
    }

    // x in pieces, rows padded with zeros, shared out over the blocks.
    const long long all = static_cast<long long>(s.tokens) * s.dp;
    for (long long i = (static_cast<long long>(block) * kThreads + threadIdx.x) * 8; i < all;
         i += static_cast<long long>(blocks) * kThreads * 8) {
        const int t = static_cast<int>(i / s.dp), k = static_cast<int>(i % s.dp);
        float v[8];
        load_eight<kIn>(x, t * ldx + k, s.d - k, v);
        u32x4 out[kP];
        cut_eight<kP>(v, out);
#pragma unroll
        for (int p = 0; p < kP; ++p) *reinterpret_cast<u32x4*>(w.x + p * all + i) = out[p];
    }

    if (!mc_split_last_arrival(w.arrived, blocks, &flag)) return;
    for (int i = threadIdx.x; i < all_logits; i += kThreads) {
        float sum = mc_split_load(w.logits + i);
        for (int z = 1; z < parts; ++z) sum += mc_split_load(w.logits + z * all_logits + i);
        logits[i] = sum;
    }
    __syncthreads();
    for (int t = wave; t < s.tokens; t += kWaves)
        choose(logits + t * s.experts, s.experts, s.top_k, normalize, lane, chosen[t], gate[t]);
    __syncthreads();
    list_jobs(w, s, chosen, gate, mask, place);
    for (int i = threadIdx.x; i < s.tokens * s.top_k; i += kThreads) {
        const int t = i / s.top_k, j = i % s.top_k;
        if (chosen_out != nullptr) chosen_out[i] = chosen[t][j];
        if (gates_out != nullptr) gates_out[i] = gate[t][j];
    }
}

// ---------------------------------------------------------------- experts' products

// Rows of an expert's weights in steps of 128: lane (r, q) supplies row r in
// four instructions s. 16-bit rows: elements 32 s + 8 q .. + 7 of the step
// (whole 64-byte pieces per instruction); mx4: 32 q + 8 s .. + 7 (block q of
// the step is the lane's own 16 bytes).
template <int kType>
struct Weights {
    static constexpr int kPiecesW = kType == kF16 ? 2 : 1;
    const void* base;
    const unsigned char* scales;
    int k, kp;

    __device__ __forceinline__ static int offset(int q, int s) { return kType == kMx4 ? 32 * q + 8 * s : 32 * s + 8 * q; }

    struct Step {
        u32x4 raw[4];
        float scale;
    };

    __device__ __forceinline__ Step load(long long row, int t, int q) const {
        Step st;
        if constexpr (kType == kMx4) {
            st.raw[0] = *reinterpret_cast<const u32x4*>(static_cast<const unsigned char*>(base) + row * (kp / 2) +
                                                        t * 64 + q * 16);
            st.scale = scale_operand(scales[row * (kp / 32) + t * 4 + q]);
        } else {
            const unsigned short* p = static_cast<const unsigned short*>(base) + row * k;
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int k0 = t * kStep + offset(q, s);
                if (k0 + 8 <= k) {
                    st.raw[s] = *reinterpret_cast<const u32x4_loose*>(p + k0);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const unsigned lo = k0 + 2 * j < k ? p[k0 + 2 * j] : 0u;
                        const unsigned hi = k0 + 2 * j + 1 < k ? p[k0 + 2 * j + 1] : 0u;
                        st.raw[s][j] = lo | hi << 16;
                    }
                }
            }
        }
        return st;
    }

    __device__ __forceinline__ static void operand(const Step& st, int s, u32x4 (&out)[kPiecesW]) {
        if constexpr (kType == kMx4) {
            out[0] = decode_eight(st.raw[0][s], st.scale);
        } else if constexpr (kType == kBf16) {
            out[0] = st.raw[s];
        } else {
            float v[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[2 * j] = to_f32<kF16>(st.raw[s][j] & 0xffffu);
                v[2 * j + 1] = to_f32<kF16>(st.raw[s][j] >> 16);
            }
            cut_eight<2>(v, out);
        }
    }
};

template <int kType, int kTiles>
__device__ __forceinline__ void load_step(const Weights<kType>& w, const long long (&rows)[kTiles], int t, int q,
                                          typename Weights<kType>::Step (&st)[kTiles]) {
#pragma unroll
    for (int i = 0; i < kTiles; ++i) st[i] = w.load(rows[i], t, q);
}

// acc[i] += step t of 16 weight rows, loaded, times the columns `col` (a lane's
// own row of the pieces, `plane` elements apart; has: there is one).
template <int kType, int kP, int kTiles>
__device__ __forceinline__ void multiply_step(const typename Weights<kType>::Step (&st)[kTiles],
                                              const unsigned short* col, long long plane, bool has, int t, int q,
                                              f32x4 (&acc)[kTiles]) {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        u32x4 x[kP];
        const int k0 = t * kStep + Weights<kType>::offset(q, s);
#pragma unroll
        for (int p = 0; p < kP; ++p)
            x[p] = has ? *reinterpret_cast<const u32x4*>(col + p * plane + k0) : u32x4{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
            u32x4 a[Weights<kType>::kPiecesW];
            Weights<kType>::operand(st[i], s, a);
#pragma unroll
            for (int wp = 0; wp < Weights<kType>::kPiecesW; ++wp)
#pragma unroll
                for (int p = 0; p < kP; ++p) acc[i] = mfma_bf16(a[wp], x[p], acc[i]);
        }
    }
}

template <int kAct>
__device__ __forceinline__ float activate(float u, float up) {
    if constexpr (kAct == MCHIP_MOE_RELU) return u > 0.0f ? u : (u == u ? 0.0f : u);
    if constexpr (kAct == MCHIP_MOE_SWIGLU) return u / (1.0f + expf(-u)) * up;
    return 0.5f * u * (1.0f + tanhf(0.79788456080286536f * (u + 0.044715f * u * u * u)));
}

// A job's h for 16 kTiles (swiglu: 16) columns from blockIdx.x on. Columns from
// h to hp are written as zeros.
template <int kType, int kP, int kHP, int kAct>
__global__ __launch_bounds__(kThreads) void moe_up(Weights<kType> w1, const float* __restrict__ b1, Workspace w,
                                                   Sizes s) {
    constexpr bool kGated = kAct == MCHIP_MOE_SWIGLU;
    constexpr int kTiles = 2, kUpCols = kGated ? 16 : 32;
    __shared__ f32x4 space[kWaves / 2 * kTiles * 64];
    const Job& job = w.job[blockIdx.y];
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int r = lane % 16, q = lane / 16;
    const int h0 = blockIdx.x * kUpCols;
    // The job is read beside the number of jobs, not after it; past the last, it is not used.
    const int jobs = *w.jobs, expert = job.expert, token = job.token[r];
    if (static_cast<int>(blockIdx.y) >= jobs) return;
    const long long all_rows = kGated ? 2LL * s.h : s.h;
    const long long first = expert * all_rows;
    long long rows[kTiles];
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
        const int col = h0 + (kGated ? 0 : 16 * i) + r;
        rows[i] = first + (col < s.h ? col : s.h - 1) + (kGated && i == 1 ? s.h : 0);
    }
    f32x4 acc[kTiles];
#pragma unroll
    for (int i = 0; i < kTiles; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const long long plane = static_cast<long long>(s.tokens) * s.dp;
    const unsigned short* col = w.x + static_cast<long long>(token == kNone ? 0 : token) * s.dp;
    if (h0 < s.h) {
        const int steps = s.dp / kStep;
        typename Weights<kType>::Step now[kTiles], next[kTiles];
        if (wave < steps) load_step<kType, kTiles>(w1, rows, wave, q, now);
        for (int t = wave; t < steps; t += kWaves) {
            if (t + kWaves < steps) load_step<kType, kTiles>(w1, rows, t + kWaves, q, next);
            multiply_step<kType, kP, kTiles>(now, col, plane, token != kNone, t, q, acc);
#pragma unroll
            for (int i = 0; i < kTiles; ++i) now[i] = next[i];
        }
    }
    add_waves<kWaves, kTiles>(acc, space, wave, lane);
    if (wave != 0) return;
    const long long h_plane = static_cast<long long>(s.max_jobs) * 16 * s.hp;
#pragma unroll
    for (int i = 0; i < (kGated ? 1 : kTiles); ++i) {
        const int c0 = h0 + 16 * i + 4 * q;
        u16x4 out[kHP];
#pragma unroll
        for (int v = 0; v < 4; ++v) {
            float u = acc[i][v], up = kGated ? acc[1][v] : 0.0f;
            const bool in = c0 + v < s.h;
            if (b1 != nullptr && in) {
                u += b1[first + c0 + v];
                if (kGated) up += b1[first + s.h + c0 + v];
            }
            float piece[kHP];
            cut<kHP>(in ? activate<kAct>(u, up) : 0.0f, piece);
#pragma unroll
            for (int p = 0; p < kHP; ++p)
                out[p][v] = static_cast<unsigned short>(__builtin_bit_cast(unsigned, piece[p]) >> 16);
        }
#pragma unroll
        for (int p = 0; p < kHP; ++p)
            *reinterpret_cast<u16x4*>(w.h + p * h_plane + (static_cast<long long>(blockIdx.y) * 16 + r) * s.hp + c0) =
                out[p];
    }
}

// 32 columns of y for all tokens and one share of the jobs' steps (all jobs' steps
// in a row, cut evenly over the shares' waves). A wave adds each of its jobs'
// parts, weighed, to its own LDS tile (no two lanes the same element); the tiles
// are added in wave order, the shares in their order by the last block to arrive.
template <int kType, int kP, int kOut>
__global__ __launch_bounds__(kThreads) void moe_down(Weights<kType> w2, const float* __restrict__ b2, Workspace w,
                                                     Sizes s, void* __restrict__ y) {
    constexpr int kTiles = kCols / 16;
    extern __shared__ float tile[];  // [kWaves][tokens][kCols]
    __shared__ int flag;
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int r = lane % 16, q = lane / 16;
    const int d0 = blockIdx.x * kCols, shares = gridDim.y;
    const int cells = s.tokens * kCols;
    float* mine = tile + wave * cells;
    for (int i = lane; i < cells; i += 64) mine[i] = 0.0f;
    const int steps = s.hp / kStep, units = *w.jobs * steps;
    const int waves = shares * kWaves, each = units / waves, more = units % waves;
    const int index = blockIdx.y * kWaves + wave;
    const int from = index * each + (index < more ? index : more), to = from + each + (index < more ? 1 : 0);
    const long long h_plane = static_cast<long long>(s.max_jobs) * 16 * s.hp;

    const auto rows_of = [&](int expert, long long (&rows)[kTiles]) {
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
            const int col = d0 + 16 * i + r;
            rows[i] = static_cast<long long>(expert) * s.d + (col < s.d ? col : s.d - 1);
        }
    };
    int u = from;
    while (u < to) {
        const int n = u / steps, last = (n + 1) * steps < to ? (n + 1) * steps : to;
        const Job& job = w.job[n];
        const int expert = job.expert, token = job.token[r];
        const float gate = job.gate[r];
        long long rows[kTiles];
        rows_of(expert, rows);
        f32x4 acc[kTiles];
#pragma unroll
        for (int i = 0; i < kTiles; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (b2 != nullptr && u == n * steps) {  // the job's first step brings the bias
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const int c = d0 + 16 * i + 4 * q + v;
                    if (c < s.d) acc[i][v] = b2[static_cast<long long>(expert) * s.d + c];
                }
        }
        const unsigned short* col = w.h + (static_cast<long long>(n) * 16 + r) * s.hp;
        typename Weights<kType>::Step now[kTiles], next[kTiles];
        load_step<kType, kTiles>(w2, rows, u - n * steps, q, now);
        for (; u < last; ++u) {
            if (u + 1 < last) load_step<kType, kTiles>(w2, rows, u + 1 - n * steps, q, next);
            multiply_step<kType, kP, kTiles>(now, col, h_plane, token != kNone, u - n * steps, q, acc);
#pragma unroll
            for (int i = 0; i < kTiles; ++i) now[i] = next[i];
        }
        if (token != kNone) {
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
#pragma unroll
                for (int v = 0; v < 4; ++v) mine[token * kCols + 16 * i + 4 * q + v] += gate * acc[i][v];
        }
    }
    __syncthreads();
    const long long row = static_cast<long long>(gridDim.x) * kCols, plane = s.tokens * row;
    for (int i = threadIdx.x; i < cells; i += kThreads) {
        const int t = i / kCols, c = i % kCols;
        float sum = 0.0f;
#pragma unroll
        for (int v = 0; v < kWaves; ++v) sum += tile[v * cells + i];
        if (shares > 1)
            mc_split_store(w.y + blockIdx.y * plane + t * row + d0 + c, sum);
        else if (d0 + c < s.d)
            store_one<kOut>(y, static_cast<long long>(t) * s.d + d0 + c, sum);
    }
    if (shares == 1 || !mc_split_last_arrival(w.arrived + 1 + blockIdx.x, shares, &flag)) return;
    for (int i = threadIdx.x; i < cells; i += kThreads) {
        const int t = i / kCols, c = i % kCols;
        if (d0 + c >= s.d) continue;
        const float* at = w.y + t * row + d0 + c;
        float sum = mc_split_load(at);
        for (int v = 1; v < shares; ++v) sum += mc_split_load(at + v * plane);
        store_one<kOut>(y, static_cast<long long>(t) * s.d + d0 + c, sum);
    }
}

// ---------------------------------------------------------------- launches

template <int kType>
Weights<kType> weights(const void* base, const void* scales, int k) {
    return {base, static_cast<const unsigned char*>(scales), k, padded(k)};
}

template <int kIn, int kType, int kAct>
int launch_experts(const mchip_moe_args& a, const Workspace& w, const Sizes& s, hipStream_t stream) {
    constexpr int kHP = kIn == kF32 ? 3 : 2;
    constexpr int kUpCols = kAct == MCHIP_MOE_SWIGLU ? 16 : 32;
    hipLaunchKernelGGL((moe_up<kType, kPieces<kIn>, kHP, kAct>),
                       dim3(static_cast<unsigned>(s.hp / kUpCols), static_cast<unsigned>(s.max_jobs)), dim3(kThreads), 0,
                       stream, weights<kType>(a.w1, a.w1_scales, s.d), a.b1, w, s);
    hipLaunchKernelGGL((moe_down<kType, kHP, kIn>), 
                       dim3(static_cast<unsigned>(column_tiles(s.d)), static_cast<unsigned>(down_shares(s))),
                       dim3(kThreads), sizeof(float) * kWaves * s.tokens * kCols, stream, weights<kType>(a.w2, a.w2_scales, s.h), a.b2, w, s, a.y);
    return hipGetLastError();
}

template <int kIn, int kType>
int launch_act(const mchip_moe_args& a, const Workspace& w, const Sizes& s, hipStream_t stream) {
    if (a.activation == MCHIP_MOE_RELU) return launch_experts<kIn, kType, MCHIP_MOE_RELU>(a, w, s, stream);
    if (a.activation == MCHIP_MOE_GELU) return launch_experts<kIn, kType, MCHIP_MOE_GELU>(a, w, s, stream);
    return launch_experts<kIn, kType, MCHIP_MOE_SWIGLU>(a, w, s, stream);
}

template <int kIn>
int launch(const mchip_moe_args& a, hipStream_t stream) {
    const Sizes s = sizes_of(a.tokens, a.d, a.h, a.experts, a.top_k);
    Workspace w;
    lay_out(s, a.dtype, static_cast<unsigned char*>(a.workspace), &w);
    hipLaunchKernelGGL(moe_router<kIn>,
                       dim3(static_cast<unsigned>((s.experts + 15) / 16), static_cast<unsigned>((s.tokens + 15) / 16),
                            static_cast<unsigned>(router_parts(s.d))),
                       dim3(kThreads), sizeof(float) * s.tokens * s.experts, stream, a.x, a.ldx, a.router, w, s, a.normalize != 0, a.chosen, a.gates);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (a.weights == kBf16) return launch_act<kIn, kBf16>(a, w, s, stream);
    if (a.weights == kF16) return launch_act<kIn, kF16>(a, w, s, stream);
    return launch_act<kIn, kMx4>(a, w, s, stream);
}

const char* refusal(const mchip_moe_args& a) {
    if (!is_float_type(a.dtype)) return "x's type is none of fp32 (0), bf16 (1), fp16 (2)";
    if (a.weights != kBf16 && a.weights != kF16 && a.weights != kMx4)
        return "the weights' type is none of bf16 (1), fp16 (2), mx4 (4)";
    if (a.activation < MCHIP_MOE_RELU || a.activation > MCHIP_MOE_SWIGLU) return "an unknown activation";
    if (a.tokens < 1 || a.d < 1 || a.h < 1 || a.experts < 1 || a.top_k < 1) return "a size below 1";
    if (a.tokens > kMaxTokens) return "more than 64 tokens";
    if (a.experts > kMaxExperts) return "more than 512 experts";
    if (a.top_k > kMaxTopK) return "more than 16 experts for a token";
    if (a.top_k > a.experts) return "more experts for a token than there are";
    if (a.d > kMaxWidth || a.h > kMaxWidth) return "rows longer than 2^20";
    if (a.ldx < a.d) return "rows of x closer together than they are long";
    if (!a.x || !a.router || !a.w1 || !a.w2 || !a.y || !a.workspace) return "a null operand";
    if (a.weights == kMx4 && (!a.w1_scales || !a.w2_scales)) return "mx4 weights without scales";
    if (!aligned(a.x, size_of(a.dtype)) || !aligned(a.y, size_of(a.dtype)) || !aligned(a.router, 4) ||
        !aligned(a.b1, 4) || !aligned(a.b2, 4) || !aligned(a.chosen, 4) || !aligned(a.gates, 4) ||
        !aligned(a.w1, a.weights == kMx4 ? 16 : 2) || !aligned(a.w2, a.weights == kMx4 ? 16 : 2))
        return "an address that is no multiple of its element's size (mx4 codes: of 16)";
    if (!aligned(a.workspace, 256)) return "a workspace that is not 256-byte aligned";
    return nullptr;
}

}  // namespace

extern "C" {

long long mchip_moe_workspace_bytes(int dtype, int tokens, int d, int h, int experts, int top_k) {
    if (!is_float_type(dtype) || tokens < 1 || tokens > kMaxTokens || d < 1 || h < 1 || d > kMaxWidth ||
        h > kMaxWidth || experts < 1 || experts > kMaxExperts || top_k < 1 || top_k > kMaxTopK)
        return 0;
    Workspace w;
    return static_cast<long long>(lay_out(sizes_of(tokens, d, h, experts, top_k), dtype, nullptr, &w));
}

int mchip_launch_moe(const mchip_moe_args* args, void* stream, const char** why) {
    *why = refusal(*args);
    if (*why != nullptr) return hipErrorInvalidValue;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (args->dtype == kF32) return launch<kF32>(*args, s);
    if (args->dtype == kBf16) return launch<kBf16>(*args, s);
    return launch<kF16>(*args, s);
}

}  // extern "C"

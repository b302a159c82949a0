// A mixture-of-experts MLP for the few tokens of a decoding step (mx4.h):
//   p = softmax(x R^T); the top_k largest experts e of each token, ties to the
//   lower index, with gates g_e = p_e, or p_e / sum of the chosen p;
//   y = sum over the chosen e of g_e (act(x W1_e^T + b1_e) W2_e^T + b2_e).
//
// Three launches, in stream order:
//   moe_router  x R^T on the FP32 matrix instruction, d shared out over blocks; x
//               cut into bf16 pieces by blocks of their own; for more than 8
//               tokens the last block of 16 tokens adds the parts of their logits
//               in order and picks their experts, and the last of all lists the
//               jobs (one per chosen expert and 16 of its tokens);
//   moe_up      per job and 32 (swiglu: 16) columns of h: act(x W1^T + b1), cut
//               into bf16 pieces. Up to 8 tokens every block picks the experts for
//               itself, which is less than waiting for one that does;
//   moe_down    per 32 columns of y and share of the jobs' steps: h W2^T weighed
//               by the gates; the last block of a column tile adds the shares
//               in order.
// Bound by the chosen experts' weights, each read once per job, and for few
// tokens by the chain of launches, routing and trips to memory. Weights are the
// matrix instruction's first operand, 16 rows of them, and a job's 16 tokens
// the second. Products are exact (bf16 pieces of x, h and the weights; what of
// fp32 numbers lies below 2^-133 is left out), sums fp32.
//
// Measured (router, up, down, medians of a kernel trace, and all of it in steady
// repetition): one token, 8 of 64 mx4 experts of 2048x1024: 4.0, 10.6, 8.7, 22.3
// us (27 MB); 16 tokens, 8 bf16 experts of 512x2048, fp32: 8.0, 10.5, 10.3, 28.8 us
// (34 MB); 64 tokens, 32 fp16 experts of 1023x777: 13.0, 31.3, 25.4, 70.7 us (153
// MB); with rows of 1024 and 768 elements 12.3, 25.2, 21.0, 58.7: rows at odd places
// cost a fifth of the time.

#include "mx4_rows.h"

#include "gemm_split_arrival.h"

namespace {

using namespace mx4;

constexpr int kMaxTokens = MCHIP_MOE_MAX_TOKENS, kMaxExperts = MCHIP_MOE_MAX_EXPERTS, kMaxTopK = MCHIP_MOE_MAX_TOP_K;
constexpr int kMaxWidth = 1 << 20;  // of d and h
constexpr int kThreads = 512, kWaves = kThreads / 64;
constexpr int kFirstColumn = 1 + kMaxTokens / 16;  // counter of the first column tile of y
constexpr int kFew = 8;    // tokens for which every block of moe_up picks the experts
constexpr int kNone = -1;  // the token of a job's empty place

// A job's tokens and what they weigh.
struct Job {
    int expert;
    int token[16];
    float gate[16];
};

// The workspace: counters (zero between calls), the jobs, then the arrays.
struct Workspace {
    unsigned* arrived;  // [1 + token tiles + column tiles of y]
    int* jobs;          // how many
    int* chosen;        // [tokens][kMaxTopK]
    float* gate;
    Job* job;           // [max_jobs]
    float* logits;      // [parts][tokens, experts]
    unsigned short* x;  // [pieces][dp / 8][tokens][8]: a token's eight elements beside its neighbours'
    unsigned short* h;  // [pieces][max_jobs][hp / 8][16][8]
    float* y;           // [shares][tokens][column tiles * 32]
};

struct Sizes {
    int tokens, d, h, experts, top_k;
    int dp, hp;  // padded to 128
    int max_jobs;
};

Sizes sizes_of(int tokens, int d, int h, int experts, int top_k) {
    // Every chosen pair a job of its own, or every expert's full tiles and one more.
    const int pairs = tokens * top_k, tiled = experts + pairs / 16;
    return {tokens, d, h, experts, top_k, padded(d), padded(h), pairs < tiled ? pairs : tiled};
}

constexpr int kCols = 32;  // of y per block

// The parts that d is cut into for the logits: 64 elements for each wave.
int router_parts(int d) { return std::min((d + 64 * kWaves - 1) / (64 * kWaves), 16); }

int column_tiles(int d) { return (d + kCols - 1) / kCols; }

// The shares that a column tile of y is cut into: a block for each CU, as long as a
// wave has a step to do. (A block is two waves to a SIMD; the kernel's registers,
// 158 of 512 with mx4 weights and 209 to 224 with 16-bit ones, leave room for three
// and for two.)
int down_shares(const Sizes& s) {
    const int want = device_cus() / column_tiles(s.d);
    const int most = (s.max_jobs * (s.hp / kStep) + kWaves - 1) / kWaves;
    return std::max(1, std::min({want, most, 64}));
}

int pieces_of(int dtype) { return dtype == kF32 ? 3 : dtype == kF16 ? 2 : 1; }  // at most
// h is an fp32 number, kept whole whatever the result's type: cut to 16 bits for 16-bit results it was up to 2^-15 too
// small, which turned last bits of y (2e-4 of a bf16 y, 4e-6 so), and moe_down took 8.2 us instead of 8.7 for one
// token, 24.2 instead of 25.4 for 64.
constexpr int kPiecesH = 3;

std::size_t round_up(std::size_t v) { return (v + 255) / 256 * 256; }

std::size_t lay_out(const Sizes& s, int dtype, unsigned char* base, Workspace* w) {
    std::size_t at = 0;
    const auto take = [&](std::size_t bytes) {
        unsigned char* p = base + at;
        at += round_up(bytes);
        return p;
    };
    w->arrived = reinterpret_cast<unsigned*>(take(sizeof(unsigned) * (kFirstColumn + column_tiles(kMaxWidth))));
    w->jobs = reinterpret_cast<int*>(take(sizeof(int)));
    w->chosen = reinterpret_cast<int*>(take(sizeof(int) * kMaxTokens * kMaxTopK));
    w->gate = reinterpret_cast<float*>(take(sizeof(float) * kMaxTokens * kMaxTopK));
    w->job = reinterpret_cast<Job*>(take(sizeof(Job) * static_cast<std::size_t>(s.max_jobs)));
    w->logits = reinterpret_cast<float*>(take(sizeof(float) * static_cast<std::size_t>(router_parts(s.d)) * s.tokens * s.experts));
    w->x = reinterpret_cast<unsigned short*>(
        take(2 * static_cast<std::size_t>(pieces_of(dtype)) * s.tokens * s.dp));
    w->h = reinterpret_cast<unsigned short*>(
        take(2 * static_cast<std::size_t>(kPiecesH) * s.max_jobs * 16 * s.hp));
    w->y = reinterpret_cast<float*>(
        take(sizeof(float) * static_cast<std::size_t>(down_shares(s)) * s.tokens * column_tiles(s.d) * kCols));
    return at;
}

// ---------------------------------------------------------------- router

// sum[n] = parts[n][0] + parts[n][plane] + ... (`count` of them, in order),
// written by other blocks. Eight loads of each are under way: one after the
// other, 16 of them took 16 us.
template <int kEach>
__device__ __forceinline__ void add_parts(const float* const (&parts)[kEach], long long plane, int count,
                                          float (&sum)[kEach]) {
#pragma unroll
    for (int n = 0; n < kEach; ++n) sum[n] = 0.0f;
    for (int v = 0; v < count; v += 8) {
        float part[kEach][8];
#pragma unroll
        for (int n = 0; n < kEach; ++n)
#pragma unroll
            for (int j = 0; j < 8; ++j) part[n][j] = v + j < count ? mc_split_load(parts[n] + (v + j) * plane) : 0.0f;
#pragma unroll
        for (int n = 0; n < kEach; ++n)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (v + j < count) sum[n] += part[n][j];
    }
}

// The experts and gates of kTokens tokens from `first` on, by one wave, from
// their logits in LDS; kEach: experts per lane. Logits are compared as unsigned
// numbers in the order of the floats, from 2 up; a NaN counts as 1, smaller than
// all, and a chosen one as 0. A NaN makes every gate NaN, as softmax does. A
// reduction over the wave is a chain of dependent instructions: several tokens'
// chains go side by side.
template <int kEach, int kTokens>
__device__ void choose(const float* logits, int from, int first, int to, const Sizes& s, bool normalize, int lane,
                       int (*chosen)[kMaxTopK], float (*gate)[kMaxTopK]) {
    unsigned key[kTokens][kEach];
    float top[kTokens], sum[kTokens];
    int mine[kTokens];  // lane i: the i-th expert
#pragma unroll
    for (int n = 0; n < kTokens; ++n) {
        const int t = (first + n < to ? first + n : to - 1) - from;
        float l[kEach];
        unsigned best = 0;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int e = lane + 64 * j;
            l[j] = e < s.experts ? logits[t * s.experts + e] + 0.0f : 0.0f;  // -0 to 0
            const unsigned u = __builtin_bit_cast(unsigned, l[j]);
            key[n][j] = e >= s.experts ? 0u : l[j] != l[j] ? 1u : u >> 31 ? ~u : u | 0x80000000u;
            best = key[n][j] > best ? key[n][j] : best;
        }
        const unsigned most = wave_max(best);
        top[n] = __builtin_bit_cast(float, most >> 31 ? most & 0x7fffffffu : ~most);
        float part = 0.0f;
#pragma unroll
        for (int j = 0; j < kEach; ++j)
            if (lane + 64 * j < s.experts) part += expf(l[j] - top[n]);
        sum[n] = wave_sum(part);
        mine[n] = 0;
    }
    for (int i = 0; i < s.top_k; ++i) {
#pragma unroll
        for (int n = 0; n < kTokens; ++n) {
            unsigned most = 0, at = 0xffffffffu;
#pragma unroll
            for (int j = 0; j < kEach; ++j)
                if (key[n][j] > most) {
                    most = key[n][j];
                    at = static_cast<unsigned>(lane + 64 * j);
                }
            const unsigned winner = wave_max(most);
            const unsigned e = wave_min(most == winner ? at : 0xffffffffu);
#pragma unroll
            for (int j = 0; j < kEach; ++j)
                if (e == static_cast<unsigned>(lane + 64 * j)) key[n][j] = 0;
            if (lane == i) mine[n] = static_cast<int>(e);
        }
    }
#pragma unroll
    for (int n = 0; n < kTokens; ++n) {
        const int t = first + n;
        if (t >= to) break;
        const float p = lane < s.top_k ? expf(logits[(t - from) * s.experts + mine[n]] - top[n]) / sum[n] : 0.0f;
        const float kept = wave_sum(p);
        if (lane < s.top_k) {
            chosen[t][lane] = mine[n];
            gate[t][lane] = normalize ? p / kept : p;
        }
    }
}

// Tokens `from` to `to` of the logits (from `logits` on, in LDS), a few for each of the block's waves.
template <int kEach, int kTokens>
__device__ __forceinline__ void choose_all(const float* logits, int from, int to, const Sizes& s, bool normalize,
                                           int wave, int waves, int lane, int (*chosen)[kMaxTopK],
                                           float (*gate)[kMaxTopK]) {
    for (int t = from + wave * kTokens; t < to; t += waves * kTokens)
        choose<kEach, kTokens>(logits, from, t, to, s, normalize, lane, chosen, gate);
}

// The logits of tokens `from` to `to` added up into LDS, and their experts and gates.
__device__ __forceinline__ void route(const Workspace& w, const Sizes& s, int parts, int from, int to, bool normalize,
                                      float* logits, int (*chosen)[kMaxTopK], float (*gate)[kMaxTopK]) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), waves = blockDim.x / 64, lane = threadIdx.x % 64;
    const long long plane = static_cast<long long>(s.tokens) * s.experts;
    const int all = (to - from) * s.experts;
    for (int i = threadIdx.x; i < all; i += 2 * blockDim.x) {
        const int second = i + static_cast<int>(blockDim.x);
        const float* at[2] = {w.logits + from * s.experts + i, w.logits + from * s.experts + (second < all ? second : i)};
        float sum[2];
        add_parts<2>(at, plane, parts, sum);
        logits[i] = sum[0];
        if (second < all) logits[second] = sum[1];
    }
    __syncthreads();
    if (s.experts > 128)
        choose_all<kMaxExperts / 64, 1>(logits, from, to, s, normalize, wave, waves, lane, chosen, gate);
    else if (to - from <= waves)
        choose_all<2, 1>(logits, from, to, s, normalize, wave, waves, lane, chosen, gate);
    else
        choose_all<2, 2>(logits, from, to, s, normalize, wave, waves, lane, chosen, gate);
    __syncthreads();
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

// The same for up to 8 tokens (a job per chosen expert) into `jobs`, by blocks
// of at least 128 threads, a thread per chosen pair; returns how many. The jobs'
// places and the masks of the experts have been cleared (clear_few_jobs).
__device__ int list_few_jobs(const Sizes& s, const int (*chosen)[kMaxTopK], const float (*gate)[kMaxTopK],
                             unsigned* mask, int* place, int* counts, Job* jobs) {
    const int i = threadIdx.x, t = i / s.top_k, j = i % s.top_k;
    const bool pair = i < s.tokens * s.top_k;
    const int e = pair ? chosen[t][j] : 0;
    const float g = pair ? gate[t][j] : 0.0f;
    if (s.tokens == 1) {  // every pair a job
        if (pair) {
            jobs[i].expert = e;
            jobs[i].token[0] = 0;
            jobs[i].gate[0] = g;
        }
        __syncthreads();
        return s.top_k;
    }
    if (pair) atomicOr(mask + e, 1u << t);
    __syncthreads();
    const unsigned before = pair ? mask[e] & ((1u << t) - 1) : 1u;
    const unsigned long long firsts = __ballot(before == 0);
    if (i % 64 == 0 && i < 128) counts[i / 64] = __builtin_popcountll(firsts);
    __syncthreads();
    if (before == 0) {
        const int n = (i >= 64 ? counts[0] : 0) + __builtin_popcountll(firsts & ((1ull << i % 64) - 1));
        place[e] = n;
        jobs[n].expert = e;
    }
    __syncthreads();
    if (pair) {
        Job& job = jobs[place[e]];
        job.token[__builtin_popcount(before)] = t;
        job.gate[__builtin_popcount(before)] = g;
    }
    __syncthreads();
    return counts[0] + counts[1];
}

__device__ __forceinline__ void clear_few_jobs(const Sizes& s, unsigned* mask, Job* jobs) {
    for (int i = threadIdx.x; i < s.experts; i += blockDim.x) mask[i] = 0;
    for (int i = threadIdx.x; i < 16 * s.max_jobs; i += blockDim.x) {
        jobs[i / 16].token[i % 16] = kNone;
        jobs[i / 16].gate[i % 16] = 0.0f;
    }
}

// x in pieces, padded with zeros, and zeros for the end of h, by `blocks` blocks
// of moe_router of their own (by those with the logits it took 1.2 of 13 us).
template <int kIn, bool kHalf>
__device__ __forceinline__ void cut_tokens(const void* __restrict__ x, long long ldx, const Workspace& w, const Sizes& s,
                                           int block, int blocks) {
    constexpr int kP = kPieces<kIn>;
    const int chunks = s.tokens * (s.dp / 8);
    for (int i = block * kThreads + threadIdx.x; i < chunks; i += blocks * kThreads) {
        const int t = i % s.tokens, k = i / s.tokens * 8;
        float v[8];
        load_eight<kIn>(x, t * ldx + k, s.d - k, v);
        if constexpr (kHalf) {
            u16x8 same;
#pragma unroll
            for (int e = 0; e < 8; ++e) same[e] = to_16<kF16>(v[e]);
            *reinterpret_cast<u16x8*>(w.x + static_cast<long long>(i) * 8) = same;
            continue;
        }
        u32x4 out[kP];
        cut_eight<kP>(v, out);
#pragma unroll
        for (int p = 0; p < kP; ++p)
            *reinterpret_cast<u32x4*>(w.x + (static_cast<long long>(p) * chunks + i) * 8) = out[p];
    }

    // h's columns past its last tile of 16, in all jobs, to zeros.
    const int pad = s.hp / 8 - (s.h + 15) / 16 * 2, pads = kPiecesH * s.max_jobs * pad * 16;
    for (int i = block * kThreads + threadIdx.x; i < pads; i += blocks * kThreads) {
        const long long row = i / (pad * 16) + 1LL;  // ends of jobs, of all pieces
        *reinterpret_cast<u32x4*>(w.h + row * 16 * s.hp - (i % (pad * 16) + 1) * 8) = u32x4{0, 0, 0, 0};
    }
}

// 16 experts by 16 tokens of the logits over one part of d, 64 elements at a time
// for each wave. v_mfma_f32_16x16x4_f32: lane (r, q) supplies row or column r,
// element q; here a lane's four elements go to four instructions.
template <int kIn, bool kHalf>
__global__ __launch_bounds__(kThreads) void moe_router(const void* __restrict__ x, long long ldx,
                                                       const float* __restrict__ router, Workspace w, Sizes s,
                                                       bool normalize, int* __restrict__ chosen_out,
                                                       float* __restrict__ gates_out) {
    extern __shared__ __attribute__((aligned(16))) float logits[];  // [16, experts], in the last block of 16 tokens
    __shared__ f32x4 space[kWaves * 64];
    __shared__ int chosen[kMaxTokens][kMaxTopK];
    __shared__ float gate[kMaxTokens][kMaxTopK];
    __shared__ unsigned long long mask[kMaxExperts];
    __shared__ int place[kMaxExperts + kWaves];
    __shared__ int flag;
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int r = lane % 16, q = lane / 16;
    const int e0 = blockIdx.x * 16, t0 = blockIdx.y * 16, parts = gridDim.z / 2;
    if (static_cast<int>(blockIdx.z) >= parts) {
        const int block = ((blockIdx.z - parts) * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x;
        cut_tokens<kIn, kHalf>(x, ldx, w, s, block, gridDim.x * gridDim.y * parts);
        return;
    }
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
    sum_waves<kWaves>(acc, space, wave, lane, [&](int, f32x4 sum) {
        float* out = w.logits + blockIdx.z * all_logits + static_cast<long long>(t0 + r) * s.experts + e0 + 4 * q;
#pragma unroll
        for (int v = 0; v < 4; ++v)
            if (t0 + r < s.tokens && e0 + 4 * q + v < s.experts) mc_split_store(out + v, sum[v]);
    });

    if (s.tokens <= kFew) return;
    if (!mc_split_last_arrival(w.arrived + 1 + blockIdx.y, gridDim.x * parts, &flag)) return;
    const int t1 = t0 + 16 < s.tokens ? t0 + 16 : s.tokens;
    route(w, s, parts, t0, t1, normalize, logits, chosen, gate);
    if (gridDim.y > 1) {
        for (int i = threadIdx.x; i < (t1 - t0) * kMaxTopK; i += kThreads) {
            mc_split_store(reinterpret_cast<float*>(w.chosen) + t0 * kMaxTopK + i,
                           __builtin_bit_cast(float, chosen[t0][i]));
            mc_split_store(w.gate + t0 * kMaxTopK + i, gate[t0][i]);
        }
        if (!mc_split_last_arrival(w.arrived, gridDim.y, &flag)) return;
        for (int i = threadIdx.x; i < s.tokens * kMaxTopK; i += kThreads) {
            chosen[0][i] = __builtin_bit_cast(int, mc_split_load(reinterpret_cast<const float*>(w.chosen) + i));
            gate[0][i] = mc_split_load(w.gate + i);
        }
        __syncthreads();
    }
    list_jobs(w, s, chosen, gate, mask, place);
    for (int i = threadIdx.x; i < s.tokens * s.top_k; i += kThreads) {
        const int t = i / s.top_k, j = i % s.top_k;
        if (chosen_out != nullptr) chosen_out[i] = chosen[t][j];
        if (gates_out != nullptr) gates_out[i] = gate[t][j];
    }
}

// ---------------------------------------------------------------- experts' products

// kTiles tiles of 16 rows of an expert's weights and 16 tokens' pieces.
template <int kType, int kTiles, int kP, bool kOdd, bool kHalf>
struct Stream : Rows<kType, kTiles, kOdd, kHalf> {
    typedef Rows<kType, kTiles, kOdd, kHalf> Base;
    using Base::offset;
    using Base::q;

    struct Step {
        typename Base::Step w;
        u32x4 x[4][kP];
    };

    const unsigned short* x;  // lane's token, at its chunk
    long long x_plane, x_chunk;
    bool has;

    // Chunks of eight elements of a token, `chunk` apart, in pieces `plane` apart; has: there is a token.
    __device__ __forceinline__ void tokens(const unsigned short* p, long long chunk, long long plane, bool has_) {
        x = p, x_chunk = chunk, x_plane = plane, has = has_;
    }

    __device__ __forceinline__ void load(int t, Step& st) const {
        Base::load(t, st.w);
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int p = 0; p < kP; ++p)
                st.x[s][p] = has ? *reinterpret_cast<const u32x4*>(x + p * x_plane + (t * kStep + offset(q, s)) / 8 * x_chunk)
                                 : u32x4{0, 0, 0, 0};
    }

    __device__ __forceinline__ void multiply(int t, Step& st, f32x4 (&acc)[kTiles]) const {
        if (Base::past_end(t)) Base::cut_off(t, st.w);
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
            float scale = 0.0f;
            if constexpr (Base::kQuant) scale = scale_operand(Base::scale(st.w, i));
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                u32x4 w[Base::kPiecesW];
                Base::operand(st.w, i, s, scale, w);
#pragma unroll
                for (int wp = 0; wp < Base::kPiecesW; ++wp)
#pragma unroll
                    for (int p = 0; p < kP; ++p)
                        acc[i] = kHalf ? mfma_f16(w[wp], st.x[s][p], acc[i]) : mfma_bf16(w[wp], st.x[s][p], acc[i]);
            }
        }
    }
};

template <int kAct>
__device__ __forceinline__ float activate(float u, float up) {
    if constexpr (kAct == MCHIP_MOE_RELU) return u > 0.0f ? u : (u == u ? 0.0f : u);
    if constexpr (kAct == MCHIP_MOE_SWIGLU) return u / (1.0f + expf(-u)) * up;
    return 0.5f * u * (1.0f + tanhf(0.79788456080286536f * (u + 0.044715f * u * u * u)));
}

// h of jobs, 32 (swiglu: 16) columns at a time: every job's column tiles in a row
// are cut evenly over the blocks, so that the grid does not depend on how many
// jobs there are. The waves take a tile's steps in turn, and the next step, of
// the next tile too, is under way while one is multiplied and while the waves'
// sums are added (a block per tile waited for its job, its weights and its sums
// in turn: 143 MB of mx4 in 42 us). Columns past h are written as zeros (past
// the last tile by moe_router).
// kHalf: x was kept in fp16, as the weights are (one piece).
template <int kType>
constexpr int kUpWaves = kType == kMx4 ? 8 : 4;  // 16-bit weights take the registers of two mx4 waves

template <int kType, int kP, int kAct, bool kOdd, bool kHalf>
__global__ __launch_bounds__(64 * kUpWaves<kType>) void moe_up(const void* __restrict__ w1,
                                                               const unsigned char* __restrict__ w1_scales,
                                                               const float* __restrict__ b1, Workspace w, Sizes s,
                                                               int parts, bool normalize,
                                                               int* __restrict__ chosen_out,
                                                               float* __restrict__ gates_out) {
    constexpr bool kGated = kAct == MCHIP_MOE_SWIGLU;
    constexpr int kTiles = 2, kUpCols = kGated ? 16 : 32, kWaves = kUpWaves<kType>, kThreads = 64 * kWaves;
    typedef Stream<kType, kTiles, kP, kOdd, kHalf> In;
    __shared__ f32x4 space[2][kWaves][kTiles][64];
    extern __shared__ __attribute__((aligned(16))) float logits[];  // for few tokens: [tokens, experts], then their jobs
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int r = lane % 16;
    const int tiles = (s.h + kUpCols - 1) / kUpCols, steps = s.dp / kStep;
    Job* jobs = reinterpret_cast<Job*>(logits);  // the block's, from `first_job` on
    int count;
    if (s.tokens <= kFew) {
        __shared__ int chosen[kFew][kMaxTopK];
        __shared__ float gate[kFew][kMaxTopK];
        __shared__ unsigned mask[kMaxExperts];
        __shared__ int place[kMaxExperts], counts[2];
        jobs = reinterpret_cast<Job*>(logits + s.tokens * s.experts);
        clear_few_jobs(s, mask, jobs);
        route(w, s, parts, 0, s.tokens, normalize, logits, chosen, gate);
        count = list_few_jobs(s, chosen, gate, mask, place, counts, jobs);
        if (blockIdx.x == 0) {  // for moe_down and the caller
            if (threadIdx.x == 0) *w.jobs = count;
            for (int i = threadIdx.x; i < count * static_cast<int>(sizeof(Job) / 4); i += kThreads)
                reinterpret_cast<int*>(w.job)[i] = reinterpret_cast<const int*>(jobs)[i];
            for (int i = threadIdx.x; i < s.tokens * s.top_k; i += kThreads) {
                if (chosen_out != nullptr) chosen_out[i] = chosen[i / s.top_k][i % s.top_k];
                if (gates_out != nullptr) gates_out[i] = gate[i / s.top_k][i % s.top_k];
            }
        }
    } else {
        count = *w.jobs;
    }
    const long long all = static_cast<long long>(count) * tiles;
    // (Said to be the same in all lanes: a descriptor that may differ is loaded through lane by lane.)
    const int from = __builtin_amdgcn_readfirstlane(static_cast<int>(blockIdx.x * all / gridDim.x));
    const int to = __builtin_amdgcn_readfirstlane(static_cast<int>((blockIdx.x + 1) * all / gridDim.x));
    if (from >= to) return;
    int first_job = 0;
    if (s.tokens > kFew) {
        first_job = from / tiles;
        const int dwords = ((to - 1) / tiles - first_job + 1) * static_cast<int>(sizeof(Job) / 4);
        for (int i = threadIdx.x; i < dwords; i += kThreads)
            reinterpret_cast<int*>(jobs)[i] = reinterpret_cast<const int*>(w.job + first_job)[i];
        __syncthreads();
    }
    const int h_rows = kGated ? 2 * s.h : s.h;
    const long long h_plane = static_cast<long long>(s.max_jobs) * 16 * s.hp;

    int job = kNone, expert = 0, token = kNone;
    const auto open = [&](int u, In& in) {
        if (u / tiles != job) {
            job = u / tiles;
            expert = __builtin_amdgcn_readfirstlane(jobs[job - first_job].expert);
            token = jobs[job - first_job].token[r];
        }
        const int h0 = u % tiles * kUpCols;
        in.open(w1, w1_scales, s.d, static_cast<long long>(s.experts) * h_rows, [&](int i) {
            return static_cast<long long>(expert) * h_rows + (kGated ? h0 + i * s.h : h0 + 16 * i < s.h ? h0 + 16 * i : 0);
        });
        in.tokens(w.x + (token == kNone ? 0 : token) * 8, 8LL * s.tokens, static_cast<long long>(s.tokens) * s.dp,
                  token != kNone);
    };
    In in;
    typename In::Step now, next;
    open(from, in);
    if (wave < steps) in.load(wave, next);
    for (int u = from; u < to; ++u) {
        const int of_job = u / tiles, of_expert = expert, h0 = u % tiles * kUpCols;
        f32x4 acc[kTiles];
#pragma unroll
        for (int i = 0; i < kTiles; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int t = wave; t < steps; t += kWaves) {
            now = next;
            const int then = t + kWaves < steps ? t + kWaves : wave;
            const bool move = then == wave;  // to the next tile (multiplying needs nothing of `in` but the lane's place)
            if (move && u + 1 < to) open(u + 1, in);
            if (!move || u + 1 < to) in.load(then, next);
            in.multiply(t, now, acc);
        }
        if (wave >= steps && u + 1 < to) open(u + 1, in);
        f32x4(&sums)[kWaves][kTiles][64] = space[u & 1];
#pragma unroll
        for (int i = 0; i < kTiles; ++i) sums[wave][i][lane] = acc[i];
        __syncthreads();
        // A thread per element: lane's values v of a tile are columns 4 q + v of token r.
        for (int o = threadIdx.x; o < (kGated ? 256 : 512); o += kThreads) {
            const int at = o % 256, tile = o / 256, er = at / 4 % 16, col = h0 + 16 * tile + at / 64 * 4 + at % 4;
            const auto sum = [&](int i) {
                float v = 0.0f;
#pragma unroll
                for (int n = 0; n < kWaves; ++n) v += reinterpret_cast<const float*>(sums[n][i])[at];
                return v;
            };
            float a = sum(tile), up = kGated ? sum(1) : 0.0f;
            const bool in_h = col < s.h;
            if (b1 != nullptr && in_h) {
                a += b1[static_cast<long long>(of_expert) * h_rows + col];
                if (kGated) up += b1[static_cast<long long>(of_expert) * h_rows + s.h + col];
            }
            float piece[kPiecesH];
            cut<kPiecesH>(in_h ? activate<kAct>(a, up) : 0.0f, piece);
#pragma unroll
            for (int p = 0; p < kPiecesH; ++p)
                w.h[p * h_plane + static_cast<long long>(of_job) * 16 * s.hp + (col / 8 * 16 + er) * 8 + col % 8] =
                    static_cast<unsigned short>(__builtin_bit_cast(unsigned, piece[p]) >> 16);
        }
    }
}

// 32 columns of y for all tokens and one share of the jobs' steps (all jobs' steps
// in a row, cut evenly over the shares' waves). A wave adds each of its jobs'
// parts, weighed, to its own LDS tile (no two lanes the same element); the tiles
// are added in wave order, the shares in their order by the last block to arrive.
template <int kType, int kOut, bool kOdd>
__global__ __launch_bounds__(kThreads) void moe_down(const void* __restrict__ w2, const unsigned char* __restrict__ w2_scales,
                                                     const float* __restrict__ b2, Workspace w, Sizes s,
                                                     void* __restrict__ y) {
    constexpr int kTiles = kCols / 16;
    extern __shared__ __attribute__((aligned(16))) float tile[];  // [kWaves][tokens][kCols]
    __shared__ int flag;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int r = lane % 16, q = lane / 16;
    const int d0 = blockIdx.x * kCols, shares = gridDim.y;
    const int cells = s.tokens * kCols;
    float* mine = tile + wave * cells;
    const int steps = s.hp / kStep, units = *w.jobs * steps;
    const int waves = shares * kWaves, each = units / waves, more = units % waves;
    const int index = blockIdx.y * kWaves + wave;
    const int from = index * each + (index < more ? index : more), to = from + each + (index < more ? 1 : 0);
    const long long h_plane = static_cast<long long>(s.max_jobs) * 16 * s.hp;

    typedef Stream<kType, kTiles, kPiecesH, kOdd, false> In;
    In in;
    typename In::Step now, next;
    int expert = 0, token = kNone;
    float gate = 0.0f;
    const auto open = [&](int n) {
        expert = __builtin_amdgcn_readfirstlane(w.job[n].expert);
        token = w.job[n].token[r];
        gate = w.job[n].gate[r];
        in.open(w2, w2_scales, s.h, static_cast<long long>(s.experts) * s.d, [&](int i) {
            return static_cast<long long>(expert) * s.d + (d0 + 16 * i < s.d ? d0 + 16 * i : d0);
        });
        in.tokens(w.h + static_cast<long long>(n) * 16 * s.hp + r * 8, 16 * 8, h_plane, token != kNone);
    };
    int n = from / steps, t = from % steps;
    if (from < to) {
        open(n);
        in.load(t, next);
    }
    for (int i = lane * 4; i < cells; i += 256) *reinterpret_cast<f32x4*>(mine + i) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int u = from; u < to;) {
        const int of_expert = expert, of_token = token;
        const float of_gate = gate;
        f32x4 acc[kTiles];
#pragma unroll
        for (int i = 0; i < kTiles; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (b2 != nullptr && t == 0) {  // the job's first step brings the bias
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const int c = d0 + 16 * i + 4 * q + v;
                    if (c < s.d) acc[i][v] = b2[static_cast<long long>(of_expert) * s.d + c];
                }
        }
        // To the job's end or the wave's; the next step, of the next job too, is under way meanwhile.
        for (bool same = true; same && u < to; ++u) {
            now = next;
            const int of_t = t;
            if (++t == steps) {
                t = 0;
                same = false;
                if (u + 1 < to) open(++n);
            }
            if (u + 1 < to) in.load(t, next);
            in.multiply(of_t, now, acc);
        }
        if (of_token != kNone) {
#pragma unroll
            for (int i = 0; i < kTiles; ++i)
#pragma unroll
                for (int v = 0; v < 4; ++v) mine[of_token * kCols + 16 * i + 4 * q + v] += of_gate * acc[i][v];
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
    if (shares == 1 || !mc_split_last_arrival(w.arrived + kFirstColumn + blockIdx.x, shares, &flag)) return;
    constexpr int kEach = kMaxTokens * kCols / kThreads;
    const float* parts[kEach];
    float sum[kEach];
#pragma unroll
    for (int n = 0; n < kEach; ++n) {  // past the last cell: the first one's, not stored
        const int i = threadIdx.x + n * kThreads, t = i / kCols, c = i % kCols;
        parts[n] = w.y + (i < cells ? t * row + d0 + c : d0);
    }
    add_parts<kEach>(parts, plane, shares, sum);
#pragma unroll
    for (int n = 0; n < kEach; ++n) {
        const int i = threadIdx.x + n * kThreads, t = i / kCols, c = i % kCols;
        if (i < cells && d0 + c < s.d) store_one<kOut>(y, static_cast<long long>(t) * s.d + d0 + c, sum[n]);
    }
}

// ---------------------------------------------------------------- launches

template <int kIn, int kType, int kAct, bool kOdd>
int launch_experts(const mchip_moe_args& a, const Workspace& w, const Sizes& s, hipStream_t stream) {
    constexpr int kUpCols = kAct == MCHIP_MOE_SWIGLU ? 16 : 32;
    constexpr bool kHalf = kIn == kF16 && kType == kF16;
    // As many blocks as the registers let run at once, about.
    const long long units = static_cast<long long>(s.max_jobs) * ((s.h + kUpCols - 1) / kUpCols);
    const long long blocks = static_cast<long long>(kType == kMx4 ? 2 : 3) * device_cus();
    // A block's jobs: all of few tokens' (behind their logits), or those of its share of the units.
    const long long grid = std::min(blocks, units);
    const std::size_t jobs = s.tokens <= kFew ? s.max_jobs : std::min<long long>(s.max_jobs, s.max_jobs / grid + 2);
    const std::size_t lds = sizeof(Job) * jobs + (s.tokens <= kFew ? sizeof(float) * s.tokens * s.experts : 0);
    const int rc = launch_kernel(moe_up<kType, kHalf ? 1 : kPieces<kIn>, kAct, kOdd, kHalf>, static_cast<unsigned>(grid),
                                 64 * kUpWaves<kType>, lds, stream, a.w1, static_cast<const unsigned char*>(a.w1_scales),
                                 a.b1, w, s, router_parts(s.d), a.normalize != 0, a.chosen, a.gates);
    if (rc != hipSuccess) return rc;
    return launch_kernel(moe_down<kType, kIn, kOdd>,
                         dim3(static_cast<unsigned>(column_tiles(s.d)), static_cast<unsigned>(down_shares(s))), kThreads,
                         sizeof(float) * kWaves * s.tokens * kCols, stream, a.w2,
                         static_cast<const unsigned char*>(a.w2_scales), a.b2, w, s, a.y);
}

template <int kIn, int kType, int kAct>
int launch_odd(const mchip_moe_args& a, const Workspace& w, const Sizes& s, hipStream_t stream) {
    if constexpr (kType != kMx4) {
        if (s.d % 2 != 0 || s.h % 2 != 0 || !aligned(a.w1, 4) || !aligned(a.w2, 4))
            return launch_experts<kIn, kType, kAct, true>(a, w, s, stream);
    }
    return launch_experts<kIn, kType, kAct, false>(a, w, s, stream);
}

template <int kIn, int kType>
int launch_act(const mchip_moe_args& a, const Workspace& w, const Sizes& s, hipStream_t stream) {
    if (a.activation == MCHIP_MOE_RELU) return launch_odd<kIn, kType, MCHIP_MOE_RELU>(a, w, s, stream);
    if (a.activation == MCHIP_MOE_GELU) return launch_odd<kIn, kType, MCHIP_MOE_GELU>(a, w, s, stream);
    return launch_odd<kIn, kType, MCHIP_MOE_SWIGLU>(a, w, s, stream);
}

template <int kIn>
int launch(const mchip_moe_args& a, hipStream_t stream) {
    const Sizes s = sizes_of(a.tokens, a.d, a.h, a.experts, a.top_k);
    Workspace w;
    lay_out(s, a.dtype, static_cast<unsigned char*>(a.workspace), &w);
    const dim3 grid(static_cast<unsigned>((s.experts + 15) / 16), static_cast<unsigned>((s.tokens + 15) / 16),
                    static_cast<unsigned>(2 * router_parts(s.d)));
    const auto router = [&](auto kernel) {
        return launch_kernel(kernel, grid, kThreads, sizeof(float) * 16 * s.experts, stream, a.x, a.ldx, a.router, w, s,
                             a.normalize != 0, a.chosen, a.gates);
    };
    const int rc = kIn == kF16 && a.weights == kF16 ? router(moe_router<kIn, kIn == kF16>) : router(moe_router<kIn, false>);
    if (rc != hipSuccess) return rc;
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
    if (a.weights == kMx4 && (!aligned(a.w1_scales, 4) || !aligned(a.w2_scales, 4))) return "scales not 4-byte aligned";
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

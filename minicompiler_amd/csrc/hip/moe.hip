// A mixture-of-experts MLP for the few tokens of a decoding step (mx4.h):
//   p = softmax(x R^T); the top_k largest experts e of each token, ties to the
//   lower index, with gates g_e = p_e, or p_e / sum of the chosen p;
//   y = sum over the chosen e of g_e (act(x W1_e^T + b1_e) W2_e^T + b2_e).
//
// Three launches, in stream order:
//   moe_router  x R^T on the FP32 matrix instruction, x cut into bf16 pieces;
//               the last block to arrive picks the experts and lists the jobs
//               (one per chosen expert and 16 of its tokens);
//   moe_up      per job and 32 (swiglu: 16) columns of h: act(x W1^T + b1), cut
//               into bf16 pieces;
//   moe_down    per 32 columns of y: all jobs, h W2^T weighed by the gates.
// Bound by the chosen experts' weights, each read once per job. Weights are the
// matrix instruction's first operand, 16 rows of them, and a job's 16 tokens
// the second. Products are exact (bf16 pieces of x, h and the weights), sums fp32.

#include "mx4_device.h"

#include "gemm_split_arrival.h"

namespace {

using namespace mx4;

constexpr int kMaxTokens = MCHIP_MOE_MAX_TOKENS, kMaxExperts = MCHIP_MOE_MAX_EXPERTS, kMaxTopK = MCHIP_MOE_MAX_TOP_K;
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
    unsigned* arrived;
    int* jobs;            // how many
    Job* job;             // [max_jobs]
    float* logits;        // [tokens, experts]
    unsigned short* x;    // [pieces][tokens][dp]
    unsigned short* h;    // [pieces][max_jobs * 16][hp]
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
    w->arrived = reinterpret_cast<unsigned*>(take(sizeof(unsigned)));
    w->jobs = reinterpret_cast<int*>(take(sizeof(int)));
    w->job = reinterpret_cast<Job*>(take(sizeof(Job) * static_cast<std::size_t>(s.max_jobs)));
    w->logits = reinterpret_cast<float*>(take(sizeof(float) * static_cast<std::size_t>(s.tokens) * s.experts));
    w->x = reinterpret_cast<unsigned short*>(
        take(2 * static_cast<std::size_t>(pieces_of(dtype)) * s.tokens * s.dp));
    w->h = reinterpret_cast<unsigned short*>(
        take(2 * static_cast<std::size_t>(h_pieces_of(dtype)) * s.max_jobs * 16 * s.hp));
    return at;
}

// ---------------------------------------------------------------- router

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o /= 2) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o /= 2) v += __shfl_xor(v, o);
    return v;
}

// One token's experts and gates, by one wave. A NaN logit never counts as
// larger; it makes every gate NaN, as softmax does.
__device__ void choose(const float* logits, int experts, int top_k, bool normalize, int lane, int* chosen, float* gate) {
    constexpr int kEach = kMaxExperts / 64;
    float l[kEach];
    float top = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        const int e = lane + 64 * j;
        l[j] = e < experts ? mc_split_load(logits + e) : -__builtin_inff();
        top = fmaxf(top, l[j]);
    }
    top = wave_max(top);
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kEach; ++j)
        if (lane + 64 * j < experts) sum += expf(l[j] - top);
    sum = wave_sum(sum);
    unsigned taken = 0;
    float kept = 0.0f;
    for (int i = 0; i < top_k; ++i) {
        float best = -__builtin_inff();
        int at = 0x7fffffff;
#pragma unroll
        for (int j = 0; j < kEach; ++j) {
            const int e = lane + 64 * j;
            if (e >= experts || (taken >> j & 1u)) continue;
            if (at == 0x7fffffff || l[j] > best) {
                best = l[j] > -__builtin_inff() ? l[j] : -__builtin_inff();
                at = e;
            }
        }
#pragma unroll
        for (int o = 32; o > 0; o /= 2) {
            const float other = __shfl_xor(best, o);
            const int e = __shfl_xor(at, o);
            if (other > best || (other == best && e < at)) {
                best = other;
                at = e;
            }
        }
        if (at % 64 == lane) taken |= 1u << (at / 64);
        // The chosen expert's own logit (NaN if it is one).
        const float p = expf(mc_split_load(logits + at) - top) / sum;
        kept += p;
        if (lane == 0) {
            chosen[i] = at;
            gate[i] = p;
        }
    }
    if (normalize && lane == 0)
        for (int i = 0; i < top_k; ++i) gate[i] /= kept;
}

// The jobs from the chosen experts in LDS, by the whole block: a thread per expert.
__device__ void list_jobs(const Workspace& w, const Sizes& s, const int (*chosen)[kMaxTopK],
                          const float (*gate)[kMaxTopK], int* scan) {
    const int e = threadIdx.x;
    unsigned long long mask = 0;
    if (e < s.experts)
        for (int t = 0; t < s.tokens; ++t)
            for (int i = 0; i < s.top_k; ++i)
                if (chosen[t][i] == e) mask |= 1ull << t;
    const int mine = (__builtin_popcountll(mask) + 15) / 16;
    scan[e] = mine;
    __syncthreads();
    for (int o = 1; o < kMaxExperts; o *= 2) {
        const int add = e >= o ? scan[e - o] : 0;
        __syncthreads();
        scan[e] += add;
        __syncthreads();
    }
    if (e == kMaxExperts - 1) *w.jobs = scan[e];
    int at = scan[e] - mine;
    for (int n = 0; n < mine; ++n, ++at) {
        Job& job = w.job[at];
        job.expert = e;
        for (int i = 0; i < 16; ++i) {
            int t = kNone;
            float g = 0.0f;
            if (mask != 0) {
                t = __builtin_ctzll(mask);
                mask &= mask - 1;
                for (int j = 0; j < s.top_k; ++j)
                    if (chosen[t][j] == e) g = gate[t][j];
            }
            job.token[i] = t;
            job.gate[i] = g;
        }
    }
}

// 16 experts by 16 tokens of the logits; the waves take 16-wide steps of d in
// turn. v_mfma_f32_16x16x4_f32: lane (r, q) supplies row or column r, element q.
template <int kIn>
__global__ __launch_bounds__(kThreads) void moe_router(const void* __restrict__ x, long long ldx,
                                                       const float* __restrict__ router, Workspace w, Sizes s,
                                                       bool normalize, int* __restrict__ chosen_out,
                                                       float* __restrict__ gates_out) {
    constexpr int kP = kPieces<kIn>;
    __shared__ f32x4 space[kWaves / 2 * 64];
    __shared__ int chosen[kMaxTokens][kMaxTopK];
    __shared__ float gate[kMaxTokens][kMaxTopK];
    __shared__ int scan[kMaxExperts];
    __shared__ int flag;
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int r = lane % 16, q = lane / 16;
    const int e0 = blockIdx.x * 16, t0 = blockIdx.y * 16;
    const int blocks = gridDim.x * gridDim.y, block = blockIdx.y * gridDim.x + blockIdx.x;

    const long long expert = e0 + r < s.experts ? e0 + r : s.experts - 1;
    const long long token = t0 + r < s.tokens ? t0 + r : s.tokens - 1;
    f32x4 acc[1] = {{0.0f, 0.0f, 0.0f, 0.0f}};
    for (int k0 = wave * 16; k0 < s.d; k0 += kWaves * 16) {
        const int k = k0 + 4 * q;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool in = k + j < s.d;
            const float a = in ? router[expert * s.d + k + j] : 0.0f;
            const float b = in ? load_one<kIn>(x, token * ldx + k + j) : 0.0f;
            acc[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, acc[0], 0, 0, 0);
        }
    }
    add_waves<kWaves, 1>(acc, space, wave, lane);
    if (wave == 0 && t0 + r < s.tokens) {
#pragma unroll
        for (int v = 0; v < 4; ++v)
            if (e0 + 4 * q + v < s.experts)
                mc_split_store(w.logits + static_cast<long long>(t0 + r) * s.experts + e0 + 4 * q + v, acc[0][v]);
    }

    // x in pieces, rows padded with zeros, shared out over the blocks.
    const long long all = static_cast<long long>(s.tokens) * s.dp;
    for (long long i = static_cast<long long>(block) * kThreads + threadIdx.x; i < all;
         i += static_cast<long long>(blocks) * kThreads) {
        const int t = static_cast<int>(i / s.dp), k = static_cast<int>(i % s.dp);
        float piece[kP];
        cut<kP>(k < s.d ? load_one<kIn>(x, t * ldx + k) : 0.0f, piece);
#pragma unroll
        for (int p = 0; p < kP; ++p)
            w.x[p * all + i] = static_cast<unsigned short>(__builtin_bit_cast(unsigned, piece[p]) >> 16);
    }

    if (!mc_split_last_arrival(w.arrived, blocks, &flag)) return;
    for (int t = wave; t < s.tokens; t += kWaves)
        choose(w.logits + static_cast<long long>(t) * s.experts, s.experts, s.top_k, normalize, lane, chosen[t], gate[t]);
    __syncthreads();
    list_jobs(w, s, chosen, gate, scan);
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
    bool wide;

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
                if (wide && k0 + 8 <= k) {
                    st.raw[s] = *reinterpret_cast<const u32x4*>(p + k0);
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

// acc[i] += rows[i] (16 weight rows) times the columns `col` (a lane's own
// row of the pieces, `plane` elements apart), over step t.
template <int kType, int kP, int kTiles>
__device__ __forceinline__ void multiply_step(const Weights<kType>& w, const long long (&rows)[kTiles],
                                              const unsigned short* col, long long plane, bool has, int t, int q,
                                              f32x4 (&acc)[kTiles]) {
    typename Weights<kType>::Step st[kTiles];
#pragma unroll
    for (int i = 0; i < kTiles; ++i) st[i] = w.load(rows[i], t, q);
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
    constexpr int kTiles = 2, kCols = kGated ? 16 : 32;
    __shared__ f32x4 space[kWaves / 2 * kTiles * 64];
    if (static_cast<int>(blockIdx.y) >= *w.jobs) return;
    const Job& job = w.job[blockIdx.y];
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int r = lane % 16, q = lane / 16;
    const int h0 = blockIdx.x * kCols;
    const int token = job.token[r];
    const long long all_rows = kGated ? 2LL * s.h : s.h;
    const long long first = job.expert * all_rows;
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
    if (h0 < s.h)
        for (int t = wave; t < s.dp / kStep; t += kWaves)
            multiply_step<kType, kP, kTiles>(w1, rows, col, plane, token != kNone, t, q, acc);
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

// 32 columns of y for all tokens. A wave adds every job's share of its steps of
// h into its own LDS tile (no two lanes the same element); the tiles are added
// in wave order.
template <int kType, int kP, int kOut>
__global__ __launch_bounds__(kThreads) void moe_down(Weights<kType> w2, const float* __restrict__ b2, Workspace w,
                                                     Sizes s, void* __restrict__ y) {
    constexpr int kTiles = 2, kCols = 16 * kTiles;
    __shared__ float tile[kWaves][kMaxTokens][kCols];
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int r = lane % 16, q = lane / 16;
    const int d0 = blockIdx.x * kCols;
    for (int i = lane; i < s.tokens * kCols; i += 64) (&tile[wave][0][0])[i] = 0.0f;
    const int jobs = *w.jobs;
    const long long h_plane = static_cast<long long>(s.max_jobs) * 16 * s.hp;
    for (int n = 0; n < jobs; ++n) {
        const Job& job = w.job[n];
        const int token = job.token[r];
        const float gate = job.gate[r];
        const long long first = static_cast<long long>(job.expert) * s.d;
        long long rows[kTiles];
        f32x4 acc[kTiles];
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
            const int col = d0 + 16 * i + r;
            rows[i] = first + (col < s.d ? col : s.d - 1);
            acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        const unsigned short* col = w.h + (static_cast<long long>(n) * 16 + r) * s.hp;
        for (int t = wave; t < s.hp / kStep; t += kWaves)
            multiply_step<kType, kP, kTiles>(w2, rows, col, h_plane, token != kNone, t, q, acc);
        if (token == kNone) continue;
#pragma unroll
        for (int i = 0; i < kTiles; ++i)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int c = 16 * i + 4 * q + v;
                float o = acc[i][v];
                if (b2 != nullptr && wave == 0 && d0 + c < s.d) o += b2[first + d0 + c];
                tile[wave][token][c] += gate * o;
            }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < s.tokens * kCols; i += kThreads) {
        const int t = i / kCols, c = i % kCols;
        if (d0 + c >= s.d) continue;
        float sum = 0.0f;
#pragma unroll
        for (int v = 0; v < kWaves; ++v) sum += tile[v][t][c];
        store_one<kOut>(y, static_cast<long long>(t) * s.d + d0 + c, sum);
    }
}

// ---------------------------------------------------------------- launches

template <int kType>
Weights<kType> weights(const void* base, const void* scales, int k) {
    return {base, static_cast<const unsigned char*>(scales), k, padded(k), k % 8 == 0 && aligned(base, 16)};
}

template <int kIn, int kType, int kAct>
int launch_experts(const mchip_moe_args& a, const Workspace& w, const Sizes& s, hipStream_t stream) {
    constexpr int kHP = kIn == kF32 ? 3 : 2;
    constexpr int kCols = kAct == MCHIP_MOE_SWIGLU ? 16 : 32;
    hipLaunchKernelGGL((moe_up<kType, kPieces<kIn>, kHP, kAct>),
                       dim3(static_cast<unsigned>(s.hp / kCols), static_cast<unsigned>(s.max_jobs)), dim3(kThreads), 0,
                       stream, weights<kType>(a.w1, a.w1_scales, s.d), a.b1, w, s);
    hipLaunchKernelGGL((moe_down<kType, kHP, kIn>), dim3(static_cast<unsigned>((s.d + 31) / 32)), dim3(kThreads), 0,
                       stream, weights<kType>(a.w2, a.w2_scales, s.h), a.b2, w, s, a.y);
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
                       dim3(static_cast<unsigned>((s.experts + 15) / 16), static_cast<unsigned>((s.tokens + 15) / 16)),
                       dim3(kThreads), 0, stream, a.x, a.ldx, a.router, w, s, a.normalize != 0, a.chosen, a.gates);
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
    if (a.d > (1 << 20) || a.h > (1 << 20)) return "rows longer than 2^20";
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
    if (!is_float_type(dtype) || tokens < 1 || tokens > kMaxTokens || d < 1 || h < 1 || d > (1 << 20) ||
        h > (1 << 20) || experts < 1 || experts > kMaxExperts || top_k < 1 || top_k > kMaxTopK)
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

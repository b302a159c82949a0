// The choice of experts: scores, groups, the top_k largest, their gates, and the
// plan (pairs of token and place by expert) that the experts' products run on.
//
// Keys are in fp64: they are compared with a bias added, or in sums of two, and two
// experts whose scores lie next to each other are then still in their order.
//
// Bound by latency, and that by the code that a launch reads into a cold instruction
// cache: sixteen lanes take a token, a lane 4 to 32 experts next to each other, keys lie
// in LDS while loops go over them and in registers while the largest are picked, over
// lanes by DPP. 8192 tokens, 8 of 256 experts in groups: 20.3 us, 14.9 of them here and 6.5 in
// the plan's launch; one token on 64 experts 4.3, plan included. (A wave a token with LDS
// permutes: 35 us for the choice alone; fp32 keys in unrolled code, with fp64 ones behind for
// what lies too near: 23.)

#include "i8_device.h"

namespace {

using namespace i8;

constexpr int kThreads = 512, kWaves = kThreads / 64, kTokens = kThreads / 16;  // of a block
constexpr int kFewPairs = 128;  // of a plan that the choosing block makes itself
constexpr double kNone = -__builtin_inf();

struct Route {
    const void* logits;
    long long ld;
    const float* bias;
    int tokens, experts, top_k, score, groups, each, top_groups, group_best, normalize;
    float scale;
    int* chosen;
    float* gates;
    int *order, *offsets;
    unsigned short* ids;  // of all pairs, for the plan's launch, or null
    bool by_logit;        // one score by itself is as large as its logit
    bool plans;           // the only block makes the plan, too
    long long first;      // the launch's first token
};

// Place j of a token. Behind the last pair the ids go on to a multiple of eight with an
// expert past all others.
__device__ __forceinline__ void put(const Route& p, unsigned short* few, long long token, int j, int expert, float gate) {
    const long long at = token * p.top_k + j;
    p.chosen[at] = expert;
    p.gates[at] = gate;
    if (p.plans) few[at] = static_cast<unsigned short>(expert);
    if (p.ids != nullptr) {
        p.ids[at] = static_cast<unsigned short>(expert);
        const long long pairs = static_cast<long long>(p.tokens) * p.top_k;
        if (at == pairs - 1)
            for (long long i = pairs; i % 8 != 0; ++i) p.ids[i] = 0xffff;
    }
}

// Over the 16 lanes of a token: the two neighbours of a pair, of four, of eight, of all.
template <int kCtrl>
__device__ __forceinline__ double of_lane(double v) {
    const u32x2 u = __builtin_bit_cast(u32x2, v);
    u32x2 r;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        r[i] = static_cast<unsigned>(
            __builtin_amdgcn_update_dpp(static_cast<int>(u[i]), static_cast<int>(u[i]), kCtrl, 0xf, 0xf, false));
    return __builtin_bit_cast(double, r);
}
template <typename Op>
__device__ __forceinline__ double over_token(double v, Op op) {
    v = op(v, of_lane<0xb1>(v));
    v = op(v, of_lane<0x4e>(v));
    v = op(v, of_lane<0x141>(v));
    return op(v, of_lane<0x140>(v));
}
// Of a number and a NaN the number.
__device__ __forceinline__ double larger(double a, double b) { return __builtin_fmax(a, b); }
__device__ __forceinline__ double both(double a, double b) { return a + b; }

// The plan of few pairs by the block that chose them: pair i's slot is how many pairs come
// before it, expert e's first how many have a lower one. `few` is padded with experts past
// the last.
__device__ __forceinline__ void plan_few(const Route& p, const unsigned short* few) {
    const int pairs = p.tokens * p.top_k, i = threadIdx.x;
    const int mine = i < pairs ? few[i] : 0;
    int before = 0, below = 0;
#pragma unroll 2
    for (int j = 0; j < pairs; j += 8) {
        const u16x8 eight = *reinterpret_cast<const u16x8*>(few + j);
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int e = eight[u];
            before += e < mine + (j + u < i);
            below += e < i;
        }
    }
    if (i < pairs) p.order[before] = i;
    if (i < p.experts) p.offsets[i] = below;
    if (i == 0) p.offsets[p.experts] = pairs;
}

// Sixteen lanes take a token, lane l experts l kPer .. + kPer - 1. An expert that may not
// be chosen (it is none, is not in a group that stays, or has been chosen) has a NaN key.
template <int kType, int kPer>
__global__ __launch_bounds__(kThreads) void route_tokens(const Route p) {
    // Two spare words behind a lane's experts and a token's: lanes and groups meet in
    // different banks.
    constexpr int kLane = kPer + 2, kWords = 16 * kLane + 2;
    __shared__ __attribute__((aligned(16))) double space[kTokens * kWords];
    __shared__ float bias[kPer * 16];  // zeros without one
    __shared__ __attribute__((aligned(16))) unsigned short few[kFewPairs];
    __shared__ int picked[kTokens][MCHIP_ROUTE_MAX_TOP_K];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, l = lane % 16, row = lane / 16;
    const long long token = p.first + (static_cast<long long>(blockIdx.x) * kWaves + wave) * 4 + row;
    const bool has = token < p.tokens;
    const long long from = (has ? token : 0) * p.ld;
    const int e0 = l * kPer;
    double* mine = space + (wave * 4 + row) * kWords;
    const auto slot = [](int e) { return e / kPer * kLane + e % kPer; };
    if (p.plans && threadIdx.x < kFewPairs) few[threadIdx.x] = 0xffff;
    f32x4 four[kPer / 4];
    if (p.experts % 4 == 0) {
#pragma unroll
        for (int i = 0; i < kPer / 4; ++i) {
            four[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (e0 + 4 * i < p.experts) four[i] = load_four<kType>(p.logits, from + e0 + 4 * i, 4);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kPer / 4; ++i) four[i] = load_four<kType>(p.logits, from + e0 + 4 * i, p.experts - e0 - 4 * i);
    }
    if (threadIdx.x < kPer * 16)
        bias[threadIdx.x] = p.bias != nullptr && static_cast<int>(threadIdx.x) < p.experts ? p.bias[threadIdx.x] : 0.0f;
    __syncthreads();
    bool bad = false;
    double key[kPer], top = kNone;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const float v = four[i / 4][i % 4];
        bad |= v != v;
        key[i] = v != v ? kNone : static_cast<double>(v);
        key[i] = e0 + i < p.experts ? key[i] : __builtin_nan("");
        top = larger(top, key[i]);
    }
    top = over_token(top, larger);
    const bool soft = p.score == MCHIP_ROUTE_SOFTMAX;
    // Over +infinity a softmax is no number, though the experts that are chosen may be others.
    bad = (__ballot(bad) >> (16 * row) & 0xffffull) != 0 || (soft && top == -kNone);
    double total = 0.0;
    if (!p.by_logit || (soft && !p.normalize) || p.groups > 1) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) mine[l * kLane + i] = key[i];
        // Four experts at a time, straight through, so that their chains of dependent steps
        // run beside each other. An expert that is masked out stays so whatever its bias.
        const auto fours = [&](auto step) {
#pragma unroll 1
            for (int i = 0; i < kPer; i += 4) {
                double* at = mine + l * kLane + i;
                double v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = at[e];
                step(v, i);
#pragma unroll
                for (int e = 0; e < 4; ++e) at[e] = v[e];
            }
        };
        // Of a softmax's score, below 0 where masked out; no expert's is no number and stays so.
        const auto key_of = [&](double s, int e) {
            const double k = s + static_cast<double>(bias[e0 + e]);
            return s != s ? s : s < 0.0 || k != k ? kNone : k;
        };
        if (!p.by_logit && !soft) {
            fours([&](double (&v)[4], int i) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const double logit = v[e], k = 1.0 / (1.0 + exp(-logit)) + static_cast<double>(bias[e0 + i + e]);
                    v[e] = logit != logit ? logit : logit == kNone || k != k ? kNone : k;
                }
            });
        } else if (soft && (!p.by_logit || !p.normalize)) {
            fours([&](double (&v)[4], int i) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const double logit = v[e], x = exp(logit - top);
                    total += logit > kNone ? x : 0.0;  // none that is masked out, or no expert
                    // (+infinity less itself is no number, either: a key of none.)
                    if (!p.by_logit) v[e] = logit != logit ? logit : logit == kNone || x != x ? -1.0 : x;
                }
            });
            total = over_token(total, both);
            if (!p.by_logit) {
                const double share = 1.0 / total;
                fours([&](double (&v)[4], int i) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const double s = v[e] * share;
                        v[e] = key_of(s != s && v[e] == v[e] ? -1.0 : s, i + e);
                    }
                });
            }
        }
    }
    unsigned long long kept = ~0ull;
    if (p.groups > 1) {
        wave_lds_order();
        // sums[g]: group g's score, over the token's keys once all lanes have theirs in registers.
        double* sums = mine;
        kept = 0;
        double sum[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            sum[q] = kNone;
            const int g = l + 16 * q;
            if (16 * q >= p.groups) continue;
            if (g < p.groups) {
                double first = kNone, second = kNone;
#pragma unroll 4
                for (int i = 0; i < p.each; ++i) {
                    const double k = mine[slot(g * p.each + i)];
                    second = larger(second, __builtin_fmin(first, k));
                    first = larger(first, k);
                }
                // An expert that is masked out takes nothing from the group's others: only a group
                // of none but such is worth none.
                sum[q] = p.group_best == 2 && second > kNone ? first + second : first;
            }
        }
        wave_lds_order();
#pragma unroll
        for (int i = 0; i < kPer; ++i) key[i] = mine[l * kLane + i];
        wave_lds_order();
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (l + 16 * q < p.groups) sums[l + 16 * q] = sum[q];
        wave_lds_order();
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (16 * q >= p.groups) continue;
            const int g = l + 16 * q;
            int before = 0;
#pragma unroll 2
            for (int o = 0; o < p.groups; ++o) {
                const double s = sums[o];
                before += s > sum[q] || (s == sum[q] && o < g);
            }
            kept |= (__ballot(g < p.groups && before < p.top_groups) >> (16 * row) & 0xffffull) << (16 * q);
        }
        int group = e0 / p.each, in_group = e0 - group * p.each;
        bool stays = (kept >> (group & 63) & 1) != 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            key[i] = stays ? key[i] : __builtin_nan("");
            if (++in_group == p.each) in_group = 0, ++group, stays = (kept >> (group & 63) & 1) != 0;
        }
    } else if (!p.by_logit) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) key[i] = mine[l * kLane + i];
    }
    // The chosen one after the other, lane j the j-th.
    int* const places = picked[wave * 4 + row];
#pragma unroll 1
    for (int j = 0; j < p.top_k; ++j) {
        double most[kPer / 2];
#pragma unroll
        for (int i = 0; i < kPer / 2; ++i) most[i] = larger(key[2 * i], key[2 * i + 1]);
#pragma unroll
        for (int n = kPer / 4; n > 0; n /= 2)
#pragma unroll
            for (int i = 0; i < n; ++i) most[i] = larger(most[2 * i], most[2 * i + 1]);
        const double best = over_token(most[0], larger);
        const unsigned lanes = static_cast<unsigned>(__ballot(most[0] == best) >> (16 * row)) & 0xffffu;
        const bool winner = l == __builtin_ctz(lanes | 0x10000u);
        int at = kPer;
#pragma unroll
        for (int i = kPer - 1; i >= 0; --i) at = key[i] == best ? i : at;
        if (winner) places[j] = e0 + at;
        at = winner ? at : kPer;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            u32x2 u = __builtin_bit_cast(u32x2, key[i]);
            u[1] = at == i ? 0x7ff80000u : u[1];
            key[i] = __builtin_bit_cast(double, u);
        }
    }
    wave_lds_order();
    const int expert = l < p.top_k ? places[l] : 0;
    double gate = 0.0;
    if (l < p.top_k) {
        const double logit = load_one<kType>(p.logits, from + expert);
        const double e = exp(soft ? logit - top : -logit);
        gate = logit == kNone ? 0.0 : soft ? e : 1.0 / (1.0 + e);
    }
    const double over = p.normalize ? over_token(gate, both) : soft ? total : 1.0;
    gate = over != 0.0 ? gate / over : 0.0;
    if (bad) gate = __builtin_nan("");
    if (has && l < p.top_k) put(p, few, token, l, expert, static_cast<float>(gate * static_cast<double>(p.scale)));
    if (!p.plans) return;
    __syncthreads();
    plan_few(p, few);
}

// A block takes an expert: how many pairs have a lower one is where its slots begin,
// and its own pairs follow in order. A wave takes 4096 pairs at a time, a lane eight of
// 512 next to each other (whole lines to a load; 64 to a lane took three times as long).
// 65536 pairs of 256 experts in 6.5 us; every block reads all ids, twice where they are
// more than 65536 (16384 tokens, 8 of 384: 64 us with the choice).
constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64, kSteps = 8;

// The sum over the lanes up to this one.
__device__ __forceinline__ unsigned sum_to(unsigned v) {
#define ROUTE_STEP(ctrl, rows) \
    v += static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), ctrl, rows, 0xf, false));
    ROUTE_STEP(0x111, 0xf) ROUTE_STEP(0x112, 0xf) ROUTE_STEP(0x114, 0xf) ROUTE_STEP(0x118, 0xf)
    ROUTE_STEP(0x142, 0xa) ROUTE_STEP(0x143, 0xc)
#undef ROUTE_STEP
    return v;
}

__global__ __launch_bounds__(kPlanThreads) void make_plan(const unsigned short* __restrict__ ids, int pairs, int experts,
                                                          int* __restrict__ order, int* __restrict__ offsets) {
    constexpr int kPart = kPlanThreads * 8 * kSteps;
    __shared__ int own[kPlanWaves], lower[kPlanWaves];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, e = static_cast<int>(blockIdx.x);
    const int parts = (pairs + kPart - 1) / kPart;
    unsigned below = 0, mine[kSteps];  // mine: bit j: the lane's pair j of the step, of the part that was read last
    int at = 0;
    const auto read = [&](int part) {
        at = part * kPart + (wave * kSteps * 64 + lane) * 8;
        u16x8 eight[kSteps];
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            const int from = at + i * 512;
            eight[i] = u16x8{0xffff, 0xffff, 0xffff, 0xffff, 0xffff, 0xffff, 0xffff, 0xffff};
            if (from < pairs) eight[i] = *reinterpret_cast<const u16x8*>(ids + from);
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            mine[i] = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int id = eight[i][j];
                below += static_cast<unsigned>(id - e) >> 31;
                mine[i] |= id == e ? 1u << j : 0u;
            }
        }
    };
    for (int part = 0; part < parts; ++part) read(part);
    below = sum_to(below);
    if (lane == 63) lower[wave] = static_cast<int>(below);
    __syncthreads();
    int first = 0;
    for (int w = 0; w < kPlanWaves; ++w) first += lower[w];
    const int start = first;
    for (int part = 0; part < parts; ++part) {
        if (parts > 1) read(part);
        // Three steps' counts to a word: at most 512 each.
        unsigned packed[3] = {0, 0, 0}, up_to[3];
#pragma unroll
        for (int i = 0; i < kSteps; ++i) packed[i / 3] += static_cast<unsigned>(__popc(mine[i])) << i % 3 * 10;
        unsigned before[kSteps], all = 0;
#pragma unroll
        for (int w = 0; w < 3; ++w) up_to[w] = sum_to(packed[w]);
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            before[i] = all + ((up_to[i / 3] - packed[i / 3]) >> i % 3 * 10 & 1023u);
            all += __builtin_amdgcn_readlane(static_cast<int>(up_to[i / 3]), 63) >> i % 3 * 10 & 1023u;
        }
        if (lane == 0) own[wave] = static_cast<int>(all);
        __syncthreads();
        int to = first;
        for (int w = 0; w < kPlanWaves; ++w) {
            if (w < wave) to += own[w];
            first += own[w];
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            int slot = to + static_cast<int>(before[i]);
            for (unsigned bits = mine[i]; bits != 0; bits &= bits - 1) order[slot++] = at + i * 512 + __builtin_ctz(bits);
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        offsets[e] = start;
        if (e == experts - 1) offsets[experts] = first;
    }
}

// As many tokens at a time as a launch takes.
template <int kType>
int launch_tokens(Route p, hipStream_t stream) {
    constexpr long long kMost = 1LL << 27;
    static_assert(kMost / kTokens * kThreads < 1LL << 32);
    const auto go = [&](auto kernel) {
        int rc = hipSuccess;
        for (p.first = 0; rc == hipSuccess && p.first < p.tokens; p.first += kMost) {
            const long long count = std::min(kMost, p.tokens - p.first);
            rc = launch_kernel(kernel, static_cast<unsigned>((count + kTokens - 1) / kTokens), kThreads, 0, stream, p);
        }
        return rc;
    };
    if (p.experts <= 64) return go(route_tokens<kType, 4>);
    if (p.experts <= 128) return go(route_tokens<kType, 8>);
    if (p.experts <= 256) return go(route_tokens<kType, 16>);
    return go(route_tokens<kType, 32>);
}

// Whether the block that chooses makes the plan, too.
bool plans_itself(int tokens, int top_k) { return tokens <= kTokens && tokens * top_k <= kFewPairs; }

const char* refusal(const mchip_route_args& x) {
    if (!is_float_type(x.dtype)) return "the type is none of fp32 (0), bf16 (1), fp16 (2)";
    if (x.score != MCHIP_ROUTE_SOFTMAX && x.score != MCHIP_ROUTE_SIGMOID)
        return "the score is none of softmax (0), sigmoid (1)";
    if (x.tokens < 1 || x.experts < 1 || x.top_k < 1 || x.groups < 1 || x.top_groups < 1) return "a size below 1";
    if (x.experts > MCHIP_ROUTE_MAX_EXPERTS) return "more than 512 experts";
    if (x.top_k > MCHIP_ROUTE_MAX_TOP_K) return "more than 16 experts for a token";
    if (x.groups > MCHIP_ROUTE_MAX_GROUPS || x.experts % x.groups != 0)
        return "more than 64 groups, or groups that do not share out the experts evenly";
    if (x.top_groups > x.groups) return "more groups to choose than there are";
    if (x.group_best != 1 && x.group_best != 2) return "a group's score is neither of its largest (1) nor of its two largest (2)";
    if (x.top_k > x.experts / x.groups * x.top_groups) return "more experts to choose than the chosen groups have";
    if (static_cast<long long>(x.tokens) * x.top_k > (1 << 30)) return "more than 2^30 pairs of a token and an expert";
    if (x.ld < x.experts) return "rows closer together than they are long";
    if (x.logits == nullptr || x.chosen == nullptr || x.gates == nullptr) return "null logits, chosen or gates";
    if ((x.order == nullptr) != (x.offsets == nullptr)) return "one half of a plan";
    if (x.order != nullptr && !plans_itself(x.tokens, x.top_k) && (x.workspace == nullptr || !aligned(x.workspace, 256)))
        return "a null workspace, or one that is not 256-byte aligned";
    if (!aligned(x.logits, size_of(x.dtype))) return "an address that is no multiple of its element's size";
    if (!aligned(x.bias, 4) || !aligned(x.chosen, 4) || !aligned(x.gates, 4) || !aligned(x.order, 4) || !aligned(x.offsets, 4))
        return "a bias or an output that is not 4-byte aligned";
    return nullptr;
}

}  // namespace

extern "C" {

long long mchip_route_workspace_bytes(int tokens, int experts, int top_k) {
    if (tokens < 1 || experts < 1 || top_k < 1 || top_k > MCHIP_ROUTE_MAX_TOP_K || plans_itself(tokens, top_k)) return 0;
    return (static_cast<long long>(tokens) * top_k * 2 + 255) / 256 * 256;  // whole eights of ids
}

int mchip_launch_route(const mchip_route_args* args, void* stream, const char** why) {
    const mchip_route_args& x = *args;
    *why = refusal(x);
    if (*why != nullptr) return hipErrorInvalidValue;
    const bool plans = x.order != nullptr && plans_itself(x.tokens, x.top_k);
    unsigned short* ids = x.order != nullptr && !plans ? static_cast<unsigned short*>(x.workspace) : nullptr;
    const Route p{x.logits, x.ld, x.bias, x.tokens, x.experts, x.top_k, x.score, x.groups, x.experts / x.groups,
                  x.top_groups, x.group_best, x.normalize, x.scale, x.chosen, x.gates, x.order, x.offsets, ids,
                  x.bias == nullptr && (x.groups == 1 || x.group_best == 1), plans, 0};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int rc = x.dtype == kF32    ? launch_tokens<kF32>(p, s)
                   : x.dtype == kBf16 ? launch_tokens<kBf16>(p, s)
                                      : launch_tokens<kF16>(p, s);
    if (rc != hipSuccess || ids == nullptr) return rc;
    return launch_kernel(make_plan, static_cast<unsigned>(x.experts), kPlanThreads, 0, s, ids, x.tokens * x.top_k,
                         x.experts, x.order, x.offsets);
}

}  // extern "C"

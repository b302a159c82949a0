// The choice of experts: scores, groups, the top_k largest, their gates, and the
// plan (pairs of token and place by expert) that the experts' products run on.
//
// Scores are in fp64: choices are compared with a bias added and in sums of two, and
// two experts whose scores lie next to each other are then still in their order.

#include "i8_device.h"

namespace {

using namespace i8;

constexpr int kWaves = 4;
constexpr double kNone = -__builtin_inf();

struct Route {
    const void* logits;
    long long ld;
    const float* bias;
    int tokens, experts, top_k, score, groups, each, top_groups, group_best, normalize;
    float scale;
    int* chosen;
    float* gates;
    bool by_logit;  // one score by itself is as large as its logit
};

__device__ __forceinline__ double wave_max(double v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v = fmax(v, __shfl_xor(v, d));
    return v;
}
__device__ __forceinline__ double wave_add(double v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    return v;
}

// The largest key of the wave and the lowest place that has it.
__device__ __forceinline__ void wave_first(double& key, int& at) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const double k = __shfl_xor(key, d);
        const int a = __shfl_xor(at, d);
        if (k > key || (k == key && a < at)) key = k, at = a;
    }
}

// A wave takes a token; lane l experts l, l + 64, ...
template <int kType, int kPer>
__global__ __launch_bounds__(kWaves * 64) void route_tokens(const Route p) {
    __shared__ double keys[kWaves][kPer * 64];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const long long token = static_cast<long long>(blockIdx.x) * kWaves + wave;
    if (token >= p.tokens) return;
    double score[kPer], key[kPer];
    bool bad = false;
    double top = kNone;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = lane + 64 * i;
        const float l = e < p.experts ? load_one<kType>(p.logits, token * p.ld + e) : -__builtin_inff();
        bad |= l != l;
        key[i] = l != l ? kNone : static_cast<double>(l);
        top = fmax(top, key[i]);
    }
    bad = __any(bad);
    top = wave_max(top);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        if (p.score == MCHIP_ROUTE_SOFTMAX)
            score[i] = top == kNone ? 0.0 : exp(key[i] - top);  // +inf - inf: no number
        else
            score[i] = 1.0 / (1.0 + exp(-key[i]));
        sum += score[i];
    }
    if (p.score == MCHIP_ROUTE_SOFTMAX) {
        sum = wave_add(sum);
#pragma unroll
        for (int i = 0; i < kPer; ++i) score[i] = sum > 0.0 || sum != sum ? score[i] / sum : 0.0;
    }
    if (!p.by_logit) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int e = lane + 64 * i;
            // An expert that is masked out stays so whatever its bias.
            if (key[i] != kNone) key[i] = score[i] + (p.bias != nullptr && e < p.experts ? static_cast<double>(p.bias[e]) : 0.0);
            if (key[i] != key[i]) key[i] = kNone;
        }
    }
    int place[kPer];  // by it ties are settled: experts of no chosen group come last
#pragma unroll
    for (int i = 0; i < kPer; ++i) place[i] = lane + 64 * i;
    if (p.groups > 1) {
#pragma unroll
        for (int i = 0; i < kPer; ++i) keys[wave][lane + 64 * i] = key[i];
        __builtin_amdgcn_wave_barrier();
        double mine = kNone;
        if (lane < p.groups) {
            double first = kNone, second = kNone;
            for (int i = 0; i < p.each; ++i) {
                const double k = keys[wave][lane * p.each + i];
                if (k > first) second = first, first = k;
                else if (k > second) second = k;
            }
            mine = p.group_best == 2 && p.each > 1 ? first + second : first;
            if (mine != mine) mine = kNone;
        }
        unsigned long long kept = 0;
        int at_mine = lane < p.groups ? lane : 1 << 20;
        for (int g = 0; g < p.top_groups; ++g) {
            double k = mine;
            int at = at_mine;
            wave_first(k, at);
            kept |= 1ull << at;
            if (lane == at) mine = kNone, at_mine = 1 << 21;
        }
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int e = lane + 64 * i;
            if (e >= p.experts || !(kept >> (e / p.each) & 1)) key[i] = kNone, place[i] = e + (1 << 20);
        }
    } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (place[i] >= p.experts) place[i] += 1 << 20;
    }
    int expert = 0;
    double gate = 0.0, total = 0.0;
    for (int j = 0; j < p.top_k; ++j) {
        double k = key[0];
        int at = place[0];
#pragma unroll
        for (int i = 1; i < kPer; ++i)
            if (key[i] > k || (key[i] == k && place[i] < at)) k = key[i], at = place[i];
        wave_first(k, at);
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < kPer; ++i)
            if (at == lane + 64 * i) s = score[i], key[i] = kNone, place[i] = at + (1 << 21);
        s = __shfl(s, at % 64);
        total += s;
        if (lane == j) expert = at, gate = s;
    }
    if (lane >= p.top_k) return;
    if (p.normalize) gate = total != 0.0 ? gate / total : 0.0;
    float g = static_cast<float>(gate * static_cast<double>(p.scale));
    if (bad) g = __builtin_nanf("");
    p.chosen[token * p.top_k + lane] = expert;
    p.gates[token * p.top_k + lane] = g;
}

// A block takes an expert: how many pairs have a lower one is where its slots begin,
// and its own pairs follow in order, each wave a range of them.
__global__ __launch_bounds__(1024) void make_plan(const int* __restrict__ chosen, int pairs, int experts,
                                                  int* __restrict__ order, int* __restrict__ offsets) {
    __shared__ int lower[16], own[16];
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, e = static_cast<int>(blockIdx.x);
    const int share = (pairs + 16 * 64 - 1) / (16 * 64) * 64;
    const int from = min(wave * static_cast<long long>(share), static_cast<long long>(pairs));
    const int to = min(from + static_cast<long long>(share), static_cast<long long>(pairs));
    int below = 0, mine = 0;
    for (int i = from + lane; i < to; i += 64) {
        const int c = chosen[i];
        below += c < e;
        mine += c == e;
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) below += __shfl_xor(below, d), mine += __shfl_xor(mine, d);
    if (lane == 0) lower[wave] = below, own[wave] = mine;
    __syncthreads();
    int at = 0, all = 0;
    for (int w = 0; w < 16; ++w) {
        at += lower[w];
        if (w < wave) at += own[w];
        all += lower[w] + own[w];
    }
    if (threadIdx.x == 0) {
        offsets[e] = at;
        if (e == experts - 1) offsets[experts] = all;
    }
    for (int i = from; i < to; i += 64) {
        const bool is = i + lane < to && chosen[i + lane] == e;
        const unsigned long long here = __ballot(is);
        if (is) order[at + __popcll(here & ((1ull << lane) - 1))] = i + lane;
        at += __popcll(here);
    }
}

template <int kType>
int launch_tokens(const Route& p, hipStream_t stream) {
    const unsigned blocks = static_cast<unsigned>((static_cast<long long>(p.tokens) + kWaves - 1) / kWaves);
    const auto go = [&](auto kernel) { return launch_kernel(kernel, blocks, kWaves * 64, 0, stream, p); };
    if (p.experts <= 64) return go(route_tokens<kType, 1>);
    if (p.experts <= 128) return go(route_tokens<kType, 2>);
    if (p.experts <= 256) return go(route_tokens<kType, 4>);
    return go(route_tokens<kType, 8>);
}

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
    if (!aligned(x.logits, size_of(x.dtype))) return "an address that is no multiple of its element's size";
    if (!aligned(x.bias, 4) || !aligned(x.chosen, 4) || !aligned(x.gates, 4) || !aligned(x.order, 4) || !aligned(x.offsets, 4))
        return "a bias or an output that is not 4-byte aligned";
    return nullptr;
}

}  // namespace

extern "C" {

long long mchip_route_workspace_bytes(int tokens, int experts, int top_k) { return 0; }

int mchip_launch_route(const mchip_route_args* args, void* stream, const char** why) {
    const mchip_route_args& x = *args;
    *why = refusal(x);
    if (*why != nullptr) return hipErrorInvalidValue;
    const Route p{x.logits, x.ld, x.bias, x.tokens, x.experts, x.top_k, x.score, x.groups, x.experts / x.groups,
                  x.top_groups, x.group_best, x.normalize, x.scale, x.chosen, x.gates,
                  x.bias == nullptr && (x.groups == 1 || x.group_best == 1)};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int rc = x.dtype == kF32    ? launch_tokens<kF32>(p, s)
                   : x.dtype == kBf16 ? launch_tokens<kBf16>(p, s)
                                      : launch_tokens<kF16>(p, s);
    if (rc != hipSuccess || x.order == nullptr) return rc;
    return launch_kernel(make_plan, static_cast<unsigned>(x.experts), 1024, 0, s, x.chosen, x.tokens * x.top_k, x.experts,
                         x.order, x.offsets);
}

}  // extern "C"

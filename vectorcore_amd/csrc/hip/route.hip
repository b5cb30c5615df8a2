// The router of a mixture of experts: each row's top_k experts and their
// weights, and the gradient of the weights with respect to the logits.
//
// score_e = softmax(l)_e or 1 / (1 + exp(-l_e)), rank_e = score_e + bias_e; of
// G groups of neighbouring experts the top_groups with the largest sum of
// their two best ranks stay open; the top_k open experts in falling rank order,
// the lower index first among equals; weight_j = score_j / sum of the chosen
// scores (renormalised) or score_j.
//
// One wavefront per row, all in double: choices next to a border between ranks
// are those of the definition.
#include "reduce_common.hpp"
#include "vc_hip_internal.hpp"

#include <string>

namespace vchip {
namespace {

using red::kWave;

constexpr int kWaves = 4;  // rows per workgroup
constexpr int kMaxExperts = 1024, kMaxPicks = 64, kMaxGroups = 64;

__device__ inline uint64_t wave_max_key(uint64_t v) {
    const int lane = red::lane_id();
    const auto step = [&](double other) {
        const uint64_t o = __builtin_bit_cast(uint64_t, other);
        v = o > v ? o : v;
    };
    step(red::partner<0>(__builtin_bit_cast(double, v), lane));
    step(red::partner<1>(__builtin_bit_cast(double, v), lane));
    step(red::partner<2>(__builtin_bit_cast(double, v), lane));
    step(red::partner<3>(__builtin_bit_cast(double, v), lane));
    step(red::partner<4>(__builtin_bit_cast(double, v), lane));
    step(red::partner<5>(__builtin_bit_cast(double, v), lane));
    return v;
}

__device__ inline int wave_min(int v) {
    const int lane = red::lane_id();
    v = min(v, red::partner<0>(v, lane));
    v = min(v, red::partner<1>(v, lane));
    v = min(v, red::partner<2>(v, lane));
    v = min(v, red::partner<3>(v, lane));
    v = min(v, red::partner<4>(v, lane));
    v = min(v, red::partner<5>(v, lane));
    return v;
}

// A number in the order of ranks: NaN above all, -0 like 0; 0 is no rank.
__device__ inline uint64_t rank_key(double rank) {
    if (rank != rank) return ~0ull;
    const uint64_t bits = __builtin_bit_cast(uint64_t, rank + 0.0);
    return bits >> 63 ? ~bits : bits | (1ull << 63);
}

template <int NV>
__device__ inline void row_scores(const float* __restrict__ row, int experts, int lane, bool sigmoid, double (&s)[NV]) {
    if (sigmoid) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = lane + kWave * i;
            s[i] = e < experts ? 1.0 / (1.0 + exp(-double(row[e]))) : 0.0;
        }
        return;
    }
    float top = -__builtin_huge_valf();
    float l[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int e = lane + kWave * i;
        l[i] = e < experts ? row[e] : -__builtin_huge_valf();
        top = l[i] > top ? l[i] : top;
    }
    top = fmaxf(top, red::partner<0>(top, lane));
    top = fmaxf(top, red::partner<1>(top, lane));
    top = fmaxf(top, red::partner<2>(top, lane));
    top = fmaxf(top, red::partner<3>(top, lane));
    top = fmaxf(top, red::partner<4>(top, lane));
    top = fmaxf(top, red::partner<5>(top, lane));
    double total = 0.0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        s[i] = lane + kWave * i < experts ? exp(double(l[i]) - double(top)) : 0.0;
        total += s[i];
    }
    total = red::wave_sum(total);
#pragma unroll
    for (int i = 0; i < NV; ++i) s[i] /= total;
}

template <int NV>
__global__ __launch_bounds__(kWave* kWaves) void route_kernel(const float* __restrict__ logits, const float* __restrict__ bias,
                                                             size_t tokens, int experts, int top_k, bool sigmoid, int groups,
                                                             int top_groups, bool renormalise, float* __restrict__ weights,
                                                             float* __restrict__ chosen) {
    __shared__ double ranks[kWaves][kWave * NV];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const size_t t = size_t(blockIdx.x) * kWaves + wave;
    const bool live = t < tokens;  // uniform in the wavefront
    double s[NV];
    uint64_t key[NV];
    if (live) {
        row_scores<NV>(logits + t * experts, experts, lane, sigmoid, s);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = lane + kWave * i;
            const double rank = s[i] + (bias && e < experts ? double(bias[e]) : 0.0);
            ranks[wave][e] = rank;
            key[i] = e < experts ? rank_key(rank) : 0;
        }
    }
    __syncthreads();
    if (!live) return;
    if (groups > 1) {
        const int size = experts / groups;
        uint64_t strength = 0;
        if (lane < groups) {
            double best = -__builtin_huge_val(), second = -__builtin_huge_val();
            bool nan = false;
            for (int i = 0; i < size; ++i) {
                const double r = ranks[wave][lane * size + i];
                nan |= r != r;
                if (r > best) {
                    second = best;
                    best = r;
                } else if (r > second) {
                    second = r;
                }
            }
            strength = rank_key(nan ? __builtin_nan("") : size > 1 ? best + second : best);
        }
        uint64_t open = 0;
        for (int j = 0; j < top_groups; ++j) {
            const uint64_t best = wave_max_key(strength);
            const int g = wave_min(strength == best && lane < groups ? lane : kWave);
            open |= 1ull << g;
            if (lane == g) strength = 0;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = lane + kWave * i;
            if (e < experts && !(open >> (e / size) & 1)) key[i] = 0;
        }
    }
    int mine = 0;
    double score = 0.0, total = 0.0;
    for (int j = 0; j < top_k; ++j) {
        uint64_t best = key[0];
#pragma unroll
        for (int i = 1; i < NV; ++i) best = key[i] > best ? key[i] : best;
        best = wave_max_key(best);
        int at = 1 << 30;
#pragma unroll
        for (int i = NV - 1; i >= 0; --i)
            if (key[i] == best) at = lane + kWave * i;
        at = wave_min(at);
        double picked = 0.0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (at == lane + kWave * i) {
                key[i] = 0;
                picked = s[i];
            }
        picked = __shfl(picked, at % kWave);
        total += picked;
        if (lane == j) {
            mine = at;
            score = picked;
        }
    }
    if (lane < top_k) {
        weights[t * top_k + lane] = float(renormalise ? score / total : score);
        chosen[t * top_k + lane] = float(mine);
    }
}

template <int NV>
__global__ __launch_bounds__(kWave* kWaves) void route_backward_kernel(const float* __restrict__ logits,
                                                                      const float* __restrict__ chosen,
                                                                      const float* __restrict__ grad, size_t tokens,
                                                                      int experts, int top_k, bool sigmoid,
                                                                      bool renormalise, float* __restrict__ out) {
    const int lane = threadIdx.x % kWave;
    const size_t t = size_t(blockIdx.x) * kWaves + threadIdx.x / kWave;
    if (t >= tokens) return;
    double s[NV], d[NV];
    row_scores<NV>(logits + t * experts, experts, lane, sigmoid, s);
#pragma unroll
    for (int i = 0; i < NV; ++i) d[i] = 0.0;
    const int at = lane < top_k ? int(chosen[t * top_k + lane]) : 0;
    const double g = lane < top_k ? double(grad[t * top_k + lane]) : 0.0;
    double total = 0.0, dot = 0.0;  // of the chosen scores, of their products with the gradients
    double p = 0.0;
    for (int j = 0; j < top_k; ++j) {
        const int e = __shfl(at, j);
        double picked = 0.0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (e == lane + kWave * i) picked = s[i];
        picked = __shfl(picked, e % kWave);
        total += picked;
        dot += picked * __shfl(g, j);
        if (lane == j) p = picked;
    }
    const double gp = renormalise ? (g - dot / total) / total : g;  // gradient of the chosen score
    const double mean = renormalise ? 0.0 : dot;  // sum of d * score: the renormalised gradients cancel
    for (int j = 0; j < top_k; ++j) {
        const int e = __shfl(at, j);
        const double v = __shfl(gp, j);
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (e == lane + kWave * i) d[i] = v;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int e = lane + kWave * i;
        if (e < experts) out[t * experts + e] = float(sigmoid ? d[i] * s[i] * (1.0 - s[i]) : s[i] * (d[i] - mean));
    }
}

void check_route(const char* name, size_t tokens, size_t experts, size_t top_k, int score) {
    if (experts == 0 || experts > kMaxExperts)
        fail(VC_HIP_ERR_INVALID_ARGUMENT, std::string(name) + ": between 1 and 1024 experts are supported, got " + std::to_string(experts));
    if (top_k == 0 || top_k > experts || top_k > kMaxPicks)
        fail(VC_HIP_ERR_INVALID_ARGUMENT, std::string(name) + ": top_k must be between 1 and the experts (at most 64), got " +
                                              std::to_string(top_k) + " of " + std::to_string(experts));
    if (score != VC_HIP_SCORE_SOFTMAX && score != VC_HIP_SCORE_SIGMOID)
        fail(VC_HIP_ERR_INVALID_ARGUMENT, std::string(name) + ": unknown score");
    if (tokens > (size_t(1) << 31)) fail(VC_HIP_ERR_INVALID_ARGUMENT, std::string(name) + ": too many tokens");
}

// f(std::integral_constant<int, NV>) with NV values per lane for a row of experts.
template <typename F>
void with_row_width(size_t experts, F&& f) {
    if (experts <= 64) f(std::integral_constant<int, 1>());
    else if (experts <= 128) f(std::integral_constant<int, 2>());
    else if (experts <= 256) f(std::integral_constant<int, 4>());
    else if (experts <= 512) f(std::integral_constant<int, 8>());
    else f(std::integral_constant<int, 16>());
}

}  // namespace
}  // namespace vchip

using namespace vchip;

extern "C" {

int vc_hip_route_forward(const float* logits, const float* bias, size_t tokens, size_t experts, size_t top_k, int score,
                         size_t groups, size_t top_groups, int renormalise, float* weights, float* chosen) {
    return guard([&] {
        Device& d = require_device();
        check_route("route", tokens, experts, top_k, score);
        if (groups == 0 || groups > kMaxGroups || experts % groups != 0 || top_groups == 0 || top_groups > groups ||
            experts / groups * top_groups < top_k)
            fail(VC_HIP_ERR_INVALID_ARGUMENT, "route: groups (at most 64) must divide the experts and the open groups hold top_k");
        if (tokens == 0) return;
        if (!logits || !weights || !chosen) fail(VC_HIP_ERR_INVALID_ARGUMENT, "route: null pointer");
        const double n = double(tokens) * experts, picks = double(tokens) * top_k;
        Profiled p("route", 6.0 * n, 4.0 * (n + 2.0 * picks));
        with_row_width(experts, [&](auto nv) {
            launch(route_kernel<nv()>, dim3(unsigned((tokens + kWaves - 1) / kWaves)), dim3(kWave * kWaves), 0, d.stream, logits,
                   bias, tokens, int(experts), int(top_k), score == VC_HIP_SCORE_SIGMOID, int(groups), int(top_groups),
                   renormalise != 0, weights, chosen);
        });
        after_launch("route");
        p.done();
    });
}

int vc_hip_route_backward(const float* logits, const float* chosen, const float* grad_weights, size_t tokens,
                          size_t experts, size_t top_k, int score, int renormalise, float* grad_logits) {
    return guard([&] {
        Device& d = require_device();
        check_route("route_backward", tokens, experts, top_k, score);
        if (tokens == 0) return;
        if (!logits || !chosen || !grad_weights || !grad_logits)
            fail(VC_HIP_ERR_INVALID_ARGUMENT, "route_backward: null pointer");
        const double n = double(tokens) * experts, picks = double(tokens) * top_k;
        Profiled p("route_backward", 6.0 * n, 4.0 * (2.0 * n + 2.0 * picks));
        with_row_width(experts, [&](auto nv) {
            launch(route_backward_kernel<nv()>, dim3(unsigned((tokens + kWaves - 1) / kWaves)), dim3(kWave * kWaves), 0,
                   d.stream, logits, chosen, grad_weights, tokens, int(experts), int(top_k), score == VC_HIP_SCORE_SIGMOID,
                   renormalise != 0, grad_logits);
        });
        after_launch("route_backward");
        p.done();
    });
}

}  // extern "C"

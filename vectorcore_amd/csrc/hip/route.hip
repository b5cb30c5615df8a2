// The router of a mixture of experts: each row's top_k experts and their
// weights, and the gradient of the weights with respect to the logits.
//
// score_e = softmax(l)_e or 1 / (1 + exp(-l_e)), rank_e = score_e + bias_e; of
// G groups of neighbouring experts the top_groups with the largest sum of
// their two best ranks stay open; the top_k open experts in falling rank order,
// the lower index first among equals; weight_j = score_j / sum of the chosen
// scores (renormalised) or score_j.
//
// Choices next to a border between ranks are those of the definition: where a
// row's 32-bit ranks cannot tell two candidates apart, its whole wavefront ranks
// it again in double, weights included. So it does where a chosen score is below
// 2^-100, which float32 would soon not hold. A bias far above the scores, as one
// that masks an expert, makes that every row, as 32-bit ranks next to it have no
// digits of the scores (65536 rows of 256 experts: 200 us with one bias of -1e4).
//
// Many rows would be bound by HBM (the logits are read, the gradient is written)
// and are, forward, by vector instructions still: sixteen lanes share a row, so
// four rows share each step of a search or sum across lanes. 65536 rows of 256
// experts: 50.9 us forward (1.4 TB/s), 18.1 us backward (67 MB written, 3.7 TB/s);
// 4096 rows of 64: 4.1 and 3.9 us, a launch's latency.
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

struct RouteArgs {
    const float *logits, *bias;
    int64_t tokens;
    int experts, top_k, groups, top_groups;
    bool sigmoid, renormalise;
    float *weights, *chosen;
};

// LDS that a wavefront has written is read by its other lanes.
__device__ inline void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Row t by a whole wavefront, in double. ranks: 64 NV of LDS.
template <int NV>
__device__ void route_row(const RouteArgs& p, int64_t t, double* ranks) {
    const int lane = threadIdx.x % kWave, experts = p.experts;
    double s[NV];
    uint64_t key[NV];
    row_scores<NV>(p.logits + t * experts, experts, lane, p.sigmoid, s);
    wave_fence();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int e = lane + kWave * i;
        const double rank = s[i] + (p.bias && e < experts ? double(p.bias[e]) : 0.0);
        ranks[e] = rank;
        key[i] = e < experts ? rank_key(rank) : 0;
    }
    wave_fence();
    if (p.groups > 1) {
        const int size = experts / p.groups;
        uint64_t strength = 0;
        if (lane < p.groups) {
            double best = -__builtin_huge_val(), second = -__builtin_huge_val();
            bool nan = false;
            for (int i = 0; i < size; ++i) {
                const double r = ranks[lane * size + i];
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
        for (int j = 0; j < p.top_groups; ++j) {
            const uint64_t best = wave_max_key(strength);
            const int g = wave_min(strength == best && lane < p.groups ? lane : kWave);
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
    for (int j = 0; j < p.top_k; ++j) {
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
    if (lane < p.top_k) {
        p.weights[t * p.top_k + lane] = float(p.renormalise ? score / total : score);
        p.chosen[t * p.top_k + lane] = float(mine);
    }
}

// A wavefront per row.
template <int NV>
__global__ __launch_bounds__(kWave* kWaves) void route_wide_kernel(RouteArgs p) {
    __shared__ double ranks[kWaves][kWave * NV];
    const int64_t t = block_id() * kWaves + threadIdx.x / kWave;
    if (t < p.tokens) route_row<NV>(p, t, ranks[threadIdx.x / kWave]);
}

// ---- sixteen lanes a row --------------------------------------------------------------
// Up to 256 experts, 16 picks and 16 groups. Lane l of a row holds experts
// 64 j + 4 l .. + 3.

constexpr int kLanes = 16, kRows = kWave / kLanes;  // of a row; rows of a wavefront

template <class F>
__device__ inline float row_all(float v, F&& f) {
    const int lane = red::lane_id();
    v = f(v, red::partner<0>(v, lane));
    v = f(v, red::partner<1>(v, lane));
    v = f(v, red::partner<2>(v, lane));
    return f(v, red::partner<3>(v, lane));
}
__device__ inline float row_sum(float v) {
    return row_all(v, [](float a, float b) { return a + b; });
}
__device__ inline float row_max(float v) {
    return row_all(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ inline uint32_t row_max_key(uint32_t v) {
    const int lane = red::lane_id();
    v = max(v, red::partner<0>(v, lane));
    v = max(v, red::partner<1>(v, lane));
    v = max(v, red::partner<2>(v, lane));
    return max(v, red::partner<3>(v, lane));
}
__device__ inline int row_min(int v) {
    const int lane = red::lane_id();
    v = min(v, red::partner<0>(v, lane));
    v = min(v, red::partner<1>(v, lane));
    v = min(v, red::partner<2>(v, lane));
    return min(v, red::partner<3>(v, lane));
}

// A number in its order (not NaN; -0 like 0), never 0.
__device__ inline uint32_t order_key(float v) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, v + 0.0f);
    return bits >> 31 ? ~bits : bits | 0x80000000u;
}
__device__ inline float order_value(uint32_t key) {
    return __builtin_bit_cast(float, key >> 31 ? key & 0x7FFFFFFFu : ~key);
}

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

// The row's logits; none past its end.
template <int NV>
__device__ inline void row_logits(const float* __restrict__ row, int experts, int l, float (&v)[NV]) {
#pragma unroll
    for (int j = 0; j < NV / 4; ++j) {
        const int e = 64 * j + 4 * l;
        if (e + 4 <= experts) {
            const f4u x = *reinterpret_cast<const f4u*>(row + e);
#pragma unroll
            for (int c = 0; c < 4; ++c) v[4 * j + c] = x[c];
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c) v[4 * j + c] = e + c < experts ? row[e + c] : -__builtin_huge_valf();
        }
    }
}

// exp(a - b), with what the difference's rounding leaves to first order: far
// below the top that would be most of the error.
__device__ inline float exp_difference(float a, float b) {
    const float d = a - b, back = d - a, rest = (a - (d - back)) - (b + back), e = expf(d);
    return fabsf(rest) < 1.0f ? fmaf(e, rest, e) : e;  // no rest of infinities
}
__device__ inline float score_of(float logit, bool sigmoid, float top, float inverse) {
    return sigmoid ? 1.0f / (1.0f + expf(-logit)) : exp_difference(logit, top) * inverse;
}

// The two largest of a set, joined with those of another set.
__device__ inline void join_best(float& best, float& second, float other, float other_second) {
    second = fmaxf(fminf(best, other), fmaxf(second, other_second));
    best = fmaxf(best, other);
}
template <int Step, int N>
__device__ inline void join_partners(float (&best)[N], float (&second)[N], int lane) {
#pragma unroll
    for (int j = 0; j < N; ++j)
        join_best(best[j], second[j], red::partner<Step>(best[j], lane), red::partner<Step>(second[j], lane));
}

// Falling order, by odd-even merges.
template <int N>
__device__ inline void sort_keys(uint32_t (&key)[N]) {
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                        const uint32_t x = key[i + j], y = key[i + j + k];
                        key[i + j] = max(x, y);
                        key[i + j + k] = min(x, y);
                    }
}

// 1 / (1 + exp(-x)) within 2^-21 of itself, or 2^-115 where x < -80: exp2(t)
// with t = -x / ln 2, and what t's rounding leaves to first order; 1 / ln 2 in
// two terms, as in Cody and Waite's reduction (Software Manual for the Elementary
// Functions, 1980).
__device__ inline float quick_sigmoid(float x) {
    const float log2e = 0x1.715476p+0f, rest = 0x1.4ae0cp-26f, ln2 = 0x1.62e43p-1f;
    x = fmaxf(x, -80.0f);
    const float t = x * -log2e, low = fmaf(x, -rest, fmaf(x, -log2e, -t)), e = __builtin_amdgcn_exp2f(t);
    return __builtin_amdgcn_rcpf(1.0f + fmaf(e, low * ln2, e));
}

// Exact: without a bias and groups the logits' own order is that of the ranks,
// as long as doubles tell the scores apart. Otherwise the 32-bit ranks decide
// where they are further apart than their errors: with M the largest score and
// bias, a score is within 2^-21 of itself, a rank (at most 2 M) within 2^-20.6 M,
// the difference of two within 2^-19.6 M and that of two groups' sums within 2^-18 M.
//
// A lane's ranks become fixed point numbers in units of 2^-26 of M's next power of
// two, above four bits of the place in the lane: they differ, and are sorted once;
// a pick is then the largest of sixteen first keys, and its lane moves up. (65536
// rows of 256 experts, 8 of them in 4 of 8 groups: 50.6 us; 75.2 with every pick
// looked for among all keys and each group's ranks read by one lane.)
template <int NV, bool Exact>
__global__ __launch_bounds__(kWave* kWaves) void route_kernel(RouteArgs p) {
    __shared__ double scratch[kWaves][kWave * NV / 2];  // floats of four rows, or doubles of one
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, l = lane % kLanes, r = lane / kLanes;
    const int64_t first = (block_id() * kWaves + wave) * kRows;
    if (first >= p.tokens) return;  // uniform in the wavefront
    const int64_t t = min(first + r, p.tokens - 1);
    const int experts = p.experts;
    const float* const row = p.logits + t * experts;
    float v[NV];
    row_logits<NV>(row, experts, l, v);
    float top = -__builtin_huge_valf(), inverse = 1.0f;
    bool again = false;  // this row in double
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        top = fmaxf(top, v[i]);
        again |= v[i] != v[i];
    }
    top = row_max(top);
    again |= !(fabsf(top) < __builtin_huge_valf());
    if (!p.sigmoid) {
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) total += expf(v[i] - top);
        inverse = 1.0f / row_sum(total);
    }
    uint32_t key[NV];
    if constexpr (Exact) {
#pragma unroll
        for (int i = 0; i < NV; ++i) key[i] = 64 * (i / 4) + 4 * l + i % 4 < experts ? order_key(v[i]) : 0;
    } else {
        float most = 0.0f, rank[NV];
        if (p.bias) {
            row_logits<NV>(p.bias, experts, l, rank);
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) rank[i] = 0.0f;
        }
        // The scores take the logits' place.
        if (p.sigmoid) {
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] = quick_sigmoid(v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] = expf(v[i] - top) * inverse;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const bool there = 64 * (i / 4) + 4 * l + i % 4 < experts;
            const float score = v[i];
            if (there) most = fmaxf(most, fmaxf(score, fabsf(rank[i])));
            rank[i] = there ? score + rank[i] : -__builtin_huge_valf();
            again |= rank[i] != rank[i];
        }
        most = row_max(most);
        again |= !(most > 0x1p-80f && most < __builtin_huge_valf());
        const int unit = 26 - __builtin_amdgcn_frexp_expf(most);  // most < 2^(26 - unit)
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int fixed = int(__builtin_amdgcn_ldexpf(rank[i], unit)) + (1 << 27);
            key[i] = 64 * (i / 4) + 4 * l + i % 4 < experts ? uint32_t(fixed) << 4 | i : 0;
        }
        if (p.groups > 1) {
            const int size = experts / p.groups;
            const bool aligned = size >= 4 && size <= 64 && (size & (size - 1)) == 0;  // size / 4 lanes share a group
            const int shift = 31 - __builtin_clz(size);
            float* const ranks = reinterpret_cast<float*>(scratch[wave]) + r * (kWave * NV / 4);
            float strength = 0.0f;
            if (aligned) {
                float best[NV / 4], second[NV / 4];
#pragma unroll
                for (int j = 0; j < NV / 4; ++j) {
                    float other = fmaxf(rank[4 * j + 2], rank[4 * j + 3]);
                    best[j] = fmaxf(rank[4 * j], rank[4 * j + 1]);
                    second[j] = fminf(rank[4 * j], rank[4 * j + 1]);
                    join_best(best[j], second[j], other, fminf(rank[4 * j + 2], rank[4 * j + 3]));
                }
                if (size > 4) join_partners<0>(best, second, lane);
                if (size > 8) join_partners<1>(best, second, lane);
                if (size > 16) join_partners<2>(best, second, lane);
                if (size > 32) join_partners<3>(best, second, lane);
                wave_fence();
#pragma unroll
                for (int j = 0; j < NV / 4; ++j) {
                    const int e = 64 * j + 4 * l;
                    if (e < experts && (e & (size - 1)) == 0) ranks[e >> shift] = best[j] + second[j];
                }
                wave_fence();
                if (l < p.groups) strength = ranks[l];
            } else {
                wave_fence();
#pragma unroll
                for (int i = 0; i < NV; ++i) ranks[64 * (i / 4) + 4 * l + i % 4] = rank[i];
                wave_fence();
                float best = -__builtin_huge_valf(), second = best;
                if (l < p.groups) {
                    int at = l % size;  // each lane begins elsewhere: other banks
                    for (int i = 0; i < size; ++i) {
                        const float next = ranks[l * size + at];
                        second = fmaxf(second, fminf(best, next));
                        best = fmaxf(best, next);
                        at = at + 1 == size ? 0 : at + 1;
                    }
                }
                strength = size > 1 ? best + second : best;
                wave_fence();
                if (l < p.groups) ranks[l] = strength;
                wave_fence();
            }
            const float margin = most * 0x1p-18f;
            int before = 0, perhaps = -1;  // the groups that are stronger, and that may be (not itself)
            for (int g = 0; g < p.groups; ++g) {
                const float ahead = ranks[g] - strength;
                before += ahead > margin;
                perhaps += !(ahead < -margin);
            }
            again |= l < p.groups && before < p.top_groups && perhaps >= p.top_groups;
            const uint32_t open = uint32_t(__ballot(l < p.groups && before < p.top_groups) >> (kLanes * r));
            if (aligned) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    if (!(open >> ((64 * (i / 4) + 4 * l) >> shift) & 1)) key[i] = 0;
            } else {
                const uint32_t inverse_size = (65536 + size - 1) / size;  // e / size for e < 256
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const uint32_t e = 64 * (i / 4) + 4 * l + i % 4;
                    if (!(open >> (e * inverse_size >> 16) & 1)) key[i] = 0;
                }
            }
        }
        sort_keys(key);
    }
    int mine = 0;
    uint32_t previous = 0;
    bool tied = false;  // the candidate after the last pick with that pick
    // Of two logits in falling order: may doubles not tell their scores apart?
    const auto near = [&](float ahead, float value) {
        const float gap = ahead - value;
        return gap > 0.0f && !(gap * (p.sigmoid ? expf(-fmaxf(value, 0.0f)) : 1.0f) > 1e-12f);
    };
    for (int j = 0; j <= p.top_k; ++j) {
        uint32_t best = key[0];
        if constexpr (Exact) {
#pragma unroll
            for (int i = 1; i < NV; ++i) best = max(best, key[i]);
        }
        best = row_max_key(best);
        // The candidate after the last pick is only compared with it.
        if constexpr (Exact) {
            const float value = order_value(best);
            if (j > 0 && best != 0) {
                again |= near(order_value(previous), value);
                tied = best == previous;
                again |= (p.sigmoid ? value : value - top) < -600.0f && j < p.top_k;
            }
        } else {
            again |= j > 0 && best != 0 && (previous >> 4) - (best >> 4) <= 128;  // of 2^26: 2^-19
        }
        previous = best;
        if (j == p.top_k) break;
        int at = 1 << 30;
        if constexpr (Exact) {
#pragma unroll
            for (int i = NV - 1; i >= 0; --i)
                if (key[i] == best) at = 64 * (i / 4) + 4 * l + i % 4;
            at = row_min(at);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (at == 64 * (i / 4) + 4 * l + i % 4) key[i] = 0;
        } else {
            const bool won = key[0] == best;
            const uint32_t winners = uint32_t(__ballot(won) >> (kLanes * r)) & 0xFFFF;
            const int i = best & 15;
            again |= (winners & (winners - 1)) != 0;  // equal keys of two lanes
            at = 64 * (i / 4) + 4 * (__ffs(winners) - 1) + i % 4;
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                const uint32_t stays = key[n], next = n + 1 < NV ? key[n + 1] : 0u;
                key[n] = won ? next : stays;
            }
        }
        if (l == j) mine = at;
    }
    if constexpr (Exact) {
        if (__ballot(tied)) {  // the next logit below the tied ones may have their score, and a lower index
            uint32_t below = 0;
#pragma unroll
            for (int i = 0; i < NV; ++i) below = max(below, key[i] < previous ? key[i] : 0);
            below = row_max_key(below);
            again |= tied && below != 0 && near(order_value(previous), order_value(below));
        }
    }
    const bool picked = l < p.top_k;
    const float score = picked ? score_of(row[min(mine, experts - 1)], p.sigmoid, top, inverse) : 0.0f;
    const float total = row_sum(score);
    again |= picked && !(score > 0x1p-100f);  // the least scores lose bits, and their quotients with them
    if (picked && first + r < p.tokens) {
        p.weights[t * p.top_k + l] = p.renormalise ? score / total : score;
        p.chosen[t * p.top_k + l] = float(mine);
    }
    uint64_t rows = __ballot(again);
    for (int i = 0; i < kRows; ++i)
        if (rows >> (kLanes * i) & 0xFFFF && first + i < p.tokens) route_row<(NV + 3) / 4>(p, first + i, scratch[wave]);
}

// The expert of a saved pick, or one of them where another library has written
// something else there since (before the conversion, which knows no NaN).
__device__ inline int expert_of(float chosen, int experts) { return int(fminf(fmaxf(chosen, 0.0f), float(experts - 1))); }

// Up to 256 experts and 64 picks. Renormalised weights and sigmoid scores leave
// the other logits no gradient, so only the chosen ones are read:
//   softmax: w_j (g_j - sum g w), w over the chosen alone;
//   sigmoid: w_j (1 - p_j) (g_j - sum g w), or p_j (1 - p_j) g_j;
// Dense (a softmax as it is): s_e (g_e - sum g p) for every expert. The weights
// w are quotients of scores over a common factor that leaves the largest near
// one, where the scores themselves may vanish, and 1 - p is the sigmoid of -l,
// which has all its bits next to p = 1.
template <int NV, bool Dense>
__global__ __launch_bounds__(kWave* kWaves) void route_gradient_kernel(const float* __restrict__ logits,
                                                                      const float* __restrict__ chosen,
                                                                      const float* __restrict__ grad, int64_t tokens,
                                                                      int experts, int top_k, bool sigmoid, bool renormalise,
                                                                      float* __restrict__ out) {
    __shared__ __align__(16) float lds[kWaves][kRows][kLanes * NV];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, l = lane % kLanes, r = lane / kLanes;
    const int64_t t = (block_id() * kWaves + wave) * kRows + r;
    const bool live = t < tokens;
    const float* const row = logits + (live ? t : 0) * experts;
    const float* const picks = chosen + (live ? t : 0) * top_k;
    const float* const g = grad + (live ? t : 0) * top_k;
    float* const place = lds[wave][r];
    f4u zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < NV / 4; ++j) *reinterpret_cast<f4u*>(place + 64 * j + 4 * l) = zero;
    float v[NV], top = -__builtin_huge_valf(), inverse = 1.0f;
    if constexpr (Dense) {
        row_logits<NV>(row, experts, l, v);
#pragma unroll
        for (int i = 0; i < NV; ++i) top = fmaxf(top, v[i]);
        top = row_max(top);
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            v[i] = expf(v[i] - top);
            total += v[i];
        }
        inverse = 1.0f / row_sum(total);
    } else if (sigmoid && !renormalise) {
        top = 0.0f;
    } else {
        for (int j = l; j < top_k; j += kLanes) top = fmaxf(top, row[expert_of(picks[j], experts)]);
        top = row_max(top);
        if (sigmoid) top = fminf(top, 0.0f);
    }
    // sigmoid(x) = exp(min(x, 0)) / (1 + exp(-|x|)), over exp(top).
    const auto score = [&](float x) {
        return sigmoid ? exp_difference(fminf(x, 0.0f), top) / (1.0f + expf(-fabsf(x))) : score_of(x, false, top, inverse);
    };
    float total = 0.0f, dot = 0.0f;
    for (int j = l; j < top_k; j += kLanes) {
        const float p = score(row[expert_of(picks[j], experts)]);
        total += p;
        dot += p * g[j];
    }
    total = row_sum(total);
    dot = row_sum(dot);
    wave_fence();
    for (int j = l; j < top_k; j += kLanes) {
        const int e = expert_of(picks[j], experts);
        const float x = row[e], p = score(x);
        float d = Dense || !renormalise ? g[j] : top_k == 1 ? 0.0f : g[j] - dot / total;  // one weight alone is always 1
        if (!Dense) d *= renormalise ? p / total : p;
        if (sigmoid) d *= score_of(-x, true, 0.0f, 1.0f);
        place[e] = d;
    }
    wave_fence();
    if (!live) return;
    float* const to = out + t * experts;
#pragma unroll
    for (int j = 0; j < NV / 4; ++j) {
        const int e = 64 * j + 4 * l;
        f4u d = *reinterpret_cast<const f4u*>(place + e);
        if constexpr (Dense) {
#pragma unroll
            for (int c = 0; c < 4; ++c) d[c] = v[4 * j + c] * inverse * (d[c] - dot);
        }
        if (e + 4 <= experts) {
            *reinterpret_cast<f4u*>(to + e) = d;
        } else {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (e + c < experts) to[e + c] = d[c];
        }
    }
}

template <int NV>
__global__ __launch_bounds__(kWave* kWaves) void route_gradient_wide_kernel(const float* __restrict__ logits,
                                                                      const float* __restrict__ chosen,
                                                                      const float* __restrict__ grad, size_t tokens,
                                                                      int experts, int top_k, bool sigmoid,
                                                                      bool renormalise, float* __restrict__ out) {
    const int lane = threadIdx.x % kWave;
    const size_t t = size_t(block_id()) * kWaves + threadIdx.x / kWave;
    if (t >= tokens) return;
    double s[NV], d[NV];
    row_scores<NV>(logits + t * experts, experts, lane, sigmoid, s);
#pragma unroll
    for (int i = 0; i < NV; ++i) d[i] = 0.0;
    const int at = lane < top_k ? expert_of(chosen[t * top_k + lane], experts) : 0;
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
        if (e < experts)
            out[t * experts + e] =
                float(sigmoid ? d[i] * s[i] / (1.0 + exp(double(logits[t * experts + e]))) : s[i] * (d[i] - mean));
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

// f(std::integral_constant<int, NV>) with NV values per lane for a row of experts, of 64 or of 16 lanes.
template <typename F>
void with_wide_rows(size_t experts, F&& f) {
    if (experts <= 64) f(std::integral_constant<int, 1>());
    else if (experts <= 128) f(std::integral_constant<int, 2>());
    else if (experts <= 256) f(std::integral_constant<int, 4>());
    else if (experts <= 512) f(std::integral_constant<int, 8>());
    else f(std::integral_constant<int, 16>());
}
template <typename F>
void with_rows(size_t experts, F&& f) {
    if (experts <= 64) f(std::integral_constant<int, 4>());
    else if (experts <= 128) f(std::integral_constant<int, 8>());
    else f(std::integral_constant<int, 16>());
}

dim3 row_grid(size_t tokens, int rows) { return grid_2d((tokens + rows - 1) / rows); }

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
        const RouteArgs args{logits, bias, int64_t(tokens), int(experts), int(top_k), int(groups), int(top_groups),
                             score == VC_HIP_SCORE_SIGMOID, renormalise != 0, weights, chosen};
        const dim3 block(kWave * kWaves);
        if (experts > 256 || top_k > size_t(kLanes) || groups > size_t(kLanes))
            with_wide_rows(experts, [&](auto nv) { launch(route_wide_kernel<nv()>, row_grid(tokens, kWaves), block, 0, d.stream, args); });
        else
            with_rows(experts, [&](auto nv) {
                const dim3 grid = row_grid(tokens, kWaves * kRows);
                if (!bias && groups == 1) launch(route_kernel<nv(), true>, grid, block, 0, d.stream, args);
                else launch(route_kernel<nv(), false>, grid, block, 0, d.stream, args);
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
        const bool sigmoid = score == VC_HIP_SCORE_SIGMOID, renorm = renormalise != 0;
        const dim3 block(kWave * kWaves);
        if (experts > 256)
            with_wide_rows(experts, [&](auto nv) {
                launch(route_gradient_wide_kernel<nv()>, row_grid(tokens, kWaves), block, 0, d.stream, logits, chosen,
                       grad_weights, tokens, int(experts), int(top_k), sigmoid, renorm, grad_logits);
            });
        else
            with_rows(experts, [&](auto nv) {
                const dim3 grid = row_grid(tokens, kWaves * kRows);
                if (!sigmoid && !renorm)
                    launch(route_gradient_kernel<nv(), true>, grid, block, 0, d.stream, logits, chosen, grad_weights,
                           int64_t(tokens), int(experts), int(top_k), sigmoid, renorm, grad_logits);
                else
                    launch(route_gradient_kernel<nv(), false>, grid, block, 0, d.stream, logits, chosen, grad_weights,
                           int64_t(tokens), int(experts), int(top_k), sigmoid, renorm, grad_logits);
            });
        after_launch("route_backward");
        p.done();
    });
}

}  // extern "C"

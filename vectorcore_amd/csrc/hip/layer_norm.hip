// Layer normalisation over the last axis of [rows, width], and its gradients.
//
// With m and v a row's mean and variance, r = 1 / sqrt(v + eps) and
// h = (x - m) r:
//   y  = h w + b
//   dx = r (d - mean(d) - h mean(d h)),  d = dy w
//   dw = the sum over rows of dy h,      db = the sum over rows of dy.
//
// Bound by HBM: the forward reads x and writes y, the backward reads x and dy
// and writes dx. So a row stays in registers between its statistics and what is
// made of it, and the backward collects dw and db on the way: a thread holds the
// same columns of every row of its workgroup, each workgroup leaves one partial
// row of either sum, and a second launch adds those in a fixed order, in double.
// The thread's own sums are float32, of at most 64 rows: of many more of one sign
// the late ones would lose their bits (1e-5 of a sum of 2^21 equal ones).
//
// A row's mean is kept as a float and what the float is off by: x - m would
// otherwise lose the bits of a row that lies far from zero, and is made of a sum in
// double, which also holds any row's. The squares' sum is float32, of at most 16
// values a lane, then a tree; rows whose largest value is past 2^50 or below 2^-40
// are scaled by a power of two for it, so rows of any length have the cpu's range.
// (Both sums in double took 53 us of 8192 rows of 4096, for 49.)
//
// Measured: 8192 rows of 4096, forward 49 us (5.5 TB/s), backward 77 us (5.2) and
// 8 us for the partial rows; 262144 rows of 64 without a weight 24 and 33 us (5.7
// and 6.1; a copy of 1 GiB reaches 5.1, these partly stay in the last cache);
// 999 rows of 515 4.6 us, and 5.7 and 5.4; one row of 4096 3.7 us. 4000 rows of
// 10000 67 us, and 106 and 26; 2048 of 16384 59 us, and 87 and 83 (x and dy again
// for the columns) and 7; 1024 of 32768 115 us, and 116, 72 and 10.
#include "reduce_common.hpp"
#include "vc_hip_internal.hpp"

#include <algorithm>
#include <cmath>
#include <string>

namespace vchip {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
// 16 bytes on any 4-byte boundary, as rows of any length start.
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

// What the forward leaves of a row: x factor - mean - rest is exact to a rounding, times scale it is h; scale factor is r. The
// factor is one, or a power of two that brings the row near one.
struct alignas(16) RowStats {
    float mean, rest, scale, factor;
    __device__ inline float normed(float x) const { return (x * factor - mean - rest) * scale; }
};
// The power of two for a row of which `most`, of the largest magnitude and the root of eps, is the larger.
__device__ inline float factor_of(float most) {
    if (most >= 0x1p-40f && most <= 0x1p50f) return 1.0f;
    return __builtin_amdgcn_ldexpf(1.0f, -min(max(__builtin_amdgcn_frexp_expf(most), -100), 120));
}
// From the mean, and the variance of the row times factor.
__device__ inline RowStats stats_of(double mean, float factor, float square, float eps) {
    RowStats st;
    st.factor = square == 0.0f ? 1.0f : factor;  // equal values: eps alone, which the factor may take away
    const double centre = mean * double(st.factor);
    st.mean = float(centre);
    st.rest = float(centre - double(st.mean));
    st.scale = 1.0f / sqrtf(square + eps * st.factor * st.factor);
    return st;
}

// G threads hold a row of up to 4 G NV values: values 4 t + 4 G u .. of thread t. Groups of up to a wavefront share a
// workgroup of 256 threads; a larger group is a workgroup.
template <int G>
constexpr int kThreadsOf = G > 256 ? G : 256;
template <int G, int NV>
struct Shape {
    static constexpr int kThreads = kThreadsOf<G>, kGroups = kThreads / G, kMost = 4 * G * NV;
    static constexpr int kWaves = G > 64 ? G / 64 : 1;  // of a group
    // Of 16 wavefronts 128 registers a thread do not hold four groups of x, dy, w, dw and db.
    static constexpr bool kHoldsSums = G < 1024 || NV < 4;
    // Wavefronts a SIMD that the registers have to leave room for, where a few more would take a workgroup's place (1269 rows of 8558
    // forward: 18 us, 22 with one workgroup of 1024 threads on a CU; 8192 rows of 4096: 49 with six of 256, 54 with five).
    static constexpr int kForwardWaves = G == 1024 && NV < 4 ? 8 : G == 256 && NV == 4 ? 6 : 1;
    static constexpr int kBackwardWaves = G == 64 && NV == 4 ? 4 : 1;
};

struct Add {
    template <class T>
    __device__ inline T operator()(T a, T b) const { return a + b; }
};
struct Larger {
    __device__ inline float operator()(float a, float b) const { return fmaxf(a, b); }
};

template <int G, class T, class Op>
__device__ inline T lanes_all(T v, Op op) {
    const int lane = red::lane_id();
    v = op(v, red::partner<0>(v, lane));
    v = op(v, red::partner<1>(v, lane));
    if constexpr (G >= 8) v = op(v, red::partner<2>(v, lane));
    if constexpr (G >= 16) v = op(v, red::partner<3>(v, lane));
    if constexpr (G >= 32) v = op(v, red::partner<4>(v, lane));
    if constexpr (G >= 64) v = op(v, red::partner<5>(v, lane));
    return v;
}

// Values of a group's threads become those of the whole group. A group of several wavefronts exchanges through one of two places
// in turn: who is a whole reduction ahead has passed a barrier that all others reached after reading.
template <int G, class A, class OpA, class B = A, class OpB = OpA>
struct Group {
    struct Pair {
        A a;
        B b;
    };
    Pair (*place)[Shape<G, 1>::kWaves];  // [2]
    int turn = 0;
    __device__ inline void operator()(A& a, B& b) {
        constexpr int kLanes = G < 64 ? G : 64;
        a = lanes_all<kLanes>(a, OpA{});
        b = lanes_all<kLanes>(b, OpB{});
        if constexpr (G > 64) {
            if (threadIdx.x % 64 == 0) place[turn][threadIdx.x / 64] = Pair{a, b};
            __syncthreads();
            a = place[turn][0].a;
            b = place[turn][0].b;
            constexpr int kAtOnce = sizeof(Pair) == 8 ? 16 : 4;  // more take registers
#pragma unroll kAtOnce
            for (int w = 1; w < Shape<G, 1>::kWaves; ++w) {
                a = OpA{}(a, place[turn][w].a);
                b = OpB{}(b, place[turn][w].b);
            }
            turn ^= 1;
        }
    }
    __device__ inline void operator()(A& a) {
        a = lanes_all<(G < 64 ? G : 64)>(a, OpA{});
        if constexpr (G > 64) {
            if (threadIdx.x % 64 == 0) place[turn][threadIdx.x / 64].a = a;
            __syncthreads();
            a = place[turn][0].a;
#pragma unroll
            for (int w = 1; w < Shape<G, 1>::kWaves; ++w) a = OpA{}(a, place[turn][w].a);
            turn ^= 1;
        }
    }
};
template <int G>
using SumAndLargest = Group<G, double, Add, float, Larger>;
template <int G>
using Sums = Group<G, float, Add>;

template <int G, int NV>
__device__ inline void load(const float* __restrict__ row, int width, int t, float fill, f4 (&v)[NV]) {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        const int a = 4 * t + 4 * G * u;
        if (a + 3 < width) {
            v[u] = *reinterpret_cast<const f4u*>(row + a);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[u][e] = a + e < width ? row[a + e] : fill;
        }
    }
}
template <int G, int NV>
__device__ inline void store(float* __restrict__ row, int width, int t, const f4 (&v)[NV]) {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
        const int a = 4 * t + 4 * G * u;
        if (a + 3 < width) {
            *reinterpret_cast<f4u*>(row + a) = v[u];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (a + e < width) row[a + e] = v[u][e];
        }
    }
}

// A value that all threads have, in scalar registers.
__device__ inline double uniform(double v) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, v);
    const uint64_t lo = uint32_t(__builtin_amdgcn_readfirstlane(int(bits))), hi = uint32_t(__builtin_amdgcn_readfirstlane(int(bits >> 32)));
    return __builtin_bit_cast(double, lo | hi << 32);
}

// The row's values, with zeros past its end, become x factor - mean - rest; the same for every thread of the group. root: of eps.
template <int G, int NV>
__device__ inline RowStats statistics(f4 (&v)[NV], int width, double n, double one_nth, int t, float eps, float root, SumAndLargest<G>& first,
                                      Sums<G>& second) {
    double sum = 0.0;
    float most = root;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            sum += double(v[u][e]);
            most = fmaxf(most, fabsf(v[u][e]));
        }
        asm volatile("" : "+v"(sum));  // the doubles of one group at a time: they take registers
    }
    first(sum, most);
    // The quotient to its last bit, as a division: of equal values it is their value.
    const double about = sum * one_nth;
    const double mean = __builtin_fma(__builtin_fma(-about, n, sum), one_nth, about);
    const float factor = factor_of(most);
    const double centre = mean * double(factor);
    const float near = float(centre), rest = float(centre - double(near));
    float squares = 0.0f;
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[u][e] = 4 * t + 4 * G * u + e < width ? v[u][e] * factor - near - rest : 0.0f;
            squares = __builtin_fmaf(v[u][e], v[u][e], squares);
        }
    second(squares);
    return stats_of(mean, factor, squares * float(one_nth), eps);
}

template <int G, int NV>
__global__ __launch_bounds__(kThreadsOf<G>, (Shape<G, NV>::kForwardWaves)) void rows_forward_kernel(
    const float* __restrict__ x, const float* __restrict__ weight, const float* __restrict__ bias, float* __restrict__ y,
    RowStats* __restrict__ stats, int64_t rows, int width, float eps) {
    constexpr int kGroups = Shape<G, NV>::kGroups;
    __shared__ typename SumAndLargest<G>::Pair first_place[2][Shape<G, 1>::kWaves];
    __shared__ typename Sums<G>::Pair second_place[2][Shape<G, 1>::kWaves];
    SumAndLargest<G> first_sum{first_place};
    Sums<G> second_sum{second_place};
    const int t = threadIdx.x % G;
    f4 w[NV], b[NV];
    if (weight) load<G>(weight, width, t, 0.0f, w);
    if (bias) load<G>(bias, width, t, 0.0f, b);
    const double n = uniform(double(width)), one_nth = uniform(1.0 / double(width));
    const float root = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, sqrtf(eps))));
    for (int64_t first = int64_t(blockIdx.x) * kGroups; first < rows; first += int64_t(gridDim.x) * kGroups) {
        const int64_t r = first + threadIdx.x / G;
        const bool there = r < rows;  // the wavefront stays whole
        f4 v[NV];
        load<G>(x + (there ? r : rows - 1) * width, width, t, 0.0f, v);
        const RowStats st = statistics<G>(v, width, n, one_nth, t, eps, root, first_sum, second_sum);
#pragma unroll
        for (int u = 0; u < NV; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float h = v[u][e] * st.scale;
                v[u][e] = weight ? h * w[u][e] : h;
                if (bias) v[u][e] += b[u][e];
            }
        if (there) {
            store<G>(y + r * width, width, t, v);
            if (stats && t == 0) stats[r] = st;
        }
    }
}

// Columns: dw and db wanted; sums [gridDim.x][2][width], this workgroup's rows.
template <int G, int NV, bool Columns>
__global__ __launch_bounds__(kThreadsOf<G>, (Shape<G, NV>::kBackwardWaves)) void rows_backward_kernel(
    const float* __restrict__ grad, const float* __restrict__ x, const float* __restrict__ weight,
    const RowStats* __restrict__ stats, float* __restrict__ dx, float* __restrict__ sums, int64_t rows, int width) {
    constexpr int kGroups = Shape<G, NV>::kGroups, kMost = Shape<G, NV>::kMost;
    __shared__ typename Sums<G>::Pair place[2][Shape<G, 1>::kWaves];
    __shared__ float columns[Columns && kGroups > 1 ? kGroups * kMost : 1];
    Sums<G> sum{place};
    const int t = threadIdx.x % G;
    const float n = float(width);
    f4 w[NV], dw[Columns ? NV : 1] = {}, db[Columns ? NV : 1] = {};
    if (weight) load<G>(weight, width, t, 0.0f, w);
    // The next row is on its way while a row is made, where few workgroups share a CU and there are registers for it (8192 rows
    // of 4096: 116 us without, 79 with).
    constexpr bool kAhead = Columns && G == 256;
    const int64_t step = int64_t(gridDim.x) * kGroups;
    f4 next_x[kAhead ? NV : 1], next_d[kAhead ? NV : 1];
    RowStats next_stats{};
    const auto fetch = [&](int64_t first, f4(&xs)[NV], f4(&ds)[NV], RowStats& st) {
        const int64_t at = min(first + threadIdx.x / G, rows - 1);
        load<G>(x + at * width, width, t, 0.0f, xs);
        load<G>(grad + at * width, width, t, 0.0f, ds);
        st = stats[at];
    };
    if constexpr (kAhead) fetch(int64_t(blockIdx.x) * kGroups, next_x, next_d, next_stats);
    for (int64_t first = int64_t(blockIdx.x) * kGroups; first < rows; first += step) {
        const int64_t r = first + threadIdx.x / G;
        const bool there = r < rows;
        f4 h[NV], d[NV];
        RowStats st;
        if constexpr (kAhead) {
#pragma unroll
            for (int u = 0; u < NV; ++u) {
                h[u] = next_x[u];
                d[u] = next_d[u];
            }
            st = next_stats;
            fetch(first + step, next_x, next_d, next_stats);
        } else {
            fetch(first, h, d, st);
        }
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int u = 0; u < NV; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                h[u][e] = 4 * t + 4 * G * u + e < width ? st.normed(h[u][e]) : 0.0f;
                if constexpr (Columns) {
                    if (there) {
                        dw[u][e] = __builtin_fmaf(d[u][e], h[u][e], dw[u][e]);
                        db[u][e] += d[u][e];
                    }
                }
                if (weight) d[u][e] *= w[u][e];
                s[0] += d[u][e];
                s[1] = __builtin_fmaf(d[u][e], h[u][e], s[1]);
            }
        if (!dx) continue;  // the same in every thread
        sum(s[0], s[1]);
        if (fabsf(s[0]) < __builtin_huge_valf() && fabsf(s[1]) < __builtin_huge_valf()) {  // the same in every thread of the group
            s[0] /= n;
            s[1] /= n;
        } else {  // again, of values so small that float32 holds the sums of any
            s[0] = s[1] = 0.0f;
#pragma unroll
            for (int u = 0; u < NV; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[0] = __builtin_fmaf(d[u][e], 0x1p-30f, s[0]);
                    s[1] = __builtin_fmaf(d[u][e] * 0x1p-30f, h[u][e], s[1]);
                }
            sum(s[0], s[1]);
            s[0] = s[0] / n * 0x1p30f;
            s[1] = s[1] / n * 0x1p30f;
        }
#pragma unroll
        for (int u = 0; u < NV; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) d[u][e] = (d[u][e] - s[0] - h[u][e] * s[1]) * st.scale * st.factor;
        if (there) store<G>(dx + r * width, width, t, d);
    }
    if constexpr (Columns) {
        float* const out = sums + int64_t(blockIdx.x) * 2 * width;
        if constexpr (kGroups == 1) {
            store<G>(out, width, t, dw);
            store<G>(out + width, width, t, db);
        } else {
#pragma unroll
            for (int which = 0; which < 2; ++which) {
                __syncthreads();
#pragma unroll
                for (int u = 0; u < NV; ++u)
                    *reinterpret_cast<f4*>(columns + threadIdx.x / G * kMost + 4 * t + 4 * G * u) = which ? db[u] : dw[u];
                __syncthreads();
                for (int c = threadIdx.x; c < width; c += Shape<G, NV>::kThreads) {
                    double total = 0.0;
#pragma unroll
                    for (int g = 0; g < kGroups; ++g) total += double(columns[g * kMost + c]);
                    out[which * width + c] = float(total);
                }
            }
        }
    }
}

// ---- rows that no workgroup holds: read once for each sum ------------------------------

constexpr int kWideThreads = 1024;

// Sums of N doubles over the workgroup, on every thread.
template <int N>
__device__ inline void workgroup_sum(double (&v)[N], double (*place)[kWideThreads / 64]) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = red::wave_sum(v[i]);
        if (threadIdx.x % 64 == 0) place[i][threadIdx.x / 64] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = 0.0;
        for (int w = 0; w < kWideThreads / 64; ++w) v[i] += place[i][w];
    }
}

__global__ __launch_bounds__(kWideThreads) void wide_forward_kernel(const float* __restrict__ x, const float* __restrict__ weight,
                                                                    const float* __restrict__ bias, float* __restrict__ y,
                                                                    RowStats* __restrict__ stats, int64_t rows, int64_t width,
                                                                    float eps) {
    __shared__ double place[2][kWideThreads / 64];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const float* const row = x + r * width;
        double s[1] = {0.0}, q[1] = {0.0};
        for (int64_t c = threadIdx.x; c < width; c += kWideThreads) s[0] += double(row[c]);
        workgroup_sum(s, place);
        const double mean = s[0] / double(width);
        for (int64_t c = threadIdx.x; c < width; c += kWideThreads) {
            const double d = double(row[c]) - mean;
            q[0] += d * d;
        }
        workgroup_sum(q, place);
        const double square = q[0] / double(width);
        const float factor = factor_of(fmaxf(float(fmin(sqrt(square), 0x1p127)), sqrtf(eps)));
        const RowStats st = stats_of(mean, factor, float(square * double(factor) * double(factor)), eps);
        for (int64_t c = threadIdx.x; c < width; c += kWideThreads) {
            float h = st.normed(row[c]);
            if (weight) h *= weight[c];
            if (bias) h += bias[c];
            y[r * width + c] = h;
        }
        if (stats && threadIdx.x == 0) stats[r] = st;
    }
}

__global__ __launch_bounds__(kWideThreads) void wide_backward_kernel(const float* __restrict__ grad, const float* __restrict__ x,
                                                                     const float* __restrict__ weight,
                                                                     const RowStats* __restrict__ stats, float* __restrict__ dx,
                                                                     int64_t rows, int64_t width) {
    __shared__ double place[2][kWideThreads / 64];
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const float *const g = grad + r * width, *const row = x + r * width;
        const RowStats st = stats[r];
        double s[2] = {0.0, 0.0};
        for (int64_t c = threadIdx.x; c < width; c += kWideThreads) {
            const float h = st.normed(row[c]), d = weight ? g[c] * weight[c] : g[c];
            s[0] += double(d);
            s[1] += double(d) * double(h);
        }
        workgroup_sum(s, place);
        const float first = float(s[0] / double(width)), second = float(s[1] / double(width));
        for (int64_t c = threadIdx.x; c < width; c += kWideThreads) {
            const float h = st.normed(row[c]), d = weight ? g[c] * weight[c] : g[c];
            dx[r * width + c] = (d - first - h * second) * st.scale * st.factor;
        }
    }
}

// Workgroup (i, j): columns 256 i .., rows j, j + gridDim.y, ...
__global__ __launch_bounds__(256) void wide_columns_kernel(const float* __restrict__ grad, const float* __restrict__ x,
                                                           const RowStats* __restrict__ stats, float* __restrict__ sums,
                                                           int64_t rows, int64_t width) {
    const int64_t c = int64_t(blockIdx.x) * 256 + threadIdx.x;
    if (c >= width) return;
    double dw = 0.0, db = 0.0;
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
        const RowStats st = stats[r];
        const float g = grad[r * width + c];
        dw += double(g) * double(st.normed(x[r * width + c]));
        db += double(g);
    }
    float* const out = sums + int64_t(blockIdx.y) * 2 * width;
    out[c] = float(dw);
    out[width + c] = float(db);
}

// ---- the partial rows -----------------------------------------------------------------

constexpr int kFinishThreads = 1024, kFinishColumns = 32, kFinishGroups = kFinishThreads / kFinishColumns, kFinishLoads = 16;

// Column c of 2 width: dw, then db. Group g of a workgroup adds the parts g, g + 32, ... of its 32 columns, 16 loads in flight,
// then the groups are added in order. Bound by those loads' latency where rows are short: 512 parts of 4096 columns 8 us, of 515
// 5.8.
__global__ __launch_bounds__(kFinishThreads) void finish_kernel(const float* __restrict__ sums, int parts, int64_t width,
                                                                float* __restrict__ dw, float* __restrict__ db) {
    __shared__ double groups[kFinishGroups][kFinishColumns];
    const int lane = threadIdx.x % kFinishColumns, group = threadIdx.x / kFinishColumns;
    const int64_t c = int64_t(blockIdx.x) * kFinishColumns + lane;
    double total = 0.0;
    if (c < 2 * width) {
        for (int p = group; p < parts; p += kFinishLoads * kFinishGroups) {
            float v[kFinishLoads];
#pragma unroll
            for (int u = 0; u < kFinishLoads; ++u) {
                const int at = p + u * kFinishGroups;
                v[u] = at < parts ? sums[int64_t(at) * 2 * width + c] : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < kFinishLoads; ++u) total += double(v[u]);
        }
    }
    groups[group][lane] = total;
    __syncthreads();
    if (group != 0 || c >= 2 * width) return;
    for (int g = 1; g < kFinishGroups; ++g) total += groups[g][lane];
    float* const out = c < width ? dw : db;
    if (out) out[c < width ? c : c - width] = float(total);
}

constexpr size_t kMostAdded = 64;  // rows of a thread's float32 sums

// f(G, NV) for the least shape that holds a row; false where none does.
template <class F>
bool with_shape(size_t width, F&& f) {
#define VC_SHAPE(G, NV) \
    if (width <= size_t(Shape<G, NV>::kMost)) return f(std::integral_constant<int, G>{}, std::integral_constant<int, NV>{}), true
    VC_SHAPE(4, 1);
    VC_SHAPE(16, 1);
    VC_SHAPE(32, 1);
    VC_SHAPE(64, 1);
    VC_SHAPE(64, 2);
    VC_SHAPE(64, 3);
    VC_SHAPE(64, 4);
    VC_SHAPE(256, 2);
    VC_SHAPE(256, 3);
    VC_SHAPE(256, 4);
    VC_SHAPE(1024, 2);
    VC_SHAPE(1024, 3);
    VC_SHAPE(1024, 4);
#undef VC_SHAPE
    return false;
}

void check_sizes(const char* op, size_t rows, size_t width) {
    if (width == 0) fail(VC_HIP_ERR_INVALID_ARGUMENT, std::string(op) + ": no values in a row");
    if (rows > (size_t(1) << 40) || width > (size_t(1) << 26) || rows > (size_t(1) << 46) / width)
        fail(VC_HIP_ERR_OVERFLOW, std::string(op) + ": too many values");
}

}  // namespace
}  // namespace vchip

using namespace vchip;

extern "C" {

int vc_hip_layer_norm_forward(const float* x, const float* weight, const float* bias, size_t rows, size_t width, float eps,
                              float* y, float* stats) {
    return guard([&] {
        Device& d = require_device();
        check_sizes("layer_norm", rows, width);
        if (!(eps >= 0.0f) || std::isinf(eps)) fail(VC_HIP_ERR_INVALID_ARGUMENT, "layer_norm: eps must be a number from zero up");
        if (rows == 0) return;
        if (!x || !y) fail(VC_HIP_ERR_INVALID_ARGUMENT, "layer_norm: null pointer");
        if (stats && !aligned16(stats)) fail(VC_HIP_ERR_INVALID_ARGUMENT, "layer_norm: stats must lie on a 16-byte boundary");
        auto* const st = reinterpret_cast<RowStats*>(stats);
        const double count = double(rows) * double(width);
        Profiled p("layer_norm", 8.0 * count, 8.0 * count);
        const bool held = with_shape(width, [&](auto g, auto nv) {
            using S = Shape<g(), nv()>;
            // Two rows of a group or more, which share the weight's loads, and 16 workgroups a CU if there are as many: 4000 rows of
            // 3500 20.5 us, 22.7 with one; 8192 rows of 4096 49 us, 55 with eight.
            const size_t pairs = rows / S::kGroups / 2, cus = size_t(d.cu_count);
            const unsigned grid = grid_1d(rows, S::kGroups, unsigned(std::clamp(pairs, 8 * cus, 16 * cus)));
            launch(rows_forward_kernel<g(), nv()>, dim3(grid), dim3(S::kThreads), 0, d.stream, x, weight, bias, y, st,
                   int64_t(rows), int(width), eps);
        });
        if (!held)
            launch(wide_forward_kernel, dim3(grid_1d(rows, 1, 2u * unsigned(d.cu_count))), dim3(kWideThreads), 0, d.stream, x, weight,
                   bias, y, st, int64_t(rows), int64_t(width), eps);
        after_launch("layer_norm");
        p.done();
    });
}

int vc_hip_layer_norm_backward(const float* grad, const float* x, const float* weight, const float* stats, size_t rows,
                               size_t width, float* grad_x, float* grad_weight, float* grad_bias) {
    return guard([&] {
        Device& d = require_device();
        check_sizes("layer_norm_backward", rows, width);
        const bool columns = grad_weight || grad_bias;
        if (!grad_x && !columns) return;
        if (rows == 0) {
            for (float* out : {grad_weight, grad_bias})
                if (out && vc_hip_fill(out, width, 0.0f) != VC_HIP_OK) fail(VC_HIP_ERR_RUNTIME, vc_hip_last_error());
            return;
        }
        if (!grad || !x || !stats) fail(VC_HIP_ERR_INVALID_ARGUMENT, "layer_norm_backward: null pointer");
        if (!aligned16(stats)) fail(VC_HIP_ERR_INVALID_ARGUMENT, "layer_norm_backward: stats must lie on a 16-byte boundary");
        const auto* const st = reinterpret_cast<const RowStats*>(stats);
        const double count = double(rows) * double(width);
        Profiled p("layer_norm_backward", 10.0 * count, 12.0 * count);
        unsigned parts = 0;
        std::unique_ptr<Scratch> sums;
        const auto scratch = [&](unsigned n) {
            parts = n;
            if (columns) sums = std::make_unique<Scratch>(size_t(n) * 2 * width * sizeof(float));
            return sums ? sums->as<float>() : nullptr;
        };
        bool collected = !columns;  // are the sums made with dx?
        const bool held = with_shape(width, [&](auto g, auto nv) {
            using S = Shape<g(), nv()>;
            if constexpr (S::kHoldsSums) {
                if (columns) {
                    const size_t least = (rows + kMostAdded * S::kGroups - 1) / (kMostAdded * S::kGroups);
                    if (least > kMostBlocks * 256 / S::kThreads) fail(VC_HIP_ERR_OVERFLOW, "layer_norm_backward: too many rows");
                    const unsigned grid = grid_1d(rows, S::kGroups, std::max(unsigned(least), 2u * unsigned(d.cu_count)));
                    launch(rows_backward_kernel<g(), nv(), true>, dim3(grid), dim3(S::kThreads), 0, d.stream, grad, x, weight, st,
                           grad_x, scratch(grid), int64_t(rows), int(width));
                    collected = true;
                    return;
                }
            }
            if (grad_x)
                launch(rows_backward_kernel<g(), nv(), false>, dim3(grid_1d(rows, S::kGroups, 8u * unsigned(d.cu_count))),
                       dim3(S::kThreads), 0, d.stream, grad, x, weight, st, grad_x, nullptr, int64_t(rows), int(width));
        });
        if (!collected || !held) {
            if (grad_x && !held)
                launch(wide_backward_kernel, dim3(grid_1d(rows, 1, 2u * unsigned(d.cu_count))), dim3(kWideThreads), 0, d.stream, grad,
                       x, weight, st, grad_x, int64_t(rows), int64_t(width));
            if (columns) {
                const unsigned across = unsigned((width + 255) / 256);
                const unsigned down = unsigned(std::min<size_t>(rows, std::max<size_t>(1, 4 * size_t(d.cu_count) / across)));
                launch(wide_columns_kernel, dim3(across, down), dim3(256), 0, d.stream, grad, x, st, scratch(down), int64_t(rows),
                       int64_t(width));
            }
        }
        after_launch("layer_norm_backward");
        if (columns) {
            launch(finish_kernel, dim3(unsigned((2 * width + kFinishColumns - 1) / kFinishColumns)), dim3(kFinishThreads), 0, d.stream,
                   sums->as<float>(), int(parts), int64_t(width), grad_weight, grad_bias);
            after_launch("layer_norm_backward columns");
        }
        p.done();
    });
}

}  // extern "C"

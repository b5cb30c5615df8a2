// Dropout whose mask is a function of a counter: kept again, not kept in memory.
//
// Element i is kept where word i % 4 of Philox 4x32 with ten rounds (Salmon,
// Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011), of
// the counter (i / 4, stream) under the key `seed`, is at least round(p 2^32).
// What is kept is divided by 1 - p. The gradient is the same function of the
// upstream gradient, so one kernel serves both.
//
// Bound by HBM (8 bytes an element, 12 with a residual): ten rounds of two 32 x 32
// products make four words, about 20 instructions an element at a quarter rate or
// better. A thread makes the words of four neighbours, which it loads and stores
// as one 16-byte access, of four such groups in flight. 8192 x 4096: 52 us (5.2
// TB/s), 85 us with a residual (4.7; a copy of 1 GiB reaches 5.1). 256 x 256: 3.3.
#include "vc_hip_internal.hpp"

#include <cmath>

namespace vchip {
namespace {

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kThreads = 256, kAtOnce = 4;  // counters of a thread whose loads are in flight together

struct Words {
    uint32_t v[4];
};

__device__ inline Words philox(uint64_t block, uint64_t stream, uint64_t seed) {
    uint32_t a = uint32_t(block), b = uint32_t(block >> 32), c = uint32_t(stream), d = uint32_t(stream >> 32);
    uint32_t k = uint32_t(seed), l = uint32_t(seed >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t first = uint64_t(0xD2511F53u) * a, second = uint64_t(0xCD9E8D57u) * c;
        a = uint32_t(second >> 32) ^ b ^ k;
        b = uint32_t(second);
        c = uint32_t(first >> 32) ^ d ^ l;
        d = uint32_t(first);
        k += 0x9E3779B9u;
        l += 0xBB67AE85u;
    }
    return Words{{a, b, c, d}};
}

template <bool Residual>
__global__ __launch_bounds__(kThreads) void dropout_kernel(const float* __restrict__ x, const float* __restrict__ residual,
                                                           float* __restrict__ out, int64_t count, uint64_t threshold,
                                                           float scale, uint64_t seed, uint64_t stream) {
    const int64_t whole = count / 4, step = int64_t(gridDim.x) * kThreads;
    const auto keep = [&](uint32_t word, float v) { return uint64_t(word) >= threshold ? v * scale : 0.0f; };
    for (int64_t first = int64_t(blockIdx.x) * kThreads + threadIdx.x; first < whole; first += kAtOnce * step) {
        f4u v[kAtOnce], r[kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u)
            if (first + u * step < whole) {
                v[u] = *reinterpret_cast<const f4u*>(x + 4 * (first + u * step));
                if constexpr (Residual) r[u] = *reinterpret_cast<const f4u*>(residual + 4 * (first + u * step));
            }
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const int64_t at = first + u * step;
            if (at >= whole) break;
            const Words words = philox(uint64_t(at), stream, seed);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                v[u][e] = keep(words.v[e], v[u][e]);
                if constexpr (Residual) v[u][e] += r[u][e];
            }
            *reinterpret_cast<f4u*>(out + 4 * at) = v[u];
        }
    }
    const int64_t tail = 4 * whole + threadIdx.x;
    if (blockIdx.x == 0 && tail < count) {
        const Words words = philox(uint64_t(whole), stream, seed);
        uint32_t word = words.v[0];
        word = threadIdx.x == 1 ? words.v[1] : word;
        word = threadIdx.x == 2 ? words.v[2] : word;
        const float v = keep(word, x[tail]);
        out[tail] = Residual ? v + residual[tail] : v;
    }
}

}  // namespace
}  // namespace vchip

using namespace vchip;

extern "C" {

int vc_hip_dropout(const float* x, const float* residual, size_t count, double p, uint64_t seed, uint64_t stream, float* out) {
    return guard([&] {
        Device& d = require_device();
        if (!(p >= 0.0 && p <= 1.0)) fail(VC_HIP_ERR_INVALID_ARGUMENT, "dropout: p must lie between zero and one");
        if (count > (size_t(1) << 46)) fail(VC_HIP_ERR_OVERFLOW, "dropout: too many values");
        if (count == 0) return;
        if (!x || !out) fail(VC_HIP_ERR_INVALID_ARGUMENT, "dropout: null pointer");
        const auto threshold = uint64_t(std::nearbyint(p * 4294967296.0));
        const float scale = p < 1.0 ? float(1.0 / (1.0 - p)) : 0.0f;
        Profiled profile("dropout", double(count), (residual ? 12.0 : 8.0) * double(count));
        const dim3 grid(grid_1d((count + 3) / 4, kThreads * kAtOnce, 16u * unsigned(d.cu_count))), block(kThreads);
        if (residual)
            launch(dropout_kernel<true>, grid, block, 0, d.stream, x, residual, out, int64_t(count), threshold, scale, seed, stream);
        else
            launch(dropout_kernel<false>, grid, block, 0, d.stream, x, residual, out, int64_t(count), threshold, scale, seed, stream);
        after_launch("dropout");
        profile.done();
    });
}

}  // extern "C"

// Orthogonalised momentum updates of weight matrices.
//
// With U = U S V^T the singular value decomposition of an update, the step is
// U V^T, approached without one: X = U / ||U|| and, `steps` times,
//   X <- a X + (b G + c G G) X,   G = X X^T (or X <- a X + X (b G + c G G), G = X^T X for a tall X),
// which maps every singular value s to a s + b s^3 + c s^5. The sums run over
// the longer side once and over the shorter twice.
#include "reduce_common.hpp"
#include "vc_hip_internal.hpp"

#include <algorithm>
#include <cmath>
#include <string>
#include <vector>

namespace vchip {
namespace {

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr int kNormBlocks = 64;  // partial sums of squares of a matrix

// u = g + mu * m after m = mu * m + g (momentum), or u = g; the squares of u are summed in double, a partial
// for each workgroup, in a fixed order.
template <bool Momentum>
__global__ __launch_bounds__(256) void update_kernel(const float* __restrict__ grad, float* __restrict__ momentum, float mu,
                                                     int64_t count, float* __restrict__ u, double* __restrict__ partials) {
    __shared__ double sums[4];
    const int64_t base = int64_t(blockIdx.y) * count;
    double sum = 0.0;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < count; i += int64_t(gridDim.x) * 256) {
        float v = grad[base + i];
        if constexpr (Momentum) {
            const float m = momentum[base + i] * mu + v;
            momentum[base + i] = m;
            v = v + mu * m;
        }
        u[base + i] = v;
        sum += double(v) * double(v);
    }
    sum = red::wave_sum(sum);
    if (threadIdx.x % 64 == 0) sums[threadIdx.x / 64] = sum;
    __syncthreads();
    if (threadIdx.x == 0) partials[blockIdx.y * gridDim.x + blockIdx.x] = sums[0] + sums[1] + sums[2] + sums[3];
}

__global__ __launch_bounds__(256) void normalise_kernel(float* __restrict__ u, int64_t count, const double* __restrict__ partials,
                                                        int blocks) {
    double sum = 0.0;
    for (int i = 0; i < blocks; ++i) sum += partials[blockIdx.y * blocks + i];
    const double norm = sqrt(sum);
    const double scale = norm == 0.0 ? 0.0 : 1.0 / norm;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < count; i += int64_t(gridDim.x) * 256)
        u[int64_t(blockIdx.y) * count + i] = float(double(u[int64_t(blockIdx.y) * count + i]) * scale);
}

__global__ __launch_bounds__(256) void mix_kernel(float a, const float* __restrict__ x, float b, const float* __restrict__ y,
                                                  int64_t count, float* __restrict__ out) {
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < count; i += int64_t(gridDim.x) * 256)
        out[i] = a * x[i] + b * y[i];
}

void mix(Device& d, float a, const float* x, float b, const float* y, size_t count, float* out) {
    launch(mix_kernel, dim3(grid_1d(count, 256, 4096)), dim3(256), 0, d.stream, a, x, b, y, int64_t(count), out);
    after_launch("muon mix");
}

void products(const float* a, const float* b, float* c, size_t m, size_t k, size_t n, size_t count, bool ta, bool tb) {
    std::vector<size_t> ao(count), bo(count);
    for (size_t i = 0; i < count; ++i) {
        ao[i] = i * m * k;
        bo[i] = i * k * n;
    }
    if (const int rc = vc_hip_matmul(a, b, c, m, k, n, ao.data(), bo.data(), count, ta, tb))
        fail(rc, std::string("orthogonalise: ") + vc_hip_last_error());
}

// x, normalised, becomes its iterate.
void iterate(Device& d, float* x, size_t count, size_t rows, size_t cols, size_t steps) {
    const size_t s = std::min(rows, cols), elements = count * rows * cols;
    const bool wide = rows <= cols;
    Scratch gram(count * s * s * sizeof(float)), square(count * s * s * sizeof(float)), y(elements * sizeof(float));
    for (size_t i = 0; i < steps; ++i) {
        if (wide) products(x, x, gram.as<float>(), rows, cols, rows, count, false, true);
        else products(x, x, gram.as<float>(), cols, rows, cols, count, true, false);
        products(gram.as<float>(), gram.as<float>(), square.as<float>(), s, s, s, count, false, false);
        mix(d, kB, gram.as<float>(), kC, square.as<float>(), count * s * s, square.as<float>());
        if (wide) products(square.as<float>(), x, y.as<float>(), rows, rows, cols, count, false, false);
        else products(x, square.as<float>(), y.as<float>(), rows, cols, cols, count, false, false);
        mix(d, kA, x, 1.0f, y.as<float>(), elements, x);
    }
}

void start(Device& d, const float* grad, float* momentum, float mu, size_t count, size_t elements, float* u) {
    const unsigned blocks = grid_1d(elements, 2048, kNormBlocks);
    Scratch partials(count * blocks * sizeof(double));
    const dim3 grid(blocks, unsigned(count));
    if (momentum)
        launch(update_kernel<true>, grid, dim3(256), 0, d.stream, grad, momentum, mu, int64_t(elements), u, partials.as<double>());
    else
        launch(update_kernel<false>, grid, dim3(256), 0, d.stream, grad, momentum, mu, int64_t(elements), u, partials.as<double>());
    after_launch("muon update");
    launch(normalise_kernel, dim3(grid_1d(elements, 256, 1024), unsigned(count)), dim3(256), 0, d.stream, u, int64_t(elements),
           static_cast<const double*>(partials.as<double>()), int(blocks));
    after_launch("muon normalise");
}

void check_matrix(size_t count, size_t rows, size_t cols) {
    if (count > 65535) fail(VC_HIP_ERR_INVALID_ARGUMENT, "orthogonalise: at most 65535 matrices");
    if (rows > 65535 * 32 || cols > 65535 * 32) fail(VC_HIP_ERR_OVERFLOW, "orthogonalise: matrix too large");
}

}  // namespace
}  // namespace vchip

using namespace vchip;

extern "C" {

int vc_hip_orthogonalise(const float* in, size_t count, size_t rows, size_t cols, size_t steps, float* out) {
    return guard([&] {
        Device& d = require_device();
        check_matrix(count, rows, cols);
        if (count == 0 || rows == 0 || cols == 0) return;
        if (!in || !out) fail(VC_HIP_ERR_INVALID_ARGUMENT, "orthogonalise: null pointer");
        start(d, in, nullptr, 0.0f, count, rows * cols, out);
        iterate(d, out, count, rows, cols, steps);
    });
}

int vc_hip_muon_step(const vc_hip_muon_item* items, size_t n_items, float rate, float mu, float decay, size_t steps) {
    return guard([&] {
        Device& d = require_device();
        if (n_items && !items) fail(VC_HIP_ERR_INVALID_ARGUMENT, "muon_step: null items");
        for (size_t i = 0; i < n_items; ++i) {
            const vc_hip_muon_item& it = items[i];
            check_matrix(it.count, it.rows, it.cols);
            if (it.count * it.rows * it.cols && (!it.param || !it.momentum || !it.grad))
                fail(VC_HIP_ERR_INVALID_ARGUMENT, "muon_step: null pointer");
        }
        for (size_t i = 0; i < n_items; ++i) {
            const vc_hip_muon_item& it = items[i];
            const size_t elements = it.rows * it.cols, all = it.count * elements;
            if (all == 0) continue;
            Scratch u(all * sizeof(float));
            start(d, it.grad, it.momentum, mu, it.count, elements, u.as<float>());
            iterate(d, u.as<float>(), it.count, it.rows, it.cols, steps);
            const float scaled = rate * float(std::sqrt(std::max(1.0, double(it.cols) / double(it.rows))));
            mix(d, 1.0f - rate * decay, it.param, -scaled, u.as<float>(), all, it.param);
        }
    });
}

}  // extern "C"

// Softmax cross entropy of a linear layer's logits that are never kept.
//
// For each row t of x [rows, width], with z = x W + b [classes]:
//   loss_t = log(sum_v exp(z_v)) - z_target,
//   dz_v   = share_t (exp(z_v) / sum - [v = target]),
//   dx = dz W^T, dW = x^T dz, db = the sum over rows of dz.
// A row whose target is no class number is left out: its loss and its part of
// every gradient are zero, whatever x holds there. The share of a row is its
// upstream gradient, or one over the number of rows that count (the mean loss).
//
// Rows are taken in pieces: the logits of a piece live in a workspace until
// their gradients are used.
#include "reduce_common.hpp"
#include "vc_hip_internal.hpp"

#include <algorithm>
#include <cmath>
#include <memory>
#include <string>

namespace vchip {
namespace {

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));

constexpr float kLowest = -__builtin_huge_valf();

// The class a target names, or -1.
__device__ inline int64_t class_of(float target, int64_t classes) {
    if (!(target >= 0.0f && target < float(classes))) return -1;
    const int64_t c = int64_t(target);
    return float(c) == target ? c : -1;
}

constexpr int kCountThreads = 1024;

// share[0] = one over the number of rows that count, or zero.
__global__ __launch_bounds__(kCountThreads) void count_kernel(const float* __restrict__ targets, int64_t rows, int64_t classes,
                                                              float* __restrict__ share) {
    __shared__ double lds[kCountThreads / 64];
    double n = 0.0;
    for (int64_t r = threadIdx.x; r < rows; r += kCountThreads) n += class_of(targets[r], classes) >= 0 ? 1.0 : 0.0;
    n = red::block_sum(n, lds);
    if (threadIdx.x == 0) share[0] = n > 0.0 ? float(1.0 / n) : 0.0f;
}

// mean[0] = share[0] times the sum of the losses.
__global__ __launch_bounds__(kCountThreads) void mean_kernel(const float* __restrict__ losses, int64_t rows,
                                                             const float* __restrict__ share, float* __restrict__ mean) {
    __shared__ double lds[kCountThreads / 64];
    double s = 0.0;
    for (int64_t r = threadIdx.x; r < rows; r += kCountThreads) s += double(losses[r]);
    s = red::block_sum(s, lds);
    if (threadIdx.x == 0) mean[0] = float(s * double(share[0]));
}

// A copy of x whose left out rows are zeros: zero times what they hold would not be zero for an infinity or a NaN.
__global__ __launch_bounds__(256) void counted_rows_kernel(const float* __restrict__ x, const float* __restrict__ targets,
                                                           float* __restrict__ out, int64_t rows, int64_t width,
                                                           int64_t classes) {
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        const bool counted = class_of(targets[r], classes) >= 0;
        for (int64_t c = threadIdx.x; c < width; c += 256) out[r * width + c] = counted ? x[r * width + c] : 0.0f;
    }
}

constexpr int kRowThreads = 256;

__device__ inline float workgroup_max(float v, float* lds) {
    const int lane = red::lane_id();
    const auto larger = [](float a, float b) { return fmaxf(a, b); };
    v = larger(v, red::partner<0>(v, lane));
    v = larger(v, red::partner<1>(v, lane));
    v = larger(v, red::partner<2>(v, lane));
    v = larger(v, red::partner<3>(v, lane));
    v = larger(v, red::partner<4>(v, lane));
    v = larger(v, red::partner<5>(v, lane));
    if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
    __syncthreads();
    float m = lds[0];
    for (int w = 1; w < kRowThreads / 64; ++w) m = fmaxf(m, lds[w]);
    return m;
}

// A workgroup a row: its loss from the logits z (without the bias), and, where Gradient, z becomes dz.
template <bool Gradient>
__global__ __launch_bounds__(kRowThreads) void logits_kernel(float* __restrict__ z, const float* __restrict__ bias,
                                                             const float* __restrict__ targets, const float* __restrict__ shares,
                                                             bool one_share, int64_t rows, int64_t classes,
                                                             float* __restrict__ losses) {
    __shared__ double sums[kRowThreads / 64];
    __shared__ float most[kRowThreads / 64];
    __shared__ double total_of_row;
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        __syncthreads();
        float* const row = z + r * classes;
        const int64_t target = class_of(targets[r], classes);
        if (target < 0) {
            if (losses && threadIdx.x == 0) losses[r] = 0.0f;
            if constexpr (Gradient)
                for (int64_t c = threadIdx.x; c < classes; c += kRowThreads) row[c] = 0.0f;
            continue;
        }
        const auto value = [&](int64_t c) { return bias ? row[c] + bias[c] : row[c]; };
        float m = kLowest;
        for (int64_t c = threadIdx.x; c < classes; c += kRowThreads) m = fmaxf(m, value(c));
        m = workgroup_max(m, most);
        double s = 0.0;
        for (int64_t c = threadIdx.x; c < classes; c += kRowThreads) s += double(expf(value(c) - m));
        s = red::block_sum(s, sums);
        if (threadIdx.x == 0) total_of_row = s;
        __syncthreads();
        s = total_of_row;
        const float at = value(target) - m;
        if (losses && threadIdx.x == 0) losses[r] = float(log(s) - double(at));
        if constexpr (Gradient) {
            const float share = one_share ? shares[0] : shares[r], scale = float(double(share) / s);
            const double own = double(expf(at));
            __syncthreads();  // every thread has read the target's logit
            for (int64_t c = threadIdx.x; c < classes; c += kRowThreads) {
                const float e = expf(value(c) - m);
                // The others' sum in double: one minus a share near one would leave no bits.
                row[c] = c == target ? float(-double(share) * ((s - own) / s)) : e * scale;
            }
        }
    }
}

void run(int status) {
    if (status != VC_HIP_OK) fail(status, vc_hip_last_error());
}

struct Call {
    const float *x, *weight, *bias, *targets;
    size_t rows, width, classes;
};

void check_call(const char* op, const Call& c) {
    const std::string name(op);
    if (c.width == 0 || c.classes == 0) fail(VC_HIP_ERR_INVALID_ARGUMENT, name + ": no features or no classes");
    if (c.classes > (size_t(1) << 24)) fail(VC_HIP_ERR_OVERFLOW, name + ": float32 class numbers reach 2^24 classes");
    if (c.width > (size_t(1) << 24) || c.rows >= (size_t(1) << 31)) fail(VC_HIP_ERR_OVERFLOW, name + ": too many rows or features");
    if (c.rows && (!c.x || !c.weight || !c.targets)) fail(VC_HIP_ERR_INVALID_ARGUMENT, name + ": null pointer");
}

// Logits of a piece: 2^28 of them, 1 GiB.
size_t rows_of_piece(const Call& c) { return std::max<size_t>(1, std::min(c.rows, (size_t(1) << 28) / c.classes)); }

void product(const float* a, const float* b, float* c, size_t m, size_t k, size_t n, bool trans_a, bool trans_b) {
    const size_t none = 0;
    run(vc_hip_matmul(a, b, c, m, k, n, &none, &none, 1, trans_a, trans_b));
}

void forward(Device& d, const Call& c, float* losses) {
    const size_t piece = rows_of_piece(c);
    Scratch logits(piece * c.classes * sizeof(float));
    for (size_t r = 0; r < c.rows; r += piece) {
        const size_t n = std::min(piece, c.rows - r);
        product(c.x + r * c.width, c.weight, logits.as<float>(), n, c.width, c.classes, false, false);
        launch(logits_kernel<false>, dim3(grid_1d(n, 1, 16u * unsigned(d.cu_count))), dim3(kRowThreads), 0, d.stream,
               logits.as<float>(), c.bias, c.targets + r, nullptr, false, int64_t(n), int64_t(c.classes), losses + r);
        after_launch("linear_cross_entropy rows");
    }
}

void gradient(Device& d, const Call& c, const float* shares, bool one_share, float* losses, float* grad_x, float* grad_weight,
              float* grad_bias) {
    const size_t piece = rows_of_piece(c), pieces = (c.rows + piece - 1) / piece;
    Scratch logits(piece * c.classes * sizeof(float));
    Scratch rows(grad_weight ? piece * c.width * sizeof(float) : 4);
    Scratch more(pieces > 1 ? std::max(grad_weight ? c.width * c.classes : 0, c.classes) * sizeof(float) : 4);
    for (size_t r = 0; r < c.rows; r += piece) {
        const size_t n = std::min(piece, c.rows - r);
        const float* const x = c.x + r * c.width;
        float* const z = logits.as<float>();
        product(x, c.weight, z, n, c.width, c.classes, false, false);
        launch(logits_kernel<true>, dim3(grid_1d(n, 1, 16u * unsigned(d.cu_count))), dim3(kRowThreads), 0, d.stream, z, c.bias,
               c.targets + r, one_share ? shares : shares + r, one_share, int64_t(n), int64_t(c.classes),
               losses ? losses + r : nullptr);
        after_launch("linear_cross_entropy rows");
        if (grad_x) product(z, c.weight, grad_x + r * c.width, n, c.classes, c.width, false, true);
        if (grad_weight) {
            launch(counted_rows_kernel, dim3(grid_1d(n, 1, 16u * unsigned(d.cu_count))), dim3(256), 0, d.stream, x, c.targets + r,
                   rows.as<float>(), int64_t(n), int64_t(c.width), int64_t(c.classes));
            after_launch("linear_cross_entropy counted rows");
            product(rows.as<float>(), z, r ? more.as<float>() : grad_weight, c.width, n, c.classes, true, false);
            if (r) run(vc_hip_axpy(grad_weight, more.as<float>(), c.width * c.classes, 1.0f));
        }
        if (grad_bias) {
            run(vc_hip_reduce_axis(z, r ? more.as<float>() : grad_bias, 1, n, c.classes, VC_REDUCE_SUM));
            if (r) run(vc_hip_axpy(grad_bias, more.as<float>(), c.classes, 1.0f));
        }
    }
}

void count(Device& d, const Call& c, float* share) {
    launch(count_kernel, dim3(1), dim3(kCountThreads), 0, d.stream, c.targets, int64_t(c.rows), int64_t(c.classes), share);
    after_launch("linear_cross_entropy count");
}
void mean_of(Device& d, const Call& c, const float* losses, const float* share, float* mean) {
    launch(mean_kernel, dim3(1), dim3(kCountThreads), 0, d.stream, losses, int64_t(c.rows), share, mean);
    after_launch("linear_cross_entropy mean");
}

}  // namespace
}  // namespace vchip

using namespace vchip;

extern "C" {

int vc_hip_linear_xent_forward(const float* x, const float* weight, const float* bias, const float* targets, size_t rows,
                               size_t width, size_t classes, float* losses, float* mean) {
    return guard([&] {
        Device& d = require_device();
        const Call c{x, weight, bias, targets, rows, width, classes};
        check_call("linear_cross_entropy", c);
        if (rows == 0) {
            if (mean) run(vc_hip_fill(mean, 1, 0.0f));
            return;
        }
        if (!losses && !mean) return;
        const double products = 2.0 * double(rows) * double(width) * double(classes);
        Profiled p("linear_cross_entropy", products, 4.0 * double(width) * double(rows + classes));
        std::unique_ptr<Scratch> own;
        if (!losses) {
            own = std::make_unique<Scratch>(rows * sizeof(float));
            losses = own->as<float>();
        }
        forward(d, c, losses);
        if (mean) {
            Scratch share(sizeof(float));
            count(d, c, share.as<float>());
            mean_of(d, c, losses, share.as<float>(), mean);
        }
        p.done();
    });
}

int vc_hip_linear_xent_gradient(const float* x, const float* weight, const float* bias, const float* targets,
                                const float* shares, size_t rows, size_t width, size_t classes, float* mean, float* grad_x,
                                float* grad_weight, float* grad_bias) {
    return guard([&] {
        Device& d = require_device();
        const Call c{x, weight, bias, targets, rows, width, classes};
        check_call("linear_cross_entropy", c);
        if (shares && mean) fail(VC_HIP_ERR_INVALID_ARGUMENT, "linear_cross_entropy: the mean has shares of its own");
        if (rows == 0) {
            if (mean) run(vc_hip_fill(mean, 1, 0.0f));
            if (grad_weight) run(vc_hip_fill(grad_weight, width * classes, 0.0f));
            if (grad_bias) run(vc_hip_fill(grad_bias, classes, 0.0f));
            return;
        }
        const double products = 2.0 * double(rows) * double(width) * double(classes);
        Profiled p("linear_cross_entropy_gradient", products * (1.0 + (grad_x != nullptr) + (grad_weight != nullptr)),
                   8.0 * double(width) * double(rows + classes));
        Scratch share(sizeof(float)), losses(mean ? rows * sizeof(float) : 4);
        if (!shares) count(d, c, share.as<float>());
        gradient(d, c, shares ? shares : share.as<float>(), !shares, mean ? losses.as<float>() : nullptr, grad_x, grad_weight,
                 grad_bias);
        if (mean) mean_of(d, c, losses.as<float>(), share.as<float>(), mean);
        p.done();
    });
}

}  // extern "C"

#pragma once
// Layer normalisation, dropout and the cross entropy of a linear layer on the
// `cpu` device: the entry points of the same names in include/vc_hip.h, on host
// memory.
#include <cstddef>
#include <cstdint>

namespace vectorcore::cpu {

// stats: of each row times factor its mean, what the float mean is off by and 1 / deviation, then the factor: one, or the power
// of two that brings a deviation past 2^100 or below 2^-100 to where its reciprocal is a normal float. Or null.
void layer_norm_forward(const float* x, const float* weight, const float* bias, std::size_t rows, std::size_t width, float eps,
                        float* y, float* stats);
// The outputs that are null are left out.
void layer_norm_backward(const float* grad, const float* x, const float* weight, const float* stats, std::size_t rows,
                         std::size_t width, float* grad_x, float* grad_weight, float* grad_bias);

void dropout(const float* x, const float* residual, std::size_t count, double p, std::uint64_t seed, std::uint64_t stream,
             float* out);

struct LinearLoss {
    const float *x, *weight, *bias, *targets;  // bias: or null
    std::size_t rows, width, classes;
};
// One over the number of rows that count, or zero.
float linear_xent_share(const LinearLoss& call);
// losses and the gradients: or null. shares: of each row, or (one_share) of all.
void linear_xent(const LinearLoss& call, const float* shares, bool one_share, float* losses, float* grad_x, float* grad_weight,
                 float* grad_bias);
float linear_xent_mean(const float* losses, std::size_t rows, float share);

}  // namespace vectorcore::cpu

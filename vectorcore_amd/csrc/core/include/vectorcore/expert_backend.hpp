#pragma once
// The expert kernels of the `cpu` device: the entry points of the same names
// in include/vc_hip.h, on host memory.
#include <cstddef>
#include <cstdint>

namespace vectorcore::cpu {

void route_forward(const float* logits, const float* bias, std::size_t tokens, std::size_t experts, std::size_t top_k,
                   bool sigmoid, std::size_t groups, std::size_t top_groups, bool renormalise, float* weights,
                   float* chosen);
void route_backward(const float* logits, const float* chosen, const float* grad_weights, std::size_t tokens,
                    std::size_t experts, std::size_t top_k, bool sigmoid, bool renormalise, float* grad_logits);

struct ExpertRows {  // a plan's words
    std::size_t tokens, top_k, experts;
    const std::int32_t *offsets, *token, *place;
    [[nodiscard]] std::size_t rows() const { return tokens * top_k; }
};
// words: offsets [experts + 2], token [rows], place [rows].
void expert_plan_build(const float* chosen, std::size_t tokens, std::size_t top_k, std::size_t experts, std::int32_t* words);
void expert_linear_forward(const float* x, const float* w, const ExpertRows& plan, std::size_t width, std::size_t columns,
                           bool ordered, float* out);
void expert_gate_forward(const float* g, const float* u, std::size_t count, float* out);
void expert_gate_backward(const float* grad, const float* g, const float* u, std::size_t count, float* grad_gate,
                          float* grad_up);
// accumulate: adds to grad_rows instead of setting it.
void expert_linear_backward_input(const float* grad, const float* w, const ExpertRows& plan, std::size_t width,
                                  std::size_t columns, bool accumulate, float* grad_rows);
void expert_linear_backward_weight(const float* x, const float* grad, const ExpertRows& plan, std::size_t width,
                                   std::size_t columns, bool ordered, float* grad_w);
void expert_combine_forward(const float* rows, const float* weights, const ExpertRows& plan, std::size_t width, float* out);
void expert_combine_backward(const float* grad, const float* rows, const float* weights, const ExpertRows& plan,
                             std::size_t width, float* grad_rows, float* grad_weights);

void orthogonalise(const float* in, std::size_t count, std::size_t rows, std::size_t cols, std::size_t steps, float* out);
void muon_update(float* param, float* momentum, const float* grad, std::size_t count, std::size_t rows, std::size_t cols,
                 float rate, float mu, float decay, std::size_t steps);

}  // namespace vectorcore::cpu

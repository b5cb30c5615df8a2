#pragma once
// A mixture of experts: the router, the plan that sorts its picks by expert,
// the products of each expert's rows, and the sum of a token's picks; and the
// orthogonalised momentum update of weight matrices. No counterpart in the
// reference.
#include "vectorcore/storage.hpp"
#include "vectorcore/tensor.hpp"

#include <cstddef>
#include <memory>
#include <optional>
#include <vector>

namespace vectorcore {

enum class RouterScore { Softmax, Sigmoid };

struct Routed {
    Tensor weights;  // [tokens, top_k]; carries the gradient to the logits
    Tensor chosen;   // [tokens, top_k] expert numbers as float32, best first
};

struct RouteOptions {
    std::optional<Tensor> bias;  // [experts], added to the scores where experts are ranked; has no gradient
    RouterScore score = RouterScore::Softmax;
    std::size_t groups = 1;      // equal groups of neighbouring experts ...
    std::size_t top_groups = 1;  // ... of which those with the largest two best ranks stay
    bool renormalise = true;     // a token's weights sum to one
};

// The top_k experts of each row of logits [tokens, experts], at most 1024
// experts and 64 picks. Equal ranks go to the lower index, a NaN ranks first.
Routed route(const Tensor& logits, std::size_t top_k, const RouteOptions& options = {});

// The picks of chosen [tokens, top_k] sorted by expert, equal experts in pick
// order: row r of the plan's tokens * top_k rows belongs to one pick. An entry
// that is no expert number is a dropped pick: its row is zero in every result.
class ExpertPlan {
public:
    ExpertPlan(const Tensor& chosen, std::size_t experts);
    [[nodiscard]] std::size_t tokens() const { return tokens_; }
    [[nodiscard]] std::size_t top_k() const { return top_k_; }
    [[nodiscard]] std::size_t experts() const { return experts_; }
    [[nodiscard]] std::size_t rows() const { return tokens_ * top_k_; }
    [[nodiscard]] Device device() const { return words_->device(); }
    // vc_hip_expert_plan's words, as int32 bits in a float storage.
    [[nodiscard]] const Storage& words() const { return *words_; }

private:
    std::shared_ptr<Storage> words_;
    std::size_t tokens_ = 0, top_k_ = 0, experts_ = 0;
};

// [rows, columns]: each row of x times the matrix of its expert in weight
// [experts, width, columns]. x: [tokens, width], read at each row's token, or
// with `ordered` [rows, width] in the plan's order.
Tensor expert_linear(const Tensor& x, const Tensor& weight, const ExpertPlan& plan, bool ordered = false);
// silu(x @ gate[e]) * (x @ up[e]) for each row, gate and up [experts, width, columns].
Tensor expert_gated(const Tensor& x, const Tensor& gate, const Tensor& up, const ExpertPlan& plan, bool ordered = false);
// [tokens, width]: the sum of each token's rows, times its weights [tokens, top_k].
Tensor expert_combine(const Tensor& rows, const Tensor& weights, const ExpertPlan& plan);

// Each matrix of value [..., rows, cols] with its singular values brought near
// one by `steps` Newton-Schulz iterations; zeros stay zeros. Not differentiable.
Tensor orthogonalise(const Tensor& value, std::size_t steps = 5);

namespace nn {

// In place, for every parameter [..., rows, cols]: momentum = mu * momentum + g;
// p = (1 - rate * decay) * p - rate * sqrt(max(1, cols / rows)) *
// orthogonalise(g + mu * momentum). g: its entry of `gradients`, or its own
// gradient where that is empty; a parameter without one is left out. What is
// written must not overlap with anything else of the call in memory.
void muon_step(const std::vector<Tensor*>& parameters, const std::vector<Tensor*>& momenta, float rate, float mu = 0.95F,
               float decay = 0.0F, std::size_t steps = 5, const std::vector<Tensor>& gradients = {});

}  // namespace nn

}  // namespace vectorcore

#pragma once
// What stands between and behind the layers of a deep model: normalisation,
// dropout, and the loss of a last linear layer over many classes. No counterpart
// in the reference.
#include "vectorcore/tensor.hpp"

#include <cstddef>
#include <cstdint>
#include <optional>
#include <vector>

namespace vectorcore::nn {

// (x - mean) / sqrt(variance + eps) over the last axis of x, times weight, plus
// bias, both [width] or left out.
Tensor layer_norm(const Tensor& x, const std::optional<Tensor>& weight = {}, const std::optional<Tensor>& bias = {},
                  float eps = 1e-5F);

// Each element of x with probability p zero, else divided by 1 - p; plus
// residual, of x's shape, if there is one. Which elements: a function of their
// flat index, seed and stream alone (word i % 4 of Philox 4x32-10 of the counter
// (i / 4, stream) under the key seed, below round(p 2^32)), so the mask is not
// kept for the gradient, and any two calls of one (seed, stream) drop the same
// elements. p = 0 is for evaluation: x (plus residual) as it is.
Tensor dropout(const Tensor& x, double p, std::uint64_t seed, std::uint64_t stream = 0,
               const std::optional<Tensor>& residual = {});

enum class Reduction { Mean, None };

// cross_entropy(x @ weight + bias, targets) without its [rows, classes] logits:
// x [rows, width], weight [width, classes], bias [classes] or left out. A target
// is a class number as a float; a row whose target is no class number (padding,
// -1) is left out. Mean: the mean loss of the rows that count, zero if none does;
// its gradients are computed with it. None: the loss of each row, zero for one
// that is left out; the gradients compute the logits again. Large calls on the
// GPU compute products from two half-precision parts of each value, 22 bits of it,
// and take longer (by two thirds) where rows of x or W hold values that are too
// unlike each other for that, say a feature of raw size, and get three parts.
Tensor linear_cross_entropy(const Tensor& x, const Tensor& weight, const Tensor& targets, const std::optional<Tensor>& bias = {},
                            Reduction reduction = Reduction::Mean);
// The same with host targets, as cross_entropy takes them; -1 leaves a row out.
Tensor linear_cross_entropy(const Tensor& x, const Tensor& weight, const std::vector<std::int64_t>& targets,
                            const std::optional<Tensor>& bias = {}, Reduction reduction = Reduction::Mean);

}  // namespace vectorcore::nn

#include "vectorcore/expert_backend.hpp"

#include "parallel.hpp"
#include "vectorcore/cpu_backend.hpp"

#include <algorithm>
#include <cmath>
#include <limits>
#include <vector>

namespace vectorcore::cpu {

namespace {

void row_scores(const float* row, std::size_t experts, bool sigmoid, std::vector<double>& s) {
    s.resize(experts);
    if (sigmoid) {
        for (std::size_t e = 0; e < experts; ++e) s[e] = 1.0 / (1.0 + std::exp(-static_cast<double>(row[e])));
        return;
    }
    double top = -std::numeric_limits<double>::infinity(), total = 0.0;
    for (std::size_t e = 0; e < experts; ++e)
        if (row[e] > top) top = row[e];
    for (std::size_t e = 0; e < experts; ++e) total += s[e] = std::exp(row[e] - top);
    for (double& v : s) v /= total;
}

// Does rank a come before rank b, NaN first? (Equal ones keep their order.)
bool before(double a, double b) { return std::isnan(a) ? !std::isnan(b) : a > b; }

std::size_t first_best(const std::vector<double>& ranks, const std::vector<char>& open) {
    std::size_t best = ranks.size();
    for (std::size_t i = 0; i < ranks.size(); ++i)
        if (open[i] && (best == ranks.size() || before(ranks[i], ranks[best]))) best = i;
    return best;
}

// The expert of a saved pick, or one of them where another library has
// written something else there since.
std::size_t expert_of(float chosen, std::size_t experts) {
    return chosen > 0.0F ? static_cast<std::size_t>(std::min(chosen, static_cast<float>(experts - 1))) : 0;
}

float sigmoid_of(float x) {
    const float e = std::exp(-std::fabs(x));
    return (x >= 0.0F ? 1.0F : e) / (1.0F + e);
}

// The rows of x that group e's rows read, side by side.
const float* group_rows(const float* x, const ExpertRows& plan, std::size_t e, std::size_t width, bool ordered,
                        std::vector<float>& gathered) {
    const std::size_t lo = static_cast<std::size_t>(plan.offsets[e]), hi = static_cast<std::size_t>(plan.offsets[e + 1]);
    if (ordered) return x + lo * width;
    gathered.resize((hi - lo) * width);
    for (std::size_t r = lo; r < hi; ++r) {
        const float* row = x + static_cast<std::size_t>(plan.token[r]) * width;
        std::copy(row, row + width, gathered.data() + (r - lo) * width);
    }
    return gathered.data();
}

void clear_dropped(const ExpertRows& plan, std::size_t columns, float* out) {
    const std::size_t kept = static_cast<std::size_t>(plan.offsets[plan.experts]);
    std::fill(out + kept * columns, out + plan.rows() * columns, 0.0F);
}

}  // namespace

void route_forward(const float* logits, const float* bias, std::size_t tokens, std::size_t experts, std::size_t top_k,
                   bool sigmoid, std::size_t groups, std::size_t top_groups, bool renormalise, float* weights,
                   float* chosen) {
    parallel_for(tokens, std::max<std::size_t>(1, 4096 / experts), [&](std::size_t t0, std::size_t t1) {
        std::vector<double> s, ranks(experts), strength(groups);
        std::vector<char> open(experts), group_open(groups);
        const std::size_t size = experts / groups;
        for (std::size_t t = t0; t < t1; ++t) {
            row_scores(logits + t * experts, experts, sigmoid, s);
            for (std::size_t e = 0; e < experts; ++e) ranks[e] = s[e] + (bias ? static_cast<double>(bias[e]) : 0.0);
            std::fill(open.begin(), open.end(), groups == 1);
            if (groups > 1) {
                for (std::size_t g = 0; g < groups; ++g) {
                    std::vector<double> best(ranks.begin() + static_cast<std::ptrdiff_t>(g * size),
                                             ranks.begin() + static_cast<std::ptrdiff_t>((g + 1) * size));
                    std::partial_sort(best.begin(), best.begin() + static_cast<std::ptrdiff_t>(std::min<std::size_t>(2, size)),
                                      best.end(), before);
                    strength[g] = size > 1 ? best[0] + best[1] : best[0];
                }
                std::fill(group_open.begin(), group_open.end(), 1);
                for (std::size_t j = 0; j < top_groups; ++j) {
                    const std::size_t g = first_best(strength, group_open);
                    group_open[g] = 0;
                    std::fill_n(open.begin() + static_cast<std::ptrdiff_t>(g * size), size, 1);
                }
            }
            double total = 0.0;
            std::vector<double> picked(top_k);
            for (std::size_t j = 0; j < top_k; ++j) {
                const std::size_t e = first_best(ranks, open);
                open[e] = 0;
                chosen[t * top_k + j] = static_cast<float>(e);
                total += picked[j] = s[e];
            }
            for (std::size_t j = 0; j < top_k; ++j)
                weights[t * top_k + j] = static_cast<float>(renormalise ? picked[j] / total : picked[j]);
        }
    });
}

void route_backward(const float* logits, const float* chosen, const float* grad_weights, std::size_t tokens,
                    std::size_t experts, std::size_t top_k, bool sigmoid, bool renormalise, float* grad_logits) {
    parallel_for(tokens, std::max<std::size_t>(1, 4096 / experts), [&](std::size_t t0, std::size_t t1) {
        std::vector<double> s, d(experts);
        for (std::size_t t = t0; t < t1; ++t) {
            row_scores(logits + t * experts, experts, sigmoid, s);
            double total = 0.0, dot = 0.0;
            for (std::size_t j = 0; j < top_k; ++j) {
                const double p = s[expert_of(chosen[t * top_k + j], experts)];
                total += p;
                dot += p * grad_weights[t * top_k + j];
            }
            std::fill(d.begin(), d.end(), 0.0);
            for (std::size_t j = 0; j < top_k; ++j) {
                const double g = grad_weights[t * top_k + j];
                d[expert_of(chosen[t * top_k + j], experts)] = renormalise ? (g - dot / total) / total : g;
            }
            const double mean = renormalise ? 0.0 : dot;  // the renormalised gradients cancel
            for (std::size_t e = 0; e < experts; ++e) {  // (1 - s of a sigmoid is that of the negated logit)
                const double rest = sigmoid && d[e] != 0.0 ? 1.0 / (1.0 + std::exp(static_cast<double>(logits[t * experts + e]))) : 0.0;
                grad_logits[t * experts + e] = static_cast<float>(sigmoid ? d[e] * s[e] * rest : s[e] * (d[e] - mean));
            }
        }
    });
}

void expert_plan_build(const float* chosen, std::size_t tokens, std::size_t top_k, std::size_t experts, std::int32_t* words) {
    const std::size_t rows = tokens * top_k;
    std::int32_t *const offsets = words, *const token = words + experts + 2, *const place = token + rows;
    std::vector<std::int32_t> group(rows);
    std::fill(offsets, offsets + experts + 2, 0);
    for (std::size_t p = 0; p < rows; ++p) {
        const float v = chosen[p];
        const bool expert = v >= 0.0F && v < static_cast<float>(experts) && v == std::trunc(v);
        group[p] = static_cast<std::int32_t>(expert ? static_cast<std::size_t>(v) : experts);
        ++offsets[group[p] + 1];
    }
    for (std::size_t e = 0; e <= experts; ++e) offsets[e + 1] += offsets[e];
    std::vector<std::int32_t> next(offsets, offsets + experts + 1);
    for (std::size_t p = 0; p < rows; ++p) {
        const std::int32_t r = next[static_cast<std::size_t>(group[p])]++;
        token[r] = static_cast<std::int32_t>(p / top_k);
        place[p] = r;
    }
}

void expert_linear_forward(const float* x, const float* w, const ExpertRows& plan, std::size_t width, std::size_t columns,
                           bool ordered, float* out) {
    std::vector<float> gathered;
    for (std::size_t e = 0; e < plan.experts; ++e) {
        const std::size_t lo = static_cast<std::size_t>(plan.offsets[e]), n = static_cast<std::size_t>(plan.offsets[e + 1]) - lo;
        if (n == 0) continue;
        matmul(group_rows(x, plan, e, width, ordered, gathered), w + e * width * columns, out + lo * columns, n, width, columns);
    }
    clear_dropped(plan, columns, out);
}

void expert_gate_forward(const float* g, const float* u, std::size_t count, float* out) {
    parallel_for(count, 1 << 14, [&](std::size_t i0, std::size_t i1) {
        for (std::size_t i = i0; i < i1; ++i) out[i] = g[i] * sigmoid_of(g[i]) * u[i];
    });
}

void expert_gate_backward(const float* grad, const float* g, const float* u, std::size_t count, float* grad_gate,
                          float* grad_up) {
    parallel_for(count, 1 << 14, [&](std::size_t i0, std::size_t i1) {
        for (std::size_t i = i0; i < i1; ++i) {
            const float s = sigmoid_of(g[i]);
            grad_up[i] = grad[i] * (g[i] * s);
            grad_gate[i] = grad[i] * u[i] * (s * (1.0F + g[i] * (1.0F - s)));
        }
    });
}

void expert_linear_backward_input(const float* grad, const float* w, const ExpertRows& plan, std::size_t width,
                                  std::size_t columns, bool accumulate, float* grad_rows) {
    std::vector<float> product;
    for (std::size_t e = 0; e < plan.experts; ++e) {
        const std::size_t lo = static_cast<std::size_t>(plan.offsets[e]), n = static_cast<std::size_t>(plan.offsets[e + 1]) - lo;
        if (n == 0) continue;
        float* out = grad_rows + lo * width;
        if (accumulate) {
            product.resize(n * width);
            out = product.data();
        }
        matmul(grad + lo * columns, w + e * width * columns, out, n, columns, width, false, true);
        if (accumulate)
            for (std::size_t i = 0; i < n * width; ++i) grad_rows[lo * width + i] += product[i];
    }
    if (!accumulate) clear_dropped(plan, width, grad_rows);
}

void expert_linear_backward_weight(const float* x, const float* grad, const ExpertRows& plan, std::size_t width,
                                   std::size_t columns, bool ordered, float* grad_w) {
    std::vector<float> gathered;
    for (std::size_t e = 0; e < plan.experts; ++e) {
        const std::size_t lo = static_cast<std::size_t>(plan.offsets[e]), n = static_cast<std::size_t>(plan.offsets[e + 1]) - lo;
        float* out = grad_w + e * width * columns;
        if (n == 0) std::fill(out, out + width * columns, 0.0F);
        else matmul(group_rows(x, plan, e, width, ordered, gathered), grad + lo * columns, out, width, n, columns, true, false);
    }
}

void expert_combine_forward(const float* rows, const float* weights, const ExpertRows& plan, std::size_t width, float* out) {
    const std::int32_t kept = plan.offsets[plan.experts];
    parallel_for(plan.tokens, std::max<std::size_t>(1, 16384 / std::max<std::size_t>(1, width)), [&](std::size_t t0, std::size_t t1) {
        for (std::size_t t = t0; t < t1; ++t) {
            float* y = out + t * width;
            std::fill(y, y + width, 0.0F);
            for (std::size_t j = 0; j < plan.top_k; ++j) {
                const std::int32_t r = plan.place[t * plan.top_k + j];
                if (r >= kept) continue;
                const float w = weights ? weights[t * plan.top_k + j] : 1.0F;
                const float* row = rows + static_cast<std::size_t>(r) * width;
                for (std::size_t i = 0; i < width; ++i) y[i] += w * row[i];
            }
        }
    });
}

void expert_combine_backward(const float* grad, const float* rows, const float* weights, const ExpertRows& plan,
                             std::size_t width, float* grad_rows, float* grad_weights) {
    const std::int32_t kept = plan.offsets[plan.experts];
    parallel_for(plan.rows(), std::max<std::size_t>(1, 16384 / std::max<std::size_t>(1, width)), [&](std::size_t p0, std::size_t p1) {
        for (std::size_t p = p0; p < p1; ++p) {
            const std::int32_t r = plan.place[p];
            const bool dropped = r >= kept;
            const float* g = grad + p / plan.top_k * width;
            if (grad_rows)
                for (std::size_t i = 0; i < width; ++i)
                    grad_rows[static_cast<std::size_t>(r) * width + i] = dropped ? 0.0F : weights[p] * g[i];
            if (grad_weights) {
                double dot = 0.0;
                if (!dropped)
                    for (std::size_t i = 0; i < width; ++i)
                        dot += static_cast<double>(g[i]) * static_cast<double>(rows[static_cast<std::size_t>(r) * width + i]);
                grad_weights[p] = static_cast<float>(dot);
            }
        }
    });
}

void orthogonalise(const float* in, std::size_t count, std::size_t rows, std::size_t cols, std::size_t steps, float* out) {
    constexpr float a = 3.4445F, b = -4.7750F, c = 2.0315F;
    const std::size_t n = rows * cols, s = std::min(rows, cols);
    const bool wide = rows <= cols;
    std::vector<float> gram(s * s), square(s * s), y(n);
    for (std::size_t z = 0; z < count; ++z) {
        float* x = out + z * n;
        double norm = 0.0;
        for (std::size_t i = 0; i < n; ++i) norm += static_cast<double>(in[z * n + i]) * static_cast<double>(in[z * n + i]);
        const double scale = norm == 0.0 ? 0.0 : 1.0 / std::sqrt(norm);
        for (std::size_t i = 0; i < n; ++i) x[i] = static_cast<float>(in[z * n + i] * scale);
        for (std::size_t step = 0; step < steps; ++step) {
            matmul(x, x, gram.data(), s, std::max(rows, cols), s, !wide, wide);
            matmul(gram.data(), gram.data(), square.data(), s, s, s);
            for (std::size_t i = 0; i < s * s; ++i) square[i] = b * gram[i] + c * square[i];
            if (wide) matmul(square.data(), x, y.data(), rows, rows, cols);
            else matmul(x, square.data(), y.data(), rows, cols, cols);
            for (std::size_t i = 0; i < n; ++i) x[i] = a * x[i] + y[i];
        }
    }
}

void muon_update(float* param, float* momentum, const float* grad, std::size_t count, std::size_t rows, std::size_t cols,
                 float rate, float mu, float decay, std::size_t steps) {
    const std::size_t all = count * rows * cols;
    if (all == 0) return;
    std::vector<float> u(all), o(all);
    for (std::size_t i = 0; i < all; ++i) {
        momentum[i] = mu * momentum[i] + grad[i];
        u[i] = grad[i] + mu * momentum[i];
    }
    orthogonalise(u.data(), count, rows, cols, steps, o.data());
    const float scaled = rate * static_cast<float>(std::sqrt(std::max(1.0, static_cast<double>(cols) / static_cast<double>(rows))));
    for (std::size_t i = 0; i < all; ++i) param[i] = (1.0F - rate * decay) * param[i] - scaled * o[i];
}

}  // namespace vectorcore::cpu

#include "vectorcore/layer_backend.hpp"

#include "parallel.hpp"
#include "vectorcore/cpu_backend.hpp"

#include <algorithm>
#include <cmath>
#include <limits>
#include <vector>

namespace vectorcore::cpu {

namespace {

std::size_t row_grain(std::size_t width) { return std::max<std::size_t>(1, 16384 / std::max<std::size_t>(1, width)); }

struct Words {
    std::uint32_t v[4];
};

// Philox 4x32 with ten rounds (Salmon, Moraes, Dror and Shaw, 2011).
Words philox(std::uint64_t block, std::uint64_t stream, std::uint64_t seed) {
    std::uint32_t a = static_cast<std::uint32_t>(block), b = static_cast<std::uint32_t>(block >> 32);
    std::uint32_t c = static_cast<std::uint32_t>(stream), d = static_cast<std::uint32_t>(stream >> 32);
    std::uint32_t k = static_cast<std::uint32_t>(seed), l = static_cast<std::uint32_t>(seed >> 32);
    for (int round = 0; round < 10; ++round) {
        const std::uint64_t first = std::uint64_t{0xD2511F53U} * a, second = std::uint64_t{0xCD9E8D57U} * c;
        a = static_cast<std::uint32_t>(second >> 32) ^ b ^ k;
        b = static_cast<std::uint32_t>(second);
        c = static_cast<std::uint32_t>(first >> 32) ^ d ^ l;
        d = static_cast<std::uint32_t>(first);
        k += 0x9E3779B9U;
        l += 0xBB67AE85U;
    }
    return {{a, b, c, d}};
}

// The class a target names, or none (classes).
std::size_t class_of(float target, std::size_t classes) {
    if (!(target >= 0.0F && target < static_cast<float>(classes))) return classes;
    const auto c = static_cast<std::size_t>(target);
    return static_cast<float>(c) == target ? c : classes;
}

}  // namespace

void layer_norm_forward(const float* x, const float* weight, const float* bias, std::size_t rows, std::size_t width, float eps,
                        float* y, float* stats) {
    parallel_for(rows, row_grain(width), [&](std::size_t begin, std::size_t end) {
        for (std::size_t r = begin; r < end; ++r) {
            const float* row = x + r * width;
            double sum = 0.0, squares = 0.0;
            for (std::size_t c = 0; c < width; ++c) sum += row[c];
            const double mean = sum / static_cast<double>(width);
            for (std::size_t c = 0; c < width; ++c) squares += (row[c] - mean) * (row[c] - mean);
            const double deviation = std::sqrt(squares / static_cast<double>(width) + eps);
            const float factor = deviation >= 0x1p100 ? 0x1p-100F : deviation > 0.0 && deviation < 0x1p-100 ? 0x1p100F : 1.0F;
            const double centre = mean * factor;
            const float near = static_cast<float>(centre), rest = static_cast<float>(centre - near);
            const float scale = static_cast<float>(1.0 / (deviation * factor));
            for (std::size_t c = 0; c < width; ++c) {
                float h = (row[c] * factor - near - rest) * scale;
                if (weight) h *= weight[c];
                if (bias) h += bias[c];
                y[r * width + c] = h;
            }
            if (stats) {
                stats[4 * r] = near;
                stats[4 * r + 1] = rest;
                stats[4 * r + 2] = scale;
                stats[4 * r + 3] = factor;
            }
        }
    });
}

void layer_norm_backward(const float* grad, const float* x, const float* weight, const float* stats, std::size_t rows,
                         std::size_t width, float* grad_x, float* grad_weight, float* grad_bias) {
    const auto normed = [&](std::size_t r, std::size_t c) {
        return (x[r * width + c] * stats[4 * r + 3] - stats[4 * r] - stats[4 * r + 1]) * stats[4 * r + 2];
    };
    if (grad_x) {
        parallel_for(rows, row_grain(width), [&](std::size_t begin, std::size_t end) {
            for (std::size_t r = begin; r < end; ++r) {
                double first = 0.0, second = 0.0;
                const auto of = [&](std::size_t c) { return weight ? grad[r * width + c] * weight[c] : grad[r * width + c]; };
                for (std::size_t c = 0; c < width; ++c) {
                    first += of(c);
                    second += static_cast<double>(of(c)) * normed(r, c);
                }
                const float m = static_cast<float>(first / static_cast<double>(width));
                const float mh = static_cast<float>(second / static_cast<double>(width));
                for (std::size_t c = 0; c < width; ++c)
                    grad_x[r * width + c] = (of(c) - m - normed(r, c) * mh) * stats[4 * r + 2] * stats[4 * r + 3];
            }
        });
    }
    if (!grad_weight && !grad_bias) return;
    parallel_for(width, 64, [&](std::size_t begin, std::size_t end) {
        std::vector<double> dw(end - begin, 0.0), db(end - begin, 0.0);
        for (std::size_t r = 0; r < rows; ++r)
            for (std::size_t c = begin; c < end; ++c) {
                const double g = grad[r * width + c];
                dw[c - begin] += g * normed(r, c);
                db[c - begin] += g;
            }
        for (std::size_t c = begin; c < end; ++c) {
            if (grad_weight) grad_weight[c] = static_cast<float>(dw[c - begin]);
            if (grad_bias) grad_bias[c] = static_cast<float>(db[c - begin]);
        }
    });
}

void dropout(const float* x, const float* residual, std::size_t count, double p, std::uint64_t seed, std::uint64_t stream,
             float* out) {
    const auto threshold = static_cast<std::uint64_t>(std::nearbyint(p * 4294967296.0));
    const float scale = p < 1.0 ? static_cast<float>(1.0 / (1.0 - p)) : 0.0F;
    parallel_for((count + 3) / 4, 4096, [&](std::size_t begin, std::size_t end) {
        for (std::size_t block = begin; block < end; ++block) {
            const Words words = philox(block, stream, seed);
            for (std::size_t i = 4 * block; i < std::min(count, 4 * block + 4); ++i) {
                const float v = words.v[i % 4] >= threshold ? x[i] * scale : 0.0F;
                out[i] = residual ? v + residual[i] : v;
            }
        }
    });
}

float linear_xent_share(const LinearLoss& call) {
    std::size_t n = 0;
    for (std::size_t r = 0; r < call.rows; ++r) n += class_of(call.targets[r], call.classes) < call.classes;
    return n ? static_cast<float>(1.0 / static_cast<double>(n)) : 0.0F;
}

float linear_xent_mean(const float* losses, std::size_t rows, float share) {
    double sum = 0.0;
    for (std::size_t r = 0; r < rows; ++r) sum += losses[r];
    return static_cast<float>(sum * share);
}

// A piece of rows at a time: its logits, which become their gradients.
void linear_xent(const LinearLoss& call, const float* shares, bool one_share, float* losses, float* grad_x, float* grad_weight,
                 float* grad_bias) {
    const std::size_t width = call.width, classes = call.classes;
    // Eight rows or more: matmul adds the products of fewer than four one by one, and of millions of classes' in float32 the
    // small ones are lost.
    const std::size_t fitting = std::max<std::size_t>(8, (std::size_t{1} << 22) / classes);
    const std::size_t pieces = std::max<std::size_t>(1, (call.rows + fitting - 1) / fitting);
    const std::size_t piece = std::max<std::size_t>(1, (call.rows + pieces - 1) / pieces);
    const bool gradient = grad_x || grad_weight || grad_bias;
    std::vector<float> z(piece * classes), counted(grad_weight ? piece * width : 0);
    std::vector<float> part(grad_weight && call.rows > piece ? width * classes : 0);
    std::vector<double> columns(grad_bias ? classes : 0, 0.0);
    for (std::size_t first = 0; first < call.rows; first += piece) {
        const std::size_t n = std::min(piece, call.rows - first);
        matmul(call.x + first * width, call.weight, z.data(), n, width, classes);
        parallel_for(n, row_grain(classes), [&](std::size_t begin, std::size_t end) {
            for (std::size_t r = begin; r < end; ++r) {
                float* row = z.data() + r * classes;
                const std::size_t target = class_of(call.targets[first + r], classes);
                if (target == classes) {
                    if (losses) losses[first + r] = 0.0F;
                    std::fill(row, row + classes, 0.0F);
                    continue;
                }
                if (call.bias)
                    for (std::size_t c = 0; c < classes; ++c) row[c] += call.bias[c];
                float most = -std::numeric_limits<float>::infinity();
                for (std::size_t c = 0; c < classes; ++c) most = row[c] > most ? row[c] : most;
                double sum = 0.0;
                for (std::size_t c = 0; c < classes; ++c) sum += std::exp(row[c] - most);
                const float at = row[target] - most;
                if (losses) losses[first + r] = static_cast<float>(std::log(sum) - at);
                if (!gradient) continue;
                const float share = one_share ? shares[0] : shares[first + r];
                const float scale = static_cast<float>(share / sum);
                for (std::size_t c = 0; c < classes; ++c) row[c] = std::exp(row[c] - most) * scale;
                row[target] = static_cast<float>(-share * ((sum - std::exp(at)) / sum));
            }
        });
        if (!gradient) continue;
        if (grad_x && n >= 4) {
            matmul(z.data(), call.weight, grad_x + first * width, n, classes, width, false, true);
        } else if (grad_x) {
            parallel_for(n * width, row_grain(classes), [&](std::size_t begin, std::size_t end) {
                for (std::size_t i = begin; i < end; ++i) {
                    const float *row = z.data() + i / width * classes, *weight = call.weight + i % width * classes;
                    double sum = 0.0;
                    for (std::size_t c = 0; c < classes; ++c) sum += static_cast<double>(row[c]) * weight[c];
                    grad_x[first * width + i] = static_cast<float>(sum);
                }
            });
        }
        if (grad_weight) {
            // Left out rows as zeros, whatever x holds there.
            for (std::size_t r = 0; r < n; ++r) {
                const bool counts = class_of(call.targets[first + r], classes) < classes;
                const float* row = call.x + (first + r) * width;
                for (std::size_t c = 0; c < width; ++c) counted[r * width + c] = counts ? row[c] : 0.0F;
            }
            matmul(counted.data(), z.data(), first ? part.data() : grad_weight, width, n, classes, true, false);
            if (first)
                for (std::size_t i = 0; i < width * classes; ++i) grad_weight[i] += part[i];
        }
        if (grad_bias)
            for (std::size_t r = 0; r < n; ++r)
                for (std::size_t c = 0; c < classes; ++c) columns[c] += z[r * classes + c];
    }
    if (grad_weight && call.rows == 0) std::fill(grad_weight, grad_weight + width * classes, 0.0F);
    if (grad_bias)
        for (std::size_t c = 0; c < classes; ++c) grad_bias[c] = static_cast<float>(columns[c]);
}

}  // namespace vectorcore::cpu

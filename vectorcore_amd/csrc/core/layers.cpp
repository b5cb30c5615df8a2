#include "vectorcore/layers.hpp"

#include "vectorcore/autograd.hpp"
#include "vectorcore/detail/tensor_impl.hpp"
#include "vectorcore/hip_backend.hpp"
#include "vectorcore/layer_backend.hpp"
#include "vectorcore/ops.hpp"

#include <cmath>
#include <stdexcept>
#include <string>
#include <utility>

namespace vectorcore::nn {

namespace {

HipBackend& hip() { return HipBackend::instance(); }
const Storage& st(const Tensor& t) { return *t.impl()->storage; }
std::size_t off(const Tensor& t) { return t.impl()->offset; }
bool on_hip(const Tensor& t) {
    if (t.device() == Device::metal())
        throw std::runtime_error("Metal is unavailable: VectorCore was built without Apple Metal");
    return t.device() == Device::hip();
}

[[noreturn]] void reject(const std::string& message) { throw std::invalid_argument(message); }

void expect(const char* op, const char* name, const Tensor& t, const Shape& shape, Device device) {
    if (t.device() != device)
        reject(std::string(op) + ": " + name + " is on " + t.device().str() + ", expected " + device.str());
    if (t.shape() != shape)
        reject(std::string(op) + " expects " + name + " of shape " + shape_string(shape) + ", got " + shape_string(t.shape()));
}

bool wants(const std::optional<Tensor>& t) { return t && t->requires_grad(); }

// The tensors that are there, in order, as parents of a node.
std::vector<Tensor> parents_of(const Tensor& x, std::initializer_list<const std::optional<Tensor>*> others) {
    std::vector<Tensor> all{x};
    for (const auto* t : others)
        if (*t) all.push_back(**t);
    return all;
}

Tensor made(std::shared_ptr<Storage> storage, const Shape& shape) { return detail::make_tensor(std::move(storage), shape, false); }

std::optional<detail::SavedTensor> saved(const std::optional<Tensor>& t) {
    if (!t) return std::nullopt;
    return detail::SavedTensor(*t);
}

}  // namespace

Tensor layer_norm(const Tensor& x, const std::optional<Tensor>& weight, const std::optional<Tensor>& bias, float eps) {
    if (x.ndim() == 0 || x.shape().back() == 0)
        reject("layer_norm expects x with values along its last axis, got " + shape_string(x.shape()));
    if (!(eps >= 0.0F) || std::isinf(eps)) reject("layer_norm: eps must be a number from zero up");
    const std::size_t width = x.shape().back(), rows = x.numel() / width;
    if (weight) expect("layer_norm", "weight", *weight, {width}, x.device());
    if (bias) expect("layer_norm", "bias", *bias, {width}, x.device());
    const bool nx = x.requires_grad(), nw = wants(weight), nb = wants(bias);
    const bool gradient = grad_enabled() && (nx || nw || nb);
    std::shared_ptr<Storage> y, stats;
    if (on_hip(x)) {
        y = hip().layer_norm_forward(st(x), off(x), weight ? &st(*weight) : nullptr, weight ? off(*weight) : 0,
                                     bias ? &st(*bias) : nullptr, bias ? off(*bias) : 0, rows, width, eps,
                                     gradient ? &stats : nullptr);
    } else {
        y = make_cpu_storage(rows * width);
        if (gradient) stats = make_cpu_storage(4 * rows);
        cpu::layer_norm_forward(x.data(), weight ? weight->data() : nullptr, bias ? bias->data() : nullptr, rows, width, eps,
                                y->mutable_data(), stats ? stats->mutable_data() : nullptr);
    }
    Tensor out = made(std::move(y), x.shape());
    if (!gradient) return out;
    const detail::SavedTensor sx(x);
    const std::optional<detail::SavedTensor> sw = saved(weight);
    const bool has_weight = weight.has_value(), has_bias = bias.has_value();
    detail::attach_grad_fn(out, parents_of(x, {&weight, &bias}), [=](const Tensor& g) {
        const Tensor xv = sx.unpack();
        const std::optional<Tensor> wv = sw ? std::optional<Tensor>(sw->unpack()) : std::nullopt;
        std::shared_ptr<Storage> dx, dw, db;
        if (on_hip(g)) {
            hip().layer_norm_backward(st(g), off(g), st(xv), off(xv), wv ? &st(*wv) : nullptr, wv ? off(*wv) : 0, *stats, rows,
                                      width, nx ? &dx : nullptr, nw ? &dw : nullptr, nb ? &db : nullptr);
        } else {
            if (nx) dx = make_cpu_storage(rows * width);
            if (nw) dw = make_cpu_storage(width);
            if (nb) db = make_cpu_storage(width);
            cpu::layer_norm_backward(g.data(), xv.data(), wv ? wv->data() : nullptr, stats->data(), rows, width,
                                     dx ? dx->mutable_data() : nullptr, dw ? dw->mutable_data() : nullptr,
                                     db ? db->mutable_data() : nullptr);
        }
        std::vector<Tensor> grads{nx ? made(std::move(dx), xv.shape()) : Tensor()};
        if (has_weight) grads.push_back(nw ? made(std::move(dw), {width}) : Tensor());
        if (has_bias) grads.push_back(nb ? made(std::move(db), {width}) : Tensor());
        return grads;
    });
    return out;
}

namespace {

std::shared_ptr<Storage> dropped(const Tensor& x, const Tensor* residual, double p, std::uint64_t seed, std::uint64_t stream) {
    if (on_hip(x))
        return hip().dropout(st(x), off(x), residual ? &st(*residual) : nullptr, residual ? off(*residual) : 0, x.numel(), p, seed,
                             stream);
    auto out = make_cpu_storage(x.numel());
    cpu::dropout(x.data(), residual ? residual->data() : nullptr, x.numel(), p, seed, stream, out->mutable_data());
    return out;
}

}  // namespace

Tensor dropout(const Tensor& x, double p, std::uint64_t seed, std::uint64_t stream, const std::optional<Tensor>& residual) {
    if (!(p >= 0.0 && p <= 1.0)) reject("dropout: p must lie between zero and one, got " + std::to_string(p));
    if (residual) expect("dropout", "residual", *residual, x.shape(), x.device());
    if (p == 0.0) return residual ? add(*residual, x) : x;
    Tensor out = made(dropped(x, residual ? &*residual : nullptr, p, seed, stream), x.shape());
    const bool nx = x.requires_grad(), joined = residual.has_value();
    detail::attach_grad_fn(out, parents_of(x, {&residual}), [=](const Tensor& g) {
        std::vector<Tensor> grads{nx ? made(dropped(g, nullptr, p, seed, stream), g.shape()) : Tensor()};
        if (joined) grads.push_back(g);
        return grads;
    });
    return out;
}

namespace {

constexpr const char* kLoss = "linear_cross_entropy";

struct LossGradients {
    std::shared_ptr<Storage> x, weight, bias;
    bool given = false;
    // The storages have been given away: a later pass reads their values as they are now, also if they are written to.
    void keep() {
        for (auto* s : {&x, &weight, &bias})
            if (*s) *s = hip().snapshot(*s, 0, (*s)->size());
        given = true;
    }
};

// backward()'s own upstream gradient, known on the host.
bool is_one(const Tensor& g) {
    return on_hip(g) && off(g) == 0 && hip_host_scalar(st(g)) == std::optional<float>(1.0F);
}

// The gradients that are wanted, with shares of their own (null: the mean loss's, which it then leaves in *mean).
LossGradients loss_gradients(const Tensor& x, const Tensor& weight, const Tensor& targets, const std::optional<Tensor>& bias,
                             const Tensor* shares, bool nx, bool nw, bool nb, std::shared_ptr<Storage>* mean) {
    const std::size_t rows = x.shape()[0], width = x.shape()[1], classes = weight.shape()[1];
    LossGradients out;
    if (on_hip(x)) {
        hip().linear_xent_gradient(st(x), off(x), st(weight), off(weight), bias ? &st(*bias) : nullptr, bias ? off(*bias) : 0,
                                   st(targets), off(targets), shares ? &st(*shares) : nullptr, shares ? off(*shares) : 0, rows,
                                   width, classes, mean, nx ? &out.x : nullptr, nw ? &out.weight : nullptr,
                                   nb ? &out.bias : nullptr);
        return out;
    }
    if (nx) out.x = make_cpu_storage(rows * width);
    if (nw) out.weight = make_cpu_storage(width * classes);
    if (nb) out.bias = make_cpu_storage(classes);
    const cpu::LinearLoss call{x.data(), weight.data(), bias ? bias->data() : nullptr, targets.data(), rows, width, classes};
    const float share = shares ? 0.0F : cpu::linear_xent_share(call);
    std::vector<float> losses(mean ? rows : 0);
    cpu::linear_xent(call, shares ? shares->data() : &share, !shares, mean ? losses.data() : nullptr,
                     out.x ? out.x->mutable_data() : nullptr, out.weight ? out.weight->mutable_data() : nullptr,
                     out.bias ? out.bias->mutable_data() : nullptr);
    if (mean) {
        const float value = cpu::linear_xent_mean(losses.data(), rows, share);
        *mean = make_cpu_storage(&value, 1);
    }
    return out;
}

std::shared_ptr<Storage> loss_of(const Tensor& x, const Tensor& weight, const Tensor& targets, const std::optional<Tensor>& bias,
                                 bool mean) {
    const std::size_t rows = x.shape()[0], width = x.shape()[1], classes = weight.shape()[1];
    if (on_hip(x))
        return hip().linear_xent_forward(st(x), off(x), st(weight), off(weight), bias ? &st(*bias) : nullptr, bias ? off(*bias) : 0,
                                         st(targets), off(targets), rows, width, classes, mean);
    const cpu::LinearLoss call{x.data(), weight.data(), bias ? bias->data() : nullptr, targets.data(), rows, width, classes};
    auto losses = make_cpu_storage(rows);
    cpu::linear_xent(call, nullptr, false, losses->mutable_data(), nullptr, nullptr, nullptr);
    if (!mean) return losses;
    const float value = cpu::linear_xent_mean(losses->data(), rows, cpu::linear_xent_share(call));
    return make_cpu_storage(&value, 1);
}

void check_loss(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias) {
    if (x.ndim() != 2) reject(std::string(kLoss) + " expects x of shape [rows, width], got " + shape_string(x.shape()));
    if (weight.ndim() != 2)
        reject(std::string(kLoss) + " expects weight of shape [width, classes], got " + shape_string(weight.shape()));
    expect(kLoss, "weight", weight, {x.shape()[1], weight.shape()[1]}, x.device());
    if (x.shape()[1] == 0 || weight.shape()[1] == 0)
        reject(std::string(kLoss) + " expects features and classes, got " + shape_string(weight.shape()));
    if (weight.shape()[1] > (std::size_t{1} << 24))
        throw std::overflow_error(std::string(kLoss) + ": float32 class numbers reach 2^24 classes");
    if (bias) expect(kLoss, "bias", *bias, {weight.shape()[1]}, x.device());
}

}  // namespace

Tensor linear_cross_entropy(const Tensor& x, const Tensor& weight, const Tensor& targets, const std::optional<Tensor>& bias,
                            Reduction reduction) {
    check_loss(x, weight, bias);
    const std::size_t rows = x.shape()[0];
    expect(kLoss, "targets", targets, {rows}, x.device());
    const bool mean = reduction == Reduction::Mean;
    if (mean && rows == 0) reject("linear_cross_entropy of an empty batch is undefined");
    const bool nx = x.requires_grad(), nw = weight.requires_grad(), nb = wants(bias);
    const bool gradient = grad_enabled() && (nx || nw || nb);
    const Shape xs = x.shape(), ws = weight.shape();
    const bool has_bias = bias.has_value();
    std::vector<Tensor> parents{x, weight};
    if (has_bias) parents.push_back(*bias);
    const auto listed = [=](const LossGradients& g, auto&& of) {
        std::vector<Tensor> grads{nx ? of(g.x, xs) : Tensor(), nw ? of(g.weight, ws) : Tensor()};
        if (has_bias) grads.push_back(nb ? of(g.bias, Shape{ws[1]}) : Tensor());
        return grads;
    };
    if (!gradient) return made(loss_of(x, weight, targets, bias, mean), mean ? Shape{} : Shape{rows});
    if (mean) {
        std::shared_ptr<Storage> value;
        const auto unit = std::make_shared<LossGradients>(loss_gradients(x, weight, targets, bias, nullptr, nx, nw, nb, &value));
        Tensor out = made(std::move(value), {});
        detail::attach_grad_fn(out, parents, [=](const Tensor& g) {
            if (!unit->given && is_one(g)) {
                const LossGradients whole = *unit;
                unit->keep();
                return listed(whole, [](const std::shared_ptr<Storage>& s, const Shape& shape) { return made(s, shape); });
            }
            return listed(*unit, [&](const std::shared_ptr<Storage>& s, const Shape& shape) { return made(s, shape) * g; });
        });
        return out;
    }
    Tensor out = made(loss_of(x, weight, targets, bias, false), {rows});
    const detail::SavedTensor sx(x), sw(weight), stargets(targets);
    const std::optional<detail::SavedTensor> sb = saved(bias);
    detail::attach_grad_fn(out, parents, [=](const Tensor& g) {
        const std::optional<Tensor> bv = sb ? std::optional<Tensor>(sb->unpack()) : std::nullopt;
        return listed(loss_gradients(sx.unpack(), sw.unpack(), stargets.unpack(), bv, &g, nx, nw, nb, nullptr),
                      [](const std::shared_ptr<Storage>& s, const Shape& shape) { return made(s, shape); });
    });
    return out;
}

Tensor linear_cross_entropy(const Tensor& x, const Tensor& weight, const std::vector<std::int64_t>& targets,
                            const std::optional<Tensor>& bias, Reduction reduction) {
    check_loss(x, weight, bias);
    const auto classes = static_cast<std::int64_t>(weight.shape()[1]);
    if (targets.size() != x.shape()[0])
        reject(std::string(kLoss) + " received " + std::to_string(targets.size()) + " targets for a batch of " +
               std::to_string(x.shape()[0]));
    std::vector<float> numbers(targets.size());
    for (std::size_t i = 0; i < targets.size(); ++i) {
        if (targets[i] < -1 || targets[i] >= classes)
            throw std::out_of_range("target class " + std::to_string(targets[i]) + " is out of range for " +
                                    std::to_string(classes) + " classes");
        numbers[i] = static_cast<float>(targets[i]);
    }
    const std::size_t rows = numbers.size();
    return linear_cross_entropy(x, weight, Tensor(std::move(numbers), {rows}, false, x.device()), bias, reduction);
}

}  // namespace vectorcore::nn

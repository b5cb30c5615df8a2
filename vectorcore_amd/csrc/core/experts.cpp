#include "vectorcore/experts.hpp"

#include "vectorcore/autograd.hpp"
#include "vectorcore/detail/tensor_impl.hpp"
#include "vectorcore/expert_backend.hpp"
#include "vectorcore/hip_backend.hpp"

#include <cstdint>
#include <stdexcept>
#include <string>
#include <tuple>
#include <utility>

namespace vectorcore {

namespace {

constexpr std::size_t kMaxExperts = 1024, kMaxPicks = 64, kMaxGroups = 64;

[[noreturn]] void metal_unavailable() {
    throw std::runtime_error("Metal is unavailable: VectorCore was built without Apple Metal");
}
HipBackend& hip() { return HipBackend::instance(); }
const Storage& st(const Tensor& t) { return *t.impl()->storage; }
std::size_t off(const Tensor& t) { return t.impl()->offset; }
bool on_hip(const Tensor& t) {
    if (t.device() == Device::metal()) metal_unavailable();
    return t.device() == Device::hip();
}

[[noreturn]] void reject(const std::string& message) { throw std::invalid_argument(message); }

void expect_shape(const char* op, const char* name, const Tensor& t, const Shape& want) {
    if (t.shape() != want)
        reject(std::string(op) + " expects " + name + " of shape " + shape_string(want) + ", got " + shape_string(t.shape()));
}
void expect_device(const char* op, const char* name, const Tensor& t, Device want) {
    if (t.device() != want)
        reject(std::string(op) + ": " + name + " is on " + t.device().str() + ", expected " + want.str());
}

cpu::ExpertRows host_rows(const ExpertPlan& plan) {
    const auto* words = reinterpret_cast<const std::int32_t*>(plan.words().data());
    return {plan.tokens(), plan.top_k(), plan.experts(), words, words + plan.experts() + 2,
            words + plan.experts() + 2 + plan.rows()};
}
HipBackend::ExpertRows device_rows(const ExpertPlan& plan) {
    return {&plan.words(), plan.tokens(), plan.top_k(), plan.experts()};
}

// x of a product: [tokens, width], or [rows, width] in the plan's order; its width.
std::size_t check_rows(const char* op, const Tensor& x, const ExpertPlan& plan, bool ordered) {
    expect_device(op, "x", x, plan.device());
    if (x.ndim() != 2) reject(std::string(op) + " expects x of two dimensions, got " + shape_string(x.shape()));
    expect_shape(op, "x", x, {ordered ? plan.rows() : plan.tokens(), x.shape()[1]});
    return x.shape()[1];
}
std::size_t check_weight(const char* op, const char* name, const Tensor& w, const ExpertPlan& plan, std::size_t width) {
    expect_device(op, name, w, plan.device());
    if (w.ndim() != 3)
        reject(std::string(op) + " expects " + name + " of shape [experts, width, columns], got " + shape_string(w.shape()));
    expect_shape(op, name, w, {plan.experts(), width, w.shape()[2]});
    return w.shape()[2];
}

Tensor linear_rows(const Tensor& x, const Tensor& w, const ExpertPlan& plan, std::size_t width, std::size_t columns, bool ordered) {
    std::shared_ptr<Storage> out;
    if (on_hip(x)) {
        out = hip().expert_linear_forward(st(x), off(x), st(w), off(w), device_rows(plan), width, columns, ordered);
    } else {
        out = make_cpu_storage(plan.rows() * columns);
        cpu::expert_linear_forward(x.data(), w.data(), host_rows(plan), width, columns, ordered, out->mutable_data());
    }
    return detail::make_tensor(std::move(out), {plan.rows(), columns}, false);
}

// The sum over a token's rows; weights: null for all ones.
Tensor sum_rows(const Tensor& rows, const Tensor* weights, const ExpertPlan& plan, std::size_t width) {
    std::shared_ptr<Storage> out;
    if (on_hip(rows)) {
        out = hip().expert_combine_forward(st(rows), off(rows), weights ? &st(*weights) : nullptr,
                                           weights ? off(*weights) : 0, device_rows(plan), width);
    } else {
        out = make_cpu_storage(plan.tokens() * width);
        cpu::expert_combine_forward(rows.data(), weights ? weights->data() : nullptr, host_rows(plan), width,
                                    out->mutable_data());
    }
    return detail::make_tensor(std::move(out), {plan.tokens(), width}, false);
}

// The gradient of x from those of one or two products with it.
Tensor input_gradient(const Tensor& g, const Tensor& w, const Tensor* g2, const Tensor* w2, const ExpertPlan& plan,
                      std::size_t width, std::size_t columns, bool ordered) {
    std::shared_ptr<Storage> out;
    if (on_hip(g)) {
        out = hip().expert_linear_backward_input(st(g), off(g), st(w), off(w), g2 ? &st(*g2) : nullptr, g2 ? off(*g2) : 0,
                                                 w2 ? &st(*w2) : nullptr, w2 ? off(*w2) : 0, device_rows(plan), width, columns);
    } else {
        out = make_cpu_storage(plan.rows() * width);
        cpu::expert_linear_backward_input(g.data(), w.data(), host_rows(plan), width, columns, false, out->mutable_data());
        if (g2) cpu::expert_linear_backward_input(g2->data(), w2->data(), host_rows(plan), width, columns, true, out->mutable_data());
    }
    const Tensor rows = detail::make_tensor(std::move(out), {plan.rows(), width}, false);
    return ordered ? rows : sum_rows(rows, nullptr, plan, width);
}

// Of one or two matrices (g2 null: one) that multiply the same x.
std::pair<Tensor, Tensor> weight_gradients(const Tensor& x, const Tensor& g, const Tensor* g2, const ExpertPlan& plan,
                                           std::size_t width, std::size_t columns, bool ordered) {
    std::shared_ptr<Storage> out, out2;
    const std::size_t count = plan.experts() * width * columns;
    if (on_hip(g)) {
        std::tie(out, out2) = hip().expert_linear_backward_weight(st(x), off(x), st(g), off(g), g2 ? &st(*g2) : nullptr,
                                                                  g2 ? off(*g2) : 0, device_rows(plan), width, columns, ordered);
    } else {
        out = make_cpu_storage(count);
        cpu::expert_linear_backward_weight(x.data(), g.data(), host_rows(plan), width, columns, ordered, out->mutable_data());
        if (g2) {
            out2 = make_cpu_storage(count);
            cpu::expert_linear_backward_weight(x.data(), g2->data(), host_rows(plan), width, columns, ordered, out2->mutable_data());
        }
    }
    const Shape shape{plan.experts(), width, columns};
    Tensor first = detail::make_tensor(std::move(out), shape, false);
    return {first, out2 ? detail::make_tensor(std::move(out2), shape, false) : first};
}

}  // namespace

Routed route(const Tensor& logits, std::size_t top_k, const RouteOptions& o) {
    if (logits.ndim() != 2) reject("route expects [tokens, experts] logits, got " + shape_string(logits.shape()));
    const std::size_t tokens = logits.shape()[0], experts = logits.shape()[1];
    if (experts == 0 || experts > kMaxExperts)
        reject("route supports between 1 and 1024 experts, got " + std::to_string(experts));
    if (top_k == 0 || top_k > experts || top_k > kMaxPicks)
        reject("route: top_k must be between 1 and the number of experts (at most 64), got " + std::to_string(top_k) + " of " +
               std::to_string(experts));
    if (o.groups == 0 || o.groups > kMaxGroups || experts % o.groups != 0)
        reject("route: " + std::to_string(o.groups) + " groups (at most 64) do not divide " + std::to_string(experts) + " experts");
    if (o.top_groups == 0 || o.top_groups > o.groups || experts / o.groups * o.top_groups < top_k)
        reject("route: " + std::to_string(o.top_groups) + " of " + std::to_string(o.groups) + " groups cannot hold " +
               std::to_string(top_k) + " picks");
    if (o.bias) {
        expect_device("route", "bias", *o.bias, logits.device());
        expect_shape("route", "bias", *o.bias, {experts});
    }
    const bool sigmoid = o.score == RouterScore::Sigmoid, renormalise = o.renormalise;
    std::shared_ptr<Storage> w, c;
    if (on_hip(logits)) {
        std::tie(w, c) = hip().route_forward(st(logits), off(logits), o.bias ? &st(*o.bias) : nullptr, o.bias ? off(*o.bias) : 0,
                                             tokens, experts, top_k, sigmoid, o.groups, o.top_groups, renormalise);
    } else {
        w = make_cpu_storage(tokens * top_k);
        c = make_cpu_storage(tokens * top_k);
        cpu::route_forward(logits.data(), o.bias ? o.bias->data() : nullptr, tokens, experts, top_k, sigmoid, o.groups,
                           o.top_groups, renormalise, w->mutable_data(), c->mutable_data());
    }
    Routed out{detail::make_tensor(std::move(w), {tokens, top_k}, false), detail::make_tensor(std::move(c), {tokens, top_k}, false)};
    if (!grad_enabled() || !logits.requires_grad()) return out;
    const detail::SavedTensor saved(logits), picks(out.chosen);
    detail::attach_grad_fn(out.weights, {logits}, [=](const Tensor& g) {
        const Tensor x = saved.unpack(), at = picks.unpack();
        std::shared_ptr<Storage> d;
        if (on_hip(g)) {
            d = hip().route_backward(st(x), off(x), st(at), off(at), st(g), off(g), tokens, experts, top_k, sigmoid, renormalise);
        } else {
            d = make_cpu_storage(tokens * experts);
            cpu::route_backward(x.data(), at.data(), g.data(), tokens, experts, top_k, sigmoid, renormalise, d->mutable_data());
        }
        return std::vector<Tensor>{detail::make_tensor(std::move(d), {tokens, experts}, false)};
    });
    return out;
}

ExpertPlan::ExpertPlan(const Tensor& chosen, std::size_t experts) : experts_(experts) {
    if (chosen.ndim() != 2 || chosen.shape()[1] == 0)
        reject("ExpertPlan expects [tokens, top_k] expert numbers, got " + shape_string(chosen.shape()));
    if (experts == 0 || experts > kMaxExperts)
        reject("ExpertPlan supports between 1 and 1024 experts, got " + std::to_string(experts));
    tokens_ = chosen.shape()[0];
    top_k_ = chosen.shape()[1];
    if (rows() >= (std::size_t(1) << 31)) throw std::overflow_error("ExpertPlan: too many picks for int32 rows");
    if (on_hip(chosen)) {
        words_ = hip().expert_plan(st(chosen), off(chosen), tokens_, top_k_, experts);
    } else {
        words_ = make_cpu_storage(experts + 2 + 2 * rows());
        cpu::expert_plan_build(chosen.data(), tokens_, top_k_, experts, reinterpret_cast<std::int32_t*>(words_->mutable_data()));
    }
}

Tensor expert_linear(const Tensor& x, const Tensor& weight, const ExpertPlan& plan, bool ordered) {
    const std::size_t width = check_rows("expert_linear", x, plan, ordered);
    const std::size_t columns = check_weight("expert_linear", "weight", weight, plan, width);
    Tensor out = linear_rows(x, weight, plan, width, columns, ordered);
    if (!grad_enabled() || !(x.requires_grad() || weight.requires_grad())) return out;
    const detail::SavedTensor sx(x), sw(weight);
    const bool nx = x.requires_grad(), nw = weight.requires_grad();
    detail::attach_grad_fn(out, {x, weight}, [=](const Tensor& g) {
        std::vector<Tensor> grads{Tensor(), Tensor()};
        const Tensor xv = sx.unpack(), wv = sw.unpack();
        if (nx) grads[0] = input_gradient(g, wv, nullptr, nullptr, plan, width, columns, ordered);
        if (nw) grads[1] = weight_gradients(xv, g, nullptr, plan, width, columns, ordered).first;
        return grads;
    });
    return out;
}

Tensor expert_gated(const Tensor& x, const Tensor& gate, const Tensor& up, const ExpertPlan& plan, bool ordered) {
    const std::size_t width = check_rows("expert_gated", x, plan, ordered);
    const std::size_t columns = check_weight("expert_gated", "gate", gate, plan, width);
    (void)check_weight("expert_gated", "up", up, plan, width);
    expect_shape("expert_gated", "up", up, gate.shape());
    const std::size_t rows = plan.rows(), count = rows * columns;
    const bool nx = x.requires_grad(), ng = gate.requires_grad(), nu = up.requires_grad();
    const bool gradient = grad_enabled() && (nx || ng || nu);
    std::shared_ptr<Storage> out, sg, su;  // sg, su: the two products, for the backward rule
    if (on_hip(x)) {
        out = hip().expert_gated_forward(st(x), off(x), st(gate), off(gate), st(up), off(up), device_rows(plan), width, columns,
                                         ordered, gradient ? &sg : nullptr, gradient ? &su : nullptr);
    } else {
        const Tensor g = linear_rows(x, gate, plan, width, columns, ordered), u = linear_rows(x, up, plan, width, columns, ordered);
        out = make_cpu_storage(count);
        cpu::expert_gate_forward(g.data(), u.data(), count, out->mutable_data());
        sg = g.impl()->storage;
        su = u.impl()->storage;
    }
    Tensor result = detail::make_tensor(std::move(out), {rows, columns}, false);
    if (!gradient) return result;
    const detail::SavedTensor sx(x), sgate(gate), sup(up);
    detail::attach_grad_fn(result, {x, gate, up}, [=](const Tensor& g) {
        std::vector<Tensor> grads{Tensor(), Tensor(), Tensor()};
        const Tensor xv = sx.unpack(), gv = sgate.unpack(), uv = sup.unpack();
        std::shared_ptr<Storage> dg, du;
        if (on_hip(g)) {
            std::tie(dg, du) = hip().expert_gated_backward(st(g), off(g), *sg, *su, count);
        } else {
            dg = make_cpu_storage(count);
            du = make_cpu_storage(count);
            cpu::expert_gate_backward(g.data(), sg->data(), su->data(), count, dg->mutable_data(), du->mutable_data());
        }
        const Tensor dgt = detail::make_tensor(std::move(dg), {rows, columns}, false);
        const Tensor dut = detail::make_tensor(std::move(du), {rows, columns}, false);
        if (nx) grads[0] = input_gradient(dgt, gv, &dut, &uv, plan, width, columns, ordered);
        if (ng || nu) std::tie(grads[1], grads[2]) = weight_gradients(xv, ng ? dgt : dut, ng && nu ? &dut : nullptr, plan, width, columns, ordered);
        return grads;
    });
    return result;
}

Tensor expert_combine(const Tensor& rows, const Tensor& weights, const ExpertPlan& plan) {
    const std::size_t width = check_rows("expert_combine", rows, plan, true);
    expect_device("expert_combine", "weights", weights, plan.device());
    expect_shape("expert_combine", "weights", weights, {plan.tokens(), plan.top_k()});
    Tensor out = sum_rows(rows, &weights, plan, width);
    if (!grad_enabled() || !(rows.requires_grad() || weights.requires_grad())) return out;
    const detail::SavedTensor sr(rows), sw(weights);
    const bool nr = rows.requires_grad(), nw = weights.requires_grad();
    detail::attach_grad_fn(out, {rows, weights}, [=](const Tensor& g) {
        std::vector<Tensor> grads{Tensor(), Tensor()};
        const Tensor rv = sr.unpack(), wv = sw.unpack();
        std::shared_ptr<Storage> dr, dw;
        if (on_hip(g)) {
            std::tie(dr, dw) = hip().expert_combine_backward(st(g), off(g), st(rv), off(rv), st(wv), off(wv), device_rows(plan),
                                                             width, nr, nw);
        } else {
            if (nr) dr = make_cpu_storage(plan.rows() * width);
            if (nw) dw = make_cpu_storage(plan.rows());
            cpu::expert_combine_backward(g.data(), rv.data(), wv.data(), host_rows(plan), width,
                                         dr ? dr->mutable_data() : nullptr, dw ? dw->mutable_data() : nullptr);
        }
        if (dr) grads[0] = detail::make_tensor(std::move(dr), {plan.rows(), width}, false);
        if (dw) grads[1] = detail::make_tensor(std::move(dw), {plan.tokens(), plan.top_k()}, false);
        return grads;
    });
    return out;
}

}  // namespace vectorcore

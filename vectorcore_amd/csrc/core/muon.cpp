#include "vectorcore/autograd.hpp"
#include "vectorcore/detail/tensor_impl.hpp"
#include "vectorcore/expert_backend.hpp"
#include "vectorcore/experts.hpp"
#include "vectorcore/hip_backend.hpp"

#include <algorithm>
#include <cstdint>
#include <stdexcept>
#include <string>
#include <unordered_set>
#include <utility>

namespace vectorcore {

namespace {

struct Matrices {
    std::size_t count, rows, cols;
};

Matrices matrices_of(const char* op, const Shape& shape) {
    if (shape.size() < 2)
        throw std::invalid_argument(std::string(op) + " takes matrices [..., rows, cols], got " + shape_string(shape));
    return {numel(Shape(shape.begin(), shape.end() - 2)), shape[shape.size() - 2], shape.back()};
}

// The memory of a tensor of n > 0 elements.
struct Range {
    std::uintptr_t begin, end;
    bool writes;
};
Range range_of(const Tensor& t, std::size_t n, bool writes) {
    const float* const data = t.device() == Device::hip() ? HipBackend::instance().address(*t.impl()->storage) + t.impl()->offset
                                                           : t.data();
    const auto begin = reinterpret_cast<std::uintptr_t>(data);
    return {begin, begin + n * sizeof(float), writes};
}

void require_known(Device device) {
    if (device == Device::metal())
        throw std::runtime_error("Metal is unavailable: VectorCore was built without Apple Metal");
}

}  // namespace

Tensor orthogonalise(const Tensor& value, std::size_t steps) {
    const Matrices m = matrices_of("orthogonalise", value.shape());
    require_known(value.device());
    std::shared_ptr<Storage> out;
    if (value.device() == Device::hip()) {
        out = HipBackend::instance().orthogonalise(*value.impl()->storage, value.impl()->offset, m.count, m.rows, m.cols, steps);
    } else {
        out = make_cpu_storage(value.numel());
        cpu::orthogonalise(value.data(), m.count, m.rows, m.cols, steps, out->mutable_data());
    }
    return detail::make_tensor(std::move(out), value.shape(), false);
}

namespace nn {

void muon_step(const std::vector<Tensor*>& parameters, const std::vector<Tensor*>& momenta, float rate, float mu, float decay,
               std::size_t steps, const std::vector<Tensor>& gradients) {
    if (parameters.size() != momenta.size())
        throw std::invalid_argument("muon_step: " + std::to_string(momenta.size()) + " momenta for " +
                                    std::to_string(parameters.size()) + " parameters");
    if (!gradients.empty() && gradients.size() != parameters.size())
        throw std::invalid_argument("muon_step: " + std::to_string(gradients.size()) + " gradients for " +
                                    std::to_string(parameters.size()) + " parameters");
    if (steps == 0) throw std::invalid_argument("muon_step needs at least one step");
    NoGradGuard guard;
    struct Item {
        Tensor *param, *momentum;
        Tensor grad;
        Matrices shape;
    };
    // Everything is checked before anything is written.
    std::vector<Item> items;
    std::unordered_set<const Storage*> written;
    for (std::size_t i = 0; i < parameters.size(); ++i) {
        Tensor *p = parameters[i], *m = momenta[i];
        if (!p || (gradients.empty() && !p->has_grad())) continue;
        if (!m) throw std::invalid_argument("muon_step: a parameter without a momentum");
        const Tensor g = gradients.empty() ? p->grad() : gradients[i];
        const Matrices shape = matrices_of("muon_step", p->shape());
        require_known(p->device());
        if (g.shape() != p->shape() || g.device() != p->device())
            throw std::invalid_argument("parameter gradient shape or device does not match");
        if (m->shape() != p->shape() || m->device() != p->device())
            throw std::invalid_argument("parameter momentum shape or device does not match");
        if (!written.insert(p->impl()->storage.get()).second || !written.insert(m->impl()->storage.get()).second)
            throw std::invalid_argument("muon_step: parameters and momenta must not share storage");
        items.push_back({p, m, g, shape});
    }
    for (const Item& it : items)
        if (written.count(it.grad.impl()->storage.get()))
            throw std::invalid_argument("muon_step: a gradient shares storage with a parameter or momentum");
    // Storages taken from another library may lie over the same memory.
    std::vector<Range> ranges;
    for (const Item& it : items)
        for (const auto& [tensor, writes] : {std::pair<const Tensor*, bool>{it.param, true}, {it.momentum, true}, {&it.grad, false}})
            if (const std::size_t n = tensor->numel()) ranges.push_back(range_of(*tensor, n, writes));
    std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
    std::uintptr_t end = 0, written_end = 0;  // of what lies before
    for (const Range& r : ranges) {
        if (r.begin < (r.writes ? end : written_end))
            throw std::invalid_argument("muon_step: parameters, momenta and gradients must not overlap in memory");
        end = std::max(end, r.end);
        if (r.writes) written_end = std::max(written_end, r.end);
    }
    std::vector<HipBackend::MuonItem> batch;
    for (const Item& it : items) {
        const auto &p = it.param->impl(), &m = it.momentum->impl(), &g = it.grad.impl();
        if (it.param->device() == Device::hip()) {
            batch.push_back({p->storage.get(), p->offset, m->storage.get(), m->offset, g->storage.get(), g->offset,
                             it.shape.count, it.shape.rows, it.shape.cols});
        } else {
            cpu::muon_update(it.param->mutable_data(), it.momentum->mutable_data(), it.grad.data(), it.shape.count,
                             it.shape.rows, it.shape.cols, rate, mu, decay, steps);
        }
    }
    if (batch.empty()) return;
    HipBackend::instance().muon_step(batch, rate, mu, decay, steps);
    for (const auto& it : batch) {
        it.param->bump_version();
        it.momentum->bump_version();
    }
}

}  // namespace nn

}  // namespace vectorcore

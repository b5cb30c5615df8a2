#pragma once
// Storage with the in-place version counter (API of include/vectorcore/storage.hpp).
#include "vectorcore/device.hpp"

#include <cstddef>
#include <cstdint>
#include <functional>
#include <memory>

namespace vectorcore {

class Storage {
public:
    virtual ~Storage() = default;
    [[nodiscard]] virtual Device device() const noexcept = 0;
    [[nodiscard]] virtual std::size_t size() const noexcept = 0;
    // Host-addressable data; device storages throw std::runtime_error.
    [[nodiscard]] virtual const float* data() const;
    [[nodiscard]] virtual float* mutable_data();

    // Shared by every view of the storage. Autograd records it when a tensor
    // is saved for backward and rejects the backward if it changed.
    [[nodiscard]] std::uint64_t version() const noexcept { return version_; }
    void bump_version() noexcept { ++version_; }

    // May another library hold the memory's address? What is to stay must then
    // not be this storage. (Of the hip device: until the library has let go.)
    [[nodiscard]] virtual bool shared() const { return shared_; }
    void set_shared() noexcept { shared_ = true; }

private:
    std::uint64_t version_{0};
    bool shared_ = false;
};

std::shared_ptr<Storage> make_cpu_storage(std::size_t elements);
std::shared_ptr<Storage> make_cpu_storage(const float* values, std::size_t elements);
// A storage over host memory that its owner keeps until `release` is called.
std::shared_ptr<Storage> adopt_cpu_storage(float* values, std::size_t elements, std::function<void()> release);

}  // namespace vectorcore

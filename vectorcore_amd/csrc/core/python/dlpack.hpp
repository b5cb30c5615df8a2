#pragma once
// Tensors shared with other libraries by the DLPack protocol
// (__dlpack__ / __dlpack_device__), without a copy: float32, contiguous, in
// host memory (the cpu device) or on the GPU (hip). The structures are those
// that the protocol fixes.
//
// Order of work: the hip device works on a stream of its own. An import makes
// it wait for what the producer's stream holds then, and an export makes the
// consumer's wait for what the hip device's holds then. Nothing orders what
// either side enqueues later: before one side writes memory that the other may
// still read, or reads what the other has written since, the program imports
// (the other side's work first) or exports (this side's first) the tensor again,
// or synchronises. Work asked for here counts as enqueued: none that reads
// shared memory stays recorded. Versions count the writes made here alone, so an
// operand that autograd has saved must not be written by the other side before
// the backward pass. A buffer that the other side frees is kept until the work
// enqueued on it is done.
#include "vectorcore/detail/tensor_impl.hpp"
#include "vectorcore/hip_backend.hpp"
#include "vectorcore/vectorcore.hpp"

#include "vc_hip.h"

#include <link.h>
#include <pybind11/pybind11.h>

#include <cstdint>
#include <memory>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

namespace vectorcore::dlpack {

namespace py = pybind11;

constexpr std::int32_t kCpu = 1, kRocm = 10;
constexpr std::uint8_t kFloat = 2;

struct DLDevice {
    std::int32_t type, id;
};
struct DLDataType {
    std::uint8_t code, bits;
    std::uint16_t lanes;
};
struct DLTensor {
    void* data;
    DLDevice device;
    std::int32_t ndim;
    DLDataType dtype;
    std::int64_t* shape;
    std::int64_t* strides;  // in elements, null for a contiguous tensor
    std::uint64_t byte_offset;
};
struct DLManagedTensor {
    DLTensor tensor;
    void* context;
    void (*deleter)(DLManagedTensor*);
};

inline void check(int status) {
    if (status != VC_HIP_OK) throw std::runtime_error(vc_hip_last_error());
}

// Streams mean nothing to another copy of the HIP runtime, and torch brings its
// own: loaded first it also serves this library, loaded later it is a second one.
inline void require_one_runtime() {
    struct Loaded {
        unsigned long long adds = ~0ULL;  // libraries ever loaded when the copies were counted
        int copies = 0;
    };
    static Loaded known;  // under the interpreter's lock
    unsigned long long adds = 0;
    dl_iterate_phdr(
        [](dl_phdr_info* info, std::size_t, void* out) {
            *static_cast<unsigned long long*>(out) = info->dlpi_adds;
            return 1;
        },
        &adds);
    if (adds != known.adds) {
        int copies = 0;
        dl_iterate_phdr(
            [](dl_phdr_info* info, std::size_t, void* out) {
                const std::string path = info->dlpi_name ? info->dlpi_name : "";
                if (path.compare(path.rfind('/') + 1, 14, "libamdhip64.so") == 0) ++*static_cast<int*>(out);
                return 0;
            },
            &copies);
        known = {adds, copies};
    }
    if (known.copies > 1)
        throw std::runtime_error("this process has loaded two HIP runtimes: import torch before vectorcore_amd to share "
                                 "GPU memory with it");
}

// The tensor of a "dltensor" capsule, which is used up.
inline Tensor take(const py::object& capsule) {
    if (!PyCapsule_IsValid(capsule.ptr(), "dltensor"))
        throw std::invalid_argument("from_dlpack: __dlpack__ gave no unused DLPack capsule");
    auto* managed = static_cast<DLManagedTensor*>(PyCapsule_GetPointer(capsule.ptr(), "dltensor"));
    const DLTensor& t = managed->tensor;
    // Until the capsule is renamed, it owns the tensor and frees it on an error.
    if (t.dtype.code != kFloat || t.dtype.bits != 32 || t.dtype.lanes != 1)
        throw std::invalid_argument("from_dlpack takes float32 tensors");
    if (t.device.type != kCpu && (t.device.type != kRocm || t.device.id != 0))
        throw std::invalid_argument("from_dlpack takes tensors in host memory or on the first ROCm GPU");
    Shape shape;
    for (std::int32_t i = 0; i < t.ndim; ++i) shape.push_back(static_cast<std::size_t>(t.shape[i]));
    const std::size_t count = numel(shape);
    if (t.strides && count > 1) {
        std::int64_t want = 1;
        for (std::int32_t i = t.ndim - 1; i >= 0; --i) {
            if (t.shape[i] != 1 && t.strides[i] != want)
                throw std::invalid_argument("from_dlpack takes contiguous tensors");
            want *= t.shape[i];
        }
    }
    auto* data = reinterpret_cast<float*>(static_cast<char*>(t.data) + t.byte_offset);
    if (reinterpret_cast<std::uintptr_t>(data) % alignof(float) != 0)
        throw std::invalid_argument("from_dlpack takes tensors aligned to their elements");
    if (count == 0)  // nothing to share: the capsule frees the tensor
        return Tensor({}, shape, false, t.device.type == kCpu ? Device::cpu() : Device::hip());
    const auto release = [managed] {
        if (managed->deleter) managed->deleter(managed);
    };
    if (t.device.type == kRocm) require_one_runtime();
    std::shared_ptr<Storage> storage = t.device.type == kCpu ? adopt_cpu_storage(data, count, release)
                                                             : HipBackend::instance().adopt(data, count, release);
    PyCapsule_SetName(capsule.ptr(), "used_dltensor");
    return detail::make_tensor(std::move(storage), std::move(shape), false);
}

inline std::uint64_t own_stream() {
    std::uint64_t stream = 0;
    check(vc_hip_stream(&stream));
    return stream;
}

// What is called of torch, looked up once it is loaded; never freed, as the
// interpreter may be gone before static objects are.
struct Torch {
    py::object tensor, to_dlpack, stream_of, current_stream;
    static const Torch* loaded() {
        static const Torch* known = nullptr;  // under the interpreter's lock
        if (!known) {
            const py::object torch = py::reinterpret_borrow<py::object>(PyImport_GetModuleDict()).attr("get")("torch", py::none());
            if (torch.is_none() || !py::hasattr(torch, "utils") || !py::hasattr(torch, "cuda")) return nullptr;  // or half loaded
            const py::object c = torch.attr("_C");
            // The stream's handle itself where torch offers it: it costs a tenth of the stream object.
            known = new Torch{torch.attr("Tensor"), torch.attr("utils").attr("dlpack").attr("to_dlpack"),
                              py::getattr(c, "_cuda_getCurrentRawStream", py::none()), torch.attr("cuda").attr("current_stream")};
        }
        return known;
    }
    [[nodiscard]] std::uint64_t stream() const {
        return (stream_of.is_none() ? current_stream().attr("cuda_stream") : stream_of(0)).cast<std::uint64_t>();
    }
};

// Tensors over the memory of `objects`, which have __dlpack__. torch's are
// exported without a wait of their own: they are all ordered by torch's current
// stream, which is waited for once.
inline py::tuple import_(const py::args& objects) {
    const Torch* const torch = Torch::loaded();
    bool waited = false;
    py::tuple out(objects.size());
    for (std::size_t i = 0; i < objects.size(); ++i) {
        const py::object object = objects[i];
        py::object capsule;
        if (torch && py::isinstance(object, torch->tensor)) {
            if (object.attr("requires_grad").cast<bool>())
                throw std::invalid_argument("from_dlpack: detach() a torch tensor that requires gradients");
            if (object.attr("is_neg")().cast<bool>())  // its memory holds the negated values
                throw std::invalid_argument("from_dlpack: resolve_neg() a torch tensor that is a negative view");
            if (!waited && object.attr("is_cuda").cast<bool>()) {
                waited = true;
                require_one_runtime();
                check(vc_hip_wait_for_stream(torch->stream()));
            }
            capsule = torch->to_dlpack(object);
        } else {
            const py::tuple device = object.attr("__dlpack_device__")();
            capsule = device[0].cast<int>() == kRocm ? object.attr("__dlpack__")(py::arg("stream") = own_stream())
                                                     : object.attr("__dlpack__")();
        }
        out[i] = py::cast(take(capsule));
    }
    return out;
}

inline std::pair<int, int> device_of(const Tensor& t) {
    return {t.device() == Device::hip() ? kRocm : kCpu, 0};
}

// A capsule of the tensor's own memory. stream: the consumer's, made to wait
// for the work enqueued here (None: the default stream, -1: nothing waits);
// once the consumer lets go, later work here waits for what is on it then.
inline py::capsule export_(const Tensor& t, const py::object& stream, const py::object& device, const py::object& copy) {
    if (t.requires_grad()) throw std::runtime_error("detach() a tensor that requires gradients before exporting it");
    if (!t.is_contiguous()) throw std::runtime_error("__dlpack__ requires contiguous storage");
    if (!copy.is_none() && copy.cast<bool>()) throw std::runtime_error("__dlpack__ shares memory: no copy can be asked for");
    const auto [type, id] = device_of(t);
    if (!device.is_none() && device.cast<std::pair<int, int>>() != std::make_pair(type, id))
        throw std::runtime_error("__dlpack__ exports to the tensor's own device");
    struct Exported {
        DLManagedTensor managed;
        std::shared_ptr<Storage> storage;
        std::vector<std::int64_t> shape, strides;
        bool ordered = false;
        std::uint64_t stream = 0;
    };
    auto e = std::make_unique<Exported>();
    e->storage = t.impl()->storage;
    float* data = nullptr;
    if (type == kRocm) {
        require_one_runtime();
        const std::int64_t consumer = stream.is_none() ? 0 : stream.cast<std::int64_t>();
        if (consumer < -1) throw std::runtime_error("__dlpack__: a stream is a handle, 0 or -1");
        data = HipBackend::instance().expose(*e->storage);
        if (consumer != -1) {
            e->ordered = true;
            e->stream = static_cast<std::uint64_t>(consumer);
            check(vc_hip_release_to_stream(e->stream));
        }
    } else {
        if (!stream.is_none()) throw std::runtime_error("__dlpack__: a tensor in host memory has no stream");
        data = e->storage->mutable_data();
        e->storage->set_shared();
    }
    e->shape.assign(t.shape().begin(), t.shape().end());
    e->strides.assign(t.strides().begin(), t.strides().end());
    e->managed.tensor = {data + t.impl()->offset, {type, id}, static_cast<std::int32_t>(e->shape.size()), {kFloat, 32, 1},
                         e->shape.data(), e->strides.data(), 0};
    e->managed.context = e.get();
    e->managed.deleter = [](DLManagedTensor* m) {
        const std::unique_ptr<Exported> mine(static_cast<Exported*>(m->context));
        // The buffer's next use here comes after the consumer's last one.
        if (mine->ordered) (void)vc_hip_wait_for_stream(mine->stream);
        if (mine->managed.tensor.device.type == kRocm) HipBackend::instance().conceal(*mine->storage);
    };
    py::capsule out(&e->managed, "dltensor", [](PyObject* capsule) {
        if (!PyCapsule_IsValid(capsule, "dltensor")) return;  // taken
        auto* m = static_cast<DLManagedTensor*>(PyCapsule_GetPointer(capsule, "dltensor"));
        m->deleter(m);
    });
    (void)e.release();
    return out;
}

}  // namespace vectorcore::dlpack

// What the dispatcher kernels of torch_binding.cpp and torch_binding_layer.cpp share.
#pragma once

#include <ATen/Context.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/native/TensorFactories.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/library.h>

#include <cstring>
#include <optional>
#include <tuple>

#include "../../include/hstu_mi355.h"

namespace ops_rec_binding {

namespace py = pybind11;

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

template <typename R, typename... A>
R in_python(PyObject* fn, const A&... args)
{
    py::gil_scoped_acquire gil;
    TORCH_CHECK(fn != nullptr, "ops_rec: the Python implementations have not been attached");
    return py::reinterpret_borrow<py::object>(fn)(args...).template cast<R>();
}

inline int dtype_code(at::ScalarType t)
{
    switch (t) {
    case at::kBFloat16: return HSTU_DT_BF16;
    case at::kHalf: return HSTU_DT_FP16;
    case at::kFloat: return HSTU_DT_FP32;
    case at::kFloat8_e4m3fn: return HSTU_DT_FP8_E4M3;
    default: return -1;
    }
}

// torch.empty without its way through the dispatcher: memory nobody has written yet holds NaN (all ones) when the program has asked
// for that (torch.use_deterministic_algorithms with torch.utils.deterministic.fill_uninitialized_memory)
inline Tensor empty(at::IntArrayRef size, at::ScalarType dtype, const at::Device& device)
{
    Tensor t(at::detail::empty_cuda(size, dtype, device, std::nullopt));
    const at::Context& context = at::globalContext();
    if (context.deterministicAlgorithms() && context.deterministicFillUninitializedMemory()) {
        at::native::fill_empty_deterministic_(t);
    }
    return t;
}

// A workspace a call can do without: none (undefined) when the allocator has no room for it.
inline Tensor empty_or_none(uint64_t bytes, const at::Device& device)
{
    if (bytes != 0) {
        try {
            return empty({static_cast<int64_t>(bytes)}, at::kByte, device);
        } catch (const c10::OutOfMemoryError&) {
        }
    }
    return Tensor();
}

inline void* ptr(const Tensor& t) { return t.defined() && t.numel() != 0 ? t.data_ptr() : nullptr; }
inline void* ptr(const OptTensor& t) { return t.has_value() ? ptr(*t) : nullptr; }

inline bool is_set(const OptTensor& t) { return t.has_value() && t->defined(); }

inline hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

template <typename F>
auto operator_handle(const char* name, const char* overload)
{
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, overload).typed<F>();
}

inline bool needs_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
inline bool needs_grad(const OptTensor& t) { return t.has_value() && needs_grad(*t); }

// Forward-mode differentiation: operators without a formula for it refuse a tangent, which would be lost below autograd.
inline bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
inline bool has_tangent(const OptTensor& t) { return t.has_value() && has_tangent(*t); }
template <typename... T>
void refuse_tangents(const char* op, const T&... inputs)
{
    TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(inputs) || ...), op, ": forward-mode differentiation is not implemented; do not pass inputs with a tangent");
}

inline Tensor unwrap(const OptTensor& t) { return t.value_or(Tensor()); }
inline OptTensor wrap(const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; }

// a tensor as the kernels read it (a view that is not contiguous is copied, as the Python implementations do)
inline const Tensor contiguous(const Tensor& t) { return t.is_contiguous() ? t : t.contiguous(); }

// the operators around attention (torch_binding_layer.cpp): the setter of their Python implementations
void define_layer(py::module_& m);

}  // namespace ops_rec_binding

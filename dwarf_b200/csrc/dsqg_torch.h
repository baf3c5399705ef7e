// What the files of the native host side share: checks, allocation, streams, errors (see dsqg_torch.cpp).
#pragma once

#include <torch/extension.h>

#include <ATen/autocast_mode.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/Exceptions.h>

#include <optional>
#include <sstream>

#include "dsqg_b200.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// An offset set, converted once and kept for the life of the process (programs use a handful): autograd nodes and
// the Python cache (ops._offsets) hold plain pointers to it.
struct Offsets {
    std::vector<int32_t> v;
    int J() const { return (int)v.size(); }
};

// Raises dwarf_b200.DSQGError for a non-zero status.
inline void check(int status, const char* where) {
    if (status == DSQG_OK) return;
    py::gil_scoped_acquire gil;
    py::module_::import("dwarf_b200._lib").attr("check")(status, where);
    throw std::runtime_error(std::string(where) + " failed");
}

// Runs the body of a backward node: the autograd engine's threads carry Python errors in its own exception type, and start
// without a CUDA context, which cuBLAS would remark on.
template <typename F> auto backward_body(const Tensor& on, F f) {
    static thread_local int ready = -1;
    if (on.defined() && on.is_cuda() && ready != on.device().index()) {
        ready = on.device().index();
        const int before = c10::cuda::current_device();
        c10::cuda::SetDevice(ready, /*force=*/true);
        c10::cuda::SetDevice(before);
    }
    try {
        return f();
    } catch (py::error_already_set& e) {
        py::gil_scoped_acquire gil;
        e.restore();
        python_error err;
        err.persist();
        throw err;
    }
}

inline int dtype_code(const Tensor& t) {
    if (t.scalar_type() == at::kBFloat16) return DSQG_DTYPE_BF16;
    if (t.scalar_type() == at::kFloat) return DSQG_DTYPE_F32;
    throw py::type_error(std::string("dsqg: q/k/v must be bfloat16 or float32, got ") + toString(t.scalar_type()));
}

inline std::string shape_of(const Tensor& t) {
    std::ostringstream s;
    s << t.sizes();
    return s.str();
}

inline void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
inline float* fptr(const Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; }
inline void* stream_of(const Tensor& t) { return at::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// Uninitialised device tensors straight from the allocator: a dispatched at::empty costs 2.6 us on an autograd thread, this
// one less than a third, and a backward call makes six.
inline Tensor new_tensor(at::IntArrayRef sizes, at::ScalarType dt, const Tensor& on) { return at::detail::empty_cuda(sizes, dt, on.device(), std::nullopt); }
inline Tensor new_like(const Tensor& t) { return t.defined() ? new_tensor(t.sizes(), t.scalar_type(), t) : t; }

// A parameter as the kernels read it: fp32 and contiguous (no copy where it is so already; it may be the caller's own tensor).
inline Tensor f32c(const Tensor& t) {
    if (!t.defined() || (t.scalar_type() == at::kFloat && t.is_contiguous())) return t;
    return t.detach().to(at::kFloat).contiguous();
}
// The kernels around the GEMMs and the GEMM plans want 16-byte pointers; a parameter that is a view of a flat buffer, or a caller's
// activation, may start anywhere and is copied then.
inline bool on_16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline Tensor aligned(const Tensor& t) { return !t.defined() || on_16(t.data_ptr()) ? t : t.detach().clone(); }
inline Tensor like_param(Tensor g, at::ScalarType dt) { return g.defined() && g.scalar_type() != dt ? g.to(dt) : g; }
inline Tensor opt(const std::optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }
inline at::ScalarType type_of(const Tensor& t) { return t.defined() ? t.scalar_type() : at::kFloat; }

inline bool shape_is(const Tensor& t, std::initializer_list<int64_t> s) { return t.sizes() == at::IntArrayRef(s); }

// The kernels get plain pointers: a tensor on the host or on another GPU would be read as if it were on this one.
inline void check_device(const char* who, const Tensor& on, std::initializer_list<const Tensor*> ts) {
    for (const Tensor* t : ts)
        if (t->defined() && t->device() != on.device()) throw py::value_error(std::string(who) + ": all tensors must be on " + on.device().str() + ", got one on " + t->device().str());
}

// Scratch for one call, returned to the caching allocator when it leaves scope.
inline at::DataPtr scratch_for(size_t bytes) { return c10::cuda::CUDACachingAllocator::get()->allocate(bytes); }

inline bool wants_grad(std::initializer_list<const Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

void bind_serving(py::module_& m);       // dsqg_torch_serving.cpp

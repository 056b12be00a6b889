// What the operators on torch tensors share (torch_ops.cc, vocabulary_ops.cc): checks of arguments, calls of the C interface, nodes of autograd.
#pragma once

#include "torch_ops.h"

#include <ATen/autocast_mode.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <cstdint>
#include <initializer_list>
#include <memory>
#include <optional>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

namespace b200ccl::python {

inline PyObject* g_error_class = nullptr;
inline const char* (*g_last_error)() = nullptr;

// What a call is refused for, and what it failed of. In a backward pass there is no Python frame to raise in: see in_backward().
struct Refused : std::invalid_argument {
    using std::invalid_argument::invalid_argument;
};
struct Failed : std::runtime_error {
    using std::runtime_error::runtime_error;
};
// A Python error is set.
struct Raised {};

[[noreturn]] inline void refuse(const std::string& why) { throw Refused(why); }

inline void need_arguments(Py_ssize_t got, Py_ssize_t want) {
    if (got == want) return;
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, got);
    throw Raised{};
}

inline int dtype_code(const char* what, const at::Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return 0;
        case at::kHalf: return 1;
        case at::kBFloat16: return 2;
        default: refuse(std::string(what) + " has dtype " + c10::toString(t.scalar_type()) + ": float32, float16 and bfloat16 are supported");
    }
}

inline const at::Tensor& on_gpu(const char* what, const at::Tensor& t) {
    // Fake tensors, subclasses that stand for other tensors, those inside torch.func's transformations.
    constexpr c10::DispatchKeySet kWrapped({c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize});
    if (t.unsafeGetTensorImpl()->is_python_dispatch() || t.key_set().has_any(kWrapped) || !t.has_storage())
        refuse(std::string(what) + " has no memory of its own: these operators know plain tensors only, and no transformations of them");
    if (!t.is_cuda() || t.layout() != at::kStrided) refuse(std::string(what) + " must be a dense CUDA tensor");
    if (t.is_neg()) refuse(std::string(what) + " is a view that stands for its negative: resolve_neg() makes a tensor of it");
    if (t._fw_grad(/*level=*/0).defined()) refuse(std::string(what) + " has a tangent: these operators have no forward-mode derivative");
    return t;
}
inline const at::Tensor& tensor_of(const char* what, PyObject* obj) {
    if (!THPVariable_Check(obj)) refuse(std::string(what) + " must be a tensor");
    return on_gpu(what, THPVariable_Unpack(obj));
}
// An argument that may be None: not defined then.
inline at::Tensor maybe_tensor(const char* what, PyObject* obj) { return obj == Py_None ? at::Tensor() : tensor_of(what, obj); }

inline void same_place(const char* what, const at::Tensor& t, const at::Tensor& first) {
    if (t.get_device() != first.get_device())
        refuse(std::string(what) + " lives on cuda:" + std::to_string(t.get_device()) + ", the other tensors on cuda:" + std::to_string(first.get_device()));
}
inline void same_dtype(const char* what, const at::Tensor& t, const at::Tensor& first) {
    if (t.scalar_type() != first.scalar_type())
        refuse(std::string(what) + " has dtype " + c10::toString(t.scalar_type()) + ", expected " + c10::toString(first.scalar_type()));
}

// What a call has no gradient of would come out of a backward pass as if it had no influence.
inline void no_gradient_of(const char* what, const at::Tensor& t) {
    if ((at::GradMode::is_enabled() && t.requires_grad()) || t._fw_grad(/*level=*/0).defined())
        refuse(std::string("a gradient is wanted of ") + what + ", and none is made of it");
}

inline double number(const char* what, PyObject* obj) {
    if (THPVariable_Check(obj)) no_gradient_of(what, THPVariable_Unpack(obj));
    const double v = PyFloat_AsDouble(obj);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse(std::string(what) + " must be a number");
    }
    return v;
}
inline bool truth(PyObject* obj) {
    const int v = PyObject_IsTrue(obj);
    if (v < 0) throw Raised{};
    return v != 0;
}

// Gives the GIL away where this thread has it, until the end of the block, by an exception too: a tensor without memory throws when asked for it.
class WithoutGil {
public:
    WithoutGil() : held_(PyGILState_Check() ? PyEval_SaveThread() : nullptr) {}
    ~WithoutGil() {
        if (held_ != nullptr) PyEval_RestoreThread(held_);
    }
    WithoutGil(const WithoutGil&) = delete;
    WithoutGil& operator=(const WithoutGil&) = delete;

private:
    PyThreadState* held_;
};

// The C interface, without the GIL.
template <typename F>
inline void call(F&& f) {
    int rc;
    {
        const WithoutGil gil;
        rc = f();
    }
    if (rc == 2) throw Refused(g_last_error());
    if (rc != 0) throw Failed(g_last_error());
}

inline void* stream_of(const at::Tensor& t) { return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(t.get_device())).stream(); }

// A tensor as rows of its last axis, `stride` elements apart; a copy without gaps where it does not lie so.
struct Rows {
    at::Tensor t;
    std::int64_t rows = 1, columns = 0, stride = 0;
};
inline Rows rows_of(const char* what, const at::Tensor& t) {
    if (t.dim() == 0) refuse(std::string(what) + " needs at least one axis");
    Rows r;
    r.columns = t.size(-1);
    bool even = r.columns == 1 || t.stride(-1) == 1;
    std::int64_t step = 0;
    for (std::int64_t d = t.dim() - 2; d >= 0 && even; --d) {
        const std::int64_t n = t.size(d);
        if (n == 1) continue;
        if (r.rows == 1) step = t.stride(d);
        else even = t.stride(d) == step * r.rows;
        r.rows *= n;
    }
    r.t = t;
    r.stride = step;
    if (!even) {
        r.t = t.contiguous();
        r.rows = r.columns == 0 ? 0 : r.t.numel() / r.columns;
        r.stride = r.columns;
    }
    if (t.numel() == 0) r.rows = 0;
    if (r.rows <= 1) r.stride = r.columns;
    return r;
}

inline at::Tensor new_bytes(const at::Tensor& like, std::int64_t n) { return at::empty({n}, like.options().dtype(at::kByte).requires_grad(false)); }
inline unsigned char* bytes_at(const at::Tensor& t, std::int64_t at) { return static_cast<unsigned char*>(t.data_ptr()) + at; }

inline PyObject* two(at::Tensor a, at::Tensor b) {
    PyObject* x = a.defined() ? THPVariable_Wrap(std::move(a)) : Py_NewRef(Py_None);
    PyObject* y = b.defined() ? THPVariable_Wrap(std::move(b)) : Py_NewRef(Py_None);
    PyObject* t = x != nullptr && y != nullptr ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return t;
}

inline at::Tensor new_like(const at::Tensor& t) { return at::empty(t.sizes(), t.options().requires_grad(false)); }

// ---- nodes of autograd -----------------------------------------------------------------------------------
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Gradients, computed by `f`. What f refuses is a ValueError where the backward pass was called, what fails a B200CclError, as in a forward pass; its
// results have no graph, and say so to whoever differentiates them again.
template <typename F>
variable_list in_backward(const char* what, F&& f) {
    variable_list grads;
    try {
        grads = f();
    } catch (const Refused& e) {
        TORCH_CHECK_VALUE(false, e.what());
    } catch (const Failed& e) {
        const pybind11::gil_scoped_acquire gil;
        PyErr_SetString(g_error_class, e.what());
        python_error error;
        error.persist();
        throw error;
    }
    if (!at::GradMode::is_enabled()) return grads;
    variable_list marked;
    for (at::Tensor& t : grads)
        if (t.defined()) marked.push_back(t.detach().requires_grad_());
    if (marked.empty()) return grads;
    auto error = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " has no second derivative", static_cast<std::int64_t>(marked.size()));
    marked = (*error)(std::move(marked));
    std::size_t i = 0;
    for (at::Tensor& t : grads)
        if (t.defined()) t = marked[i++];
    return grads;
}

inline bool wants_gradient(std::initializer_list<const at::Tensor*> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const at::Tensor* t : tensors)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

// By autocast's rules and through its cache: a weight is cast once, and 64-bit tensors are not. In a capture without the cache: a replay would not see
// the weights of its time, and the cache would hold memory of the graph's. While the guard lives, operators see no autocast.
inline std::optional<c10::impl::ExcludeDispatchKeyGuard> cast_by_autocast(const at::Tensor& first, std::initializer_list<at::Tensor*> tensors) {
    if (!at::autocast::is_autocast_enabled(at::kCUDA)) return std::nullopt;
    const at::ScalarType type = at::autocast::get_autocast_dtype(at::kCUDA);
    const c10::cuda::CUDAGuard guard(first.device());
    const bool captured = c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None;
    for (at::Tensor* t : tensors) {
        if (!t->defined() || !at::autocast::is_eligible(*t, at::kCUDA)) continue;
        *t = captured ? t->to(type) : at::autocast::cached_cast(type, *t, at::kCUDA);
    }
    return std::optional<c10::impl::ExcludeDispatchKeyGuard>(std::in_place, c10::DispatchKey::AutocastCUDA);
}

template <PyObject* (*kFunction)(PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS  // an allocation that fails raises torch's own error
    if (g_last_error == nullptr) {
        PyErr_SetString(PyExc_RuntimeError, "bind_train() first");
        return nullptr;
    }
    try {
        // Whoever records torch's operators would record the allocation of a result, and not the kernel that fills it.
        using Modes = c10::impl::TorchDispatchModeTLS;
        using Mode = c10::impl::TorchDispatchModeKey;
        if (torch::jit::tracer::isTracing() ||
            (Modes::any_modes_set() &&
             (Modes::get_mode(Mode::PROXY).has_value() || Modes::get_mode(Mode::FAKE).has_value() || Modes::get_mode(Mode::FUNCTIONAL).has_value())))
            refuse("these operators are no torch operators and cannot be traced");
        return kFunction(args, nargs);
    } catch (const Refused& e) {
        PyErr_SetString(PyExc_ValueError, e.what());
    } catch (const Failed& e) {
        PyErr_SetString(g_error_class, e.what());
    } catch (const Raised&) {
    }
    return nullptr;
    END_HANDLE_TH_ERRORS
}

}  // namespace b200ccl::python

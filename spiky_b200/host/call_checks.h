// What the native host sides of calls (layer_calls.cpp, residual_calls.cpp) check alike: which tensors and contexts are theirs.
#pragma once

#include <torch/extension.h>

#include <ATen/FuncTorchTLS.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/jit/frontend/tracer.h>

namespace {

struct Ref {   // owned reference
    PyObject *p = nullptr;
    explicit Ref(PyObject *q = nullptr) : p(q) {}
    Ref(const Ref &) = delete;
    Ref &operator=(const Ref &) = delete;
    ~Ref() { Py_XDECREF(p); }
    PyObject *get() const { return p; }
    explicit operator bool() const { return p != nullptr; }
};

[[noreturn]] void raise_current() {
    python_error e;
    e.persist();
    throw std::move(e);
}

bool plain_cuda(const at::Tensor &t, at::ScalarType type, c10::DeviceIndex device) {
    if (!t.defined() || t.layout() != at::kStrided || t.scalar_type() != type || !t.is_cuda() || t.device().index() != device) return false;
    const auto keys = t.unsafeGetTensorImpl()->key_set();
    return !keys.has_any(c10::python_ks) && !keys.has(c10::DispatchKey::FuncTorchGradWrapper) && !keys.has(c10::DispatchKey::FuncTorchBatched) &&
           !keys.has(c10::DispatchKey::Functionalize) && !keys.has(c10::DispatchKey::Batched) && !t.is_neg() && !t.is_conj() && !t._is_zerotensor();
}
bool ordinary_context() {
    return !torch::jit::tracer::isTracing() && !c10::impl::TorchDispatchModeTLS::any_modes_set() && !at::impl::torch_function_mode_enabled() &&
           (at::functorch::functorchTLSAccessor() == nullptr ||   // (it stays after the first transform; a key is there while one is active)
            !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode));
}

}  // namespace

// What the translation units of the module _sa2_torch share: errors, streams, and which tensors a kernel may be launched on.
#pragma once

#include <torch/extension.h>

#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include "sa2.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// norm, optimizer and loss (sa2_torch_train.cpp)
void bind_training(py::module_ &m);

namespace {

void check(int status) {
    if (status == SA2_OK) return;
    // the exception class of the package (Sa2Error) is raised by its own check function
    py::gil_scoped_acquire gil;
    py::module_::import("simplicial_attention_amd._native").attr("check_failed")(status, std::string(sa2_last_error()));
}

[[noreturn]] void raise(PyObject *type, const std::string &text) {
    py::gil_scoped_acquire gil;
    PyErr_SetString(type, text.c_str());
    throw py::error_already_set();
}

void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }

int element_of(const Tensor &t) {
    switch (t.scalar_type()) {
        case at::kBFloat16: return SA2_ELEMENT_BF16;
        case at::kHalf: return SA2_ELEMENT_F16;
        case at::kFloat: return SA2_ELEMENT_F32;
        default: return -1;
    }
}

// a call that autograd has to see: a backward may follow, or an input carries a forward-mode tangent (which the node refuses,
// also without a graph: the derivative would be lost without a word)
bool in_autograd(std::initializer_list<const Tensor *> inputs) {
    for (const Tensor *t : inputs)
        if ((at::GradMode::is_enabled() && t->requires_grad()) || t->_fw_grad(0).defined()) return true;
    return false;
}

// batched tensors (vmap's and is_grads_batched's), functorch's wrappers, subclasses with a dispatch of their own and
// forward-mode tangents: a kernel launched on their data pointers would miss what they carry
bool foreign(const Tensor &t) {
    static const c10::DispatchKeySet keys({c10::DispatchKey::Batched, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                                           c10::DispatchKey::Python, c10::DispatchKey::Functionalize});
    return t.key_set().has_any(keys) || t._fw_grad(0).defined();
}

// Recorders (torch.jit.trace, make_fx, fake tensors) see torch's operators alone: they would keep the allocation of a result without the kernel that fills it, and a
// replay would return what was in memory.  (torch.jit.trace sees Python Functions too, by which the calls go that it may record: those refuse the others.)
void refuse_modes(const char *what, bool recorded = false) {
    using c10::impl::TorchDispatchModeKey;
    for (const auto mode : {TorchDispatchModeKey::FAKE, TorchDispatchModeKey::PROXY, TorchDispatchModeKey::FUNCTIONAL})
        recorded = recorded || c10::impl::TorchDispatchModeTLS::get_mode(mode).has_value();
    if (recorded) raise(PyExc_RuntimeError, std::string(what) + " cannot be traced: a recorder does not see its kernels");
}
void refuse_recorder(const char *what) { refuse_modes(what, torch::jit::tracer::isTracing()); }

void refuse_autograd(const char *what, std::initializer_list<const Tensor *> inputs) {
    refuse_recorder(what);
    for (const Tensor *t : inputs)
        if (in_autograd({t}) || foreign(*t)) raise(PyExc_RuntimeError, std::string(what) + " has no derivative and takes plain tensors: call it under torch.no_grad()");
}

std::string shape_text(const Tensor &t) { return std::string(py::str(py::cast(t.sizes().vec()))); }

}  // namespace

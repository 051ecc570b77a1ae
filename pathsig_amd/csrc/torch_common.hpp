// What the registrations of the operators with torch share: raw pointers, scratch, the current stream, and the test for calls
// that may skip the dispatcher.
#pragma once

#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/autograd.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/python_arg_parser.h>
#include <torch/library.h>

#include "pathsig_hip.h"

namespace psig_torch {

using at::Tensor;

inline void *ptr(const Tensor &t) { return t.defined() && t.numel() > 0 ? t.data_ptr() : nullptr; }

inline void check_rc(int rc) { TORCH_CHECK(rc == PATHSIG_OK, "pathsig: ", pathsig_last_error(), " (error ", rc, ")"); }

inline void *stream_of(const Tensor &t) { return (void *)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

inline Tensor scratch(size_t nbytes, const Tensor &like) {
    if (nbytes == 0) return Tensor();
    return at::empty({(int64_t)nbytes}, like.options().dtype(at::kByte));
}

template <typename Signature>
auto typed_op(const char *name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Signature>();
}

// a plain CUDA tensor in plain eager mode
inline bool plain(const Tensor &t) {
    using c10::DispatchKey;
    if (!t.defined() || !t.is_cuda() || t._fw_grad(/*level=*/0).defined()) return false;
    if (at::impl::torch_function_mode_enabled()) return false;
    const auto tls = c10::impl::tls_local_dispatch_key_set();
    const c10::DispatchKeySet ordinary({DispatchKey::CUDA, DispatchKey::ADInplaceOrView, DispatchKey::AutogradCUDA,
                                        DispatchKey::AutogradOther, DispatchKey::BackendSelect, DispatchKey::AutocastCUDA,
                                        DispatchKey::AutocastCPU});
    const c10::DispatchKeySet rest = ((t.key_set() | tls.included_) - tls.excluded_) - ordinary;
    return (rest.raw_repr() & ~c10::full_backend_mask) == 0;
}

inline bool tensor_arg(PyObject *obj, Tensor &out) {
    if (!THPVariable_CheckExact(obj)) return false;
    out = THPVariable_Unpack(obj);
    return true;
}

// functions of the extension for the sequence operators (torch_seq.cpp)
PyObject *py_linear_attention(PyObject *, PyObject *const *args, Py_ssize_t nargs);
PyObject *py_linear_attention_step(PyObject *, PyObject *const *args, Py_ssize_t nargs);
PyObject *py_norm_join(PyObject *, PyObject *const *args, Py_ssize_t nargs);

}  // namespace psig_torch

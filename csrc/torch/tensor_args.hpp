/**
 * What the host sides of the operators share: the arguments of a call as plain CUDA tensors, whether something observes the call, outputs from torch's allocator,
 * and what nodes of the autograd graph need.
 */
#pragma once
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/utils/object_ptr.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/TracerMode.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/impl/PyInterpreterHooks.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>

namespace host_side {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

/** ncclDataType_t of the types that the kernels take, or -1. */
inline int dtype_of(const Tensor& t) {
    const at::ScalarType s = t.scalar_type();
    return s == at::kHalf ? 6 : s == at::kFloat ? 7 : s == at::kBFloat16 ? 9 : -1;
}

/** A tensor of values in CUDA memory, and none that stands for others (fake, functional, a subclass that takes over dispatch). */
inline bool is_plain(const Tensor& t) {
    return t.is_cuda() && t.layout() == at::kStrided && !t.unsafeGetTensorImpl()->is_python_dispatch() && !t.key_set().has(c10::DispatchKey::FuncTorchGradWrapper)
           && !t.key_set().has(c10::DispatchKey::FuncTorchBatched) && !t.key_set().has(c10::DispatchKey::Functionalize) && !t._is_zerotensor();
}

/** `o` as a tensor: false where it is none, or not plain. None leaves `t` undefined, if `optional`. */
inline bool tensor_of(PyObject* o, bool optional, Tensor* t) {
    if (o == Py_None) return optional;
    if (!THPVariable_Check(o)) return false;
    *t = THPVariable_Unpack(o);
    return is_plain(*t);
}

/** Python objects that calls are compared with, for the life of the process. An import may let other threads run, which a static's own guard would
 *  keep from it: two of them find the same object instead. */
struct Known {
    const char *module, *name;
    PyObject* object = nullptr;
    PyObject* get() {
        if (object) return object;
        THPObjectPtr m(PyImport_ImportModule(module));
        PyObject* o = m ? PyObject_GetAttrString(m.get(), name) : nullptr;
        if (!o) throw python_error();
        return object = o;
    }
};
inline Known parameter{"torch.nn", "Parameter"}, disabled{"torch._C", "_disabled_torch_function_impl"}, device_context{"torch.utils._device", "DeviceContext"};

/** Whether this is a tensor whose class takes torch's functions over. (Only what is left after the first lines costs anything.) */
inline bool takes_functions_over(PyObject* o) {
    PyObject* type = reinterpret_cast<PyObject*>(Py_TYPE(o));
    if (type == THPVariableClass || o == Py_None || PyFloat_Check(o) || PyLong_Check(o) || type == parameter.get() || !THPVariable_Check(o)) return false;
    THPObjectPtr f(PyObject_GetAttrString(type, "__torch_function__"));
    if (!f) throw python_error();
    return f.get() != disabled.get();
}

/** Whether something would see torch's operations of this call: a mode, a tracer, or a subclass of Tensor among the arguments. */
inline bool observed(PyObject* const* args, Py_ssize_t nargs) {
    using Functions = at::impl::PythonTorchFunctionTLS;
    if (c10::impl::dispatch_mode_enabled() || at::tracer::impl::is_dispatch_enabled()) return true;
    if (at::impl::torch_function_mode_enabled())        // the one behind torch.device and the default device only places new tensors
        for (int64_t i = 0; i < Functions::stack_len(); i++)
            if (reinterpret_cast<PyObject*>(Py_TYPE(Functions::get_stack_at(i)->ptr(c10::impl::getGlobalPyInterpreter()))) != device_context.get()) return true;
    if (Functions::get_disabled_state() == at::impl::TorchFunctionDisabledState::ENABLED)
        for (Py_ssize_t i = 0; i < nargs; i++)
            if (takes_functions_over(args[i])) return true;
    return false;
}

inline Tensor dense(const Tensor& t) {
    if (!t.defined()) return t;
    const Tensor v = t.is_neg() ? t.resolve_neg() : t;
    return v.is_contiguous() ? v : v.contiguous();
}

/** What a node saved, as the kernels read it: hooks may hand back a copy that lies otherwise in memory. */
inline Tensor unpacked(const SavedVariable& v) { return dense(v.unpack()); }

inline Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) { return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt); }
inline Tensor fresh_like(const Tensor& t) { return fresh(t.sizes(), t.scalar_type(), t); }

template <typename T = void> T* ptr(const Tensor& t) { return t.defined() ? reinterpret_cast<T*>(t.data_ptr()) : nullptr; }
inline void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

inline bool records(std::initializer_list<const Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

inline void check_forward_mode(const char* what, std::initializer_list<const Tensor*> ts) {
    for (const Tensor* t : ts)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), what, " has no derivative in forward mode");
}

/** Gradients of gradients are an error, when somebody asks for them. */
inline variable_list only_once(const char* what, variable_list grads, std::initializer_list<const Tensor*> used) {
    if (!at::GradMode::is_enabled() || !records(used)) return grads;
    variable_list out(grads.size());
    for (size_t i = 0; i < grads.size(); i++)
        if (grads[i].defined()) {
            auto error = std::make_shared<torch::autograd::DelayedError>(std::string(what) + " can be differentiated once only", 1);
            out[i] = (*error)({std::move(grads[i])})[0];
        }
    return out;
}

/** One or two tensors for Python. */
inline PyObject* wrap(Tensor a) { return THPVariable_Wrap(std::move(a)); }
inline PyObject* wrap(Tensor a, Tensor b) {
    THPObjectPtr pair(PyTuple_New(2));
    if (!pair) return nullptr;
    PyObject* x = THPVariable_Wrap(std::move(a));
    if (!x) return nullptr;
    PyTuple_SET_ITEM(pair.get(), 0, x);
    PyObject* y = THPVariable_Wrap(std::move(b));
    if (!y) return nullptr;
    PyTuple_SET_ITEM(pair.get(), 1, y);
    return pair.release();
}

inline bool number(PyObject* o, double* v) {
    if (!PyFloat_Check(o) && !PyLong_Check(o)) return false;
    *v = PyFloat_AsDouble(o);
    if (*v == -1.0 && PyErr_Occurred()) { PyErr_Clear(); return false; }
    return true;
}

} // namespace host_side

/**
 * Host side of the operators of a decoder block (csrc/decoder/decoder_ops.hpp) for dccl_b200/ops/decoder.py: their checks, outputs,
 * workspaces, launches on torch's current stream, and nodes of the autograd graph. The kernels of a decoding step take two to
 * three microseconds; from Python a call took 16 to 20, forward and backward together 130.
 *
 * A function that finds anything but plain CUDA tensors of the right types and shapes returns NotImplemented: dccl_b200/ops/decoder.py then
 * says what is wrong. Where something follows torch's operations (a mode, a tracer, a subclass of Tensor) it returns None, and the same call
 * comes back through an operator that torch knows. Plain CPython functions: their arguments are borrowed. Everything that could throw is
 * caught at this border.
 */
#include "decoder_ops.hpp"
#include "../decoder/decoder_ops.hpp"
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

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

/** The library's entry points, by address: the library that is loaded need not be the one that this file was linked with. */
struct Entries {
    decltype(&dccl_residual_norm) norm;
    decltype(&dccl_residual_norm_workspace) norm_workspace;
    decltype(&dccl_residual_norm_backward) norm_backward;
    decltype(&dccl_rotary) rotary;
    decltype(&dccl_gated_linear_workspace) gated_workspace;
    decltype(&dccl_gated_linear_pads) gated_pads;
    decltype(&dccl_gated_linear) gated;
    decltype(&dccl_gated_linear_backward) gated_backward;
} entry;

/** ncclDataType_t of the types that the kernels take, or -1. */
int dtype_of(const Tensor& t) {
    const at::ScalarType s = t.scalar_type();
    return s == at::kHalf ? 6 : s == at::kFloat ? 7 : s == at::kBFloat16 ? 9 : -1;
}

/** A tensor of values in CUDA memory, and none that stands for others (fake, functional, a subclass that takes over dispatch). */
bool is_plain(const Tensor& t) {
    return t.is_cuda() && t.layout() == at::kStrided && !t.unsafeGetTensorImpl()->is_python_dispatch() && !t.key_set().has(c10::DispatchKey::FuncTorchGradWrapper)
           && !t.key_set().has(c10::DispatchKey::FuncTorchBatched) && !t.key_set().has(c10::DispatchKey::Functionalize) && !t._is_zerotensor();
}

/** `o` as a tensor: false where it is none, or not plain. None leaves `t` undefined, if `optional`. */
bool tensor_of(PyObject* o, bool optional, Tensor* t) {
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
} parameter{"torch.nn", "Parameter"}, disabled{"torch._C", "_disabled_torch_function_impl"}, device_context{"torch.utils._device", "DeviceContext"};

/** Whether this is a tensor whose class takes torch's functions over. (Only what is left after the first lines costs anything.) */
bool takes_functions_over(PyObject* o) {
    PyObject* type = reinterpret_cast<PyObject*>(Py_TYPE(o));
    if (type == THPVariableClass || o == Py_None || PyFloat_Check(o) || PyLong_Check(o) || type == parameter.get() || !THPVariable_Check(o)) return false;
    THPObjectPtr f(PyObject_GetAttrString(type, "__torch_function__"));
    if (!f) throw python_error();
    return f.get() != disabled.get();
}

/** Whether something would see torch's operations of this call: a mode, a tracer, or a subclass of Tensor among the arguments. */
bool observed(PyObject* const* args, Py_ssize_t nargs) {
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

Tensor dense(const Tensor& t) {
    if (!t.defined()) return t;
    const Tensor v = t.is_neg() ? t.resolve_neg() : t;
    return v.is_contiguous() ? v : v.contiguous();
}

/** What a node saved, as the kernels read it: hooks may hand back a copy that lies otherwise in memory. */
Tensor unpacked(const SavedVariable& v) { return dense(v.unpack()); }

Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) { return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt); }
Tensor fresh_like(const Tensor& t) { return fresh(t.sizes(), t.scalar_type(), t); }

template <typename T = void> T* ptr(const Tensor& t) { return t.defined() ? reinterpret_cast<T*>(t.data_ptr()) : nullptr; }
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

bool records(std::initializer_list<const Tensor*> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : ts)
        if (t->defined() && t->requires_grad()) return true;
    return false;
}

void check_forward_mode(const char* what, std::initializer_list<const Tensor*> ts) {
    for (const Tensor* t : ts)
        TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), what, " has no derivative in forward mode");
}

/** Gradients of gradients are an error, when somebody asks for them. */
variable_list only_once(const char* what, variable_list grads, std::initializer_list<const Tensor*> used) {
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
PyObject* wrap(Tensor a) { return THPVariable_Wrap(std::move(a)); }
PyObject* wrap(Tensor a, Tensor b) {
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

bool number(PyObject* o, double* v) {
    if (!PyFloat_Check(o) && !PyLong_Check(o)) return false;
    *v = PyFloat_AsDouble(o);
    if (*v == -1.0 && PyErr_Occurred()) { PyErr_Clear(); return false; }
    return true;
}

/* ---------------------------------------------------------------------------------------------- norms */

/** Rows of gates, each for as many consecutive rows of x; 0 without a gate, -1 where the shapes do not fit. */
int64_t gates_of(const Tensor& x, const Tensor& gate) {
    if (!gate.defined()) return 0;
    const int64_t width = x.size(-1);
    if (gate.dim() < 1 || gate.size(-1) != width) return -1;
    if (gate.dim() == 1) return 1;
    if (gate.dim() != x.dim()) return -1;
    int64_t n = 1, k = 0;
    while (k < x.dim() - 1 && gate.size(k) == x.size(k)) n *= gate.size(k++);
    for (; k < x.dim() - 1; k++)
        if (gate.size(k) != 1) return -1;
    return n;
}

int f32_vectors(const Tensor& x, const Tensor& weight, const Tensor& post, const Tensor& gate) {
    if (x.scalar_type() == at::kFloat) return 0;
    return (weight.scalar_type() == at::kFloat ? DCCL_NORM_WEIGHT_F32 : 0) | (post.defined() && post.scalar_type() == at::kFloat ? DCCL_NORM_POST_F32 : 0)
           | (gate.defined() && gate.scalar_type() == at::kFloat ? DCCL_NORM_GATE_F32 : 0);
}

struct NormBackward : public Node {
    SavedVariable x, branch, weight, post, gate, rstd, rstd_post;       // saved like any, so that checkpointing and hooks see them
    double scale = 1;
    int64_t gates = 0;
    bool has_branch = false, own_branch = false;      // own_branch: its gradient is not that of x

    variable_list apply(variable_list&& grads) override {
        const Tensor x_ = unpacked(x), b = unpacked(branch), w = unpacked(weight), p = unpacked(post), g = unpacked(gate), ry = unpacked(rstd), rb = unpacked(rstd_post);
        const Tensor dy = has_branch ? dense(grads[0]) : Tensor(), dn = dense(grads[has_branch ? 1 : 0]);
        variable_list out(5);
        if (!dy.defined() && !dn.defined()) return out;
        const int64_t width = x_.size(-1), rows = x_.numel() / width;
        const Tensor dx = fresh_like(x_), db = own_branch ? fresh_like(b) : has_branch ? dx : Tensor();
        const Tensor dw = dn.defined() && task_should_compute_output(2) ? fresh_like(w) : Tensor();
        const Tensor dp = p.defined() && task_should_compute_output(3) ? fresh_like(p) : Tensor(), dg = g.defined() && task_should_compute_output(4) ? fresh_like(g) : Tensor();
        if (rows) {
            const int device = x_.device().index();
            const size_t bytes = entry.norm_workspace(device, dtype_of(x_), rows, width, gates, p.defined(), b.defined());
            const Tensor work = fresh({(int64_t)bytes}, at::kByte, x_);
            const int rc = entry.norm_backward(device, dtype_of(x_), rows, width, ptr(dy), ptr(dn), ptr(x_), ptr(b), ptr(w), ptr(p), ptr(g), gates ? rows / gates : 0,
                                               f32_vectors(x_, w, p, g), scale, ptr(ry), ptr(rb), ptr(dx), own_branch ? ptr(db) : nullptr, ptr(dw), ptr(dp), ptr(dg),
                                               ptr(work), bytes, stream_of(x_));
            TORCH_CHECK(rc == 0, "residual_norm: the backward pass was not launched (see stderr)");
        } else {
            for (const Tensor* t : {&dw, &dp, &dg})
                if (t->defined()) t->zero_();
        }
        out = {dx, db, dw, dp, dg};
        return only_once("residual_norm", std::move(out), {&grads[0], &grads.back(), &x_, &b, &w, &p, &g});
    }
    std::string name() const override { return "ResidualNormBackward"; }
    void release_variables() override {
        for (SavedVariable* v : {&x, &branch, &weight, &post, &gate, &rstd, &rstd_post}) v->reset_data();
    }
};

/** residual_norm(x, branch or None, weight, eps, post_weight or None, gate or None, scale): (y, n), or n without a branch. */
PyObject* residual_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(nargs == 7, "residual_norm takes seven arguments");
    Tensor x, branch, weight, post, gate;
    double eps, scale;
    if (!tensor_of(args[0], false, &x) || !tensor_of(args[1], true, &branch) || !tensor_of(args[2], false, &weight) || !tensor_of(args[4], true, &post)
        || !tensor_of(args[5], true, &gate) || !number(args[3], &eps) || !number(args[6], &scale))
        Py_RETURN_NOTIMPLEMENTED;
    const int dtype = dtype_of(x);
    if (dtype < 0 || x.dim() < 1) Py_RETURN_NOTIMPLEMENTED;
    const int64_t width = x.size(-1), gates = gates_of(x, gate);
    if (width < 1 || width > DCCL_NORM_MAX_WIDTH || gates < 0) Py_RETURN_NOTIMPLEMENTED;
    const int64_t rows = x.numel() / width;
    if (rows > INT32_MAX || (branch.defined() && (branch.sizes() != x.sizes() || branch.scalar_type() != x.scalar_type() || branch.device() != x.device()))) Py_RETURN_NOTIMPLEMENTED;
    if (!branch.defined() && (post.defined() || gate.defined())) Py_RETURN_NOTIMPLEMENTED;
    for (const Tensor* v : {&weight, &post, &gate}) {
        if (!v->defined()) continue;
        if ((v->scalar_type() != x.scalar_type() && v->scalar_type() != at::kFloat) || v->device() != x.device()) Py_RETURN_NOTIMPLEMENTED;
        if (v != &gate && (v->dim() != 1 || v->size(0) != width)) Py_RETURN_NOTIMPLEMENTED;
    }
    if (observed(args, nargs)) Py_RETURN_NONE;
    check_forward_mode("residual_norm", {&x, &branch, &weight, &post, &gate});
    Tensor y, n;
    {
        pybind11::gil_scoped_release no_gil;
        x = dense(x), branch = dense(branch), weight = dense(weight), post = dense(post), gate = dense(gate);
        const bool keep = records({&x, &branch, &weight, &post, &gate});
        n = fresh_like(x);
        if (branch.defined()) y = fresh_like(x);
        Tensor rstd, rstd_post;
        if (keep) rstd = fresh({rows}, at::kFloat, x);
        if (keep && post.defined()) rstd_post = fresh({rows}, at::kFloat, x);
        if (rows) {
            const int rc = entry.norm(x.device().index(), dtype, rows, width, ptr(x), ptr(branch), ptr(weight), ptr(post), ptr(gate), gates ? rows / gates : 0,
                                      f32_vectors(x, weight, post, gate), eps, scale, ptr(y), ptr(n), ptr(rstd), ptr(rstd_post), stream_of(x));
            TORCH_CHECK(rc == 0, "residual_norm was not launched (see stderr)");
        }
        if (keep) {
            std::shared_ptr<NormBackward> node(new NormBackward(), torch::autograd::deleteNode);
            node->set_next_edges(torch::autograd::collect_next_edges(x, branch, weight, post, gate));
            node->scale = scale;
            node->gates = gates;
            node->has_branch = branch.defined();
            node->own_branch = branch.defined() && (post.defined() || gate.defined() || scale != 1.0);
            node->x = SavedVariable(x, false);
            node->branch = SavedVariable(branch, false);
            node->weight = SavedVariable(weight, false);
            node->post = SavedVariable(post, false);
            node->gate = SavedVariable(gate, false);
            node->rstd = SavedVariable(rstd, false);
            node->rstd_post = SavedVariable(rstd_post, false);
            if (branch.defined()) torch::autograd::set_history(y, node);
            torch::autograd::set_history(n, node);
        }
    }
    return branch.defined() ? wrap(std::move(y), std::move(n)) : wrap(std::move(n));
    END_HANDLE_TH_ERRORS
}

/* ---------------------------------------------------------------------------------------------- rotary positions */

/** x as [batch, seq, heads, dim] by its strides; of three dimensions the batch is missing. */
DcclHeads heads_of(const Tensor& x, const Tensor& out) {
    if (!x.defined()) return DcclHeads{};
    const auto i = x.strides(), o = out.strides();
    if (x.dim() == 3) return {x.data_ptr(), out.data_ptr(), 0, i[0], i[1], 0, o[0], o[1], (int)x.size(1)};
    return {x.data_ptr(), out.data_ptr(), i[0], i[1], i[2], o[0], o[1], o[2], (int)x.size(2)};
}

Tensor dense_head(const Tensor& t) {
    if (!t.defined()) return t;
    const Tensor v = t.is_neg() ? t.resolve_neg() : t;
    return v.stride(-1) == 1 || v.size(-1) == 1 ? v : v.contiguous();
}

struct Turn {
    Tensor freqs, positions;
    int64_t first = 0;
    double scale = 1;
    bool interleaved = false;

    std::pair<Tensor, Tensor> operator()(const Tensor& q, const Tensor& k, bool back) const {
        Tensor out[2];
        const Tensor* in[2] = {&q, &k};
        for (int j = 0; j < 2; j++)
            if (in[j]->defined())      // laid out as it came, where that leaves no holes
                out[j] = in[j]->is_non_overlapping_and_dense() ? at::detail::empty_strided_cuda(in[j]->sizes(), in[j]->strides(), in[j]->scalar_type(), in[j]->device())
                                                               : fresh_like(*in[j]);
        const Tensor& like = q.defined() ? q : k;
        const int64_t batch = like.dim() == 3 ? 1 : like.size(0), seq = like.size(like.dim() - 3);
        if (batch && seq) {
            const DcclHeads hq = heads_of(q, out[0]), hk = heads_of(k, out[1]);
            const bool tensor = positions.defined();
            const int rc = entry.rotary(like.device().index(), dtype_of(like), batch, seq, (int)like.size(-1), (int)freqs.size(0), interleaved, back, &hq, &hk,
                                        reinterpret_cast<const double*>(freqs.data_ptr()), ptr(positions), tensor && positions.scalar_type() == at::kLong,
                                        tensor && positions.dim() == 2 ? positions.stride(0) : 0, tensor ? positions.stride(-1) : 0, first, scale, stream_of(like));
            TORCH_CHECK(rc == 0, "rotary was not launched (see stderr)");
        }
        return {out[0], out[1]};
    }
};

struct RotaryBackward : public Node {
    Turn turn;                              // without its tensors
    SavedVariable freqs, positions;
    bool has_k = false;

    variable_list apply(variable_list&& grads) override {
        Turn t = turn;
        t.freqs = unpacked(freqs);
        t.positions = positions.unpack();
        const Tensor dq = task_should_compute_output(0) ? dense_head(grads[0]) : Tensor(), dk = has_k && task_should_compute_output(1) ? dense_head(grads[1]) : Tensor();
        variable_list out(2);
        if (!dq.defined() && !dk.defined()) return out;
        std::tie(out[0], out[1]) = t(dq, dk, true);
        return only_once("rotary", std::move(out), {&grads[0], &grads.back()});
    }
    std::string name() const override { return "RotaryBackward"; }
    void release_variables() override { freqs.reset_data(); positions.reset_data(); }
};

/** rotary(q, k or None, freqs, first position or tensor of positions, interleaved, scale): (q, k), or q without k. */
PyObject* rotary(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(nargs == 6, "rotary takes six arguments");
    Tensor q, k;
    Turn turn;
    if (!tensor_of(args[0], false, &q) || !tensor_of(args[1], true, &k) || !tensor_of(args[2], false, &turn.freqs) || !number(args[5], &turn.scale)) Py_RETURN_NOTIMPLEMENTED;
    if (PyLong_CheckExact(args[3])) {
        turn.first = PyLong_AsLongLong(args[3]);
        if (turn.first == -1 && PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NOTIMPLEMENTED; }
        if (turn.first <= -(1ll << 62) || turn.first >= 1ll << 62) Py_RETURN_NOTIMPLEMENTED;
    } else if (args[3] == Py_None || !tensor_of(args[3], false, &turn.positions)) {
        Py_RETURN_NOTIMPLEMENTED;
    }
    if (args[4] != Py_True && args[4] != Py_False) Py_RETURN_NOTIMPLEMENTED;
    turn.interleaved = args[4] == Py_True;
    if (dtype_of(q) < 0 || (q.dim() != 3 && q.dim() != 4)) Py_RETURN_NOTIMPLEMENTED;
    const int64_t dim = q.size(-1), seq = q.size(q.dim() - 3), batch = q.dim() == 4 ? q.size(0) : 1;
    int64_t heads = q.size(-2);
    if (k.defined()) {
        if (k.dim() != q.dim() || k.scalar_type() != q.scalar_type() || k.device() != q.device() || k.size(-1) != dim || k.size(k.dim() - 3) != seq || (q.dim() == 4 && k.size(0) != batch))
            Py_RETURN_NOTIMPLEMENTED;
        heads += k.size(-2);
    }
    const Tensor& f = turn.freqs;
    if (f.dim() != 1 || f.scalar_type() != at::kDouble || f.device() != q.device() || f.requires_grad() || f.size(0) < 1 || 2 * f.size(0) > dim || f.size(0) > DCCL_ROTARY_MAX_PAIRS
        || heads * dim > DCCL_ROTARY_MAX_TOKEN || seq > INT32_MAX)
        Py_RETURN_NOTIMPLEMENTED;
    const Tensor& p = turn.positions;
    if (p.defined()) {
        const bool one = p.dim() == 1 && p.size(0) == seq, each = q.dim() == 4 && p.dim() == 2 && p.size(0) == batch && p.size(1) == seq;
        if ((!one && !each) || (p.scalar_type() != at::kLong && p.scalar_type() != at::kInt) || p.device() != q.device()) Py_RETURN_NOTIMPLEMENTED;
    }
    if (observed(args, nargs)) Py_RETURN_NONE;
    check_forward_mode("rotary", {&q, &k});
    std::pair<Tensor, Tensor> out;
    {
        pybind11::gil_scoped_release no_gil;
        q = dense_head(q), k = dense_head(k);
        turn.freqs = dense(turn.freqs);
        out = turn(q, k, false);
        if (records({&q, &k})) {
            std::shared_ptr<RotaryBackward> node(new RotaryBackward(), torch::autograd::deleteNode);
            node->set_next_edges(torch::autograd::collect_next_edges(q, k));
            node->freqs = SavedVariable(turn.freqs, false);
            node->positions = SavedVariable(turn.positions, false);
            node->turn.first = turn.first;
            node->turn.scale = turn.scale;
            node->turn.interleaved = turn.interleaved;
            node->has_k = k.defined();
            torch::autograd::set_history(out.first, node);
            if (k.defined()) torch::autograd::set_history(out.second, node);
        }
    }
    return k.defined() ? wrap(std::move(out.first), std::move(out.second)) : wrap(std::move(out.first));
    END_HANDLE_TH_ERRORS
}

/* ---------------------------------------------------------------------------------------------- gated linear */

bool gated_aligned(const Tensor& x, const Tensor& w_gate, const Tensor& w_up) {
    return ((uintptr_t)x.data_ptr() | (uintptr_t)w_gate.data_ptr() | (uintptr_t)w_up.data_ptr()) % 16 == 0;
}

Tensor on_16_bytes(const Tensor& t) { return t.defined() && (uintptr_t)t.data_ptr() % 16 ? t.clone() : t; }

/** The workspace of a call; undefined where it needs none. */
Tensor gated_work(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, bool backward) {
    const long long bytes = entry.gated_workspace(x.device().index(), x.numel() / x.size(-1), x.size(-1), w_gate.size(0), gated_aligned(x, w_gate, w_up), backward);
    TORCH_CHECK(bytes >= 0, "gated_linear: sizes that it does not take");
    return bytes ? fresh({(int64_t)bytes}, at::kByte, x) : Tensor();
}

struct GatedBackward : public Node {
    SavedVariable x, w_gate, w_up, gate, up, padded;
    int act = 0;

    variable_list apply(variable_list&& grads) override {
        Tensor x_ = unpacked(x), wg = unpacked(w_gate), wu = unpacked(w_up);
        const Tensor g = on_16_bytes(unpacked(gate)), u = on_16_bytes(unpacked(up)), copies = on_16_bytes(unpacked(padded)), dh = dense(grads[0]);
        variable_list out(3);
        if (!dh.defined()) return out;
        if (!copies.defined()) x_ = on_16_bytes(x_), wg = on_16_bytes(wg), wu = on_16_bytes(wu);      // so the forward pass had them
        const bool weights = task_should_compute_output(1) || task_should_compute_output(2);
        const Tensor dx = task_should_compute_output(0) ? fresh_like(x_) : Tensor();
        const Tensor dg = weights ? fresh_like(wg) : Tensor(), du = weights ? fresh_like(wu) : Tensor();
        const int64_t width = x_.size(-1), tokens = x_.numel() / width;
        if (tokens) {
            const Tensor work = gated_work(x_, wg, wu, true);
            const int rc = entry.gated_backward(x_.device().index(), dtype_of(x_), tokens, width, wg.size(0), ptr(dh), ptr<float>(g), ptr<float>(u), g.size(1), ptr(x_), ptr(wg), ptr(wu),
                                                ptr(copies), act, ptr(dx), ptr(dg), ptr(du), ptr(work), work.defined() ? (long long)work.numel() : 0, stream_of(x_));
            TORCH_CHECK(rc == 0, "gated_linear: the backward pass was not launched (see stderr)");
        } else if (weights) {
            dg.zero_();
            du.zero_();
        }
        out = {dx, task_should_compute_output(1) ? dg : Tensor(), task_should_compute_output(2) ? du : Tensor()};
        return only_once("gated_linear", std::move(out), {&grads[0], &x_, &wg, &wu});
    }
    std::string name() const override { return "GatedLinearBackward"; }
    void release_variables() override {
        for (SavedVariable* v : {&x, &w_gate, &w_up, &gate, &up, &padded}) v->reset_data();
    }
};

/** gated_linear(x, w_gate, w_up, number of the activation): h. */
PyObject* gated_linear(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(nargs == 4, "gated_linear takes four arguments");
    Tensor x, wg, wu;
    if (!tensor_of(args[0], false, &x) || !tensor_of(args[1], false, &wg) || !tensor_of(args[2], false, &wu) || !PyLong_CheckExact(args[3])) Py_RETURN_NOTIMPLEMENTED;
    const int act = (int)PyLong_AsLong(args[3]);
    const int dtype = dtype_of(x);
    if ((dtype != 6 && dtype != 9) || x.dim() < 1 || wg.dim() != 2 || act < DCCL_ACT_SILU || act > DCCL_ACT_GELU_TANH) Py_RETURN_NOTIMPLEMENTED;
    const int64_t width = x.size(-1), ffn = wg.size(0);
    if (width < 1 || ffn < 1 || wg.size(1) != width || wu.sizes() != wg.sizes() || wg.scalar_type() != x.scalar_type() || wu.scalar_type() != x.scalar_type() || wg.device() != x.device()
        || wu.device() != x.device())
        Py_RETURN_NOTIMPLEMENTED;
    const int64_t tokens = x.numel() / width;
    if (std::max({tokens, width, ffn}) >= DCCL_GATED_MAX_DIMENSION) Py_RETURN_NOTIMPLEMENTED;
    if (observed(args, nargs)) Py_RETURN_NONE;
    check_forward_mode("gated_linear", {&x, &wg, &wu});
    Tensor h;
    {
        pybind11::gil_scoped_release no_gil;
        x = dense(x), wg = dense(wg), wu = dense(wu);
        const bool keep = records({&x, &wg, &wu});
        c10::SmallVector<int64_t, 6> sizes(x.sizes().begin(), x.sizes().end());
        sizes.back() = ffn;
        h = fresh(sizes, x.scalar_type(), x);
        Tensor g, u;
        const int64_t stride = (ffn + 3) / 4 * 4;
        if (keep) {
            g = fresh({tokens, stride}, at::kFloat, x);
            u = fresh({tokens, stride}, at::kFloat, x);
        }
        Tensor work;
        if (tokens) {
            work = gated_work(x, wg, wu, false);
            const int rc = entry.gated(x.device().index(), dtype, tokens, width, ffn, ptr(x), ptr(wg), ptr(wu), act, ptr(h), ptr<float>(g), ptr<float>(u), stride, ptr(work),
                                       work.defined() ? (long long)work.numel() : 0, stream_of(x));
            TORCH_CHECK(rc == 0, "gated_linear was not launched (see stderr)");
        }
        if (keep) {
            std::shared_ptr<GatedBackward> node(new GatedBackward(), torch::autograd::deleteNode);
            node->set_next_edges(torch::autograd::collect_next_edges(x, wg, wu));
            node->x = SavedVariable(x, false);
            node->w_gate = SavedVariable(wg, false);
            node->w_up = SavedVariable(wu, false);
            node->gate = SavedVariable(g, false);
            node->up = SavedVariable(u, false);
            node->padded = SavedVariable(entry.gated_pads(width, gated_aligned(x, wg, wu)) ? work : Tensor(), false);
            node->act = act;
            torch::autograd::set_history(h, node);
        }
    }
    return wrap(std::move(h));
    END_HANDLE_TH_ERRORS
}

/** decoder_ops_bind(addresses of the entry points, in the order of Entries). */
PyObject* decoder_ops_bind(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    void* at[8];
    TORCH_CHECK(nargs == 8, "decoder_ops_bind takes eight addresses");
    for (int i = 0; i < 8; i++) {
        at[i] = PyLong_AsVoidPtr(args[i]);
        if (PyErr_Occurred()) return nullptr;
        TORCH_CHECK(at[i], "decoder_ops_bind: an address is missing");
    }
    entry = {reinterpret_cast<decltype(entry.norm)>(at[0]), reinterpret_cast<decltype(entry.norm_workspace)>(at[1]), reinterpret_cast<decltype(entry.norm_backward)>(at[2]),
             reinterpret_cast<decltype(entry.rotary)>(at[3]), reinterpret_cast<decltype(entry.gated_workspace)>(at[4]), reinterpret_cast<decltype(entry.gated_pads)>(at[5]),
             reinterpret_cast<decltype(entry.gated)>(at[6]), reinterpret_cast<decltype(entry.gated_backward)>(at[7])};
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"residual_norm", (PyCFunction)(void (*)())residual_norm, METH_FASTCALL, "(y, n), or n without a branch; NotImplemented where the arguments do not fit, None where the call is observed"},
    {"rotary", (PyCFunction)(void (*)())rotary, METH_FASTCALL, "turned q and k; NotImplemented and None likewise"},
    {"gated_linear", (PyCFunction)(void (*)())gated_linear, METH_FASTCALL, "act(x Wg^T) * (x Wu^T); NotImplemented and None likewise"},
    {"decoder_ops_bind", (PyCFunction)(void (*)())decoder_ops_bind, METH_FASTCALL, "hands over the addresses of the library's entry points"},
    {nullptr, nullptr, 0, nullptr},
};

} // namespace

int add_decoder_ops(PyObject* module) { return PyModule_AddFunctions(module, methods); }

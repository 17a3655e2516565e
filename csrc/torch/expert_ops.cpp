/**
 * Host side of the operators of a mixture of experts (csrc/experts/expert_ops.hpp) for dccl_b200/ops/experts.py, in the manner of decoder_ops.cpp: a function
 * that finds anything but plain CUDA tensors of the right types and shapes returns NotImplemented, and None where something observes the call.
 */
#include "expert_ops.hpp"
#include "../experts/expert_ops.hpp"
#include "../decoder/decoder_ops.hpp"
#include "tensor_args.hpp"

namespace {

using namespace host_side;

struct Entries {
    decltype(&dccl_route) route;
    decltype(&dccl_route_backward) route_backward;
    decltype(&dccl_expert_plan) plan;
    decltype(&dccl_dispatch) dispatch;
    decltype(&dccl_combine) combine;
    decltype(&dccl_combine_backward) combine_backward;
    decltype(&dccl_expert_linear_workspace) linear_workspace;
    decltype(&dccl_expert_linear_pads) linear_pads;
    decltype(&dccl_expert_linear) linear;
    decltype(&dccl_expert_linear_backward) linear_backward;
} entry;

bool integer(PyObject* o, int64_t low, int64_t high, int64_t* v) {
    if (!PyLong_Check(o) || PyBool_Check(o)) return false;
    *v = PyLong_AsLongLong(o);
    if (*v == -1 && PyErr_Occurred()) { PyErr_Clear(); return false; }
    return *v >= low && *v <= high;
}

bool truth(PyObject* o, bool* v) {
    if (o != Py_True && o != Py_False) return false;
    *v = o == Py_True;
    return true;
}

/** Three tensors for Python. */
PyObject* wrap3(Tensor a, Tensor b, Tensor c) {
    THPObjectPtr all(PyTuple_New(3));
    if (!all) return nullptr;
    Tensor* from[3] = {&a, &b, &c};
    for (int i = 0; i < 3; i++) {
        PyObject* o = THPVariable_Wrap(std::move(*from[i]));
        if (!o) return nullptr;
        PyTuple_SET_ITEM(all.get(), i, o);
    }
    return all.release();
}

/** The leading sizes of `t` and one more. */
c10::SmallVector<int64_t, 6> with_last(const Tensor& t, int64_t last) {
    c10::SmallVector<int64_t, 6> s(t.sizes().begin(), t.sizes().end());
    s.back() = last;
    return s;
}

/* ---------------------------------------------------------------------------------------------- routing */

struct RouteBackward : public Node {
    SavedVariable logits, chosen;
    DcclRouting how = {};

    variable_list apply(variable_list&& grads) override {
        const Tensor z = unpacked(logits), c = unpacked(chosen), dw = dense(grads[0]);
        variable_list out(1);
        if (!dw.defined()) return out;
        const Tensor dz = fresh_like(z);
        const int64_t experts = z.size(-1), tokens = z.numel() / experts;
        if (tokens) {
            const int rc = entry.route_backward(z.device().index(), dtype_of(z), tokens, (int)experts, ptr(z), ptr<int>(c), ptr<float>(dw), &how, ptr(dz), stream_of(z));
            TORCH_CHECK(rc == 0, "route: the backward pass was not launched (see stderr)");
        }
        out[0] = dz;
        return only_once("route", std::move(out), {&grads[0], &z});
    }
    std::string name() const override { return "RouteBackward"; }
    void release_variables() override { logits.reset_data(); chosen.reset_data(); }
};

/** route(logits, k, sigmoid, bias or None, groups, top_groups, top2, renormalize, scale): (weights, experts). */
PyObject* route(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(nargs == 9, "route takes nine arguments");
    Tensor z, bias;
    int64_t k, groups, top_groups;
    bool sigmoid, top2, renormalize;
    double scale;
    if (!tensor_of(args[0], false, &z) || !tensor_of(args[3], true, &bias) || !integer(args[1], 1, DCCL_EXPERTS_MAX_CHOSEN, &k) || !truth(args[2], &sigmoid)
        || !integer(args[4], 1, DCCL_EXPERTS_MAX_GROUPS, &groups) || !integer(args[5], 1, groups, &top_groups) || !truth(args[6], &top2) || !truth(args[7], &renormalize)
        || !number(args[8], &scale))
        Py_RETURN_NOTIMPLEMENTED;
    const int dtype = dtype_of(z);
    if (dtype < 0 || z.dim() < 1) Py_RETURN_NOTIMPLEMENTED;
    const int64_t experts = z.size(-1);
    if (experts < 1 || experts > DCCL_EXPERTS_MAX || experts % groups || k > top_groups * (experts / groups) || z.numel() / experts * k > DCCL_EXPERTS_MAX_PLACES) Py_RETURN_NOTIMPLEMENTED;
    if (bias.defined() && (bias.scalar_type() != at::kFloat || bias.dim() != 1 || bias.size(0) != experts || bias.device() != z.device())) Py_RETURN_NOTIMPLEMENTED;
    if (observed(args, nargs)) Py_RETURN_NONE;
    check_forward_mode("route", {&z});
    Tensor weights, chosen;
    {
        pybind11::gil_scoped_release no_gil;
        z = dense(z), bias = dense(bias);
        const auto sizes = with_last(z, k);
        weights = fresh(sizes, at::kFloat, z);
        chosen = fresh(sizes, at::kInt, z);
        const DcclRouting how = {sigmoid, (int)k, (int)groups, (int)top_groups, top2, renormalize, (float)scale};
        const int64_t tokens = z.numel() / experts;
        if (tokens) {
            const int rc = entry.route(z.device().index(), dtype, tokens, (int)experts, ptr(z), ptr<float>(bias), &how, ptr<float>(weights), ptr<int>(chosen), stream_of(z));
            TORCH_CHECK(rc == 0, "route was not launched (see stderr)");
        }
        if (records({&z})) {
            std::shared_ptr<RouteBackward> node(new RouteBackward(), torch::autograd::deleteNode);
            node->set_next_edges(torch::autograd::collect_next_edges(z));
            node->logits = SavedVariable(z, false);
            node->chosen = SavedVariable(chosen, false);
            node->how = how;
            torch::autograd::set_history(weights, node);
        }
    }
    return wrap(std::move(weights), std::move(chosen));
    END_HANDLE_TH_ERRORS
}

/** expert_plan(experts, number of them): (rows, counts, starts). */
PyObject* expert_plan(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(nargs == 2, "expert_plan takes two arguments");
    Tensor chosen;
    int64_t experts;
    if (!tensor_of(args[0], false, &chosen) || !integer(args[1], 1, DCCL_EXPERTS_MAX, &experts)) Py_RETURN_NOTIMPLEMENTED;
    if ((chosen.scalar_type() != at::kInt && chosen.scalar_type() != at::kLong) || chosen.dim() < 1 || chosen.size(-1) < 1 || chosen.size(-1) > DCCL_EXPERTS_MAX_CHOSEN
        || chosen.numel() > DCCL_EXPERTS_MAX_PLACES)
        Py_RETURN_NOTIMPLEMENTED;
    if (observed(args, nargs)) Py_RETURN_NONE;
    Tensor rows, counts, starts;
    {
        pybind11::gil_scoped_release no_gil;
        chosen = dense(chosen);
        rows = fresh(chosen.sizes(), at::kInt, chosen);
        counts = fresh({experts}, at::kInt, chosen);
        starts = fresh({experts + 1}, at::kInt, chosen);
        const int rc = entry.plan(chosen.device().index(), chosen.numel(), (int)experts, ptr(chosen), chosen.scalar_type() == at::kLong, ptr<int>(rows), ptr<int>(counts), ptr<int>(starts),
                                  stream_of(chosen));
        TORCH_CHECK(rc == 0, "expert_plan was not launched (see stderr)");
    }
    return wrap3(std::move(rows), std::move(counts), std::move(starts));
    END_HANDLE_TH_ERRORS
}

/* ---------------------------------------------------------------------------------------------- dispatch and combine */

bool plan_fits(const Tensor& rows, const Tensor& starts, const Tensor& like) {
    return rows.scalar_type() == at::kInt && rows.dim() >= 1 && rows.size(-1) >= 1 && rows.size(-1) <= DCCL_EXPERTS_MAX_CHOSEN && rows.numel() <= DCCL_EXPERTS_MAX_PLACES
           && starts.scalar_type() == at::kInt && starts.dim() == 1 && starts.size(0) >= 2 && starts.size(0) <= DCCL_EXPERTS_MAX + 1 && rows.device() == like.device()
           && starts.device() == like.device();
}
bool width_fits(const Tensor& t) { return t.dim() >= 1 && t.size(-1) >= 1 && t.size(-1) <= DCCL_EXPERTS_MAX_WIDTH; }

/** Whether each row that a plan uses has a place: said by whoever knows, or because `rows` and `starts` are still the tensors that expert_plan made, as it made them. */
bool whole_plan(PyObject* made, PyObject* rows, PyObject* starts, bool* whole) {
    if (made == Py_None) return *whole = false, true;
    if (!PyTuple_Check(made)) return truth(made, whole);
    const auto unchanged = [](PyObject* o) {
        at::TensorImpl* const t = THPVariable_Unpack(o).unsafeGetTensorImpl();
        return t->is_inference() || t->version_counter().current_version() == 0;
    };
    *whole = PyTuple_GET_SIZE(made) == 2 && PyTuple_GET_ITEM(made, 0) == rows && PyTuple_GET_ITEM(made, 1) == starts && unchanged(rows) && unchanged(starts);
    return true;
}
/** How many rows a whole plan uses, each of which has a place. Of another one it is not known which have. */
const int* used_of(const Tensor& starts, bool whole) { return whole ? ptr<int>(starts) + starts.size(0) - 1 : nullptr; }
/** What rows are written to that one of the plan's places has: others are zeros. */
Tensor rows_for(bool whole, at::IntArrayRef sizes, const Tensor& like) {
    const Tensor t = fresh(sizes, like.scalar_type(), like);
    if (!whole) t.zero_();
    return t;
}

Tensor run_combine(const Tensor& in, const Tensor& rows, const Tensor& weights, at::IntArrayRef sizes) {
    const Tensor y = fresh(sizes, in.scalar_type(), in);
    const int64_t k = rows.size(-1), tokens = rows.numel() / k;
    if (tokens) {
        const int rc = entry.combine(in.device().index(), dtype_of(in), tokens, (int)k, in.size(-1), ptr(in), ptr<int>(rows), ptr(weights),
                                     weights.defined() && weights.scalar_type() == at::kFloat, ptr(y), stream_of(in));
        TORCH_CHECK(rc == 0, "combine was not launched (see stderr)");
    }
    return y;
}

struct DispatchBackward : public Node {
    SavedVariable rows;
    c10::SmallVector<int64_t, 6> sizes;

    variable_list apply(variable_list&& grads) override {
        const Tensor r = unpacked(rows), g = dense(grads[0]);
        variable_list out(1);
        if (!g.defined()) return out;
        out[0] = run_combine(g, r, Tensor(), sizes);
        return only_once("dispatch", std::move(out), {&grads[0]});
    }
    std::string name() const override { return "DispatchBackward"; }
    void release_variables() override { rows.reset_data(); }
};

/** dispatch(x, rows, starts, whether each row that is used has a place, or what whole_plan tells it by): x's rows in the order of the experts. */
PyObject* dispatch(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(nargs == 4, "dispatch takes four arguments");
    Tensor x, rows, starts;
    bool whole;
    if (!tensor_of(args[0], false, &x) || !tensor_of(args[1], false, &rows) || !tensor_of(args[2], false, &starts) || !whole_plan(args[3], args[1], args[2], &whole))
        Py_RETURN_NOTIMPLEMENTED;
    const int dtype = dtype_of(x);
    if (dtype < 0 || !width_fits(x) || !plan_fits(rows, starts, x) || x.dim() != rows.dim() || x.sizes().slice(0, x.dim() - 1) != rows.sizes().slice(0, x.dim() - 1)) Py_RETURN_NOTIMPLEMENTED;
    if (observed(args, nargs)) Py_RETURN_NONE;
    check_forward_mode("dispatch", {&x});
    Tensor out;
    {
        pybind11::gil_scoped_release no_gil;
        x = dense(x), rows = dense(rows), starts = dense(starts);
        const int64_t width = x.size(-1), k = rows.size(-1), tokens = rows.numel() / k;
        out = rows_for(whole, {tokens * k, width}, x);
        if (tokens) {
            const int rc = entry.dispatch(x.device().index(), dtype, tokens, (int)k, width, ptr(x), ptr<int>(rows), used_of(starts, whole), ptr(out), stream_of(x));
            TORCH_CHECK(rc == 0, "dispatch was not launched (see stderr)");
        }
        if (records({&x})) {
            std::shared_ptr<DispatchBackward> node(new DispatchBackward(), torch::autograd::deleteNode);
            node->set_next_edges(torch::autograd::collect_next_edges(x));
            node->rows = SavedVariable(rows, false);
            node->sizes.assign(x.sizes().begin(), x.sizes().end());
            torch::autograd::set_history(out, node);
        }
    }
    return wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

struct CombineBackward : public Node {
    SavedVariable in, rows, starts, weights;
    bool whole = false;

    variable_list apply(variable_list&& grads) override {
        const Tensor v = unpacked(in), r = unpacked(rows), s = unpacked(starts), w = unpacked(weights), dy = dense(grads[0]);
        variable_list out(2);
        if (!dy.defined()) return out;
        const Tensor din = task_should_compute_output(0) ? rows_for(whole, v.sizes(), v) : Tensor(), dw = w.defined() && task_should_compute_output(1) ? fresh_like(w) : Tensor();
        const int64_t k = r.size(-1), tokens = r.numel() / k;
        if (tokens && (din.defined() || dw.defined())) {
            const int rc = entry.combine_backward(v.device().index(), dtype_of(v), tokens, (int)k, v.size(-1), ptr(dy), ptr(v), ptr<int>(r), used_of(s, whole), ptr(w),
                                                  w.defined() && w.scalar_type() == at::kFloat, ptr(din), ptr(dw), stream_of(v));
            TORCH_CHECK(rc == 0, "combine: the backward pass was not launched (see stderr)");
        }
        out = {din, dw};
        return only_once("combine", std::move(out), {&grads[0], &v, &w});
    }
    std::string name() const override { return "CombineBackward"; }
    void release_variables() override {
        for (SavedVariable* v : {&in, &rows, &starts, &weights}) v->reset_data();
    }
};

/** combine(in, rows, starts, weights or None, whether each row that is used has a place, or likewise): the weighted sums of each token's rows. */
PyObject* combine(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(nargs == 5, "combine takes five arguments");
    Tensor in, rows, starts, weights;
    bool whole;
    if (!tensor_of(args[0], false, &in) || !tensor_of(args[1], false, &rows) || !tensor_of(args[2], false, &starts) || !tensor_of(args[3], true, &weights) || !whole_plan(args[4], args[1], args[2], &whole))
        Py_RETURN_NOTIMPLEMENTED;
    if (dtype_of(in) < 0 || in.dim() != 2 || !width_fits(in) || !plan_fits(rows, starts, in) || in.size(0) != rows.numel()) Py_RETURN_NOTIMPLEMENTED;
    if (weights.defined() && (weights.sizes() != rows.sizes() || weights.device() != in.device() || (weights.scalar_type() != at::kFloat && weights.scalar_type() != in.scalar_type())))
        Py_RETURN_NOTIMPLEMENTED;
    if (observed(args, nargs)) Py_RETURN_NONE;
    check_forward_mode("combine", {&in, &weights});
    Tensor y;
    {
        pybind11::gil_scoped_release no_gil;
        in = dense(in), rows = dense(rows), starts = dense(starts), weights = dense(weights);
        y = run_combine(in, rows, weights, with_last(rows, in.size(-1)));
        if (records({&in, &weights})) {
            std::shared_ptr<CombineBackward> node(new CombineBackward(), torch::autograd::deleteNode);
            node->set_next_edges(torch::autograd::collect_next_edges(in, weights));
            node->in = SavedVariable(in, false);
            node->rows = SavedVariable(rows, false);
            node->starts = SavedVariable(starts, false);
            node->weights = SavedVariable(weights, false);
            node->whole = whole;
            torch::autograd::set_history(y, node);
        }
    }
    return wrap(std::move(y));
    END_HANDLE_TH_ERRORS
}

/* ---------------------------------------------------------------------------------------------- the experts' products */

bool on_16(const Tensor& a, const Tensor& b) { return ((uintptr_t)a.data_ptr() | (uintptr_t)b.data_ptr()) % 16 == 0; }

Tensor moved_to_16(const Tensor& t) { return t.defined() && (uintptr_t)t.data_ptr() % 16 ? t.clone() : t; }

/** The workspace of a call; undefined where it needs none. */
Tensor linear_work(const Tensor& x, const Tensor& w, bool backward) {
    const long long bytes = entry.linear_workspace(x.device().index(), x.size(0), (int)w.size(0), w.size(2), w.size(1), on_16(x, w), backward);
    TORCH_CHECK(bytes >= 0, "expert_linear: sizes that it does not take");
    return bytes ? fresh({(int64_t)bytes}, at::kByte, x) : Tensor();
}

struct ExpertLinearBackward : public Node {
    SavedVariable x, w, starts, z, padded;
    int act = -1;

    variable_list apply(variable_list&& grads) override {
        Tensor x_ = unpacked(x), w_ = unpacked(w);
        const Tensor s = unpacked(starts), z_ = moved_to_16(unpacked(z)), copies = moved_to_16(unpacked(padded)), dh = dense(grads[0]);
        variable_list out(2);
        if (!dh.defined()) return out;
        if (!copies.defined()) x_ = moved_to_16(x_), w_ = moved_to_16(w_);      // so the forward pass had them
        const Tensor dx = task_should_compute_output(0) ? fresh_like(x_) : Tensor(), dw = task_should_compute_output(1) ? fresh_like(w_) : Tensor();
        if (x_.size(0)) {
            const Tensor work = linear_work(x_, w_, true);
            const int rc = entry.linear_backward(x_.device().index(), dtype_of(x_), x_.size(0), (int)w_.size(0), w_.size(2), w_.size(1), ptr(dh), ptr<float>(z_), z_.defined() ? z_.size(1) : 0,
                                                 ptr(x_), ptr(w_), ptr<int>(s), ptr(copies), act, ptr(dx), ptr(dw), ptr(work), work.defined() ? (long long)work.numel() : 0, stream_of(x_));
            TORCH_CHECK(rc == 0, "expert_linear: the backward pass was not launched (see stderr)");
        } else if (dw.defined()) {
            dw.zero_();
        }
        out = {dx, dw};
        return only_once("expert_linear", std::move(out), {&grads[0], &x_, &w_});
    }
    std::string name() const override { return "ExpertLinearBackward"; }
    void release_variables() override {
        for (SavedVariable* v : {&x, &w, &starts, &z, &padded}) v->reset_data();
    }
};

/** expert_linear(x, w, starts, number of the activation or -1): h. */
PyObject* expert_linear(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(nargs == 4, "expert_linear takes four arguments");
    Tensor x, w, starts;
    int64_t act;
    if (!tensor_of(args[0], false, &x) || !tensor_of(args[1], false, &w) || !tensor_of(args[2], false, &starts) || !integer(args[3], -1, DCCL_ACT_GELU_TANH, &act)) Py_RETURN_NOTIMPLEMENTED;
    const int dtype = dtype_of(x);
    if ((dtype != 6 && dtype != 9) || x.dim() != 2 || w.dim() != 3 || w.scalar_type() != x.scalar_type() || w.device() != x.device() || starts.device() != x.device()
        || starts.scalar_type() != at::kInt || starts.dim() != 1)
        Py_RETURN_NOTIMPLEMENTED;
    const int64_t rows = x.size(0), experts = w.size(0), out = w.size(1), width = w.size(2);
    if (x.size(1) != width || experts < 1 || experts > DCCL_EXPERTS_MAX || starts.size(0) != experts + 1 || width < 1 || out < 1 || width > DCCL_EXPERTS_MAX_WIDTH
        || out > DCCL_EXPERTS_MAX_WIDTH || rows > DCCL_EXPERTS_MAX_PLACES)
        Py_RETURN_NOTIMPLEMENTED;
    if (observed(args, nargs)) Py_RETURN_NONE;
    check_forward_mode("expert_linear", {&x, &w});
    Tensor h;
    {
        pybind11::gil_scoped_release no_gil;
        x = dense(x), w = dense(w), starts = dense(starts);
        const bool keep = records({&x, &w});
        h = fresh({rows, out}, x.scalar_type(), x);
        Tensor z, work;
        const int64_t stride = (out + 3) / 4 * 4;
        if (keep && act >= 0) z = fresh({rows, stride}, at::kFloat, x);
        if (rows) {
            work = linear_work(x, w, false);
            const int rc = entry.linear(x.device().index(), dtype, rows, (int)experts, width, out, ptr(x), ptr(w), ptr<int>(starts), (int)act, ptr(h), ptr<float>(z), z.defined() ? stride : 0,
                                        ptr(work), work.defined() ? (long long)work.numel() : 0, stream_of(x));
            TORCH_CHECK(rc == 0, "expert_linear was not launched (see stderr)");
        }
        if (keep) {
            std::shared_ptr<ExpertLinearBackward> node(new ExpertLinearBackward(), torch::autograd::deleteNode);
            node->set_next_edges(torch::autograd::collect_next_edges(x, w));
            node->x = SavedVariable(x, false);
            node->w = SavedVariable(w, false);
            node->starts = SavedVariable(starts, false);
            node->z = SavedVariable(z, false);
            node->padded = SavedVariable(entry.linear_pads(width, on_16(x, w)) ? work : Tensor(), false);
            node->act = (int)act;
            torch::autograd::set_history(h, node);
        }
    }
    return wrap(std::move(h));
    END_HANDLE_TH_ERRORS
}

/** expert_ops_bind(addresses of the entry points, in the order of Entries). */
PyObject* expert_ops_bind(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    void* at[10];
    TORCH_CHECK(nargs == 10, "expert_ops_bind takes ten addresses");
    for (int i = 0; i < 10; i++) {
        at[i] = PyLong_AsVoidPtr(args[i]);
        if (PyErr_Occurred()) return nullptr;
        TORCH_CHECK(at[i], "expert_ops_bind: an address is missing");
    }
    entry = {reinterpret_cast<decltype(entry.route)>(at[0]), reinterpret_cast<decltype(entry.route_backward)>(at[1]), reinterpret_cast<decltype(entry.plan)>(at[2]),
             reinterpret_cast<decltype(entry.dispatch)>(at[3]), reinterpret_cast<decltype(entry.combine)>(at[4]), reinterpret_cast<decltype(entry.combine_backward)>(at[5]),
             reinterpret_cast<decltype(entry.linear_workspace)>(at[6]), reinterpret_cast<decltype(entry.linear_pads)>(at[7]), reinterpret_cast<decltype(entry.linear)>(at[8]),
             reinterpret_cast<decltype(entry.linear_backward)>(at[9])};
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"route", (PyCFunction)(void (*)())route, METH_FASTCALL, "(weights, experts); NotImplemented where the arguments do not fit, None where the call is observed"},
    {"expert_plan", (PyCFunction)(void (*)())expert_plan, METH_FASTCALL, "(rows, counts, starts); NotImplemented and None likewise"},
    {"dispatch", (PyCFunction)(void (*)())dispatch, METH_FASTCALL, "rows in the order of the experts; NotImplemented and None likewise"},
    {"combine", (PyCFunction)(void (*)())combine, METH_FASTCALL, "weighted sums of each token's rows; NotImplemented and None likewise"},
    {"expert_linear", (PyCFunction)(void (*)())expert_linear, METH_FASTCALL, "act(x W^T) by experts; NotImplemented and None likewise"},
    {"expert_ops_bind", (PyCFunction)(void (*)())expert_ops_bind, METH_FASTCALL, "hands over the addresses of the library's entry points"},
    {nullptr, nullptr, 0, nullptr},
};

} // namespace

int add_expert_ops(PyObject* module) { return PyModule_AddFunctions(module, methods); }

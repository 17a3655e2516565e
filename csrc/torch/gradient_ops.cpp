/**
 * Host side of the norm of many tensors and of clipping (csrc/gradients/grad_norm.hpp) for dccl_b200/ops/gradients.py, in the manner of decoder_ops.cpp. Nothing
 * here has a gradient.
 */
#include "gradient_ops.hpp"
#include "../gradients/grad_norm.hpp"
#include "tensor_args.hpp"
#include <algorithm>

namespace {

using namespace host_side;

struct Entries {
    decltype(&dccl_grad_parts) parts;
    decltype(&dccl_grad_squares) squares;
    decltype(&dccl_grad_total) total;
    decltype(&dccl_grad_clip) clip;
} entry;

/** The tensors of a sequence, as they lie: dense, of one device. What does not fit is left to Python. */
struct List {
    THPObjectPtr seq;
    std::vector<Tensor> tensors;
    bool observed_ = false;

    bool read(PyObject* o) {
        seq = THPObjectPtr(PySequence_Fast(o, "a sequence of tensors"));
        if (!seq) throw python_error();
        const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq.get());
        PyObject** items = PySequence_Fast_ITEMS(seq.get());
        if (!n) return false;
        tensors.resize(n);
        for (Py_ssize_t i = 0; i < n; i++) {
            if (!tensor_of(items[i], false, &tensors[i])) return false;
            const Tensor& t = tensors[i];
            if (dtype_of(t) < 0 || t.device() != tensors[0].device() || !t.is_non_overlapping_and_dense() || t.is_neg()) return false;
        }
        observed_ = observed(items, n);
        return true;
    }
};

bool same_layout(const Tensor& a, const Tensor& b) {
    if (a.sizes() != b.sizes()) return false;
    for (int64_t d = 0; d < a.dim(); d++)
        if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
    return true;
}

std::vector<DcclGradient> table(const std::vector<Tensor>& in, const std::vector<Tensor>& out) {
    std::vector<DcclGradient> t;
    t.reserve(in.size());
    for (size_t i = 0; i < in.size(); i++)
        if (in[i].numel()) t.push_back({in[i].data_ptr(), out[i].data_ptr(), (size_t)in[i].numel(), dtype_of(in[i]), dtype_of(out[i])});
    return t;
}

/** Whether what is written overlaps anything but, as a whole and of the same type, the tensor that it comes from. What is only read may be read twice. */
bool overlaps(const std::vector<DcclGradient>& t, bool apart) {
    const auto bytes = [](size_t n, int dtype) { return n * (dtype == 7 ? 4 : 2); };
    struct Range { uintptr_t from, to; bool written; };
    std::vector<Range> r;
    r.reserve(t.size() * (apart ? 2 : 1));
    for (const DcclGradient& g : t) {
        r.push_back({(uintptr_t)g.out, (uintptr_t)g.out + bytes(g.elements, g.out_dtype), true});
        if (apart && (g.in != g.out || g.dtype != g.out_dtype)) r.push_back({(uintptr_t)g.in, (uintptr_t)g.in + bytes(g.elements, g.dtype), false});
    }
    std::sort(r.begin(), r.end(), [](const Range& a, const Range& b) { return a.from < b.from; });
    uintptr_t written = 0, any = 0;         // the ends of those before
    for (const Range& g : r) {
        if (g.from < (g.written ? any : written)) return true;
        any = std::max(any, g.to);
        if (g.written) written = std::max(written, g.to);
    }
    return false;
}

Tensor parts_of(const std::vector<DcclGradient>& t, const Tensor& like) {
    const size_t count = t.empty() ? 0 : entry.parts(like.device().index(), t.size(), t.data());
    TORCH_CHECK(t.empty() || count, "grad_norm: tensors that it does not take");
    const Tensor parts = fresh({(int64_t)count}, at::kDouble, like);
    if (count) {
        const int rc = entry.squares(like.device().index(), t.size(), t.data(), ptr<double>(parts), stream_of(like));
        TORCH_CHECK(rc == 0, "grad_norm was not launched (see stderr)");
    }
    return parts;
}

/** grad_norm(tensors, whether the sum of squares is wanted): the norm as a float, or the sum as a double, of no dimensions. */
PyObject* grad_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(nargs == 2, "grad_norm takes two arguments");
    List in;
    if (!in.read(args[0])) Py_RETURN_NOTIMPLEMENTED;
    const bool sum = args[1] == Py_True;
    if (in.observed_) Py_RETURN_NONE;
    Tensor out;
    {
        pybind11::gil_scoped_release no_gil;
        const Tensor& like = in.tensors[0];
        const Tensor parts = parts_of(table(in.tensors, in.tensors), like);
        out = fresh({}, sum ? at::kDouble : at::kFloat, like);
        const int rc = entry.total(like.device().index(), ptr<double>(parts), parts.numel(), sum ? ptr<double>(out) : nullptr, sum ? nullptr : ptr<float>(out), stream_of(like));
        TORCH_CHECK(rc == 0, "grad_norm was not launched (see stderr)");
    }
    return wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

/** clip_grad_norm(tensors, outs or None, limit, sum of squares or None): the norm, with the tensors or outs clipped. False where what is written overlaps. */
PyObject* clip_grad_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(nargs == 4, "clip_grad_norm takes four arguments");
    List in, out;
    double limit;
    Tensor sum;
    if (!in.read(args[0]) || !number(args[2], &limit) || !(limit >= 0) || !tensor_of(args[3], true, &sum)) Py_RETURN_NOTIMPLEMENTED;
    const bool apart = args[1] != Py_None;
    if (apart) {
        if (!out.read(args[1]) || out.tensors.size() != in.tensors.size() || out.tensors[0].device() != in.tensors[0].device()) Py_RETURN_NOTIMPLEMENTED;
        for (size_t i = 0; i < in.tensors.size(); i++)
            if (!same_layout(in.tensors[i], out.tensors[i]) || (out.tensors[i].scalar_type() != in.tensors[i].scalar_type() && out.tensors[i].scalar_type() != at::kFloat))
                Py_RETURN_NOTIMPLEMENTED;
    }
    if (sum.defined() && (sum.scalar_type() != at::kDouble || sum.numel() != 1 || sum.device() != in.tensors[0].device())) Py_RETURN_NOTIMPLEMENTED;
    if (in.observed_ || out.observed_) Py_RETURN_NONE;
    const std::vector<Tensor>& to = apart ? out.tensors : in.tensors;
    for (const Tensor& t : to)
        if (t.unsafeGetTensorImpl()->is_inference() && !c10::InferenceMode::is_enabled()) Py_RETURN_NOTIMPLEMENTED;
    Tensor norm;
    bool bad = false;
    {
        pybind11::gil_scoped_release no_gil;
        const Tensor& like = in.tensors[0];
        const std::vector<DcclGradient> t = table(in.tensors, to);
        bad = overlaps(t, apart);
        if (!bad) {
            const Tensor parts = sum.defined() ? sum : parts_of(t, like);
            norm = fresh({}, at::kFloat, like);
            const int rc = t.empty() ? entry.total(like.device().index(), ptr<double>(parts), parts.numel(), nullptr, ptr<float>(norm), stream_of(like))
                                     : entry.clip(like.device().index(), t.size(), t.data(), ptr<double>(parts), parts.numel(), limit, ptr<float>(norm), stream_of(like));
            TORCH_CHECK(rc == 0, "clip_grad_norm was not launched (see stderr)");
            for (const Tensor& o : to) o.unsafeGetTensorImpl()->bump_version();
        }
    }
    if (bad) Py_RETURN_FALSE;
    return wrap(std::move(norm));
    END_HANDLE_TH_ERRORS
}

/** gradient_ops_bind(addresses of the entry points, in the order of Entries). */
PyObject* gradient_ops_bind(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
    HANDLE_TH_ERRORS
    void* at[4];
    TORCH_CHECK(nargs == 4, "gradient_ops_bind takes four addresses");
    for (int i = 0; i < 4; i++) {
        at[i] = PyLong_AsVoidPtr(args[i]);
        if (PyErr_Occurred()) return nullptr;
        TORCH_CHECK(at[i], "gradient_ops_bind: an address is missing");
    }
    entry = {reinterpret_cast<decltype(entry.parts)>(at[0]), reinterpret_cast<decltype(entry.squares)>(at[1]), reinterpret_cast<decltype(entry.total)>(at[2]),
             reinterpret_cast<decltype(entry.clip)>(at[3])};
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"grad_norm", (PyCFunction)(void (*)())grad_norm, METH_FASTCALL, "the norm, or the sum of squares; NotImplemented where the arguments do not fit, None where the call is observed"},
    {"clip_grad_norm", (PyCFunction)(void (*)())clip_grad_norm, METH_FASTCALL, "the norm, and the tensors clipped; NotImplemented and None likewise, False where what is written overlaps"},
    {"gradient_ops_bind", (PyCFunction)(void (*)())gradient_ops_bind, METH_FASTCALL, "hands over the addresses of the library's entry points"},
    {nullptr, nullptr, 0, nullptr},
};

} // namespace

int add_gradient_ops(PyObject* module) { return PyModule_AddFunctions(module, methods); }

// What the native host paths of the operators over rows of tokens share (native_sequence.cc, native_language.cc): strided rows as
// operands, results, and gradients that can be differentiated once.
#ifndef BPL_CSRC_NATIVE_ROWS_H_
#define BPL_CSRC_NATIVE_ROWS_H_

#include "native.h"

#include <torch/csrc/autograd/functions/basic_ops.h>

#include <optional>

namespace {

bool plain_cotangent_keys(const Tensor &t) { return plain_keys(t) && plain_thread() && !t._fw_grad(0).defined(); }
bool strided_plain(const Tensor &t) {
    return t.defined() && plain_keys(t) && !(c10::isFloatingType(t.scalar_type()) && t._fw_grad(0).defined());
}
// None counts as absent; anything but None or a plain CUDA tensor makes the call not plain
bool operand(PyObject *o, const Tensor *&t, bool optional = false) {
    t = nullptr;
    if (o == Py_None) return optional;
    if (!THPVariable_CheckExact(o)) return false;
    const Tensor &v = THPVariable_Unpack(o);
    if (!strided_plain(v) || !v.is_cuda()) return false;
    t = &v;
    return true;
}

int dtype_of(const Tensor &t) {
    switch (t.scalar_type()) {
        case at::kFloat: return BPL_FLOAT;
        case at::kHalf: return BPL_HALF;
        case at::kBFloat16: return BPL_BFLOAT16;
        default: return -1;
    }
}

// (tokens, ...) or (batch, length, ...) with `inner` trailing dimensions, read as rows: the distance of neighbouring rows, or
// false where the rows have no single one
struct Rows {
    int64_t batch = 0, length = 0, rows = 0, stride = 0;
    bool batched = false;
};
bool rows_of(const Tensor &t, int64_t inner, Rows &r) {
    const int64_t lead = t.dim() - inner;
    if (lead != 1 && lead != 2) return false;
    r.batched = lead == 2;
    r.batch = r.batched ? t.size(0) : 1;
    r.length = t.size(lead - 1);
    r.rows = r.batch * r.length;
    if (t.numel() == 0) return true;        // nothing to address (and no stride says anything: an empty tensor is contiguous)
    r.stride = t.stride(lead - 1);
    if (r.batched && r.batch > 1) {
        if (r.length == 1) r.stride = t.stride(0);
        else if (t.stride(0) != r.length * r.stride) return false;
    }
    return t.size(-1) <= 1 || t.stride(-1) == 1;
}
bool same_rows(const Rows &a, const Rows &b) { return a.batched == b.batched && a.batch == b.batch && a.length == b.length; }

bool dense(const Tensor *t, at::ScalarType type, at::IntArrayRef size, const Tensor &like) {
    return t->scalar_type() == type && t->sizes() == size && t->is_contiguous() && t->device() == like.device();
}

bool truth(PyObject *o) { return o == Py_True; }
// (what else counts as true goes the Python way)
bool is_flag(PyObject *o) { return o == Py_True || o == Py_False; }

// a write that autograd does not see: tensors saved before it count as changed
void written(const Tensor &t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void *ptr_of(const Tensor *t) { return t ? ptr(*t) : nullptr; }
PyObject *wrap(Tensor t) {
    if (t.defined()) return THPVariable_Wrap(std::move(t));
    Py_RETURN_NONE;
}
PyObject *tuple_of(std::initializer_list<Tensor> tensors) {
    PyObject *res = PyTuple_New(static_cast<Py_ssize_t>(tensors.size()));
    if (res == nullptr) return nullptr;
    Py_ssize_t i = 0;
    for (const Tensor &t : tensors) {
        PyObject *o = wrap(t);
        if (o == nullptr) {
            Py_DECREF(res);
            return nullptr;
        }
        PyTuple_SET_ITEM(res, i++, o);
    }
    return res;
}

// ---- both passes ------------------------------------------------------------------------------------------------------
void *at_or_null(const Tensor &t) { return t.defined() ? ptr(t) : nullptr; }
const Tensor *or_null(const Tensor &t) { return t.defined() ? &t : nullptr; }
std::optional<Tensor> maybe(const Tensor *t) { return t ? std::optional<Tensor>(*t) : std::nullopt; }
Tensor value(const std::optional<Tensor> &t) { return t.value_or(Tensor()); }

// the cotangent of an output as the kernels read it: dense, zeros where there is none
Tensor cotangent(const Tensor &g, const Tensor &like) {
    if (!g.defined()) return at::zeros(like.sizes(), like.options());
    if (!plain_cotangent_keys(g)) throw std::runtime_error("gradients of the operators over sequences are plain CUDA tensors only");
    return g.contiguous();
}
// A second derivative is refused where it is asked for, not here.
variable_list differentiable_once(variable_list grads, const char *name) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list out;
    for (const Tensor &g : grads)
        out.push_back(g.defined() ? g.detach().set_requires_grad(true) : g);
    auto refuse = std::make_shared<torch::autograd::DelayedError>(std::string(name) + " is differentiable once only",
                                                                  static_cast<int64_t>(out.size()));
    return (*refuse)(std::move(out));
}

PyObject *one_or_two(const variable_list &v) { return v.size() == 2 ? tuple_of({v[0], v[1]}) : wrap(v[0]); }

}  // namespace

#endif  // BPL_CSRC_NATIVE_ROWS_H_

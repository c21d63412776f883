// What the files of the extension module `_native` share: which operands the native host path takes, scratch memory, the
// current device and stream, and the status of a call.
#ifndef BPL_CSRC_NATIVE_H_
#define BPL_CSRC_NATIVE_H_

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/TracerMode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <stdexcept>
#include <string>

#include "abi.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

using Target = void (*)(bpl_stream_t, void **, const char *, size_t);

// ---------------------------------------------------------------------------------------------------------
// operands
// ---------------------------------------------------------------------------------------------------------
// A plain strided CUDA tensor carries these keys only; a wrapped one (functorch, fake, functional, subclass) more.
bool plain_keys(const Tensor &t) {
    static const uint64_t allowed = c10::DispatchKeySet({c10::DispatchKey::CUDA, c10::DispatchKey::ADInplaceOrView,
                                                         c10::DispatchKey::AutogradCUDA,
                                                         c10::DispatchKey::AutocastCUDA}).raw_repr();
    return (t.key_set().raw_repr() & ~allowed) == 0;
}

// no functorch transform and no dispatch mode is active on this thread
bool untransformed() {
    return !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode) &&
           !c10::impl::TorchDispatchModeTLS::any_modes_set();
}
// nor a tracer: torch.jit.trace records the Python autograd functions
bool plain_thread() { return untransformed() && !at::tracer::impl::is_dispatch_enabled(); }

bool plain(const Tensor &t) {
    return t.defined() && plain_keys(t) && t.is_contiguous() &&
           !(c10::isFloatingType(t.scalar_type()) && t._fw_grad(0).defined());
}

const Tensor *tensor_of(PyObject *o) {
    if (!THPVariable_CheckExact(o)) return nullptr;
    const Tensor &t = THPVariable_Unpack(o);
    return plain(t) ? &t : nullptr;
}

bool int32_like(const Tensor &t) { return t.scalar_type() == at::kInt || t.scalar_type() == at::kUInt32; }
bool float_like(const Tensor &t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kDouble; }
bool is_double(const Tensor &t) { return t.scalar_type() == at::kDouble; }

bool shape_of(PyObject *o, int64_t &a, int64_t &b) {
    if (!PyTuple_CheckExact(o) || PyTuple_GET_SIZE(o) != 2) return false;
    PyObject *x = PyTuple_GET_ITEM(o, 0), *y = PyTuple_GET_ITEM(o, 1);
    if (!PyLong_CheckExact(x) || !PyLong_CheckExact(y)) return false;
    int over_a = 0, over_b = 0;
    a = PyLong_AsLongLongAndOverflow(x, &over_a);
    b = PyLong_AsLongLongAndOverflow(y, &over_b);
    return !over_a && !over_b && a >= 0 && b >= 0 && a <= 0xffffffffll && b <= 0xffffffffll;
}

// Python numbers of the exact types only: what else converts to a number goes the Python way
bool number_of(PyObject *o, double &v) {
    if (PyFloat_CheckExact(o)) {
        v = PyFloat_AS_DOUBLE(o);
        return true;
    }
    if (PyLong_CheckExact(o)) {
        v = PyLong_AsDouble(o);
        if (v == -1.0 && PyErr_Occurred()) {
            PyErr_Clear();
            return false;
        }
        return true;
    }
    return false;
}

bool wants_grad(const Tensor &t) { return t.requires_grad() && at::GradMode::is_enabled(); }

// ---------------------------------------------------------------------------------------------------------
// calling a target
// ---------------------------------------------------------------------------------------------------------
// A launch waits where the stream's queue is full, an allocation where memory has to be freed: other Python threads run
// meanwhile.  (Backward passes come here without the lock.)
struct NoGil {
    PyThreadState *state = PyGILState_Check() ? PyEval_SaveThread() : nullptr;
    NoGil() = default;
    ~NoGil() {
        if (state) PyEval_RestoreThread(state);
    }
    NoGil(const NoGil &) = delete;
    NoGil &operator=(const NoGil &) = delete;
};

// Scratch of one call, from torch's stream-ordered allocator: taken and given back around the launches, so calls of
// several threads and streams never share it, and the memory serves other tensors in between.
struct Scratch {
    void *ptr = nullptr;
    Scratch(size_t bytes, cudaStream_t stream) {
        if (bytes) ptr = c10::cuda::CUDACachingAllocator::raw_alloc_with_stream(bytes, stream);
    }
    ~Scratch() {
        if (ptr) c10::cuda::CUDACachingAllocator::raw_delete(ptr);
    }
    Scratch(const Scratch &) = delete;
    Scratch &operator=(const Scratch &) = delete;
};

void check_status() {
    if (bpl_last_status(nullptr, 0) == 0) return;
    char message[256];
    const int code = bpl_last_status(message, sizeof(message));
    bpl_clear_status();
    if (code == BPL_ERR_OPAQUE_SIZE) throw std::runtime_error(message[0] ? message : "Invalid opaque object size");
    throw std::runtime_error("brainpylib_b200 kernel error (" + std::to_string(code) + "): " + message);
}

Tensor new_tensor(at::IntArrayRef size, at::ScalarType dtype, const c10::Device &device) {
    return Tensor(at::detail::empty_cuda(size, dtype, device, std::nullopt));
}

// the device of `t` is current while this lives
struct OnDevice {
    c10::cuda::OptionalCUDAGuard guard;
    cudaStream_t stream;
    explicit OnDevice(const Tensor &t) {
        const auto index = t.device().index();
        if (c10::cuda::current_device() != index) guard.set_index(index);
        stream = c10::cuda::getCurrentCUDAStream(index).stream();
    }
};

void *ptr(const Tensor &t) { return const_cast<void *>(t.const_data_ptr()); }

#define NONE_UNLESS(condition) \
    do {                       \
        if (!(condition)) Py_RETURN_NONE; \
    } while (0)

}  // namespace

#endif  // BPL_CSRC_NATIVE_H_

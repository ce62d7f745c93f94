// What the native training operators share: the library's entry points, the forms of operands, the way to Python and back.
#pragma once
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <array>
#include <cstdint>
#include <map>
#include <mutex>
#include <memory>
#include <stdexcept>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/vtdge.h"

namespace vtdge_training {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

#define VT_FUNCTIONS(X)                                                                                                \
    X(last_error) X(cross_entropy) X(cross_entropy_backward) X(cross_entropy_workspace) X(cross_entropy_laid_out)      \
    X(gate_balance) X(gate_balance_backward) X(gate_balance_workspace) X(adamw)                                        \
    X(blocks_bytes) X(quantize_blocks) X(dequantize_blocks) X(gelu_8bit) X(gelu_8bit_backward)                         \
    X(layernorm_8bit) X(layernorm_8bit_backward) X(layernorm_8bit_backward_workspace)                                  \
    X(linear_8bit) X(linear_8bit_workspace) X(linear_8bit_backward) X(linear_8bit_backward_workspace)
struct Library {
#define VT_MEMBER(name) decltype(&vtdge_##name) name = nullptr;
    VT_FUNCTIONS(VT_MEMBER)
#undef VT_MEMBER
};
inline Library lib;
inline PyObject *error_type = nullptr;                 // vtpack_amd._lib.VtdgeError

struct Failure : std::runtime_error {
    using std::runtime_error::runtime_error;
};
inline void must(int rc, const char *what)
{
    if (rc != VTDGE_OK) throw Failure(std::string(what) + " failed (" + std::to_string(rc) + "): " + lib.last_error());
}

inline int code_of(const Tensor &t) { return t.scalar_type() == at::kFloat ? VTDGE_F32 : VTDGE_BF16; }
// from one row to the next; one row alone has no distance
inline int64_t pitch_of(const Tensor &t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
inline void *at_of(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
inline void *stream_of(const Tensor &t) { return (void *)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
inline Tensor fresh(const Tensor &like, at::IntArrayRef sizes, at::ScalarType type) { return at::empty(sizes, like.options().dtype(type).requires_grad(false)); }

// A workspace's bytes by the sizes it is for (working them out looks through many cuts of a sum).
template <size_t N, class F> int64_t bytes_of(const std::array<int64_t, N> &key, F ask)
{
    static std::mutex lock;
    static std::map<std::array<int64_t, N>, int64_t> known;
    std::lock_guard<std::mutex> hold(lock);
    const auto it = known.find(key);
    if (it != known.end()) return it->second;
    const int64_t bytes = ask();
    if (bytes < 0) throw Failure(lib.last_error());
    if (known.size() >= 1024) known.clear();
    return known[key] = bytes;
}

// ------------------------------------------------------------------------------------------------ forms of operands
inline bool rows_of_any_place(const Tensor &t)
{
    return t.defined() && t.dim() == 2 && t.numel() > 0 && (t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16) &&
           t.layout() == at::kStrided && (t.is_contiguous() || (t.stride(1) == 1 && t.stride(0) >= t.size(1)));
}
inline bool plain_rows(const Tensor &t) { return t.defined() && t.is_cuda() && rows_of_any_place(t); }
inline bool plain_beside(const Tensor &t, const Tensor &x, at::ScalarType type)
{
    return t.defined() && t.device() == x.device() && t.scalar_type() == type && t.layout() == at::kStrided && t.is_contiguous();
}

// Operands that are taken as they are: one that does not fit is named before anything is launched, the place of all of them last.
struct OperandChecks {
    const char *name;
    void need(bool fits, const char *what) const
    {
        if (!fits) throw std::runtime_error(std::string(name) + ": " + what);
    }
    void on_gpu(const Tensor &x) const { need(x.is_cuda(), "operands have to be on a GPU"); }
};

inline void no_second_order(const char *name)
{
    if (at::GradMode::is_enabled()) throw std::runtime_error(std::string(name) + ": gradients of the gradients are not supported");
}

inline void no_forward_mode(const char *name, std::initializer_list<const Tensor *> operands)
{
    for (const Tensor *t : operands)
        if (t->defined() && t->_fw_grad(0).defined()) throw std::runtime_error(std::string(name) + ": forward-mode derivatives are not supported");
}

// A trace would record the allocation of the results and not what fills them.
inline void no_tracing(const char *name)
{
    using Key = c10::impl::TorchDispatchModeKey;
    using Modes = c10::impl::TorchDispatchModeTLS;
    bool traced = torch::jit::tracer::isTracing();
    if (Modes::any_modes_set())
        for (const Key key : {Key::FAKE, Key::PROXY, Key::FUNCTIONAL}) traced = traced || Modes::get_mode(key).has_value();
    if (traced) throw std::runtime_error(std::string(name) + " cannot be traced");
}

// ------------------------------------------------------------------------------------------------ for Python
struct NoGil {
    PyThreadState *state = PyEval_SaveThread();
    ~NoGil() { PyEval_RestoreThread(state); }
};
inline Tensor tensor(PyObject *o)
{
    if (o == Py_None) return Tensor();
    if (!THPVariable_Check(o)) throw std::runtime_error("expected a tensor or None");
    return THPVariable_Unpack(o);
}
inline int64_t whole(PyObject *o)
{
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}
inline double real(PyObject *o)
{
    const double v = PyFloat_AsDouble(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}
inline PyObject *wrap(const Tensor &t)
{
    if (!t.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(t);
}
inline PyObject *tuple(std::initializer_list<Tensor> ts)
{
    PyObject *out = PyTuple_New((Py_ssize_t)ts.size());
    Py_ssize_t i = 0;
    for (const Tensor &t : ts) PyTuple_SET_ITEM(out, i++, wrap(t));
    return out;
}

// f(arguments) with `count` of them, what it throws as a Python exception
template <class F> PyObject *call(PyObject *const *args, Py_ssize_t given, Py_ssize_t count, F f)
{
    HANDLE_TH_ERRORS
    try {
        if (given != count) throw std::runtime_error("expected " + std::to_string(count) + " arguments, got " + std::to_string(given));
        return f();
    } catch (const Failure &e) {
        PyErr_SetString(error_type, e.what());
        return nullptr;
    }
    END_HANDLE_TH_ERRORS
}

// a tensor, or None where that may be
inline Tensor operand(const OperandChecks &check, PyObject *o, const char *what)
{
    check.need(o == Py_None || THPVariable_Check(o), what);
    return tensor(o);
}

#define VT_METHOD(name) {#name, (PyCFunction)(void (*)(void))py_##name, METH_FASTCALL, nullptr}

// in eight_bit.cpp
PyObject *py_quantize_blocks(PyObject *, PyObject *const *a, Py_ssize_t n);
PyObject *py_dequantize_blocks(PyObject *, PyObject *const *a, Py_ssize_t n);
PyObject *py_linear_8bit(PyObject *, PyObject *const *a, Py_ssize_t n);
PyObject *py_gelu_8bit(PyObject *, PyObject *const *a, Py_ssize_t n);
PyObject *py_layer_norm_8bit(PyObject *, PyObject *const *a, Py_ssize_t n);

}  // namespace vtdge_training

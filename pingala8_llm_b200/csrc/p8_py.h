// p8_py.h -- what the Python modules of the cache operators share: tensors and numbers taken from Python, refusals as ValueError,
// the device and stream of a call. `C` is what a call found out about its cache; its `dev` is the device.
#pragma once
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/DeviceGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>
#include <string>

#include "pingala8.h"

namespace {

using at::Tensor;

bool g_bound = false;  // bind() has been called

struct Refused {
    std::string what;
};
[[noreturn]] void refuse(std::string what) { throw Refused{std::move(what)}; }

const Tensor &tensor(PyObject *o, const char *name) {
    if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
    return THPVariable_Unpack(o);
}

const char *type_name(at::ScalarType t) { return t == at::kInt ? "int32" : t == at::kLong ? "int64" : t == at::kFloat ? "float32" : "the cache's type"; }
std::string shape_name(at::IntArrayRef s) {
    std::string r = "[";
    for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
    return r + "]";
}

// a contiguous tensor of exactly this shape, or NULL for None
template <typename T, typename C>
T *flat(PyObject *o, const char *name, at::ScalarType type, at::IntArrayRef shape, const C &c, bool optional = false) {
    if (optional && o == Py_None) return nullptr;
    const Tensor &t = tensor(o, name);
    if (t.scalar_type() != type || t.sizes() != shape || !t.is_cuda() || t.get_device() != c.dev || !t.is_contiguous())
        refuse(std::string(name) + " must be contiguous " + type_name(type) + " " + shape_name(shape) + " on the cache's device");
    return static_cast<T *>(t.data_ptr());
}
// [.., width]: address and outer strides
template <typename T, typename C, size_t N>
T *rows(PyObject *o, const char *name, at::ScalarType type, at::IntArrayRef shape, const C &c, int64_t (&st)[N]) {
    const Tensor &t = tensor(o, name);
    if (t.scalar_type() != type || t.sizes() != shape || !t.is_cuda() || t.get_device() != c.dev || t.stride((int64_t)N) != 1)
        refuse(std::string(name) + " must be " + type_name(type) + " " + shape_name(shape) + " with unit stride in its last dimension, on the cache's device");
    for (size_t i = 0; i < N; ++i) st[i] = t.stride((int64_t)i);
    return static_cast<T *>(t.data_ptr());
}

double number(PyObject *o) {
    const double x = PyFloat_AsDouble(o);
    if (x == -1.0 && PyErr_Occurred()) throw nullptr;
    return x;
}
int64_t integer(PyObject *o) {
    const long long x = PyLong_AsLongLong(o);
    if (x == -1 && PyErr_Occurred()) throw nullptr;
    return x;
}

// The tensors' device current for the launch, and its current stream.
struct On {
    std::optional<c10::DeviceGuard> guard;
    void *stream;
    template <typename C>
    explicit On(const C &c) {
        const c10::Device d(c10::kCUDA, (c10::DeviceIndex)c.dev);
        guard.emplace(d);
        stream = c10::cuda::getCurrentCUDAStream(d.index()).stream();
    }
};

#define ENTRY(name, count)                                                                  \
    PyObject *name(PyObject *, PyObject *const *a, Py_ssize_t n) {                          \
        try {                                                                               \
            if (n != (count)) refuse(#name " takes " #count " arguments");                  \
            if (!g_bound) refuse("bind() comes first");                                 \
            return PyLong_FromLong(name##_(a));                                             \
        } catch (const Refused &r) {                                                        \
            PyErr_SetString(PyExc_ValueError, r.what.c_str());                              \
        } catch (const std::exception &e) {                                                 \
            PyErr_SetString(PyExc_RuntimeError, e.what());                                  \
        } catch (std::nullptr_t) { /* the Python error is set */                            \
        }                                                                                   \
        return nullptr;                                                                     \
    }

}  // namespace

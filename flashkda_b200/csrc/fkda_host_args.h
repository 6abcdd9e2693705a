// What the host sides of the operators share: reading Python arguments, refusing them, and the workspace of a call.
#pragma once

#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <initializer_list>
#include <stdexcept>
#include <string>

#include "../../include/flashkda_b200.h"

namespace fkda_host {

struct Refused : std::runtime_error {
    using std::runtime_error::runtime_error;
};
inline void check(bool ok, const char* msg) {
    if (!ok) throw Refused(msg);
}
inline void check_named(bool ok, const char* name, const char* msg) {
    if (!ok) throw Refused(std::string(name) + msg);
}

inline const at::Tensor& tensor_arg(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) throw Refused(std::string(name) + " must be a torch.Tensor");
    return THPVariable_Unpack(o);
}
inline const at::Tensor* optional_tensor_arg(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor_arg(o, name); }

// Whatever float() takes: numpy scalars, one-element tensors, strings.
inline double number_arg(PyObject* o) {
    if (PyFloat_Check(o)) return PyFloat_AS_DOUBLE(o);
    PyObject* f = PyNumber_Float(o);
    if (f == nullptr) throw std::bad_cast();
    const double x = PyFloat_AS_DOUBLE(f);
    Py_DECREF(f);
    return x;
}
// Whatever int() takes.
inline long integer_arg(PyObject* o) {
    if (PyLong_Check(o)) {
        const long x = PyLong_AsLong(o);
        if (x == -1 && PyErr_Occurred()) throw std::bad_cast();
        return x;
    }
    PyObject* i = PyNumber_Long(o);
    if (i == nullptr) throw std::bad_cast();
    const long x = PyLong_AsLong(i);
    Py_DECREF(i);
    if (x == -1 && PyErr_Occurred()) throw std::bad_cast();
    return x;
}

inline bool shape_is(const at::Tensor& t, std::initializer_list<int64_t> want) {
    const auto s = t.sizes();
    return s.size() == want.size() && std::equal(want.begin(), want.end(), s.begin());
}

// Runs the body of one entry point; what it throws becomes a Python exception.
template <typename Body>
PyObject* refusing(const char* name, Py_ssize_t wants, Py_ssize_t n, const Body& body) {
    if (n != wants) {
        PyErr_Format(PyExc_TypeError, "%s takes %zd arguments", name, wants);
        return nullptr;
    }
    try {
        body();
    } catch (const std::bad_cast&) {
        if (!PyErr_Occurred()) PyErr_Format(PyExc_TypeError, "%s: an argument has the wrong type", name);
        return nullptr;
    } catch (const c10::OutOfMemoryError& e) {
        PyObject* torch = PyImport_ImportModule("torch");
        PyObject* cls = torch != nullptr ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
        PyErr_SetString(cls != nullptr ? cls : PyExc_RuntimeError, e.what_without_backtrace());
        Py_XDECREF(cls);
        Py_XDECREF(torch);
        return nullptr;
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
    }
    Py_RETURN_NONE;
}

}  // namespace fkda_host

// fkda_host_ops.cpp
PyObject* host_linear_attention_fwd(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* host_latent_attention_fwd(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* host_latent_attention_decode(PyObject*, PyObject* const* args, Py_ssize_t n);

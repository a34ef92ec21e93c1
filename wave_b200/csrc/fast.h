// What the sources of `wave_b200._fast` share.
#pragma once
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <exception>

namespace wbfast {

bool plain_or_parameter(PyObject* o);     // an ordinary CUDA tensor, or one as a module's parameter (fast_call.cpp)
PyObject* fail(const std::exception& e);  // raises it, returns null

PyObject* bind_adapt(PyObject*, PyObject* args);
PyObject* adapters(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* router(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* combine_rows(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* input_grad(PyObject*, PyObject* const* args, Py_ssize_t n);

}  // namespace wbfast

// Functions of the native module that csrc/host_layer.cpp adds to those of csrc/host_binding.cpp.
#pragma once

#include <Python.h>

PyObject* fhob_py_rotary(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* fhob_py_layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* fhob_py_layer_norm_forward(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* fhob_py_layer_norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* fhob_py_layer_norm_bwdbwd(PyObject*, PyObject* const* a, Py_ssize_t n);

// Functions of the native module that csrc/host_layer.cpp adds to those of csrc/host_binding.cpp, and what both need.
#pragma once

#include <ATen/core/Tensor.h>
#include <Python.h>
#include <c10/core/AutogradState.h>

#include <initializer_list>

// Does one of these (undefined ones count as none) carry a tangent of forward-mode differentiation?  No operator here has a rule
// for them: such a call goes through an autograd function, where torch raises, or is refused; kernels called directly would drop it.
inline bool has_tangent(std::initializer_list<const at::Tensor*> ts) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return false;
  for (const at::Tensor* t : ts)
    if (t->defined() && t->_fw_grad(/*level=*/0).defined()) return true;
  return false;
}

PyObject* fhob_py_rotary(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* fhob_py_layer_norm(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* fhob_py_layer_norm_forward(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* fhob_py_layer_norm_backward(PyObject*, PyObject* const* a, Py_ssize_t n);
PyObject* fhob_py_layer_norm_bwdbwd(PyObject*, PyObject* const* a, Py_ssize_t n);

// Recorded calls of host_autograd.cpp and the rollout's of host_rollout.cpp, as methods of the module that host_calls.cpp makes.
#pragma once
#define PY_SSIZE_T_CLEAN
#include <Python.h>

PyObject* metis_recorded_residual_norm(PyObject*, PyObject* const* args, Py_ssize_t count);
PyObject* metis_recorded_swiglu(PyObject*, PyObject* const* args, Py_ssize_t count);
PyObject* metis_recorded_rotary(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* metis_host_rotary_append(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* metis_host_paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* metis_host_copy_pages(PyObject*, PyObject* const* args, Py_ssize_t n);
PyObject* metis_host_sample_tokens(PyObject*, PyObject* const* args, Py_ssize_t n);

// Recorded calls of host_autograd.cpp, as methods of the module that host_calls.cpp makes.
#pragma once
#define PY_SSIZE_T_CLEAN
#include <Python.h>

PyObject* metis_recorded_residual_norm(PyObject*, PyObject* const* args, Py_ssize_t count);
PyObject* metis_recorded_swiglu(PyObject*, PyObject* const* args, Py_ssize_t count);
PyObject* metis_recorded_rotary(PyObject*, PyObject* const* args, Py_ssize_t n);

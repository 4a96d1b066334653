// What operators.cpp adds to the module of host.cpp.
#pragma once
#include <Python.h>

PyObject* cx_py_linear(PyObject*, PyObject* const* a, Py_ssize_t nargs);
PyObject* cx_py_vocab_loss(PyObject*, PyObject* const* a, Py_ssize_t nargs);
PyObject* cx_py_bind_operators(PyObject*, PyObject* args);

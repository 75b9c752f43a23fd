// the paged cache's functions of the b200_host module (paged_host.cpp)
#pragma once
#include <Python.h>

PyObject* attach_paged(PyObject*, PyObject* args);
PyObject* paged_step(PyObject*, PyObject* const* a, Py_ssize_t n_args);
PyObject* paged_append(PyObject*, PyObject* const* a, Py_ssize_t n_args);
PyObject* sdp_paged(PyObject*, PyObject* const* a, Py_ssize_t n_args);
PyObject* sdp_packed(PyObject*, PyObject* const* a, Py_ssize_t n_args);

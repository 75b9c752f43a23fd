// the functions of the b200_host module for a server's steps: the paged cache (paged_host.cpp), and what a step has beside its attention (step_host.cpp)
#pragma once
#include <Python.h>

PyObject* attach_paged(PyObject*, PyObject* args);
PyObject* paged_step(PyObject*, PyObject* const* a, Py_ssize_t n_args);
PyObject* paged_append(PyObject*, PyObject* const* a, Py_ssize_t n_args);
PyObject* sdp_paged(PyObject*, PyObject* const* a, Py_ssize_t n_args);
PyObject* sdp_packed(PyObject*, PyObject* const* a, Py_ssize_t n_args);
PyObject* attach_step(PyObject*, PyObject* args);
PyObject* paged_norm_append(PyObject*, PyObject* const* a, Py_ssize_t n_args);
PyObject* paged_fork(PyObject*, PyObject* const* a, Py_ssize_t n_args);
PyObject* paged_share_release(PyObject*, PyObject* const* a, Py_ssize_t n_args);
PyObject* paged_compact(PyObject*, PyObject* const* a, Py_ssize_t n_args);
PyObject* paged_copy(PyObject*, PyObject* const* a, Py_ssize_t n_args);
PyObject* lora_add(PyObject*, PyObject* const* a, Py_ssize_t n_args);
PyObject* token_logprobs(PyObject*, PyObject* const* a, Py_ssize_t n_args);

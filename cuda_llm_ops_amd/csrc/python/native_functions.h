// The native module's functions of other files: positional arguments as their Python
// callers pass them.
#pragma once

#include <Python.h>

namespace fgqa_native {

// rope_native.cpp
PyObject* rope(PyObject* const* o);
PyObject* rope_backward(PyObject* const* o);

// pages_native.cpp
PyObject* fork(PyObject* const* o);
PyObject* compact(PyObject* const* o);
PyObject* decode_shared(PyObject* const* o);

}  // namespace fgqa_native

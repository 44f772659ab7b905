// phz_describe.cpp — from torch tensors to phz_tensor in one call.
//
// A small operator's time is mostly its call: describing four to ten tensors
// from Python costs more than their kernel. This module reads what phz_tensor
// holds (data_ptr(), shape, stride(), dtype, get_device()) through Python's C
// interface and calls the library's entry point with it. It needs torch's
// Python objects, not its C++ library.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "../../include/phyz_amd.h"

namespace {

typedef const phz_tensor* T;
// The entry points, in the order of phyz_amd/ops.py's table.
struct Entries {
  int (*scan)(phz_ops*, void*, int, T, T, T, T, T, T);
  int (*scan_backward)(phz_ops*, void*, int, T, T, T, T, T, T, T, T, T, T);
  int (*step)(phz_ops*, void*, int, T, T, T, T);
  int (*linear)(phz_ops*, void*, int, T, T, T, T, T, T);
  int (*linear_backward)(phz_ops*, void*, int, T, T, T, T, T, T, T);
  int (*orthogonalize)(phz_ops*, void*, const phz_muon_cfg*, T, T);
  int (*muon)(phz_ops*, void*, const phz_muon_cfg*, T, T, T);
};
union {
  Entries fn;
  void* at[7];
} g_entries;
const int kTensors[7] = {6, 10, 4, 6, 7, 2, 3};
// Whose results a user may expect autograd to know: not the gradients' own
// operators and the update's.
const bool kForward[7] = {true, false, true, true, false, true, false};

PyObject *g_dtypes[5], *g_data_ptr, *g_shape, *g_stride, *g_dtype, *g_get_device, *g_requires_grad;
const int kCodes[5] = {PHZ_F32, PHZ_F64, PHZ_BF16, PHZ_U8, PHZ_U8};

// False, with no Python error left, where `o` is no tensor that can be
// described (the caller finds out why and says so).
bool describe(PyObject* o, long device, phz_tensor* t) {
  PyObject* v = PyObject_CallMethodNoArgs(o, g_get_device);
  bool ok = v && PyLong_AsLong(v) == device;
  Py_XDECREF(v);
  if (ok) {
    v = PyObject_GetAttr(o, g_dtype);
    int code = -1;
    for (int i = 0; i < 5; i++)
      if (v == g_dtypes[i]) code = kCodes[i];
    Py_XDECREF(v);
    t->dtype = code;
    ok = code >= 0;
  }
  if (ok) {
    v = PyObject_CallMethodNoArgs(o, g_data_ptr);
    ok = v != nullptr;
    if (ok) t->data = PyLong_AsVoidPtr(v);
    Py_XDECREF(v);
  }
  PyObject* shape = ok ? PyObject_GetAttr(o, g_shape) : nullptr;
  PyObject* stride = shape ? PyObject_CallMethodNoArgs(o, g_stride) : nullptr;
  ok = ok && shape && stride && PyTuple_Check(shape) && PyTuple_Check(stride);
  if (ok) {
    const Py_ssize_t n = PyTuple_GET_SIZE(shape);
    ok = n >= 1 && n <= 3 && PyTuple_GET_SIZE(stride) == n;
    for (Py_ssize_t i = 0; ok && i < n; i++) {
      t->size[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, i));
      t->stride[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(stride, i));
    }
    t->ndim = (int32_t)n;
  }
  Py_XDECREF(shape);
  Py_XDECREF(stride);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    ok = false;
  }
  return ok;
}

// call(op, handle, stream, device, head, tensors, unrecorded): the entry point's
// result, -1 - i where tensor i cannot be described, or, unless `unrecorded`,
// -101 - i where a forward operator's tensor i requires gradients.
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 7 || !PyTuple_Check(args[5])) {
    PyErr_SetString(PyExc_TypeError, "call(op, handle, stream, device, head, tensors, unrecorded)");
    return nullptr;
  }
  const long op = PyLong_AsLong(args[0]), device = PyLong_AsLong(args[3]);
  auto* ops = (phz_ops*)PyLong_AsVoidPtr(args[1]);
  void* stream = PyLong_AsVoidPtr(args[2]);
  const long long head = PyLong_AsLongLong(args[4]);
  if (PyErr_Occurred()) return nullptr;
  if (op < 0 || op > 6 || PyTuple_GET_SIZE(args[5]) != kTensors[op] || !g_entries.at[op]) {
    PyErr_SetString(PyExc_ValueError, "unknown operator, or not its tensors");
    return nullptr;
  }
  phz_tensor d[10];
  T t[10] = {};
  for (int i = 0; i < kTensors[op]; i++) {
    PyObject* o = PyTuple_GET_ITEM(args[5], i);
    if (o == Py_None) continue;
    if (!describe(o, device, &d[i])) return PyLong_FromLong(-1 - i);
    if (kForward[op] && args[6] == Py_False) {
      PyObject* v = PyObject_GetAttr(o, g_requires_grad);
      if (!v) return nullptr;
      Py_DECREF(v);
      if (v == Py_True) return PyLong_FromLong(-101 - i);
    }
    t[i] = &d[i];
  }
  const Entries& f = g_entries.fn;
  const int h = (int)head;
  const auto* cfg = (const phz_muon_cfg*)(intptr_t)head;
  int rc = 1;
  switch (op) {
    case 0: rc = f.scan(ops, stream, h, t[0], t[1], t[2], t[3], t[4], t[5]); break;
    case 1: rc = f.scan_backward(ops, stream, h, t[0], t[1], t[2], t[3], t[4], t[5], t[6], t[7], t[8], t[9]); break;
    case 2: rc = f.step(ops, stream, h, t[0], t[1], t[2], t[3]); break;
    case 3: rc = f.linear(ops, stream, h, t[0], t[1], t[2], t[3], t[4], t[5]); break;
    case 4: rc = f.linear_backward(ops, stream, h, t[0], t[1], t[2], t[3], t[4], t[5], t[6]); break;
    case 5: rc = f.orthogonalize(ops, stream, cfg, t[0], t[1]); break;
    case 6: rc = f.muon(ops, stream, cfg, t[0], t[1], t[2]); break;
  }
  return PyLong_FromLong(rc);
}

// bind(entry points' addresses, (float32, float64, bfloat16, uint8, bool))
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 2 || !PyTuple_Check(args[0]) || PyTuple_GET_SIZE(args[0]) != 7 || !PyTuple_Check(args[1]) ||
      PyTuple_GET_SIZE(args[1]) != 5) {
    PyErr_SetString(PyExc_TypeError, "bind(seven addresses, five dtypes)");
    return nullptr;
  }
  for (int i = 0; i < 7; i++) g_entries.at[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(args[0], i));
  if (PyErr_Occurred()) return nullptr;
  for (int i = 0; i < 5; i++) {
    PyObject* o = PyTuple_GET_ITEM(args[1], i);
    Py_INCREF(o);
    Py_XSETREF(g_dtypes[i], o);
  }
  Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {{"call", (PyCFunction)(void*)call, METH_FASTCALL, nullptr},
                           {"bind", (PyCFunction)(void*)bind, METH_FASTCALL, nullptr},
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_describe", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__describe() {
  static_assert(sizeof(phz_tensor) == 64, "phz_tensor");
  const struct { PyObject** at; const char* name; } names[] = {
      {&g_data_ptr, "data_ptr"}, {&g_shape, "shape"}, {&g_stride, "stride"}, {&g_dtype, "dtype"}, {&g_get_device, "get_device"},
      {&g_requires_grad, "requires_grad"}};
  for (auto& s : names)
    if (!(*s.at = PyUnicode_InternFromString(s.name))) return nullptr;
  return PyModule_Create(&g_module);
}

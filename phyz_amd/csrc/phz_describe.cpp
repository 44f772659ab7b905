// phz_describe.cpp — from torch tensors to phz_tensor in one call.
//
// A small operator's time is mostly its call: describing four to ten tensors
// from Python costs more than their kernel. This module reads what phz_tensor
// holds (data_ptr(), shape, stride(), dtype, get_device()) through Python's C
// interface and calls the library's entry point with it. It needs torch's
// Python objects, not its C++ library.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <new>
#include <vector>

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
  int (*attention)(phz_ops*, void*, const phz_attention_cfg*, T, T, T, T, T, T, T, T);
  int (*attention_backward)(phz_ops*, void*, const phz_attention_cfg*, T, T, T, T, T, T, T, T, T, T, T, T, T);
  int (*attention_step)(phz_ops*, void*, const phz_attention_cfg*, T, T, T, T, T, T, T);
  int (*rotary)(phz_ops*, void*, const phz_rotary_cfg*, T, T, T, T);
  int (*adamw)(phz_ops*, void*, const phz_adamw_cfg*, int64_t, T, T, T, T, T, T);
  int (*adamw_values)(phz_ops*, void*, int64_t, T, T, T, T, T);
};
constexpr int kEntries = 13, kPlain = 11, kMost = 13, kDtypes = 7;  // the last two take lists (call_lists)
union {
  Entries fn;
  void* at[kEntries];
} g_entries;
const int kTensors[kPlain] = {6, 10, 4, 6, 7, 2, 3, 8, 13, 7, 4};
// Whose results a user may expect autograd to know: not the gradients' own
// operators and the update's.
const bool kForward[kPlain] = {true, false, true, true, false, true, false, true, false, true, true};

PyObject *g_dtypes[kDtypes], *g_data_ptr, *g_shape, *g_stride, *g_dtype, *g_get_device, *g_requires_grad,
    *g_is_contiguous, *g_numel;
const int kCodes[kDtypes] = {PHZ_F32, PHZ_F64, PHZ_BF16, PHZ_U8, PHZ_U8, PHZ_I32, PHZ_I64};

// False, with no Python error left, where `o` is no tensor that can be
// described (the caller finds out why and says so). `flat`: as a vector, which a
// contiguous tensor of any number of axes is; its shape goes to `shape`, where that is
// asked for.
bool describe(PyObject* o, long device, phz_tensor* t, bool flat = false, PyObject** of_shape = nullptr) {
  PyObject* v = PyObject_CallMethodNoArgs(o, g_get_device);
  bool ok = v && PyLong_AsLong(v) == device;
  Py_XDECREF(v);
  if (ok) {
    v = PyObject_GetAttr(o, g_dtype);
    int code = -1;
    for (int i = 0; i < kDtypes; i++)
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
  if (flat) {
    // Two calls that make no tuples; strides do not matter then.
    v = ok ? PyObject_CallMethodNoArgs(o, g_is_contiguous) : nullptr;
    ok = v == Py_True;
    Py_XDECREF(v);
    t->stride[0] = 1;
    t->ndim = 1;
    if (of_shape) {
      v = ok ? PyObject_GetAttr(o, g_shape) : nullptr;
      ok = v && PyTuple_Check(v);
      t->size[0] = 1;
      for (Py_ssize_t i = 0; ok && i < PyTuple_GET_SIZE(v); i++) t->size[0] *= PyLong_AsLongLong(PyTuple_GET_ITEM(v, i));
      *of_shape = v;
    } else {
      v = ok ? PyObject_CallMethodNoArgs(o, g_numel) : nullptr;
      ok = v != nullptr;
      if (ok) t->size[0] = PyLong_AsLongLong(v);
      Py_XDECREF(v);
    }
    if (PyErr_Occurred()) {
      PyErr_Clear();
      ok = false;
    }
    return ok;
  }
  PyObject* shape = ok ? PyObject_GetAttr(o, g_shape) : nullptr;
  PyObject* stride = shape ? PyObject_CallMethodNoArgs(o, g_stride) : nullptr;
  ok = ok && shape && stride && PyTuple_Check(shape) && PyTuple_Check(stride);
  if (ok) {
    const Py_ssize_t n = PyTuple_GET_SIZE(shape);
    ok = PyTuple_GET_SIZE(stride) == n && n >= 1 && n <= 3;
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

// Whether elements of two shapes with as many of them, one after the other, are at
// the same places: axes of one element aside the shapes are one, or either is a vector.
bool same_places(PyObject* a, PyObject* b) {
  const Py_ssize_t na = PyTuple_GET_SIZE(a), nb = PyTuple_GET_SIZE(b);
  Py_ssize_t i = 0, j = 0, axes[2] = {};
  bool same = true;
  for (;;) {
    long long x = 1, y = 1;
    while (i < na && (x = PyLong_AsLongLong(PyTuple_GET_ITEM(a, i))) == 1) i++;
    while (j < nb && (y = PyLong_AsLongLong(PyTuple_GET_ITEM(b, j))) == 1) j++;
    if (i >= na && j >= nb) break;
    same = same && i < na && j < nb && x == y;
    if (i < na) axes[0]++, i++;
    if (j < nb) axes[1]++, j++;
  }
  return same || axes[0] < 2 || axes[1] < 2;
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
  if (op < 0 || op >= kPlain || PyTuple_GET_SIZE(args[5]) != kTensors[op] || !g_entries.at[op]) {
    PyErr_SetString(PyExc_ValueError, "unknown operator, or not its tensors");
    return nullptr;
  }
  phz_tensor d[kMost];
  T t[kMost] = {};
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
  const auto* att = (const phz_attention_cfg*)(intptr_t)head;
  const auto* rot = (const phz_rotary_cfg*)(intptr_t)head;
  int rc = 1;
  switch (op) {
    case 0: rc = f.scan(ops, stream, h, t[0], t[1], t[2], t[3], t[4], t[5]); break;
    case 1: rc = f.scan_backward(ops, stream, h, t[0], t[1], t[2], t[3], t[4], t[5], t[6], t[7], t[8], t[9]); break;
    case 2: rc = f.step(ops, stream, h, t[0], t[1], t[2], t[3]); break;
    case 3: rc = f.linear(ops, stream, h, t[0], t[1], t[2], t[3], t[4], t[5]); break;
    case 4: rc = f.linear_backward(ops, stream, h, t[0], t[1], t[2], t[3], t[4], t[5], t[6]); break;
    case 5: rc = f.orthogonalize(ops, stream, cfg, t[0], t[1]); break;
    case 6: rc = f.muon(ops, stream, cfg, t[0], t[1], t[2]); break;
    case 7: rc = f.attention(ops, stream, att, t[0], t[1], t[2], t[3], t[4], t[5], t[6], t[7]); break;
    case 8:
      rc = f.attention_backward(ops, stream, att, t[0], t[1], t[2], t[3], t[4], t[5], t[6], t[7], t[8], t[9], t[10], t[11],
                                t[12]);
      break;
    case 9: rc = f.attention_step(ops, stream, att, t[0], t[1], t[2], t[3], t[4], t[5], t[6]); break;
    case 10: rc = f.rotary(ops, stream, rot, t[0], t[1], t[2], t[3]); break;
  }
  return PyLong_FromLong(rc);
}

// call_lists(op, handle, stream, device, head, lists, single): an entry point of
// lists of tensors, each a vector. Lists are tuples of one length, or None;
// `single` is a tensor or None. The result as in call(), -1 - (5 i + l) for tensor
// i of list l (l = 0 .. 4) and -1 - 5 n for the single one, -2^40 - i where the
// update's gradient i has another shape than its weights.
PyObject* call_lists(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 7 || !PyTuple_Check(args[5]) || PyTuple_GET_SIZE(args[5]) != 5) {
    PyErr_SetString(PyExc_TypeError, "call_lists(op, handle, stream, device, head, five lists, single)");
    return nullptr;
  }
  const long op = PyLong_AsLong(args[0]), device = PyLong_AsLong(args[3]);
  auto* ops = (phz_ops*)PyLong_AsVoidPtr(args[1]);
  void* stream = PyLong_AsVoidPtr(args[2]);
  const auto* cfg = (const phz_adamw_cfg*)(intptr_t)PyLong_AsLongLong(args[4]);
  if (PyErr_Occurred()) return nullptr;
  PyObject* const* lists = &PyTuple_GET_ITEM(args[5], 0);
  Py_ssize_t n = -1;
  bool fits = op >= kPlain && op < kEntries && g_entries.at[op];
  for (int l = 0; l < 5; l++) {
    if (lists[l] == Py_None) continue;
    fits = fits && PyTuple_Check(lists[l]) && (n < 0 || PyTuple_GET_SIZE(lists[l]) == n);
    if (fits) n = PyTuple_GET_SIZE(lists[l]);
  }
  if (!fits || n < 0) {
    PyErr_SetString(PyExc_ValueError, "unknown operator, or not its lists");
    return nullptr;
  }
  std::vector<phz_tensor> d;
  try {
    d.resize((size_t)n * 5 + 1);
  } catch (const std::bad_alloc&) {
    return PyErr_NoMemory();
  }
  T t[6] = {};
  for (int l = 0; l < 5; l++)
    if (lists[l] != Py_None) t[l] = d.data() + n * l;
  const bool pairs = op == kPlain && t[0] && t[1];  // weights and their gradients
  for (Py_ssize_t i = 0; pairs && i < n; i++) {
    PyObject *a = nullptr, *b = nullptr;
    const bool wa = describe(PyTuple_GET_ITEM(lists[0], i), device, &d[i], true, &a);
    // (A vector's gradient is not asked: a shape is an object made.)
    const bool wb = wa && describe(PyTuple_GET_ITEM(lists[1], i), device, &d[n + i], true, PyTuple_GET_SIZE(a) > 1 ? &b : nullptr);
    const bool apart = wb && b && d[i].size[0] == d[n + i].size[0] && d[i].size[0] > 1 && !same_places(a, b);
    Py_XDECREF(a);
    Py_XDECREF(b);
    if (!wb) return PyLong_FromSsize_t(-1 - (5 * i + wa));
    if (apart) return PyLong_FromLongLong(-(1ll << 40) - i);
  }
  for (int l = pairs ? 2 : 0; l < 5; l++) {
    if (!t[l]) continue;
    for (Py_ssize_t i = 0; i < n; i++)
      if (!describe(PyTuple_GET_ITEM(lists[l], i), device, &d[n * l + i], true)) return PyLong_FromSsize_t(-1 - (5 * i + l));
  }
  if (args[6] != Py_None) {
    if (!describe(args[6], device, &d[n * 5], true)) return PyLong_FromSsize_t(-1 - 5 * n);
    t[5] = &d[n * 5];
  }
  const Entries& f = g_entries.fn;
  return PyLong_FromLong(op == kPlain ? f.adamw(ops, stream, cfg, n, t[0], t[1], t[2], t[3], t[4], t[5])
                                      : f.adamw_values(ops, stream, n, t[0], t[1], t[2], t[3], t[4]));
}

// bind(entry points' addresses, (float32, float64, bfloat16, uint8, bool, int32, int64))
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 2 || !PyTuple_Check(args[0]) || PyTuple_GET_SIZE(args[0]) != kEntries || !PyTuple_Check(args[1]) ||
      PyTuple_GET_SIZE(args[1]) != kDtypes) {
    PyErr_SetString(PyExc_TypeError, "bind(the entry points' addresses, the dtypes)");
    return nullptr;
  }
  for (int i = 0; i < kEntries; i++) g_entries.at[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(args[0], i));
  if (PyErr_Occurred()) return nullptr;
  for (int i = 0; i < kDtypes; i++) {
    PyObject* o = PyTuple_GET_ITEM(args[1], i);
    Py_INCREF(o);
    Py_XSETREF(g_dtypes[i], o);
  }
  Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {{"call", (PyCFunction)(void*)call, METH_FASTCALL, nullptr},
                           {"call_lists", (PyCFunction)(void*)call_lists, METH_FASTCALL, nullptr},
                           {"bind", (PyCFunction)(void*)bind, METH_FASTCALL, nullptr},
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_describe", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__describe() {
  static_assert(sizeof(phz_tensor) == 64, "phz_tensor");
  const struct { PyObject** at; const char* name; } names[] = {
      {&g_data_ptr, "data_ptr"}, {&g_shape, "shape"}, {&g_stride, "stride"}, {&g_dtype, "dtype"}, {&g_get_device, "get_device"},
      {&g_requires_grad, "requires_grad"}, {&g_is_contiguous, "is_contiguous"}, {&g_numel, "numel"}};
  for (auto& s : names)
    if (!(*s.at = PyUnicode_InternFromString(s.name))) return nullptr;
  return PyModule_Create(&g_module);
}

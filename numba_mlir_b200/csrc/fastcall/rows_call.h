// Native call path of the row operators (numba_mlir_b200.rows): reads the
// arguments out of torch tensors and device arrays, makes the checks and calls
// the C entry, without building anything in Python.
//
// It takes the ordinary call only: results given, every array on the queue's own
// stream, nothing out of order.  Whatever it does not take -- an argument that
// has to be refused, arrays of other streams, results to allocate -- it leaves
// to the Python implementation by answering 0, so the rules and the messages
// stand there alone.  Answers: 0 not taken, 1 done, 2 the entry failed.  (A
// lookup of 16 rows of 2048 took 13.7 us of host time through ctypes.)
#pragma once

#include "../../../include/numba_mlir_gpu_runtime_cuda.h"

namespace rowscall {

using TakeFn = int (*)(void *, const GPUXRows *, const GPUXIndex *, double, const GPUXRows *);
using TakeGradFn = int (*)(void *, const GPUXRows *, const GPUXIndex *, double, const GPUXRows *, int, void *, size_t);
using GroupFn = int (*)(void *, const GPUXIndex *, int64_t, int32_t *, int32_t *, int32_t *, void *, size_t);
using DispatchFn = int (*)(void *, const GPUXRows *, int64_t, const int32_t *, const int32_t *, const GPUXRows *);
using SortDispatchFn = int (*)(void *, const GPUXRows *, const GPUXIndex *, int64_t, int32_t *, int32_t *, int32_t *,
                               void *, size_t, const GPUXRows *);
using CombineFn = int (*)(void *, const GPUXRows *, int64_t, const int32_t *, const int32_t *, const void *, int,
                          const GPUXRows *);
using CombineGradFn = int (*)(void *, const GPUXRows *, const GPUXRows *, int64_t, const int32_t *, const int32_t *,
                              const void *, int, const GPUXRows *, void *);
struct Entries {
  TakeFn take;
  TakeGradFn takeGrad;
  GroupFn group;
  DispatchFn dispatch;
  CombineFn combine;
  CombineGradFn combineGrad;
  SortDispatchFn sortDispatch;
};
inline Entries gEntries{};
inline PyObject *gTypes = nullptr;       // dtype -> (float code or -1, index bytes, item size)
inline PyObject *gArrayType = nullptr;   // DeviceArray
inline PyObject *gTensorType = nullptr;  // torch.Tensor, once torch is in use
inline PyObject *gCurrentStream = nullptr; // device index -> raw current stream of torch

inline PyObject *name(const char *text) { return PyUnicode_InternFromString(text); }
struct Names {
  PyObject *dtype = name("dtype"), *shape = name("shape"), *strides = name("strides"), *stride = name("stride"),
           *addr = name("_addr"), *buf = name("_buf"), *queue = name("queue"), *data_ptr = name("data_ptr"),
           *requires_grad = name("requires_grad"), *is_neg = name("is_neg"), *get_device = name("get_device"),
           *handle = name("handle"), *device = name("device"), *raw = name("_raw_stream");
};
inline Names &names() {
  static Names n;
  return n;
}

// A queue, and whether torch's current stream is its stream (asked once).
struct Queue {
  PyObject *obj;
  void *handle = nullptr;
  int64_t device = -1, raw = -1;
  int torchHere = -1;
};

constexpr int kMaxDims = 8;
struct Operand {
  int64_t ptr = 0, shape[kMaxDims], stride[kMaxDims];
  int nd = 0, kind = -1, index = 0, item = 1;
  int64_t rows = 0, cols = 0, step = 0; // as a set of rows
  int64_t size() const {
    int64_t n = 1;
    for (int i = 0; i < nd; ++i)
      n *= shape[i];
    return n;
  }
  bool contiguous() const {
    int64_t s = 1;
    for (int i = nd - 1; i >= 0; --i) {
      if (shape[i] == 0)
        return true;
      if (shape[i] != 1 && stride[i] != s)
        return false;
      s *= shape[i];
    }
    return true;
  }
  bool asRows() {
    if (kind < 0 || nd < 1)
      return false;
    cols = shape[nd - 1];
    if (cols > 1 && stride[nd - 1] != 1)
      return false;
    rows = 1;
    step = cols;
    bool found = false;
    int64_t span = 0;
    for (int i = nd - 2; i >= 0; --i) {
      rows *= shape[i];
      if (shape[i] == 1)
        continue;
      if (!found) {
        step = stride[i];
        found = true;
      } else if (stride[i] != span) {
        return false;
      }
      span = stride[i] * shape[i];
    }
    return true;
  }
  GPUXRows asArg() const { return {reinterpret_cast<void *>(ptr), rows, cols, step, kind, 0}; }
  GPUXIndex indexArg() const { return {reinterpret_cast<const void *>(ptr), size(), index, 0}; }
  bool sameShape(const Operand &o) const {
    if (nd != o.nd)
      return false;
    for (int i = 0; i < nd; ++i)
      if (shape[i] != o.shape[i])
        return false;
    return true;
  }
  void range(int64_t &lo, int64_t &hi) const {
    lo = hi = ptr;
    for (int i = 0; i < nd; ++i) {
      if (shape[i] == 0) {
        lo = hi = 0;
        return;
      }
      (stride[i] >= 0 ? hi : lo) += (shape[i] - 1) * stride[i] * item;
    }
    hi += item;
  }
};

inline bool takeInt(PyObject *o, int64_t &v) { // steals o
  if (!o)
    return false;
  v = PyLong_AsLongLong(o);
  Py_DECREF(o);
  return !(v == -1 && PyErr_Occurred());
}

inline bool takeInts(PyObject *o, int64_t *out, int &n, int64_t divide) { // steals o, a tuple
  if (!o)
    return false;
  bool ok = PyTuple_Check(o) && PyTuple_GET_SIZE(o) <= kMaxDims;
  n = ok ? (int)PyTuple_GET_SIZE(o) : 0;
  for (int i = 0; ok && i < n; ++i) {
    const int64_t v = PyLong_AsLongLong(PyTuple_GET_ITEM(o, i));
    ok = !(v == -1 && PyErr_Occurred()) && v % divide == 0;
    out[i] = v / divide;
  }
  Py_DECREF(o);
  return ok;
}

inline bool readType(PyObject *obj, Operand &op) {
  PyObject *dt = PyObject_GetAttr(obj, names().dtype);
  if (!dt)
    return false;
  PyObject *hit = PyDict_GetItemWithError(gTypes, dt); // borrowed
  Py_DECREF(dt);
  if (!hit)
    return false;
  op.kind = (int)PyLong_AsLong(PyTuple_GET_ITEM(hit, 0));
  op.index = (int)PyLong_AsLong(PyTuple_GET_ITEM(hit, 1));
  op.item = (int)PyLong_AsLong(PyTuple_GET_ITEM(hit, 2));
  return true;
}

inline bool isTrue(PyObject *obj, PyObject *attr, bool call = false) {
  PyObject *v = call ? PyObject_CallMethodNoArgs(obj, attr) : PyObject_GetAttr(obj, attr);
  const bool t = v == Py_True;
  Py_XDECREF(v);
  return t;
}

inline bool readQueue(PyObject *obj, Queue &q) {
  q.obj = obj;
  int64_t handle;
  if (!takeInt(PyObject_GetAttr(obj, names().handle), handle) ||
      !takeInt(PyObject_GetAttr(obj, names().device), q.device) || !takeInt(PyObject_GetAttr(obj, names().raw), q.raw))
    return false;
  q.handle = reinterpret_cast<void *>(handle);
  return q.handle != nullptr;
}

inline bool read(PyObject *obj, Queue &q, Operand &op) {
  Names &n = names();
  int strides = 0;
  if ((PyObject *)Py_TYPE(obj) == gArrayType) {
    PyObject *buf = PyObject_GetAttr(obj, n.buf);
    PyObject *queue = buf ? PyObject_GetAttr(buf, n.queue) : nullptr;
    Py_XDECREF(buf);
    const bool mine = queue == q.obj;
    Py_XDECREF(queue);
    return mine && readType(obj, op) && takeInt(PyObject_GetAttr(obj, n.addr), op.ptr) &&
           takeInts(PyObject_GetAttr(obj, n.shape), op.shape, op.nd, 1) &&
           takeInts(PyObject_GetAttr(obj, n.strides), op.stride, strides, op.item) && strides == op.nd;
  }
  if (!gTensorType || !PyObject_TypeCheck(obj, (PyTypeObject *)gTensorType) || isTrue(obj, n.requires_grad))
    return false;
  int64_t device; // -1 for a tensor that is not on a GPU
  if (!takeInt(PyObject_CallMethodNoArgs(obj, n.get_device), device) || device != q.device)
    return false;
  if (q.torchHere < 0) {
    PyObject *index = PyLong_FromLongLong(device);
    int64_t raw = 0;
    const bool ok = index && takeInt(PyObject_CallOneArg(gCurrentStream, index), raw);
    Py_XDECREF(index);
    if (!ok)
      return false;
    q.torchHere = raw == q.raw;
  }
  if (!q.torchHere || !readType(obj, op))
    return false;
  // the negative bit is that of parts of complex values: never of indices
  if (op.kind >= 0 && isTrue(obj, n.is_neg, true))
    return false;
  return takeInt(PyObject_CallMethodNoArgs(obj, n.data_ptr), op.ptr) &&
         takeInts(PyObject_GetAttr(obj, n.shape), op.shape, op.nd, 1) &&
         takeInts(PyObject_CallMethodNoArgs(obj, n.stride), op.stride, strides, 1) && strides == op.nd;
}

// No result shares a byte range with anything else.
inline bool apart(const Operand *const *all, int results, int count) {
  int64_t lo[16], hi[16];
  for (int i = 0; i < count; ++i)
    all[i]->range(lo[i], hi[i]);
  for (int i = 0; i < results; ++i)
    for (int j = i + 1; j < count; ++j)
      if (lo[i] < hi[j] && lo[j] < hi[i])
        return false;
  return true;
}

inline bool pairAllowed(int a, int b) {
  return a == b || ((a == GPUX_ELEM_F32 || b == GPUX_ELEM_F32) && a != GPUX_ELEM_F64 && b != GPUX_ELEM_F64);
}

inline PyObject *answer(int code) {
  if (code == 0 && PyErr_Occurred())
    PyErr_Clear(); // the Python path reports it
  return PyLong_FromLong(code);
}
inline PyObject *called(int failed) { return answer(failed ? 2 : 1); }

inline bool int32s(const Operand &o) { return o.index == 4 && o.contiguous(); }

// place and offsets of a plan (order too when `order` is given)
inline bool readPlan(PyObject *plan, Queue &q, Operand *order, Operand &place, Operand &offsets) {
  if (!PyTuple_Check(plan) || PyTuple_GET_SIZE(plan) != 3)
    return false;
  if (order && !(read(PyTuple_GET_ITEM(plan, 0), q, *order) && int32s(*order)))
    return false;
  return read(PyTuple_GET_ITEM(plan, 1), q, place) && int32s(place) && read(PyTuple_GET_ITEM(plan, 2), q, offsets) &&
         int32s(offsets) && offsets.size() > 0;
}
inline const int32_t *ints(const Operand &o, int64_t at = 0) { return reinterpret_cast<const int32_t *>(o.ptr) + at; }

// rows_init(entry addresses, types, array type): binds the C entries.
inline PyObject *py_rows_init(PyObject *, PyObject *args) {
  unsigned long long a[7];
  PyObject *types, *array;
  if (!PyArg_ParseTuple(args, "(KKKKKKK)OO", &a[0], &a[1], &a[2], &a[3], &a[4], &a[5], &a[6], &types, &array))
    return nullptr;
  gEntries = {reinterpret_cast<TakeFn>(a[0]),      reinterpret_cast<TakeGradFn>(a[1]),
              reinterpret_cast<GroupFn>(a[2]),     reinterpret_cast<DispatchFn>(a[3]),
              reinterpret_cast<CombineFn>(a[4]),   reinterpret_cast<CombineGradFn>(a[5]),
              reinterpret_cast<SortDispatchFn>(a[6])};
  Py_INCREF(types);
  Py_XSETREF(gTypes, types);
  Py_INCREF(array);
  Py_XSETREF(gArrayType, array);
  Py_RETURN_NONE;
}

// rows_torch(Tensor type, current stream function): tensors are taken from now on.
inline PyObject *py_rows_torch(PyObject *, PyObject *args) {
  PyObject *tensor, *stream;
  if (!PyArg_ParseTuple(args, "OO", &tensor, &stream))
    return nullptr;
  Py_INCREF(tensor);
  Py_XSETREF(gTensorType, tensor);
  Py_INCREF(stream);
  Py_XSETREF(gCurrentStream, stream);
  Py_RETURN_NONE;
}

// rows_take(queue, table, ids, scale, out)
inline PyObject *py_rows_take(PyObject *, PyObject *const *a, Py_ssize_t n) {
  Queue q;
  Operand table, ids, out;
  if (n != 5 || !readQueue(a[0], q) || !read(a[1], q, table) || !read(a[2], q, ids) || !read(a[4], q, out))
    return answer(0);
  const double scale = PyFloat_AsDouble(a[3]);
  bool ok = !PyErr_Occurred() && ids.index && ids.contiguous() && table.nd == 2 && table.asRows() && out.asRows() &&
            pairAllowed(table.kind, out.kind) && out.nd == ids.nd + 1 && out.cols == table.cols;
  for (int i = 0; ok && i < ids.nd; ++i)
    ok = out.shape[i] == ids.shape[i];
  const Operand *all[] = {&out, &table, &ids};
  if (!ok || !apart(all, 1, 3))
    return answer(0);
  const GPUXRows t = table.asArg(), o = out.asArg();
  const GPUXIndex i = ids.indexArg();
  return called(gEntries.take(q.handle, &t, &i, scale, &o));
}

// rows_take_grad(queue, dout, ids, scale, out, accumulate)
inline PyObject *py_rows_take_grad(PyObject *, PyObject *const *a, Py_ssize_t n) {
  Queue q;
  Operand dout, ids, out;
  if (n != 6 || !readQueue(a[0], q) || !read(a[1], q, dout) || !read(a[2], q, ids) || !read(a[4], q, out))
    return answer(0);
  const double scale = PyFloat_AsDouble(a[3]);
  bool ok = !PyErr_Occurred() && ids.index && ids.contiguous() && dout.asRows() && out.nd == 2 && out.asRows() &&
            pairAllowed(dout.kind, out.kind) && dout.nd == ids.nd + 1 && out.cols == dout.cols;
  for (int i = 0; ok && i < ids.nd; ++i)
    ok = dout.shape[i] == ids.shape[i];
  const Operand *all[] = {&out, &dout, &ids};
  if (!ok || !apart(all, 1, 3))
    return answer(0);
  const GPUXRows d = dout.asArg(), o = out.asArg();
  const GPUXIndex i = ids.indexArg();
  return called(gEntries.takeGrad(q.handle, &d, &i, scale, &o, a[5] == Py_True, nullptr, 0));
}

// rows_group(queue, ids, groups, plan)
inline PyObject *py_rows_group(PyObject *, PyObject *const *a, Py_ssize_t n) {
  Queue q;
  Operand ids, order, place, offsets;
  if (n != 4 || !readQueue(a[0], q) || !read(a[1], q, ids) || !readPlan(a[3], q, &order, place, offsets))
    return answer(0);
  const int64_t groups = PyLong_AsLongLong(a[2]);
  const Operand *all[] = {&order, &place, &offsets, &ids};
  if (PyErr_Occurred() || groups < 0 || !ids.index || !ids.contiguous() || order.size() != ids.size() ||
      place.size() != ids.size() || offsets.size() != groups + 1 || !apart(all, 3, 4))
    return answer(0);
  const GPUXIndex i = ids.indexArg();
  return called(gEntries.group(q.handle, &i, groups, const_cast<int32_t *>(ints(order)),
                               const_cast<int32_t *>(ints(place)), const_cast<int32_t *>(ints(offsets)), nullptr, 0));
}

// rows_dispatch(queue, x, ids or None, groups, plan, out): sorts the ids into
// the plan first unless they are None
inline PyObject *py_rows_dispatch(PyObject *, PyObject *const *a, Py_ssize_t n) {
  Queue q;
  Operand x, ids, order, place, offsets, out;
  if (n != 6 || !readQueue(a[0], q) || !read(a[1], q, x) || !read(a[5], q, out))
    return answer(0);
  const bool sort = a[2] != Py_None;
  if (!readPlan(a[4], q, sort ? &order : nullptr, place, offsets) || (sort && !read(a[2], q, ids)))
    return answer(0);
  const int64_t groups = sort ? PyLong_AsLongLong(a[3]) : 0;
  const Operand &entries = sort ? ids : place;
  if (PyErr_Occurred() || x.nd != 2 || !x.asRows() || out.nd != 2 || !out.asRows() || out.kind != x.kind ||
      out.cols != x.cols || entries.nd < 1 || entries.nd > 2 || entries.shape[0] != x.rows)
    return answer(0);
  const int64_t k = entries.nd == 2 ? entries.shape[1] : 1;
  if (out.rows < x.rows * k)
    return answer(0);
  const GPUXRows xr = x.asArg(), o = out.asArg();
  if (sort) {
    const Operand *all[] = {&out, &order, &place, &offsets, &x, &ids};
    if (groups < 0 || !ids.index || !ids.contiguous() || order.size() != ids.size() || place.size() != ids.size() ||
        offsets.size() != groups + 1 || !apart(all, 4, 6))
      return answer(0);
    const GPUXIndex i = ids.indexArg();
    return called(gEntries.sortDispatch(q.handle, &xr, &i, groups, const_cast<int32_t *>(ints(order)),
                                        const_cast<int32_t *>(ints(place)), const_cast<int32_t *>(ints(offsets)),
                                        nullptr, 0, &o));
  }
  const Operand *all[] = {&out, &x, &place, &offsets};
  if (!apart(all, 1, 4))
    return answer(0);
  return called(gEntries.dispatch(q.handle, &xr, k, ints(place), ints(offsets, offsets.size() - 1), &o));
}

// rows_combine(queue, ys, plan, weights or None, out)
inline PyObject *py_rows_combine(PyObject *, PyObject *const *a, Py_ssize_t n) {
  Queue q;
  Operand ys, place, offsets, weights, out;
  if (n != 5 || !readQueue(a[0], q) || !read(a[1], q, ys) || !readPlan(a[2], q, nullptr, place, offsets) ||
      !read(a[4], q, out))
    return answer(0);
  const bool weighted = a[3] != Py_None;
  if (weighted && !(read(a[3], q, weights) && weights.kind >= 0 && weights.sameShape(place) && weights.contiguous()))
    return answer(0);
  const Operand *all[] = {&out, &ys, &place, &offsets, &weights};
  if (ys.nd != 2 || !ys.asRows() || out.nd != 2 || !out.asRows() || out.kind != ys.kind || out.cols != ys.cols ||
      place.nd < 1 || place.nd > 2 || place.shape[0] != out.rows || !apart(all, 1, weighted ? 5 : 4))
    return answer(0);
  const int64_t k = place.nd == 2 ? place.shape[1] : 1;
  const GPUXRows y = ys.asArg(), o = out.asArg();
  return called(gEntries.combine(q.handle, &y, k, ints(place), ints(offsets, offsets.size() - 1),
                                 weighted ? reinterpret_cast<const void *>(weights.ptr) : nullptr,
                                 weighted ? weights.kind : 0, &o));
}

// rows_combine_grad(queue, dout, ys, plan, weights or None, out, dweights)
inline PyObject *py_rows_combine_grad(PyObject *, PyObject *const *a, Py_ssize_t n) {
  Queue q;
  Operand dout, ys, place, offsets, weights, out, dweights;
  if (n != 7 || !readQueue(a[0], q) || !read(a[1], q, dout) || !read(a[2], q, ys) ||
      !readPlan(a[3], q, nullptr, place, offsets) || !read(a[5], q, out) || !read(a[6], q, dweights))
    return answer(0);
  const bool weighted = a[4] != Py_None;
  if (weighted && !(read(a[4], q, weights) && weights.kind >= 0 && weights.sameShape(place) && weights.contiguous()))
    return answer(0);
  const int type = weighted ? weights.kind : 0;
  const Operand *all[] = {&out, &dweights, &dout, &ys, &place, &offsets, &weights};
  if (dout.nd != 2 || !dout.asRows() || ys.nd != 2 || !ys.asRows() || !out.sameShape(ys) || !out.asRows() ||
      dout.kind != ys.kind || out.kind != ys.kind || dout.cols != ys.cols || place.nd < 1 || place.nd > 2 ||
      place.shape[0] != dout.rows || dweights.kind != type || !dweights.sameShape(place) || !dweights.contiguous() ||
      !apart(all, 2, weighted ? 7 : 6))
    return answer(0);
  const int64_t k = place.nd == 2 ? place.shape[1] : 1;
  if (ys.rows != dout.rows * k)
    return answer(0);
  const GPUXRows d = dout.asArg(), y = ys.asArg(), o = out.asArg();
  return called(gEntries.combineGrad(q.handle, &d, &y, k, ints(place), ints(offsets, offsets.size() - 1),
                                     weighted ? reinterpret_cast<const void *>(weights.ptr) : nullptr, type, &o,
                                     reinterpret_cast<void *>(dweights.ptr)));
}

#define ROWSCALL_FAST(fn, text)                                                                                  \
  { #fn, (PyCFunction)(void (*)(void))rowscall::py_##fn, METH_FASTCALL, text }
#define ROWSCALL_METHODS                                                                                          \
  {"rows_init", rowscall::py_rows_init, METH_VARARGS, "rows_init(entries, types, array_type)"},                   \
      {"rows_torch", rowscall::py_rows_torch, METH_VARARGS, "rows_torch(tensor_type, current_stream)"},           \
      ROWSCALL_FAST(rows_take, "rows_take(queue, table, ids, scale, out)"),                                      \
      ROWSCALL_FAST(rows_take_grad, "rows_take_grad(queue, dout, ids, scale, out, accumulate)"),                 \
      ROWSCALL_FAST(rows_group, "rows_group(queue, ids, groups, plan)"),                                         \
      ROWSCALL_FAST(rows_dispatch, "rows_dispatch(queue, x, ids, groups, plan, out)"),                           \
      ROWSCALL_FAST(rows_combine, "rows_combine(queue, ys, plan, weights, out)"),                                \
      ROWSCALL_FAST(rows_combine_grad, "rows_combine_grad(queue, dout, ys, plan, weights, out, dweights)")

} // namespace rowscall

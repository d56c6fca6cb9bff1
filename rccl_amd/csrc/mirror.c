/* The short way from Python into the local operators: a CPython module that checks torch tensors and calls the library in one
 * step.  It takes the plain case only (contiguous tensors of the named type on the current device, host tables as C-contiguous
 * 64-bit integers) and returns -1 for everything else, which nccl.py then takes the long way, with the checks that say what is
 * wrong.  While tensors are small a call takes what its host side takes: expert_combine 7.0 us through ctypes, 4.7 this way,
 * of which the launch is 3.  Without the module nccl.py takes the long way for all calls.
 * Functions are handed over by address (bind), so the module needs neither the library nor torch to be built. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>
#include <string.h>

#include "rccl_amd.h"

static PyObject *sGetDevice, *sDtype, *sNumel, *sIsContiguous, *sDataPtr, *sShape, *sElementSize, *sCudaStream;
static PyObject* types[ncclNumTypes];      /* torch's element types by their code, or NULL */
static PyObject *currentDevice, *currentStream;

static struct {
  __typeof__(&rcclAmdAdamW) adamw;
  __typeof__(&rcclAmdSumSquares) sumSquares;
  __typeof__(&rcclAmdExpertSort) sort;
  __typeof__(&rcclAmdExpertDispatch) dispatch;
  __typeof__(&rcclAmdExpertCombine) combine;
  __typeof__(&rcclAmdExpertCombineBackward) combineBackward;
  __typeof__(&rcclAmdSumSquaresBytes) sumSquaresBytes;
  __typeof__(&rcclAmdExpertSortBytes) sortBytes;
} fn;

/* A call that is being put together: `ok` falls to 0 with the first argument that is not plain. */
typedef struct { int ok; long device; } Call;

static long long integer(Call* c, PyObject* x) {
  long long v = PyLong_Check(x) ? PyLong_AsLongLong(x) : (c->ok = 0, 0);
  if (v == -1 && PyErr_Occurred()) { PyErr_Clear(); c->ok = 0; }
  return v;
}
static size_t size(Call* c, PyObject* x) {
  const long long v = integer(c, x);
  if (v < 0 || v > (1ll << 40)) { c->ok = 0; return 0; }
  return (size_t)v;
}
static int small(Call* c, PyObject* x) {
  const long long v = integer(c, x);
  if (v < INT_MIN || v > INT_MAX) { c->ok = 0; return 0; }
  return (int)v;
}
static double number(Call* c, PyObject* x) {
  const double v = PyFloat_Check(x) || PyLong_Check(x) ? PyFloat_AsDouble(x) : (c->ok = 0, 0.0);
  if (v == -1.0 && PyErr_Occurred()) { PyErr_Clear(); c->ok = 0; }
  return v;
}
static long long ask(Call* c, PyObject* x, PyObject* method) {
  PyObject* r = c->ok ? PyObject_CallMethodNoArgs(x, method) : NULL;
  long long v = 0;
  if (r) { v = PyLong_Check(r) ? PyLong_AsLongLong(r) : (c->ok = 0, 0); Py_DECREF(r); }
  else { PyErr_Clear(); c->ok = 0; }
  if (v == -1 && PyErr_Occurred()) { PyErr_Clear(); c->ok = 0; }
  return v;
}
static void begin(Call* c) {
  c->ok = currentDevice != NULL;
  PyObject* r = c->ok ? PyObject_CallNoArgs(currentDevice) : NULL;
  c->device = r ? PyLong_AsLong(r) : (c->ok = 0, 0);
  Py_XDECREF(r);
  if (PyErr_Occurred()) { PyErr_Clear(); c->ok = 0; }
}
/* On the current device, of type `type` (-1: any), contiguous. */
static void placed(Call* c, PyObject* x, int type) {
  if (!c->ok) return;
  if (PyLong_Check(x) || ask(c, x, sGetDevice) != c->device) { c->ok = 0; return; }
  if (type >= 0) {
    PyObject* t = type < ncclNumTypes && types[type] ? PyObject_GetAttr(x, sDtype) : NULL;
    if (!t) PyErr_Clear();
    if (!t || t != types[type]) c->ok = 0;
    Py_XDECREF(t);
  }
  PyObject* r = c->ok ? PyObject_CallMethodNoArgs(x, sIsContiguous) : NULL;
  if (r != Py_True) c->ok = 0;
  Py_XDECREF(r);
  PyErr_Clear();
}
static void* whole(Call* c, PyObject* x, size_t n, int type) {
  if (x == Py_None || !c->ok) return NULL;
  placed(c, x, type);
  if (ask(c, x, sNumel) < (long long)n) c->ok = 0;
  return (void*)(uintptr_t)ask(c, x, sDataPtr);
}
static void* matrix(Call* c, PyObject* x, size_t rows, size_t hidden, int type) {
  if (x == Py_None) c->ok = 0;
  if (!c->ok) return NULL;
  placed(c, x, type);
  PyObject* shape = c->ok ? PyObject_GetAttr(x, sShape) : NULL;
  if (!shape) PyErr_Clear();
  if (!shape || !PyTuple_Check(shape) || PyTuple_GET_SIZE(shape) != 2 || PyLong_AsLongLong(PyTuple_GET_ITEM(shape, 0)) < (long long)rows ||
      PyLong_AsLongLong(PyTuple_GET_ITEM(shape, 1)) != (long long)hidden) c->ok = 0;
  Py_XDECREF(shape);
  PyErr_Clear();
  return (void*)(uintptr_t)ask(c, x, sDataPtr);
}
static void* workspace(Call* c, PyObject* x, size_t* bytes) {
  *bytes = 0;
  if (x == Py_None || !c->ok) return NULL;
  placed(c, x, -1);
  *bytes = (size_t)ask(c, x, sNumel) * (size_t)ask(c, x, sElementSize);
  return (void*)(uintptr_t)ask(c, x, sDataPtr);
}
static hipStream_t streamOf(Call* c, PyObject* x) {
  if (!c->ok) return NULL;
  PyObject* r = NULL;
  if (x == Py_None) { PyObject* d = PyLong_FromLong(c->device); r = d ? PyObject_CallOneArg(currentStream, d) : NULL; Py_XDECREF(d); }
  else if (PyLong_Check(x)) { Py_INCREF(x); r = x; }
  else r = PyObject_GetAttr(x, sCudaStream);
  void* p = r ? PyLong_AsVoidPtr(r) : NULL;
  if (!r || PyErr_Occurred()) { PyErr_Clear(); c->ok = 0; }
  Py_XDECREF(r);
  return (hipStream_t)p;
}
/* A C-contiguous host table of 64-bit integers with `columns` columns (1: one dimension). */
static int64_t* table(Call* c, PyObject* x, Py_ssize_t columns, Py_buffer* b, Py_ssize_t* rows) {
  b->obj = NULL;
  *rows = 0;
  if (!c->ok || !PyObject_CheckBuffer(x) || PyObject_GetBuffer(x, b, PyBUF_C_CONTIGUOUS | PyBUF_FORMAT) != 0) { PyErr_Clear(); c->ok = 0; return NULL; }
  const char* f = b->format ? b->format : "B";
  if (b->itemsize != 8 || !f[0] || f[1] != 0 || !strchr("lqLQ", f[0]) || b->ndim != (columns == 1 ? 1 : 2) || (columns > 1 && b->shape[1] != columns) || b->shape[0] > INT_MAX) { c->ok = 0; return NULL; }
  *rows = b->shape[0];
  return (int64_t*)b->buf;
}
static PyObject* done(Call* c, int rc) { return PyLong_FromLong(c->ok ? rc : -1); }
#define NEED(n) do { if (nargs != (n)) { PyErr_Format(PyExc_TypeError, "%d arguments are needed", (n)); return NULL; } } while (0)
#define CALL(expr) do { if (c.ok) { Py_BEGIN_ALLOW_THREADS rc = (expr); Py_END_ALLOW_THREADS } } while (0)

static PyObject* mExpertSort(PyObject* self, PyObject* const* a, Py_ssize_t nargs) {
  NEED(13);
  Call c; begin(&c);
  int rc = 0;
  const int type = small(&c, a[1]), topk = small(&c, a[3]), n = small(&c, a[5]), align = small(&c, a[6]);
  const size_t tokens = size(&c, a[2]);
  const long long first = integer(&c, a[4]);
  if (topk < 1 || topk > 64 || n < 1 || n > 1024 || align < 1 || align > 1024) c.ok = 0;
  const size_t slots = tokens * (size_t)topk;
  size_t bytes;
  void* ids = whole(&c, a[0], slots, type);
  int32_t* position = whole(&c, a[7], slots, ncclInt32);
  int32_t* source = whole(&c, a[8], slots + (size_t)n * (size_t)(align - 1), ncclInt32);
  int32_t* offsets = whole(&c, a[9], (size_t)n + 1, ncclInt32);
  int32_t* counts = whole(&c, a[10], (size_t)n, ncclInt32);
  void* work = workspace(&c, a[11], &bytes);
  hipStream_t s = streamOf(&c, a[12]);
  CALL(fn.sort(ids, type, tokens, topk, first, n, align, position, source, offsets, counts, work, bytes, s));
  return done(&c, rc);
}

/* The segments that say where padding rows are: offsets and counts of n experts, or nothing. */
static void segments(Call* c, PyObject* offsets, PyObject* counts, PyObject* experts, const int32_t** o, const int32_t** k, int* n) {
  *n = small(c, experts);
  if (*n < 0 || *n > 1024) c->ok = 0;
  *o = whole(c, offsets, (size_t)*n + 1, ncclInt32);
  *k = whole(c, counts, (size_t)*n, ncclInt32);
}
static int slotsOf(Call* c, size_t tokens, int topk) { if (topk < 1 || topk > 64 || tokens > 0x7FFFFFFF) c->ok = 0; return c->ok; }

static PyObject* mExpertDispatch(PyObject* self, PyObject* const* a, Py_ssize_t nargs) {
  NEED(12);
  Call c; begin(&c);
  int rc = 0, n;
  const size_t rows = size(&c, a[2]), tokens = size(&c, a[4]), hidden = size(&c, a[6]);
  const int type = small(&c, a[3]), topk = small(&c, a[5]);
  const int32_t *offsets, *counts;
  slotsOf(&c, tokens, topk);
  void* x = matrix(&c, a[0], tokens, hidden, type);
  void* out = matrix(&c, a[1], rows, hidden, type);
  const int32_t* position = whole(&c, a[7], tokens * (size_t)topk, ncclInt32);
  segments(&c, a[8], a[9], a[10], &offsets, &counts, &n);
  hipStream_t s = streamOf(&c, a[11]);
  CALL(fn.dispatch(x, hidden, out, hidden, rows, type, tokens, topk, hidden, position, offsets, counts, n, s));
  return done(&c, rc);
}

static PyObject* mExpertCombine(PyObject* self, PyObject* const* a, Py_ssize_t nargs) {
  NEED(11);
  Call c; begin(&c);
  int rc = 0;
  const size_t rows = size(&c, a[1]), tokens = size(&c, a[6]), hidden = size(&c, a[8]);
  const int wtype = small(&c, a[3]), type = small(&c, a[5]), topk = small(&c, a[7]);
  slotsOf(&c, tokens, topk);
  void* z = matrix(&c, a[0], rows, hidden, type);
  void* w = a[2] == Py_None ? NULL : wtype < 0 ? (c.ok = 0, NULL) : whole(&c, a[2], tokens * (size_t)topk, wtype);
  void* y = matrix(&c, a[4], tokens, hidden, type);
  const int32_t* position = whole(&c, a[9], tokens * (size_t)topk, ncclInt32);
  hipStream_t s = streamOf(&c, a[10]);
  CALL(fn.combine(z, hidden, rows, w, wtype, y, hidden, type, tokens, topk, hidden, position, s));
  return done(&c, rc);
}

static PyObject* mExpertCombineBackward(PyObject* self, PyObject* const* a, Py_ssize_t nargs) {
  NEED(16);
  Call c; begin(&c);
  int rc = 0, n;
  const size_t rows = size(&c, a[2]), tokens = size(&c, a[8]), hidden = size(&c, a[10]);
  const int wtype = small(&c, a[4]), type = small(&c, a[7]), topk = small(&c, a[9]);
  const int32_t *offsets, *counts;
  if (wtype < 0) c.ok = 0;
  slotsOf(&c, tokens, topk);
  void* dy = matrix(&c, a[0], tokens, hidden, type);
  void* z = matrix(&c, a[1], rows, hidden, type);
  void* w = whole(&c, a[3], tokens * (size_t)topk, wtype);
  void* dz = matrix(&c, a[5], rows, hidden, type);
  void* dw = whole(&c, a[6], tokens * (size_t)topk, wtype);
  const int32_t* position = whole(&c, a[11], tokens * (size_t)topk, ncclInt32);
  segments(&c, a[12], a[13], a[14], &offsets, &counts, &n);
  hipStream_t s = streamOf(&c, a[15]);
  CALL(fn.combineBackward(dy, hidden, z, hidden, rows, w, wtype, dz, hidden, dw, type, tokens, topk, hidden, position, offsets, counts, n, s));
  return done(&c, rc);
}

static PyObject* mSumSquares(PyObject* self, PyObject* const* a, Py_ssize_t nargs) {
  NEED(7);
  Call c; begin(&c);
  int rc = 0;
  Py_buffer bt, bc;
  Py_ssize_t n, m;
  size_t bytes;
  const int type = small(&c, a[2]), accumulate = PyObject_IsTrue(a[5]);
  int64_t* tensors = table(&c, a[0], 1, &bt, &n);
  int64_t* counts = table(&c, a[1], 1, &bc, &m);
  if (n != m || accumulate < 0) { PyErr_Clear(); c.ok = 0; }
  double* out = whole(&c, a[3], 1, ncclFloat64);
  void* work = workspace(&c, a[4], &bytes);
  hipStream_t s = streamOf(&c, a[6]);
  CALL(fn.sumSquares((const void* const*)tensors, (const size_t*)counts, (int)n, type, out, accumulate, work, bytes, s));
  PyBuffer_Release(&bt);
  PyBuffer_Release(&bc);
  return done(&c, rc);
}

static PyObject* mAdamW(PyObject* self, PyObject* const* a, Py_ssize_t nargs) {
  NEED(18);
  Call c; begin(&c);
  int rc = 0;
  Py_buffer b;
  Py_ssize_t n;
  rcclAmdAdamWConfig_t k;
  int64_t* tensors = table(&c, a[0], 8, &b, &n);
  const int ptype = small(&c, a[1]), gtype = small(&c, a[2]), ctype = small(&c, a[3]), stype = small(&c, a[4]);
  k.lr = number(&c, a[5]); k.beta1 = number(&c, a[6]); k.beta2 = number(&c, a[7]); k.eps = number(&c, a[8]); k.weightDecay = number(&c, a[9]);
  k.step = integer(&c, a[10]);
  k.stepPtr = whole(&c, a[11], 1, ncclInt64);
  k.lrPtr = whole(&c, a[12], 1, ncclFloat32);
  k.gradScale = number(&c, a[13]);
  k.sumSq = whole(&c, a[14], 1, ncclFloat64);
  k.maxNorm = number(&c, a[15]);
  k.seed = PyLong_Check(a[16]) ? PyLong_AsUnsignedLongLongMask(a[16]) : (c.ok = 0, 0);
  if (PyErr_Occurred()) { PyErr_Clear(); c.ok = 0; }
  hipStream_t s = streamOf(&c, a[17]);
  CALL(fn.adamw((const rcclAmdAdamWTensor_t*)tensors, (int)n, ptype, gtype, ctype, stype, &k, s));
  PyBuffer_Release(&b);
  return done(&c, rc);
}

/* The sizes of workspaces: the bytes, or -1 where the arguments are not plain or are refused. */
static PyObject* mExpertSortBytes(PyObject* self, PyObject* const* a, Py_ssize_t nargs) {
  NEED(3);
  Call c = {fn.sortBytes != NULL, 0};
  size_t bytes = 0;
  const size_t tokens = size(&c, a[0]);
  const int topk = small(&c, a[1]), n = small(&c, a[2]);
  if (c.ok && fn.sortBytes(tokens, topk, n, &bytes) != ncclSuccess) c.ok = 0;
  return PyLong_FromSsize_t(c.ok ? (Py_ssize_t)bytes : -1);
}
static PyObject* mSumSquaresBytes(PyObject* self, PyObject* const* a, Py_ssize_t nargs) {
  NEED(1);
  Call c = {fn.sumSquaresBytes != NULL, 0};
  size_t bytes = 0;
  const int n = small(&c, a[0]);
  if (c.ok && fn.sumSquaresBytes(n, &bytes) != ncclSuccess) c.ok = 0;
  return PyLong_FromSsize_t(c.ok ? (Py_ssize_t)bytes : -1);
}

/* bind(element types by code, current device, current stream of a device, addresses of the library's functions) */
static PyObject* mBind(PyObject* self, PyObject* args) {
  PyObject *t, *d, *s, *f;
  if (!PyArg_ParseTuple(args, "O!OOO!", &PyDict_Type, &t, &d, &s, &PyTuple_Type, &f)) return NULL;
  void* p[8];
  if (PyTuple_GET_SIZE(f) != 8) { PyErr_SetString(PyExc_TypeError, "eight functions are needed"); return NULL; }
  for (int i = 0; i < 8; i++) { p[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(f, i)); if (!p[i]) { if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "a null function"); return NULL; } }
  fn.adamw = (__typeof__(fn.adamw))p[0]; fn.sumSquares = (__typeof__(fn.sumSquares))p[1]; fn.sort = (__typeof__(fn.sort))p[2];
  fn.dispatch = (__typeof__(fn.dispatch))p[3]; fn.combine = (__typeof__(fn.combine))p[4]; fn.combineBackward = (__typeof__(fn.combineBackward))p[5];
  fn.sumSquaresBytes = (__typeof__(fn.sumSquaresBytes))p[6]; fn.sortBytes = (__typeof__(fn.sortBytes))p[7];
  for (int i = 0; i < ncclNumTypes; i++) {
    PyObject* key = PyLong_FromLong(i);
    PyObject* v = key ? PyDict_GetItem(t, key) : NULL;
    Py_XDECREF(key);
    Py_XINCREF(v);
    Py_XSETREF(types[i], v);
  }
  Py_INCREF(d); Py_XSETREF(currentDevice, d);
  Py_INCREF(s); Py_XSETREF(currentStream, s);
  Py_RETURN_NONE;
}

static PyMethodDef methods[] = {
  {"bind", mBind, METH_VARARGS, NULL},
  {"expert_sort", (PyCFunction)(void (*)(void))mExpertSort, METH_FASTCALL, NULL},
  {"expert_dispatch", (PyCFunction)(void (*)(void))mExpertDispatch, METH_FASTCALL, NULL},
  {"expert_combine", (PyCFunction)(void (*)(void))mExpertCombine, METH_FASTCALL, NULL},
  {"expert_combine_backward", (PyCFunction)(void (*)(void))mExpertCombineBackward, METH_FASTCALL, NULL},
  {"sum_squares", (PyCFunction)(void (*)(void))mSumSquares, METH_FASTCALL, NULL},
  {"adamw", (PyCFunction)(void (*)(void))mAdamW, METH_FASTCALL, NULL},
  {"expert_sort_bytes", (PyCFunction)(void (*)(void))mExpertSortBytes, METH_FASTCALL, NULL},
  {"sum_squares_bytes", (PyCFunction)(void (*)(void))mSumSquaresBytes, METH_FASTCALL, NULL},
  {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_mirror", "Plain calls of the local operators (see nccl.py).", -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__mirror(void) {
  if (!(sGetDevice = PyUnicode_InternFromString("get_device")) || !(sDtype = PyUnicode_InternFromString("dtype")) || !(sNumel = PyUnicode_InternFromString("numel")) ||
      !(sIsContiguous = PyUnicode_InternFromString("is_contiguous")) || !(sDataPtr = PyUnicode_InternFromString("data_ptr")) || !(sShape = PyUnicode_InternFromString("shape")) ||
      !(sElementSize = PyUnicode_InternFromString("element_size")) || !(sCudaStream = PyUnicode_InternFromString("cuda_stream"))) return NULL;
  return PyModule_Create(&module);
}

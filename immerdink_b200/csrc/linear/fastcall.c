/* The host side of a call of the quantised linear layer with PyTorch tensors: reads the tensors, checks types,
 * shapes and strides and enters the C ABI. At one row a call costs as much on the host as on the GPU, and most of
 * that is the interpreter and the conversion of some seventeen arguments; here it is the tensors' own accessors.
 *
 * A function returns the call's status, or None for whatever it does not take (other array libraries, another
 * device, anything that has to be refused): the caller then goes through immerdink_b200/linear.py's general path,
 * which accepts or refuses with a message. Built against Python.h alone: the addresses of the C entry points and
 * of cudaGetDevice come from the loaded libraries. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>

enum { kF32 = 0, kBF16 = 1, kF16 = 2, kI8 = 3, kE4M3 = 4, kU8 = 5, kMaxTypes = 16 };

typedef int (*norm_fn)(int64_t, int64_t, int32_t, const void*, int64_t, const void*, int64_t, int32_t, const void*, double,
                       void*, int64_t, int32_t, void*, int64_t, float*, void*);
typedef int (*scaled_fn)(int64_t, int64_t, int64_t, int32_t, const void*, int64_t, const void*, int64_t, const float*,
                         const float*, int32_t, void*, int64_t, void*);
typedef int (*w4_fn)(int64_t, int64_t, int64_t, int32_t, int32_t, const void*, int64_t, const void*, int64_t, int32_t,
                     const void*, int64_t, const void*, int64_t, int32_t, void*, int64_t, void*);
typedef int (*device_fn)(int*);

static PyObject *s_dtype, *s_shape, *s_stride, *s_data_ptr, *s_get_device;
/* dtype objects (immortal singletons of their library) and their types */
static PyObject* g_dtype[kMaxTypes];
static int g_type[kMaxTypes], g_types;

typedef struct {
  void* ptr;
  int64_t extent[2], stride[2];
  int rank, type;
} view_t;

/* 1: read; 0: not for this path (no exception is left). */
static int read_tensor(PyObject* x, int device, view_t* v) {
  PyObject* o = PyObject_GetAttr(x, s_dtype);
  if (o == NULL) goto no;
  v->type = -1;
  for (int i = 0; i < g_types; ++i)
    if (g_dtype[i] == o) v->type = g_type[i];
  Py_DECREF(o);
  if (v->type < 0) return 0;
  if ((o = PyObject_CallMethodNoArgs(x, s_get_device)) == NULL) goto no;
  const long on = PyLong_AsLong(o);
  Py_DECREF(o);
  if (on != device) goto no;
  if ((o = PyObject_GetAttr(x, s_shape)) == NULL) goto no;
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) < 1 || PyTuple_GET_SIZE(o) > 2) {
    Py_DECREF(o);
    return 0;
  }
  v->rank = (int)PyTuple_GET_SIZE(o);
  for (int i = 0; i < v->rank; ++i) v->extent[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(o, i));
  Py_DECREF(o);
  if ((o = PyObject_CallMethodNoArgs(x, s_stride)) == NULL) goto no;
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != v->rank) {
    Py_DECREF(o);
    return 0;
  }
  for (int i = 0; i < v->rank; ++i) v->stride[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(o, i));
  Py_DECREF(o);
  if (v->stride[v->rank - 1] != 1) goto no;
  if ((o = PyObject_CallMethodNoArgs(x, s_data_ptr)) == NULL) goto no;
  v->ptr = PyLong_AsVoidPtr(o);
  Py_DECREF(o);
  if (PyErr_Occurred()) goto no;
  return 1;
no:
  PyErr_Clear();
  return 0;
}
static int is_float(int t) { return t == kF32 || t == kBF16 || t == kF16; }
static int is_matrix(const view_t* v, int64_t rows, int64_t cols) {
  return v->rank == 2 && v->extent[0] == rows && v->extent[1] == cols;
}
static int is_vector(const view_t* v, int64_t n) { return v->rank == 1 && v->extent[0] == n; }

/* The addresses of a library and the device and stream of a call: (functions, ..., stream). */
static int context(PyObject* address, PyObject* get_device, PyObject* stream, void** fn, int* device, void** s) {
  *fn = PyLong_AsVoidPtr(address);
  device_fn dev = (device_fn)PyLong_AsVoidPtr(get_device);
  *s = PyLong_AsVoidPtr(stream);
  if (PyErr_Occurred()) return 0;
  return *fn != NULL && dev != NULL && dev(device) == 0;
}
static PyObject* status(int st) { return PyLong_FromLong(st); }

/* norm_quantize(address, get_device, stream, x, weight, q, scale, eps, residual, residual_out) */
static PyObject* norm_quantize(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  view_t x, w, q, sc, r = {0}, h = {0};
  void *fn, *stream;
  int device = 0;
  if (n != 10) Py_RETURN_NONE;
  if (!context(a[0], a[1], a[2], &fn, &device, &stream)) goto no;
  const double eps = PyFloat_AsDouble(a[7]);
  if (PyErr_Occurred() || !read_tensor(a[3], device, &x) || x.rank != 2 || !is_float(x.type)) goto no;
  const int64_t rows = x.extent[0], dim = x.extent[1];
  if (!read_tensor(a[4], device, &w) || !is_vector(&w, dim) || (w.type != x.type && w.type != kF32) ||
      !read_tensor(a[5], device, &q) || !is_matrix(&q, rows, dim) || (q.type != kI8 && q.type != kE4M3) ||
      !read_tensor(a[6], device, &sc) || !is_vector(&sc, rows) || sc.type != kF32)
    goto no;
  if (a[8] != Py_None && (!read_tensor(a[8], device, &r) || !is_matrix(&r, rows, dim) || r.type != x.type)) goto no;
  if (a[9] != Py_None && (a[8] == Py_None || !read_tensor(a[9], device, &h) || !is_matrix(&h, rows, dim) || h.type != x.type))
    goto no;
  int st;
  Py_BEGIN_ALLOW_THREADS;
  st = ((norm_fn)fn)(rows, dim, x.type, x.ptr, x.stride[0], r.ptr, r.stride[0], w.type, w.ptr, eps, h.ptr, h.stride[0], q.type,
                     q.ptr, q.stride[0], (float*)sc.ptr, stream);
  Py_END_ALLOW_THREADS;
  return status(st);
no:
  PyErr_Clear();
  Py_RETURN_NONE;
}

/* scaled_linear(address, get_device, stream, x, w, out, x_scale, w_scale) */
static PyObject* scaled_linear(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  view_t x, w, o, xs, ws;
  void *fn, *stream;
  int device = 0;
  if (n != 8) Py_RETURN_NONE;
  if (!context(a[0], a[1], a[2], &fn, &device, &stream)) goto no;
  if (!read_tensor(a[3], device, &x) || x.rank != 2 || (x.type != kI8 && x.type != kE4M3) || !read_tensor(a[4], device, &w) ||
      w.rank != 2 || w.type != x.type || w.extent[1] != x.extent[1])
    goto no;
  const int64_t rows = x.extent[0], cols = w.extent[0], k = x.extent[1];
  if (!read_tensor(a[5], device, &o) || !is_matrix(&o, rows, cols) || !is_float(o.type) || !read_tensor(a[6], device, &xs) ||
      !is_vector(&xs, rows) || xs.type != kF32 || !read_tensor(a[7], device, &ws) || !is_vector(&ws, cols) || ws.type != kF32)
    goto no;
  int st;
  Py_BEGIN_ALLOW_THREADS;
  st = ((scaled_fn)fn)(rows, cols, k, x.type, x.ptr, x.stride[0], w.ptr, w.stride[0], (const float*)xs.ptr,
                       (const float*)ws.ptr, o.type, o.ptr, o.stride[0], stream);
  Py_END_ALLOW_THREADS;
  return status(st);
no:
  PyErr_Clear();
  Py_RETURN_NONE;
}

/* linear_w4(address, get_device, stream, x, w, out, w_scale, zeros, group) */
static PyObject* linear_w4(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  view_t x, w, o, sc, z = {0};
  void *fn, *stream;
  int device = 0;
  if (n != 9) Py_RETURN_NONE;
  if (!context(a[0], a[1], a[2], &fn, &device, &stream)) goto no;
  const long group = PyLong_AsLong(a[8]);
  if (PyErr_Occurred() || (group != 32 && group != 64 && group != 128)) goto no;
  if (!read_tensor(a[3], device, &x) || x.rank != 2 || (x.type != kBF16 && x.type != kF16)) goto no;
  const int64_t rows = x.extent[0], k = x.extent[1], groups = (k + group - 1) / group;
  if (!read_tensor(a[4], device, &w) || w.rank != 2 || w.type != kU8 || w.extent[1] != (k + 1) / 2) goto no;
  const int64_t cols = w.extent[0];
  if (!read_tensor(a[5], device, &o) || !is_matrix(&o, rows, cols) || (o.type != kF32 && o.type != x.type) ||
      !read_tensor(a[6], device, &sc) || !is_matrix(&sc, cols, groups) || !is_float(sc.type))
    goto no;
  if (a[7] != Py_None && (!read_tensor(a[7], device, &z) || !is_matrix(&z, cols, groups) || z.type != kU8)) goto no;
  int st;
  Py_BEGIN_ALLOW_THREADS;
  st = ((w4_fn)fn)(rows, cols, k, (int32_t)group, x.type, x.ptr, x.stride[0], w.ptr, w.stride[0], sc.type, sc.ptr,
                   sc.stride[0], z.ptr, z.stride[0], o.type, o.ptr, o.stride[0], stream);
  Py_END_ALLOW_THREADS;
  return status(st);
no:
  PyErr_Clear();
  Py_RETURN_NONE;
}

/* learn(dtype, type): a dtype object that the general path has met. */
static PyObject* learn(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  if (n != 2) Py_RETURN_NONE;
  const long type = PyLong_AsLong(a[1]);
  if (PyErr_Occurred()) return NULL;
  for (int i = 0; i < g_types; ++i)
    if (g_dtype[i] == a[0]) Py_RETURN_NONE;
  if (g_types < kMaxTypes) {
    g_dtype[g_types] = Py_NewRef(a[0]);
    g_type[g_types++] = (int)type;
  }
  Py_RETURN_NONE;
}

static PyMethodDef methods[] = {
    {"norm_quantize", (PyCFunction)(void (*)(void))norm_quantize, METH_FASTCALL, NULL},
    {"scaled_linear", (PyCFunction)(void (*)(void))scaled_linear, METH_FASTCALL, NULL},
    {"linear_w4", (PyCFunction)(void (*)(void))linear_w4, METH_FASTCALL, NULL},
    {"learn", (PyCFunction)(void (*)(void))learn, METH_FASTCALL, NULL},
    {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fastcall", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__fastcall(void) {
  s_dtype = PyUnicode_InternFromString("dtype");
  s_shape = PyUnicode_InternFromString("shape");
  s_stride = PyUnicode_InternFromString("stride");
  s_data_ptr = PyUnicode_InternFromString("data_ptr");
  s_get_device = PyUnicode_InternFromString("get_device");
  if (!s_dtype || !s_shape || !s_stride || !s_data_ptr || !s_get_device) return NULL;
  return PyModule_Create(&module);
}

/*
 * CPython fast path of the 4-bit entry points in ops.py.
 *
 * A 4-bit product takes about 7 us on the device for a few tokens, less than checking its eight
 * tensors from Python and passing twenty arguments through ctypes.  These functions ask the same
 * questions of the tensors (type, shape, stride, device, address) through the C API, apply the
 * common case of the argument rules and launch on torch's current stream, or the given one.
 *
 *   -> True: launched.  False: not the common case; the caller's general path decides, and
 *      raises the precise error.  int: the library's status, not T8G_OK.
 *
 * Nothing is kept between calls but the objects given to setup(): torch.uint8, torch.float32,
 * torch.bfloat16 and torch's function from a device index to its current raw stream.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>

#include "../../include/thor_int8_gemm_b200.h"

static PyObject *s_dtype, *s_shape, *s_stride, *s_get_device, *s_data_ptr, *s_numel, *s_is_contiguous;
static PyObject *t_u8, *t_f32, *t_bf16, *f_raw_stream;

/* Each helper returns 0 when the object does not answer as a tensor of the wanted kind. */
static int i64_of(PyObject* o, int64_t* v) {
  if (!o) return 0;
  const long long x = PyLong_AsLongLong(o);
  Py_DECREF(o);
  if (x == -1 && PyErr_Occurred()) return 0;
  *v = x;
  return 1;
}
static int is_dtype(PyObject* t, PyObject* dtype) {
  PyObject* d = PyObject_GetAttr(t, s_dtype);
  Py_XDECREF(d);
  return d == dtype;
}
static int address(PyObject* t, void** p) {
  int64_t v;
  if (!i64_of(PyObject_CallMethodNoArgs(t, s_data_ptr), &v)) return 0;
  *p = (void*)(intptr_t)v;
  return 1;
}
static int device_is(PyObject* t, int64_t dev) {
  int64_t v;
  return i64_of(PyObject_CallMethodNoArgs(t, s_get_device), &v) && v == dev;
}
static int pair_of(PyObject* o, int64_t* a, int64_t* b) {
  int ok = o && PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 2;
  if (ok) {
    *a = PyLong_AsLongLong(PyTuple_GET_ITEM(o, 0));
    *b = PyLong_AsLongLong(PyTuple_GET_ITEM(o, 1));
    ok = !PyErr_Occurred();
  }
  Py_XDECREF(o);
  return ok;
}

typedef struct {
  int64_t rows, cols, ld;
  void* p;
} Matrix;

/* A non-empty matrix with unit stride along its rows; a single row has a pitch of its own choosing
 * (its length rounded up to `multiple` elements). */
static int matrix(PyObject* t, PyObject* dtype, int64_t multiple, Matrix* m) {
  int64_t inner;
  if (!is_dtype(t, dtype) || !pair_of(PyObject_GetAttr(t, s_shape), &m->rows, &m->cols) || m->rows < 1 || m->cols < 1)
    return 0;
  if (!pair_of(PyObject_CallMethodNoArgs(t, s_stride), &m->ld, &inner) || inner != 1) return 0;
  if (m->rows == 1) m->ld = (m->cols + multiple - 1) / multiple * multiple;
  return address(t, &m->p);
}

/* A contiguous vector of `n` elements (or `other`), or None (0 elements, a null address). */
static int vector(PyObject* t, PyObject* dtype, int64_t n, int64_t other, int64_t dev, void** p, int64_t* count) {
  *p = NULL;
  *count = 0;
  if (t == Py_None) return 1;
  if (!is_dtype(t, dtype) || !device_is(t, dev) || !i64_of(PyObject_CallMethodNoArgs(t, s_numel), count)) return 0;
  if (*count != n && *count != other) return 0;
  PyObject* c = PyObject_CallMethodNoArgs(t, s_is_contiguous);
  Py_XDECREF(c);
  return c == Py_True && address(t, p);
}

/* The block scales: at least `bytes` contiguous bytes. */
static int scales(PyObject* t, int64_t bytes, int64_t dev, void** p) {
  int64_t n;
  if (!is_dtype(t, t_u8) || !device_is(t, dev) || !i64_of(PyObject_CallMethodNoArgs(t, s_numel), &n) || n < bytes) return 0;
  PyObject* shape = PyObject_GetAttr(t, s_shape);
  const int flat = shape && PyTuple_Check(shape) && PyTuple_GET_SIZE(shape) == 1;
  Py_XDECREF(shape);
  if (!flat) return 0;
  PyObject* c = PyObject_CallMethodNoArgs(t, s_is_contiguous);
  Py_XDECREF(c);
  return c == Py_True && address(t, p);
}

/* `stream`: None (torch's current stream of the device) or a raw handle. */
static int stream_of(PyObject* stream, int64_t dev, void** p) {
  PyObject* handle = stream;
  if (stream == Py_None) {
    PyObject* d = PyLong_FromLongLong(dev);
    if (!d) return 0;
    handle = PyObject_CallOneArg(f_raw_stream, d);
    Py_DECREF(d);
    if (!handle) return 0;
  } else {
    if (!PyLong_Check(stream)) return 0;
    Py_INCREF(handle);
  }
  *p = PyLong_AsVoidPtr(handle);
  Py_DECREF(handle);
  return !(*p == NULL && PyErr_Occurred());
}

/* The device that is current and holds `t`. */
static int current_device_of(PyObject* t, int64_t* dev) {
  int cur;
  return i64_of(PyObject_CallMethodNoArgs(t, s_get_device), dev) && *dev >= 0 && t8g_get_device(&cur) == T8G_OK && cur == *dev;
}

typedef struct {
  Matrix x, w;
  void *x_sf, *w_sf, *x_scale, *w_scale, *bias;
  int64_t dev, n_xs, n_ws, n_bias, K;
} Product;

/* args: x, w, x_sf, w_sf, x_scale, w_scale, bias */
static int product(PyObject* const* a, PyObject* out_dtype, int kind, Product* p) {
  if (!current_device_of(a[0], &p->dev) || !matrix(a[0], t_u8, 16, &p->x) || !matrix(a[1], t_u8, 16, &p->w)) return 0;
  p->K = 2 * p->x.cols;
  return p->w.cols == p->x.cols && p->K % 8 == 0 && device_is(a[1], p->dev) &&
         scales(a[2], t8g_fp4_scale_bytes(p->x.rows, p->K, kind), p->dev, &p->x_sf) &&
         scales(a[3], t8g_fp4_scale_bytes(p->w.rows, p->K, kind), p->dev, &p->w_sf) &&
         vector(a[4], t_f32, p->x.rows, p->x.rows, p->dev, &p->x_scale, &p->n_xs) &&
         vector(a[5], t_f32, p->w.rows, 1, p->dev, &p->w_scale, &p->n_ws) &&
         vector(a[6], out_dtype, p->w.rows, 0, p->dev, &p->bias, &p->n_bias);
}

static PyObject* result(int rc) {
  if (rc == T8G_OK) Py_RETURN_TRUE;
  return PyLong_FromLong(rc);
}
static PyObject* uncommon(void) {
  PyErr_Clear();
  Py_RETURN_FALSE;
}
static int small_int(PyObject* o, int* v) {
  const long x = PyLong_AsLong(o);
  if ((x == -1 && PyErr_Occurred()) || x < INT32_MIN || x > INT32_MAX) return 0;
  *v = (int)x;
  return 1;
}

/* gemm(x, w, x_sf, w_sf, x_scale, w_scale, bias, out, out_dtype, out_code, per_16_bytes, kind, stream) */
static PyObject* gemm(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  (void)self;
  Product p;
  Matrix out;
  void* stream;
  int out_code, per, kind;
  if (n != 13 || !t_u8) {
    PyErr_SetString(PyExc_TypeError, "gemm: 13 arguments, after setup()");
    return NULL;
  }
  if (!small_int(a[9], &out_code) || !small_int(a[10], &per) || !small_int(a[11], &kind) || !product(a, a[8], kind, &p) ||
      !matrix(a[7], a[8], per, &out) || out.rows != p.x.rows || out.cols != p.w.rows || !device_is(a[7], p.dev) ||
      !stream_of(a[12], p.dev, &stream))
    return uncommon();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = t8g_gemm_fp4(p.x.p, p.x_sf, p.x_scale, p.w.p, p.w_sf, p.w_scale, p.n_ws, p.bias, p.n_bias, out.p, out_code, p.x.rows,
                    p.w.rows, p.K, p.x.ld, p.w.ld, out.ld, kind, stream);
  Py_END_ALLOW_THREADS
  return result(rc);
}

/* gated(x, w, x_sf, w_sf, x_scale, w_scale, bias, res, gate, out, rows_per_gate, kind, stream) */
static PyObject* gated(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  (void)self;
  Product p;
  Matrix res, gate, out;
  void* stream;
  int rows_per_gate, kind;
  if (n != 13 || !t_u8) {
    PyErr_SetString(PyExc_TypeError, "gated: 13 arguments, after setup()");
    return NULL;
  }
  if (!small_int(a[10], &rows_per_gate) || !small_int(a[11], &kind) || !product(a, t_bf16, kind, &p) ||
      !matrix(a[7], t_bf16, 8, &res) || !matrix(a[8], t_bf16, 8, &gate) || !matrix(a[9], t_bf16, 8, &out) ||
      res.rows != p.x.rows || res.cols != p.w.rows || out.rows != p.x.rows || out.cols != p.w.rows || gate.cols != p.w.rows ||
      rows_per_gate < 1 || (p.x.rows - 1) / rows_per_gate >= gate.rows || !device_is(a[7], p.dev) ||
      !device_is(a[8], p.dev) || !device_is(a[9], p.dev) || !stream_of(a[12], p.dev, &stream))
    return uncommon();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = t8g_gemm_fp4_gated(p.x.p, p.x_sf, p.x_scale, p.w.p, p.w_sf, p.w_scale, p.n_ws, p.bias, p.n_bias, res.p, res.ld, gate.p,
                          gate.ld, NULL, rows_per_gate, out.p, p.x.rows, p.w.rows, p.K, p.x.ld, p.w.ld, out.ld, kind, stream);
  Py_END_ALLOW_THREADS
  return result(rc);
}

/* A 4-bit output that the caller has just allocated for [S, D]: q, sf, q_scale (or None).  Only the
 * addresses are asked for. */
typedef struct {
  void *q, *sf, *scale;
  int64_t ld;
} Out4;
static int out4(PyObject* const* a, int64_t D, Out4* o) {
  o->ld = (D + 31) / 32 * 16;
  o->scale = NULL;
  return address(a[0], &o->q) && address(a[1], &o->sf) && (a[2] == Py_None || address(a[2], &o->scale));
}

/* quant_rows(x, q, sf, q_scale, kind, stream) */
static PyObject* quant_rows(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  (void)self;
  Matrix x;
  Out4 o;
  int64_t dev;
  void* stream;
  int kind;
  if (n != 6 || !t_u8) {
    PyErr_SetString(PyExc_TypeError, "quant_rows: 6 arguments, after setup()");
    return NULL;
  }
  if (!small_int(a[4], &kind) || !current_device_of(a[0], &dev) || !matrix(a[0], t_bf16, 8, &x) || x.cols % 8 ||
      !out4(a + 1, x.cols, &o) || !stream_of(a[5], dev, &stream))
    return uncommon();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = t8g_quant_rows_fp4(x.p, x.ld, o.q, o.ld, o.sf, (float*)o.scale, x.rows, x.cols, kind, stream);
  Py_END_ALLOW_THREADS
  return result(rc);
}

/* swiglu_fc1(y, q, sf, q_scale, kind, stream): y [M, 2F], its first half the gate */
static PyObject* swiglu_fc1(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  (void)self;
  Matrix y;
  Out4 o;
  int64_t dev;
  void* stream;
  int kind;
  if (n != 6 || !t_u8) {
    PyErr_SetString(PyExc_TypeError, "swiglu_fc1: 6 arguments, after setup()");
    return NULL;
  }
  if (!small_int(a[4], &kind) || !current_device_of(a[0], &dev) || !matrix(a[0], t_bf16, 8, &y) || y.cols % 16 ||
      !out4(a + 1, y.cols / 2, &o) || !stream_of(a[5], dev, &stream))
    return uncommon();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = t8g_swiglu_quant_fp4(y.p, (const char*)y.p + y.cols, y.ld, o.q, o.ld, o.sf, (float*)o.scale, y.rows, y.cols / 2, kind,
                            stream);   /* half a row is cols / 2 elements of two bytes */
  Py_END_ALLOW_THREADS
  return result(rc);
}

/* rms_mod_quant(x, shift, scale, rows_per_mod, scale_is_multiplier, eps, q, sf, q_scale, kind, stream) */
static PyObject* rms_mod_quant(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  (void)self;
  Matrix x, shift, scale;
  Out4 o;
  int64_t dev;
  void* stream;
  int kind, rows_per_mod, multiplier;
  if (n != 11 || !t_u8) {
    PyErr_SetString(PyExc_TypeError, "rms_mod_quant: 11 arguments, after setup()");
    return NULL;
  }
  const double eps = PyFloat_AsDouble(a[5]);
  if (PyErr_Occurred() || !small_int(a[3], &rows_per_mod) || !small_int(a[4], &multiplier) || !small_int(a[9], &kind) ||
      !current_device_of(a[0], &dev) || !matrix(a[0], t_bf16, 8, &x) || x.cols % 8 || !matrix(a[1], t_bf16, 8, &shift) ||
      !matrix(a[2], t_bf16, 8, &scale) || shift.cols != x.cols || scale.cols != x.cols || shift.rows != scale.rows ||
      shift.ld != scale.ld || rows_per_mod < 1 || (x.rows - 1) / rows_per_mod >= shift.rows || !device_is(a[1], dev) ||
      !device_is(a[2], dev) || !out4(a + 6, x.cols, &o) || !stream_of(a[10], dev, &stream))
    return uncommon();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = t8g_rms_mod_quant_fp4(x.p, x.ld, NULL, shift.p, scale.p, shift.ld, NULL, rows_per_mod, multiplier, (float)eps, o.q, o.ld,
                             o.sf, (float*)o.scale, x.rows, x.cols, kind, stream);
  Py_END_ALLOW_THREADS
  return result(rc);
}

/* dequant(q, sf, q_scale, out, out_code, kind, stream): out [S, D], contiguous, just allocated by the caller */
static PyObject* dequant(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  (void)self;
  Matrix q;
  int64_t dev, n_scale;
  void *sf, *scale, *out, *stream;
  int out_code, kind;
  if (n != 7 || !t_u8) {
    PyErr_SetString(PyExc_TypeError, "dequant: 7 arguments, after setup()");
    return NULL;
  }
  if (!small_int(a[4], &out_code) || !small_int(a[5], &kind) || !current_device_of(a[0], &dev) ||
      !matrix(a[0], t_u8, 16, &q) || q.cols % 4 || !scales(a[1], t8g_fp4_scale_bytes(q.rows, 2 * q.cols, kind), dev, &sf) ||
      !vector(a[2], t_f32, q.rows, q.rows, dev, &scale, &n_scale) || !device_is(a[3], dev) || !address(a[3], &out) ||
      !stream_of(a[6], dev, &stream))
    return uncommon();
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = t8g_dequant_rows_fp4(q.p, q.ld, sf, (const float*)scale, out, out_code, 2 * q.cols, q.rows, 2 * q.cols, kind, stream);
  Py_END_ALLOW_THREADS
  return result(rc);
}

/* setup(torch.uint8, torch.float32, torch.bfloat16, raw_stream) */
static PyObject* setup(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  (void)self;
  if (n != 4) {
    PyErr_SetString(PyExc_TypeError, "setup(uint8, float32, bfloat16, raw_stream)");
    return NULL;
  }
  PyObject** keep[4] = {&t_u8, &t_f32, &t_bf16, &f_raw_stream};
  for (int i = 0; i < 4; ++i) {
    Py_INCREF(a[i]);
    Py_XSETREF(*keep[i], a[i]);
  }
  Py_RETURN_NONE;
}

#define FAST(f) (PyCFunction)(void (*)(void))f, METH_FASTCALL
static PyMethodDef methods[] = {{"setup", FAST(setup), "Keep torch's dtype objects and its current-stream function."},
                                {"gemm", FAST(gemm), "t8g_gemm_fp4 on torch tensors, the common case."},
                                {"gated", FAST(gated), "t8g_gemm_fp4_gated on torch tensors, the common case."},
                                {"quant_rows", FAST(quant_rows), "t8g_quant_rows_fp4, the common case."},
                                {"swiglu_fc1", FAST(swiglu_fc1), "t8g_swiglu_quant_fp4 of an fc1 output, the common case."},
                                {"rms_mod_quant", FAST(rms_mod_quant), "t8g_rms_mod_quant_fp4, the common case."},
                                {"dequant", FAST(dequant), "t8g_dequant_rows_fp4, the common case."},
                                {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_t8g_fp4", NULL, -1, methods};

PyMODINIT_FUNC PyInit__t8g_fp4(void) {
  struct {
    PyObject** at;
    const char* name;
  } names[] = {{&s_dtype, "dtype"},           {&s_shape, "shape"},       {&s_stride, "stride"},
               {&s_get_device, "get_device"}, {&s_data_ptr, "data_ptr"}, {&s_numel, "numel"},
               {&s_is_contiguous, "is_contiguous"}};
  for (size_t i = 0; i < sizeof(names) / sizeof(names[0]); ++i)
    if (!(*names[i].at = PyUnicode_InternFromString(names[i].name))) return NULL;
  return PyModule_Create(&module);
}

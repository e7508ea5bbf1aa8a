/* CPython binding of the per-token (small-M) INT4 + LoRA forward and of the MXFP4,
 * adapter bank, dropout and block boundary entry points.
 *
 * Such an eager call spends more time on the host than on the GPU, and
 * ctypes' per-argument conversion is a large share of it. These functions
 * take the same arguments as the C ABI (device pointers as Python ints, NULL
 * as None) through METH_FASTCALL and forward them unchanged; each returns the
 * C function's status or size. They add nothing else: validation, errors
 * (rpx_last_error) and launches are the library's.
 *
 * Built against librepresentax_amd.so in the same directory (rpath $ORIGIN),
 * so the process holds one instance of the library whichever binding it uses.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <stdint.h>
#include <string.h>

#include "../../include/representax_amd.h"

#define MAX_PROJECTIONS 16
#define PROJECTION_FIELDS 11

static int get_i64(PyObject* o, int64_t* v) {
  long long x = PyLong_AsLongLong(o);
  if (x == -1 && PyErr_Occurred()) return 0;
  *v = (int64_t)x;
  return 1;
}

static int get_int(PyObject* o, int* v) {
  long x = PyLong_AsLong(o);
  if (x == -1 && PyErr_Occurred()) return 0;
  if (x < INT32_MIN || x > INT32_MAX) {
    PyErr_SetString(PyExc_OverflowError, "value does not fit a C int");
    return 0;
  }
  *v = (int)x;
  return 1;
}

static int get_ptr(PyObject* o, void** p) {
  if (o == Py_None) {
    *p = NULL;
    return 1;
  }
  unsigned long long x = PyLong_AsUnsignedLongLong(o);
  if (x == (unsigned long long)-1 && PyErr_Occurred()) return 0;
  *p = (void*)(uintptr_t)x;
  return 1;
}

static int get_f32(PyObject* o, float* v) {
  double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) return 0;
  *v = (float)x;
  return 1;
}

static int check_nargs(const char* name, Py_ssize_t nargs, Py_ssize_t want) {
  if (nargs == want) return 1;
  PyErr_Format(PyExc_TypeError, "%s takes %zd arguments (%zd given)", name, want, nargs);
  return 0;
}

/* int4lora_forward(x, dtype, m, k, packed, scale_bits, n, group_size,
 *                  bias_bits, lora_a, lora_b, rank, scaling, y, h,
 *                  workspace, workspace_bytes, stream) -> status */
static PyObject* fast_int4lora_forward(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  void *x, *packed, *scales, *bias, *a, *b, *y, *h, *ws, *stream;
  int dtype;
  int64_t m, k, n, group, rank, ws_bytes;
  float scaling;
  if (!check_nargs("int4lora_forward", nargs, 18)) return NULL;
  if (!get_ptr(args[0], &x) || !get_int(args[1], &dtype) || !get_i64(args[2], &m) ||
      !get_i64(args[3], &k) || !get_ptr(args[4], &packed) || !get_ptr(args[5], &scales) ||
      !get_i64(args[6], &n) || !get_i64(args[7], &group) || !get_ptr(args[8], &bias) ||
      !get_ptr(args[9], &a) || !get_ptr(args[10], &b) || !get_i64(args[11], &rank) ||
      !get_f32(args[12], &scaling) || !get_ptr(args[13], &y) || !get_ptr(args[14], &h) ||
      !get_ptr(args[15], &ws) || !get_i64(args[16], &ws_bytes) || !get_ptr(args[17], &stream))
    return NULL;
  if (ws_bytes < 0) {
    PyErr_SetString(PyExc_ValueError, "workspace_bytes must be non-negative");
    return NULL;
  }
  int status = rpx_int4lora_forward(x, dtype, m, k, (const uint8_t*)packed,
                                    (const uint16_t*)scales, n, group, (const uint16_t*)bias, a, b,
                                    rank, scaling, y, h, ws, (size_t)ws_bytes, stream);
  return PyLong_FromLong(status);
}

/* int4lora_forward_workspace(m, n, k, group_size, rank, dtype) -> bytes */
static PyObject* fast_int4lora_forward_workspace(PyObject* self, PyObject* const* args,
                                                 Py_ssize_t nargs) {
  (void)self;
  int64_t m, n, k, group, rank;
  int dtype;
  if (!check_nargs("int4lora_forward_workspace", nargs, 6)) return NULL;
  if (!get_i64(args[0], &m) || !get_i64(args[1], &n) || !get_i64(args[2], &k) ||
      !get_i64(args[3], &group) || !get_i64(args[4], &rank) || !get_int(args[5], &dtype))
    return NULL;
  return PyLong_FromSize_t(rpx_int4lora_forward_workspace(m, n, k, group, rank, dtype));
}

/* Fills table[0, count) from a tuple of count x 11 fields in the order of
 * rpx_int4lora_projection: packed, scale_bits, n, group_size, bias_bits,
 * lora_a, lora_b, rank, scaling, y, h. */
static int fill_projections(PyObject* flat, rpx_int4lora_projection* table, int* count) {
  if (!PyTuple_Check(flat)) {
    PyErr_SetString(PyExc_TypeError, "projections must be a flat tuple");
    return 0;
  }
  Py_ssize_t len = PyTuple_GET_SIZE(flat);
  if (len % PROJECTION_FIELDS != 0 || len / PROJECTION_FIELDS > MAX_PROJECTIONS) {
    PyErr_Format(PyExc_ValueError,
                 "projections: expected a multiple of %d fields for at most %d projections",
                 PROJECTION_FIELDS, MAX_PROJECTIONS);
    return 0;
  }
  *count = (int)(len / PROJECTION_FIELDS);
  for (int i = 0; i < *count; ++i) {
    PyObject* const* f = &PyTuple_GET_ITEM(flat, (Py_ssize_t)i * PROJECTION_FIELDS);
    void *packed, *scales, *bias, *a, *b, *y, *h;
    rpx_int4lora_projection* p = &table[i];
    if (!get_ptr(f[0], &packed) || !get_ptr(f[1], &scales) || !get_i64(f[2], &p->n) ||
        !get_i64(f[3], &p->group_size) || !get_ptr(f[4], &bias) || !get_ptr(f[5], &a) ||
        !get_ptr(f[6], &b) || !get_i64(f[7], &p->rank) || !get_f32(f[8], &p->scaling) ||
        !get_ptr(f[9], &y) || !get_ptr(f[10], &h))
      return 0;
    p->packed = (const uint8_t*)packed;
    p->scale_bits = (const uint16_t*)scales;
    p->bias_bits = (const uint16_t*)bias;
    p->lora_a = a;
    p->lora_b = b;
    p->y = y;
    p->h = h;
  }
  return 1;
}

/* int4lora_forward_multi_workspace(m, k, projections, dtype) -> bytes */
static PyObject* fast_int4lora_forward_multi_workspace(PyObject* self, PyObject* const* args,
                                                       Py_ssize_t nargs) {
  (void)self;
  int64_t m, k;
  int dtype, count;
  rpx_int4lora_projection table[MAX_PROJECTIONS];
  if (!check_nargs("int4lora_forward_multi_workspace", nargs, 4)) return NULL;
  if (!get_i64(args[0], &m) || !get_i64(args[1], &k) || !fill_projections(args[2], table, &count) ||
      !get_int(args[3], &dtype))
    return NULL;
  return PyLong_FromSize_t(rpx_int4lora_forward_multi_workspace(m, k, count, table, dtype));
}

/* int4lora_forward_multi(x, dtype, m, k, projections, workspace,
 *                        workspace_bytes, stream) -> status */
static PyObject* fast_int4lora_forward_multi(PyObject* self, PyObject* const* args,
                                             Py_ssize_t nargs) {
  (void)self;
  void *x, *ws, *stream;
  int dtype, count;
  int64_t m, k, ws_bytes;
  rpx_int4lora_projection table[MAX_PROJECTIONS];
  if (!check_nargs("int4lora_forward_multi", nargs, 8)) return NULL;
  if (!get_ptr(args[0], &x) || !get_int(args[1], &dtype) || !get_i64(args[2], &m) ||
      !get_i64(args[3], &k) || !fill_projections(args[4], table, &count) ||
      !get_ptr(args[5], &ws) || !get_i64(args[6], &ws_bytes) || !get_ptr(args[7], &stream))
    return NULL;
  if (ws_bytes < 0) {
    PyErr_SetString(PyExc_ValueError, "workspace_bytes must be non-negative");
    return NULL;
  }
  int status = rpx_int4lora_forward_multi(x, dtype, m, k, count, table, ws, (size_t)ws_bytes,
                                          stream);
  return PyLong_FromLong(status);
}

/* get_tuning(knob) -> value: the library's knob as this binding sees it (the
 * check that both bindings share one loaded library). */
static PyObject* fast_get_tuning(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  int knob;
  if (!check_nargs("get_tuning", nargs, 1)) return NULL;
  if (!get_int(args[0], &knob)) return NULL;
  return PyLong_FromLong(rpx_get_tuning(knob));
}

typedef union {
  void* p;
  int64_t l;
  int i;
  float f;
} Value;

/* Arguments by a format: p pointer, l int64, s size (not negative), i int, f float. */
static int parse(const char* name, const char* format, PyObject* const* args, Py_ssize_t nargs,
                 Value* v) {
  if (!check_nargs(name, nargs, (Py_ssize_t)strlen(format))) return 0;
  for (Py_ssize_t j = 0; j < nargs; ++j) {
    const int ok = format[j] == 'p'   ? get_ptr(args[j], &v[j].p)
                   : format[j] == 'i' ? get_int(args[j], &v[j].i)
                   : format[j] == 'f' ? get_f32(args[j], &v[j].f)
                                      : get_i64(args[j], &v[j].l);
    if (!ok) return 0;
    if (format[j] == 's' && v[j].l < 0) {
      PyErr_Format(PyExc_ValueError, "%s: buffer sizes must be non-negative", name);
      return 0;
    }
  }
  return 1;
}

/* The MXFP4 calls take the C functions' arguments (mxfp4_quantize: of its one part). */
static PyObject* fast_mxfp4_linear(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  Value v[12];
  if (!parse("mxfp4_linear", "pilllpplppsp", args, nargs, v)) return NULL;
  return PyLong_FromLong(rpx_mxfp4_linear(v[0].p, v[1].i, v[2].l, v[3].l, v[4].l, v[5].p, v[6].p,
                                          v[7].l, v[8].p, v[9].p, (size_t)v[10].l, v[11].p));
}

static PyObject* fast_mxfp4_gated(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  Value v[14];
  if (!parse("mxfp4_gated", "pilllpppplppsp", args, nargs, v)) return NULL;
  return PyLong_FromLong(rpx_mxfp4_gated(v[0].p, v[1].i, v[2].l, v[3].l, v[4].l, v[5].p, v[6].p,
                                         v[7].p, v[8].p, v[9].l, v[10].p, v[11].p,
                                         (size_t)v[12].l, v[13].p));
}

/* mxfp4_quantize(t, rows, columns, row_stride, codes, scales, codes_t, scales_t, dtype,
 * stream): one matrix, its codes dense. */
static PyObject* fast_mxfp4_quantize(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  Value v[10];
  if (!parse("mxfp4_quantize", "plllppppip", args, nargs, v)) return NULL;
  const rpx_mxfp4_part part = {v[0].p, v[1].l, v[2].l, v[3].l, v[4].p, v[5].p,
                               0,      v[6].p, v[7].p, 0,      v[8].i};
  return PyLong_FromLong(rpx_mxfp4_quantize(&part, 1, v[9].p));
}

static PyObject* fast_mxfp4_dequantize(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  Value v[7];
  if (!parse("mxfp4_dequantize", "ppllpip", args, nargs, v)) return NULL;
  return PyLong_FromLong(
      rpx_mxfp4_dequantize(v[0].p, v[1].p, v[2].l, v[3].l, v[4].p, v[5].i, v[6].p));
}

static PyObject* fast_mxfp4_linear_forward(PyObject* self, PyObject* const* args,
                                           Py_ssize_t nargs) {
  (void)self;
  Value v[19];
  if (!parse("mxfp4_linear_forward", "pilllpilllpipsiipsp", args, nargs, v)) return NULL;
  return PyLong_FromLong(rpx_mxfp4_linear_forward(
      v[0].p, v[1].i, v[2].l, v[3].l, v[4].l, v[5].p, v[6].i, v[7].l, v[8].l, v[9].l, v[10].p,
      v[11].i, v[12].p, (size_t)v[13].l, v[14].i, v[15].i, v[16].p, (size_t)v[17].l, v[18].p));
}

static PyObject* fast_mxfp4_linear_backward(PyObject* self, PyObject* const* args,
                                            Py_ssize_t nargs) {
  (void)self;
  Value v[17];
  if (!parse("mxfp4_linear_backward", "pilllpsliipipipsp", args, nargs, v)) return NULL;
  return PyLong_FromLong(rpx_mxfp4_linear_backward(
      v[0].p, v[1].i, v[2].l, v[3].l, v[4].l, v[5].p, (size_t)v[6].l, v[7].l, v[8].i, v[9].i,
      v[10].p, v[11].i, v[12].p, v[13].i, v[14].p, (size_t)v[15].l, v[16].p));
}

static PyObject* fast_mxfp4_gated_forward(PyObject* self, PyObject* const* args,
                                          Py_ssize_t nargs) {
  (void)self;
  Value v[25];
  if (!parse("mxfp4_gated_forward", "pilllpillpilllpppipsiipsp", args, nargs, v)) return NULL;
  return PyLong_FromLong(rpx_mxfp4_gated_forward(
      v[0].p, v[1].i, v[2].l, v[3].l, v[4].l, v[5].p, v[6].i, v[7].l, v[8].l, v[9].p, v[10].i,
      v[11].l, v[12].l, v[13].l, v[14].p, v[15].p, v[16].p, v[17].i, v[18].p, (size_t)v[19].l,
      v[20].i, v[21].i, v[22].p, (size_t)v[23].l, v[24].p));
}

static PyObject* fast_mxfp4_gated_backward(PyObject* self, PyObject* const* args,
                                           Py_ssize_t nargs) {
  (void)self;
  Value v[18];
  if (!parse("mxfp4_gated_backward_products", "pppillpsliipipipsp", args, nargs, v)) return NULL;
  return PyLong_FromLong(rpx_mxfp4_gated_backward_products(
      v[0].p, v[1].p, v[2].p, v[3].i, v[4].l, v[5].l, v[6].p, (size_t)v[7].l, v[8].l, v[9].i,
      v[10].i, v[11].p, v[12].i, v[13].p, v[14].i, v[15].p, (size_t)v[16].l, v[17].p));
}

/* mxfp4_bytes(what, m, n, k, need_left, need_right) -> bytes; what: 0 linear, 1
 * gated (serving workspaces), 2 and 3 their saved buffers, 4 and 5 their forward,
 * 6 and 7 their backward workspaces */
static PyObject* fast_mxfp4_bytes(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  Value v[6];
  if (!parse("mxfp4_bytes", "illlii", args, nargs, v)) return NULL;
  const int64_t m = v[1].l, n = v[2].l, k = v[3].l;
  const int left = v[4].i, right = v[5].i;
  switch (v[0].i) {
    case 0: return PyLong_FromSize_t(rpx_mxfp4_linear_workspace(m, n, k));
    case 1: return PyLong_FromSize_t(rpx_mxfp4_gated_workspace(m, n, k));
    case 2: return PyLong_FromSize_t(rpx_mxfp4_linear_saved_bytes(m, n, k, left, right));
    case 3: return PyLong_FromSize_t(rpx_mxfp4_gated_saved_bytes(m, n, k, left, right));
    case 4: return PyLong_FromSize_t(rpx_mxfp4_linear_forward_workspace(m, n, k));
    case 5: return PyLong_FromSize_t(rpx_mxfp4_gated_forward_workspace(m, n, k));
    case 6: return PyLong_FromSize_t(rpx_mxfp4_linear_backward_workspace(m, n, k, left, right));
    case 7: return PyLong_FromSize_t(rpx_mxfp4_gated_backward_workspace(m, n, k, left, right));
  }
  PyErr_SetString(PyExc_ValueError, "mxfp4_bytes: unknown size");
  return NULL;
}

static PyObject* fast_dropout(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  Value v[8];
  if (!parse("dropout", "pilpllpp", args, nargs, v)) return NULL;
  return PyLong_FromLong(
      rpx_dropout(v[0].p, v[1].i, v[2].l, v[3].p, v[4].l, v[5].l, v[6].p, v[7].p));
}

/* The fields of an rpx_block, its norms' in their places: x, u, gate, rows_per_gate, post
 * (weight, bias, dtype, kind, eps), norm (the same), key, site, threshold, rows, size, t,
 * h, dtype, gate_dtype, scale. */
#define BLOCK "ppplppiifppiifpllllppiif"
static rpx_block block_of(const Value* v) {
  const rpx_block b = {v[0].p,
                       v[1].p,
                       v[2].p,
                       v[3].l,
                       {v[4].p, v[5].p, v[6].i, v[7].i, v[8].f},
                       {v[9].p, v[10].p, v[11].i, v[12].i, v[13].f},
                       v[14].p,
                       v[15].l,
                       v[16].l,
                       v[17].l,
                       v[18].l,
                       v[19].p,
                       v[20].p,
                       v[21].i,
                       v[22].i,
                       v[23].f};
  return b;
}

static PyObject* fast_block_forward(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  Value v[25];
  if (!parse("block_forward", BLOCK "p", args, nargs, v)) return NULL;
  const rpx_block b = block_of(v);
  return PyLong_FromLong(rpx_block_forward(&b, v[24].p));
}

static rpx_block_gradients gradients_of(const Value* v) {
  const rpx_block_gradients g = {v[0].p, v[1].p, v[2].p, v[3].p, v[4].p,
                                 v[5].p, v[6].p, v[7].p, v[8].p};
  return g;
}

/* block_backward_workspace(block fields, gradients) -> bytes */
static PyObject* fast_block_backward_workspace(PyObject* self, PyObject* const* args,
                                               Py_ssize_t nargs) {
  (void)self;
  Value v[33];
  if (!parse("block_backward_workspace", BLOCK "ppppppppp", args, nargs, v)) return NULL;
  const rpx_block b = block_of(v);
  const rpx_block_gradients g = gradients_of(v + 24);
  return PyLong_FromSize_t(rpx_block_backward_workspace(&b, &g));
}

static PyObject* fast_block_backward(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  Value v[36];
  if (!parse("block_backward", BLOCK "ppppppppppsp", args, nargs, v)) return NULL;
  const rpx_block b = block_of(v);
  const rpx_block_gradients g = gradients_of(v + 24);
  return PyLong_FromLong(rpx_block_backward(&b, &g, v[33].p, (size_t)v[34].l, v[35].p));
}

/* The fields of an rpx_bank in their order. */
#define BANK "pllppllppppllpspll"
static rpx_bank bank_of(const Value* v) {
  const rpx_bank b = {v[0].p,  v[1].l,  v[2].l, v[3].p, v[4].p,  v[5].l,          v[6].l,
                      v[7].p,  v[8].p,  v[9].p, v[10].p, v[11].l, v[12].l,         v[13].p,
                      (size_t)v[14].l, v[15].p, v[16].l, v[17].l};
  return b;
}

/* bank_forward_workspace(bank fields, h_given) -> bytes */
static PyObject* fast_bank_forward_workspace(PyObject* self, PyObject* const* args,
                                             Py_ssize_t nargs) {
  (void)self;
  Value v[19];
  if (!parse("bank_forward_workspace", BANK "i", args, nargs, v)) return NULL;
  const rpx_bank b = bank_of(v);
  return PyLong_FromSize_t(rpx_bank_forward_workspace(&b, v[18].i));
}

static PyObject* fast_bank_forward(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  Value v[23];
  if (!parse("bank_forward", BANK "pppsp", args, nargs, v)) return NULL;
  const rpx_bank b = bank_of(v);
  return PyLong_FromLong(
      rpx_bank_forward(&b, v[18].p, v[19].p, v[20].p, (size_t)v[21].l, v[22].p));
}

/* bank_backward_workspace(bank fields, need_x, need_a, need_b) -> bytes */
static PyObject* fast_bank_backward_workspace(PyObject* self, PyObject* const* args,
                                              Py_ssize_t nargs) {
  (void)self;
  Value v[21];
  if (!parse("bank_backward_workspace", BANK "iii", args, nargs, v)) return NULL;
  const rpx_bank b = bank_of(v);
  return PyLong_FromSize_t(rpx_bank_backward_workspace(&b, v[18].i, v[19].i, v[20].i));
}

static PyObject* fast_bank_backward(PyObject* self, PyObject* const* args, Py_ssize_t nargs) {
  (void)self;
  Value v[28];
  if (!parse("bank_backward", BANK "ppppipipsp", args, nargs, v)) return NULL;
  const rpx_bank b = bank_of(v);
  return PyLong_FromLong(rpx_bank_backward(&b, v[18].p, v[19].p, v[20].p, v[21].p, v[22].i,
                                           v[23].p, v[24].i, v[25].p, (size_t)v[26].l, v[27].p));
}

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))fast_##name, METH_FASTCALL, "rpx_" #name}

static PyMethodDef methods[] = {
    METHOD(dropout),
    METHOD(block_forward),
    METHOD(block_backward_workspace),
    METHOD(block_backward),
    METHOD(bank_forward_workspace),
    METHOD(bank_forward),
    METHOD(bank_backward_workspace),
    METHOD(bank_backward),
    {"get_tuning", (PyCFunction)(void (*)(void))fast_get_tuning, METH_FASTCALL, "rpx_get_tuning"},
    {"int4lora_forward", (PyCFunction)(void (*)(void))fast_int4lora_forward, METH_FASTCALL,
     "rpx_int4lora_forward"},
    {"int4lora_forward_workspace", (PyCFunction)(void (*)(void))fast_int4lora_forward_workspace,
     METH_FASTCALL, "rpx_int4lora_forward_workspace"},
    {"int4lora_forward_multi", (PyCFunction)(void (*)(void))fast_int4lora_forward_multi,
     METH_FASTCALL, "rpx_int4lora_forward_multi"},
    {"int4lora_forward_multi_workspace",
     (PyCFunction)(void (*)(void))fast_int4lora_forward_multi_workspace, METH_FASTCALL,
     "rpx_int4lora_forward_multi_workspace"},
    {"mxfp4_linear", (PyCFunction)(void (*)(void))fast_mxfp4_linear, METH_FASTCALL,
     "rpx_mxfp4_linear"},
    {"mxfp4_gated", (PyCFunction)(void (*)(void))fast_mxfp4_gated, METH_FASTCALL,
     "rpx_mxfp4_gated"},
    {"mxfp4_quantize", (PyCFunction)(void (*)(void))fast_mxfp4_quantize, METH_FASTCALL,
     "rpx_mxfp4_quantize of one matrix"},
    {"mxfp4_dequantize", (PyCFunction)(void (*)(void))fast_mxfp4_dequantize, METH_FASTCALL,
     "rpx_mxfp4_dequantize"},
    {"mxfp4_linear_forward", (PyCFunction)(void (*)(void))fast_mxfp4_linear_forward,
     METH_FASTCALL, "rpx_mxfp4_linear_forward"},
    {"mxfp4_linear_backward", (PyCFunction)(void (*)(void))fast_mxfp4_linear_backward,
     METH_FASTCALL, "rpx_mxfp4_linear_backward"},
    {"mxfp4_gated_forward", (PyCFunction)(void (*)(void))fast_mxfp4_gated_forward, METH_FASTCALL,
     "rpx_mxfp4_gated_forward"},
    {"mxfp4_gated_backward_products", (PyCFunction)(void (*)(void))fast_mxfp4_gated_backward,
     METH_FASTCALL, "rpx_mxfp4_gated_backward_products"},
    {"mxfp4_bytes", (PyCFunction)(void (*)(void))fast_mxfp4_bytes, METH_FASTCALL,
     "the MXFP4 calls' buffer sizes"},
    {NULL, NULL, 0, NULL}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_rpxfast",
                                    "Fast-call binding of the small-M forward entry points.", -1,
                                    methods};

PyMODINIT_FUNC PyInit__rpxfast(void) { return PyModule_Create(&module); }

/* kh_pyops.c - the operator calls of a decoder layer (kuiperllama_amd/ops.py) from Python to the C-ABI without ctypes: checks of
 * the tensors, conversions and the call in one C function each.  A call through ctypes took 4.9 us on the host, 2.5 of them the
 * launch itself; a layer is 14 calls of kernels that run for 2 to 14 us each.
 *
 * Knows nothing of torch's C++ interface: tensors are asked through their Python attributes, as ops.py asked them.  The addresses
 * of the C-ABI's functions come from the ctypes handle (bind), so that there is one libkuiper_hip.so in a process. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <math.h>
#include <stdint.h>

#include "../../include/kuiper_hip.h"

static PyObject *s_dtype, *s_is_cuda, *s_is_contiguous, *s_data_ptr, *s_numel, *s_shape, *s_stride, *s_get_device;
/* from bind() */
static PyObject *o_f32, *o_i32, *o_i8, *o_tensor, *o_device, *o_raw_stream, *o_stream, *o_check, *o_arg_error;
static PyObject *o_bf16, *o_i64, *o_u8, *o_set_device;

typedef int (*add_fn)(const void*, const void*, void*, int32_t, void*);
typedef int (*matmul_fn)(const void*, const void*, void*, int32_t, int32_t, float, void*);
typedef int (*matmul_q8_fn)(const void*, const void*, const void*, int32_t, void*, int32_t, int32_t, void*);
typedef int (*rmsnorm_fn)(const void*, const void*, void*, int32_t, float, void*);
typedef int (*rope_fn)(int32_t, int32_t, int32_t, void*, void*, const void*, int32_t, const void*, const void*, int32_t, void*);
typedef int (*mha_fn)(const void*, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, int32_t, void*, const void*, void*, const void*,
                      const void*, void*);
static add_fn f_add, f_swiglu;
static matmul_fn f_matmul;
static matmul_q8_fn f_matmul_q8;
static rmsnorm_fn f_rmsnorm;
static rope_fn f_rope;
static mha_fn f_mha;
typedef int (*rope_tokens_fn)(const kh_rope_rows*, void*);
typedef int (*rope_store_fn)(const kh_rope_rows*, const void*, int64_t, int64_t, int32_t, const kh_page_cache*, const int32_t*, void*);
typedef int (*attn_packed_fn)(const kh_attn_rows*, const void*, int64_t, int64_t, const void*, int64_t, int64_t, void*);
typedef int (*attn_paged_fn)(const kh_attn_rows*, const kh_page_cache*, const int32_t*, int64_t, int32_t, const int32_t*, int32_t, void*, int64_t,
                             void*);
static rope_tokens_fn f_rope_tokens;
static rope_store_fn f_rope_store;
static attn_packed_fn f_attn_packed;
static attn_paged_fn f_attn_paged;

/* The address of a tensor on the GPU, contiguous and of the type; None: null.  0, or -1 with an exception. */
static int ptr(PyObject* t, PyObject* dtype, void** out) {
  *out = NULL;
  if (t == Py_None) return 0;
  PyObject* v = PyObject_GetAttr(t, s_is_cuda);
  if (!v) return -1;
  int yes = PyObject_IsTrue(v);
  Py_DECREF(v);
  if (yes < 0) return -1;
  if (!yes) {
    PyErr_SetString(PyExc_ValueError, "kuiperllama_amd.ops: tensors must be on the GPU (no CPU fallback)");
    return -1;
  }
  if (!(v = PyObject_VectorcallMethod(s_is_contiguous, &t, 1 | PY_VECTORCALL_ARGUMENTS_OFFSET, NULL))) return -1;
  yes = PyObject_IsTrue(v);
  Py_DECREF(v);
  if (yes < 0) return -1;
  if (!yes) {
    PyErr_SetString(PyExc_ValueError, "kuiperllama_amd.ops: tensors must be contiguous");
    return -1;
  }
  if (!(v = PyObject_GetAttr(t, s_dtype))) return -1;
  yes = v == dtype ? 1 : PyObject_RichCompareBool(v, dtype, Py_EQ);
  if (yes == 0) PyErr_Format(PyExc_TypeError, "expected %S, got %S", dtype, v);
  Py_DECREF(v);
  if (yes <= 0) return -1;
  if (!(v = PyObject_VectorcallMethod(s_data_ptr, &t, 1 | PY_VECTORCALL_ARGUMENTS_OFFSET, NULL))) return -1;
  *out = PyLong_AsVoidPtr(v);
  Py_DECREF(v);
  return *out == NULL && PyErr_Occurred() ? -1 : 0;
}
/* Numbers as ctypes takes them: integers masked to 32 bits, no floats for integers. */
static int wrong(const char* what) {
  PyErr_Clear();
  PyErr_Format(o_arg_error, "%s expected", what);
  return -1;
}
static int i32(PyObject* o, int32_t* out) {
  if (PyFloat_Check(o)) return wrong("int");
  const unsigned long v = PyLong_AsUnsignedLongMask(o);
  if (v == (unsigned long)-1 && PyErr_Occurred()) return wrong("int");
  *out = (int32_t)(uint32_t)v;
  return 0;
}
static int f32(PyObject* o, float* out) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) return wrong("float");
  *out = (float)v;
  return 0;
}
static int numel(PyObject* t, int32_t* out) {
  PyObject* v = PyObject_VectorcallMethod(s_numel, &t, 1 | PY_VECTORCALL_ARGUMENTS_OFFSET, NULL);
  if (!v) return -1;
  const int rc = i32(v, out);
  Py_DECREF(v);
  return rc;
}
/* rows and columns of a matrix */
static int shape2(PyObject* t, int32_t* rows, int32_t* cols) {
  PyObject* v = PyObject_GetAttr(t, s_shape);
  if (!v) return -1;
  int rc = -1;
  if (!PyTuple_Check(v) || PyTuple_GET_SIZE(v) != 2) PyErr_SetString(PyExc_ValueError, "a matrix is expected (two dimensions to unpack)");
  else rc = i32(PyTuple_GET_ITEM(v, 0), rows) || i32(PyTuple_GET_ITEM(v, 1), cols) ? -1 : 0;
  Py_DECREF(v);
  return rc;
}
/* torch's current stream of the current device */
static int stream(void** out) {
  PyObject* v;
  if (o_raw_stream != Py_None) {
    PyObject* d = PyObject_CallNoArgs(o_device);
    if (!d) return -1;
    v = PyObject_CallOneArg(o_raw_stream, d);
    Py_DECREF(d);
  } else {
    v = PyObject_CallNoArgs(o_stream);
  }
  if (!v) return -1;
  *out = PyLong_AsVoidPtr(v);
  Py_DECREF(v);
  return *out == NULL && PyErr_Occurred() ? -1 : 0;
}
/* a device tensor of one int32 or a number */
static int position(PyObject* o, void** d_pos, int32_t* pos) {
  *d_pos = NULL;
  *pos = 0;
  if (!PyLong_CheckExact(o)) {
    const int is = PyObject_IsInstance(o, o_tensor);
    if (is < 0) return -1;
    if (is) return ptr(o, o_i32, d_pos);
    PyObject* v = PyNumber_Long(o);
    if (!v) return -1;
    const int rc = i32(v, pos);
    Py_DECREF(v);
    return rc;
  }
  return i32(o, pos);
}
/* raises what the library reports, else returns a new reference to `out` */
static PyObject* done(int rc, const char* what, PyObject* out) {
  if (rc) {
    PyObject* v = PyObject_CallFunction(o_check, "is", rc, what);
    if (!v) return NULL;
    Py_DECREF(v);
  }
  Py_INCREF(out);
  return out;
}
static int count(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return 0;
  PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", want, n);
  return -1;
}
#define CALL(rc, ...)       \
  Py_BEGIN_ALLOW_THREADS    \
  rc = __VA_ARGS__;         \
  Py_END_ALLOW_THREADS

static PyObject* elementwise(PyObject* const* a, Py_ssize_t n, add_fn f, const char* name) {
  void *x, *y, *o, *s;
  int32_t len;
  int rc;
  if (count(n, 3) || ptr(a[0], o_f32, &x) || ptr(a[1], o_f32, &y) || ptr(a[2], o_f32, &o) || numel(a[0], &len) || stream(&s)) return NULL;
  CALL(rc, f(x, y, o, len, s))
  return done(rc, name, a[2]);
}
static PyObject* py_add(PyObject* m, PyObject* const* a, Py_ssize_t n) { return elementwise(a, n, f_add, "kh_add_f32"); }
static PyObject* py_swiglu(PyObject* m, PyObject* const* a, Py_ssize_t n) { return elementwise(a, n, f_swiglu, "kh_swiglu_f32"); }
static PyObject* py_matmul(PyObject* m, PyObject* const* a, Py_ssize_t n) { /* x, w, out, scale */
  void *x, *w, *o, *s;
  int32_t K, M;
  float scale;
  int rc;
  if (count(n, 4) || shape2(a[1], &K, &M) || ptr(a[0], o_f32, &x) || ptr(a[1], o_f32, &w) || ptr(a[2], o_f32, &o) || f32(a[3], &scale) ||
      stream(&s))
    return NULL;
  CALL(rc, f_matmul(x, w, o, M, K, scale, s))
  return done(rc, "kh_matmul_f32", a[2]);
}
static PyObject* py_matmul_q8(PyObject* m, PyObject* const* a, Py_ssize_t n) { /* x, w8, scales, group, out */
  void *x, *w, *sc, *o, *s;
  int32_t K, M, group;
  int rc;
  if (count(n, 5) || shape2(a[1], &K, &M) || ptr(a[0], o_f32, &x) || ptr(a[1], o_i8, &w) || ptr(a[2], o_f32, &sc) || i32(a[3], &group) ||
      ptr(a[4], o_f32, &o) || stream(&s))
    return NULL;
  CALL(rc, f_matmul_q8(x, w, sc, group, o, M, K, s))
  return done(rc, "kh_matmul_q8", a[4]);
}
static PyObject* py_rmsnorm(PyObject* m, PyObject* const* a, Py_ssize_t n) { /* x, w, out, eps */
  void *x, *w, *o, *s;
  int32_t len;
  float eps;
  int rc;
  if (count(n, 4) || ptr(a[0], o_f32, &x) || ptr(a[1], o_f32, &w) || ptr(a[2], o_f32, &o) || numel(a[0], &len) || f32(a[3], &eps) || stream(&s))
    return NULL;
  CALL(rc, f_rmsnorm(x, w, o, len, eps, s))
  return done(rc, "kh_rmsnorm_f32", a[2]);
}
static PyObject* py_rope(PyObject* m, PyObject* const* a, Py_ssize_t n) { /* q, k, pos, sin, cos, head_size, mode */
  void *q, *k, *d_pos, *sn, *cs, *s;
  int32_t pos, nq, nk, hs, mode;
  int rc;
  if (count(n, 7) || position(a[2], &d_pos, &pos) || numel(a[0], &nq) || numel(a[1], &nk) || i32(a[5], &hs) || ptr(a[0], o_f32, &q) ||
      ptr(a[1], o_f32, &k) || ptr(a[3], o_f32, &sn) || ptr(a[4], o_f32, &cs) || i32(a[6], &mode) || stream(&s))
    return NULL;
  CALL(rc, f_rope(nq, nk, hs, q, k, d_pos, pos, sn, cs, mode, s))
  return done(rc, "kh_rope_f32", Py_None);
}
/* pos, head_num, layer_index, seq_len, kv_dim, kv_mul, head_size, mha_out, q, score, kcache, vcache */
static PyObject* py_mha(PyObject* m, PyObject* const* a, Py_ssize_t n) {
  void *d_pos, *o, *q, *sc, *k, *v, *s;
  int32_t pos, i[6];
  int rc;
  if (count(n, 12) || position(a[0], &d_pos, &pos)) return NULL;
  for (int j = 0; j < 6; ++j)
    if (i32(a[1 + j], &i[j])) return NULL;
  if (ptr(a[7], o_f32, &o) || ptr(a[8], o_f32, &q) || ptr(a[9], o_f32, &sc) || ptr(a[10], o_f32, &k) || ptr(a[11], o_f32, &v) || stream(&s))
    return NULL;
  CALL(rc, f_mha(d_pos, pos, i[0], i[1], i[2], i[3], i[4], i[5], o, q, sc, k, v, s))
  return done(rc, "kh_mha_f32", a[7]);
}

/* ---- many tokens of several sequences ------------------------------------------------------------------------------- */
typedef struct {
  void* p;
  int dims;
  int64_t n[4], s[4];
} Rows;
static int numbers(PyObject* v, int dims, int64_t* out) {
  for (int i = 0; i < dims; ++i) {
    out[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(v, i));
    if (out[i] == -1 && PyErr_Occurred()) return -1;
  }
  return 0;
}
/* A tensor on *device (-1: not known yet) of the type and number of dimensions, the last one side by side. */
static int rows(PyObject* t, PyObject* dtype, int dims, int* device, const char* what, Rows* out) {
  PyObject* v = PyObject_VectorcallMethod(s_get_device, &t, 1 | PY_VECTORCALL_ARGUMENTS_OFFSET, NULL);
  if (!v) return -1;
  const long d = PyLong_AsLong(v);
  Py_DECREF(v);
  if (d == -1 && PyErr_Occurred()) return -1;
  if (d < 0) {
    PyErr_SetString(PyExc_ValueError, "kuiperllama_amd.ops: tensors must be on the GPU (no CPU fallback)");
    return -1;
  }
  if (*device < 0) *device = (int)d;
  if (*device != d) {
    PyErr_Format(PyExc_ValueError, "kuiperllama_amd.ops: tensors on device %d and %ld", *device, d);
    return -1;
  }
  if (!(v = PyObject_GetAttr(t, s_dtype))) return -1;
  int yes = v == dtype ? 1 : PyObject_RichCompareBool(v, dtype, Py_EQ);
  if (yes == 0) PyErr_Format(PyExc_TypeError, "%s: expected %S, got %S", what, dtype, v);
  Py_DECREF(v);
  if (yes <= 0) return -1;
  if (!(v = PyObject_GetAttr(t, s_shape))) return -1;
  yes = PyTuple_Check(v) && PyTuple_GET_SIZE(v) == dims;
  if (!yes) PyErr_Format(PyExc_ValueError, "%s: %d dimensions expected, got shape %S", what, dims, v);
  else yes = numbers(v, dims, out->n) ? 0 : 1;
  Py_DECREF(v);
  if (!yes) return -1;
  if (!(v = PyObject_VectorcallMethod(s_stride, &t, 1 | PY_VECTORCALL_ARGUMENTS_OFFSET, NULL))) return -1;
  yes = PyTuple_Check(v) && PyTuple_GET_SIZE(v) == dims && !numbers(v, dims, out->s);
  if (yes && out->n[dims - 1] > 1 && out->s[dims - 1] != 1) {
    PyErr_Format(PyExc_ValueError, "%s: the last dimension has to be contiguous, got strides %S", what, v);
    yes = 0;
  }
  Py_DECREF(v);
  if (!yes) {
    if (!PyErr_Occurred()) PyErr_Format(PyExc_ValueError, "%s: strides expected", what);
    return -1;
  }
  if (!(v = PyObject_VectorcallMethod(s_data_ptr, &t, 1 | PY_VECTORCALL_ARGUMENTS_OFFSET, NULL))) return -1;
  out->p = PyLong_AsVoidPtr(v);
  out->dims = dims;
  Py_DECREF(v);
  return out->p == NULL && PyErr_Occurred() ? -1 : 0;
}
/* bfloat16 or float32, as the C-ABI calls it; *dtype borrowed */
static int storage(PyObject* t, PyObject** dtype, int32_t* code) {
  PyObject* v = PyObject_GetAttr(t, s_dtype);
  if (!v) return -1;
  *code = v == o_bf16 ? KH_DTYPE_BF16 : (v == o_f32 ? KH_DTYPE_F32 : -1);
  *dtype = v == o_bf16 ? o_bf16 : o_f32;
  if (*code < 0) PyErr_Format(PyExc_TypeError, "expected bfloat16 or float32, got %S", v);
  Py_DECREF(v);
  return *code < 0 ? -1 : 0;
}
static int sizes(const char* what, const Rows* r, const int64_t* want) {
  for (int i = 0; i < r->dims; ++i)
    if (r->n[i] != want[i]) {
      PyErr_Format(PyExc_ValueError, "%s: %lld expected in dimension %d, got %lld", what, (long long)want[i], i, (long long)r->n[i]);
      return -1;
    }
  return 0;
}
static int fits(int64_t n, int32_t* out) {
  *out = (int32_t)n;
  if (*out == n) return 0;
  PyErr_Format(PyExc_ValueError, "%lld is more than the library counts", (long long)n);
  return -1;
}
/* torch's current stream of a device; *before: the device to go back to, where it is another */
static int enter(int device, void** out, long* before) {
  PyObject *v, *d = PyObject_CallNoArgs(o_device);
  if (!d) return -1;
  *before = PyLong_AsLong(d);
  if (*before == -1 && PyErr_Occurred()) {
    Py_DECREF(d);
    return -1;
  }
  if (*before == device) {
    *before = -1;
  } else {
    Py_DECREF(d);
    if (!(d = PyLong_FromLong(device))) return -1;
    if (!(v = PyObject_CallOneArg(o_set_device, d))) {
      Py_DECREF(d);
      return -1;
    }
    Py_DECREF(v);
  }
  v = o_raw_stream != Py_None ? PyObject_CallOneArg(o_raw_stream, d) : PyObject_CallNoArgs(o_stream);
  Py_DECREF(d);
  if (!v) return -1;
  *out = PyLong_AsVoidPtr(v);
  Py_DECREF(v);
  return *out == NULL && PyErr_Occurred() ? -1 : 0;
}
static int leave(long before) {
  if (before < 0) return 0;
  PyObject *t, *e, *tb, *d = PyLong_FromLong(before), *v = NULL;
  PyErr_Fetch(&t, &e, &tb);
  if (d) v = PyObject_CallOneArg(o_set_device, d);
  Py_XDECREF(d);
  Py_XDECREF(v);
  if (t) PyErr_Restore(t, e, tb);
  return PyErr_Occurred() ? -1 : 0;
}
/* the call on the tensors' device and its current stream */
#define ON_DEVICE(rc, device, ...)                       \
  {                                                      \
    long before = -1;                                    \
    int ok = !enter(device, &s, &before);                \
    if (ok) {                                            \
      CALL(rc, __VA_ARGS__)                              \
    }                                                    \
    if (leave(before) || !ok) return NULL;               \
  }

/* q, k, positions, turns, rot_dim, magnitude, mode, q_out, k_out (None: not wanted) from a[0] on */
static int rope_rows(PyObject* const* a, kh_rope_rows* r, PyObject** dtype, int* device) {
  Rows q, k, p, t, qo, ko;
  float mag;
  *device = -1;
  if (storage(a[0], dtype, &r->dtype) || rows(a[0], *dtype, 3, device, "q", &q) || rows(a[1], *dtype, 3, device, "k", &k) ||
      rows(a[2], o_i32, 1, device, "positions", &p) || rows(a[3], o_i64, 1, device, "table", &t) || i32(a[4], &r->rot_dim) || f32(a[5], &mag) ||
      i32(a[6], &r->mode) || rows(a[7], *dtype, 3, device, "q_out", &qo))
    return -1;
  const int64_t kn[3] = {q.n[0], k.n[1], q.n[2]}, pairs = r->rot_dim / 2;
  if (sizes("k", &k, kn) || sizes("positions", &p, q.n) || sizes("table", &t, &pairs) || sizes("q_out", &qo, q.n) || fits(q.n[0], &r->n_tokens) ||
      fits(q.n[1], &r->head_num) || fits(k.n[1], &r->kv_head_num) || fits(q.n[2], &r->head_size))
    return -1;
  r->magnitude = mag;
  r->turns = t.p;
  r->positions = p.p;
  r->q = q.p;
  r->k = k.p;
  r->q_out = qo.p;
  r->q_token = q.s[0], r->q_head = q.s[1], r->k_token = k.s[0], r->k_head = k.s[1], r->qo_token = qo.s[0], r->qo_head = qo.s[1];
  r->k_out = NULL;
  r->ko_token = r->ko_head = 0;
  if (a[8] != Py_None) {
    if (rows(a[8], *dtype, 3, device, "k_out", &ko) || sizes("k_out", &ko, k.n)) return -1;
    r->k_out = ko.p;
    r->ko_token = ko.s[0], r->ko_head = ko.s[1];
  }
  return 0;
}
static int page_cache(PyObject* kc, PyObject* vc, PyObject* dtype, int* device, kh_page_cache* c, Rows* k, Rows* v) {
  if (rows(kc, dtype, 4, device, "kcache", k) || rows(vc, dtype, 4, device, "vcache", v)) return -1;
  const int64_t vn[4] = {k->n[0], k->n[1], k->n[2], v->n[3]};
  if (sizes("vcache", v, vn) || fits(k->n[0], &c->n_pages) || fits(k->n[1], &c->page_size)) return -1;
  c->k = k->p;
  c->v = v->p;
  c->k_page = k->s[0], c->k_slot = k->s[1], c->k_head = k->s[2], c->v_page = v->s[0], c->v_slot = v->s[1], c->v_head = v->s[2];
  return 0;
}
static PyObject* py_rope_tokens(PyObject* m, PyObject* const* a, Py_ssize_t n) {
  kh_rope_rows r;
  PyObject* dtype;
  void* s;
  int rc = 0, device;
  if (count(n, 9) || rope_rows(a, &r, &dtype, &device)) return NULL;
  ON_DEVICE(rc, device, f_rope_tokens(&r, s))
  return done(rc, "kh_rope_tokens", Py_None);
}
/* ... None, v, kcache, vcache, slots */
static PyObject* py_rope_store(PyObject* m, PyObject* const* a, Py_ssize_t n) {
  kh_rope_rows r;
  kh_page_cache c;
  Rows v, kc, vc, sl;
  PyObject* dtype;
  void* s;
  int rc = 0, device;
  int32_t size;
  if (count(n, 13) || rope_rows(a, &r, &dtype, &device) || rows(a[9], dtype, 3, &device, "v", &v) ||
      page_cache(a[10], a[11], dtype, &device, &c, &kc, &vc) || rows(a[12], o_i32, 1, &device, "slots", &sl))
    return NULL;
  const int64_t vn[3] = {r.n_tokens, r.kv_head_num, vc.n[3]}, kn[4] = {kc.n[0], kc.n[1], r.kv_head_num, r.head_size}, tokens = r.n_tokens;
  if (sizes("v", &v, vn) || sizes("kcache", &kc, kn) || sizes("slots", &sl, &tokens) || fits(v.n[2], &size)) return NULL;
  ON_DEVICE(rc, device, f_rope_store(&r, v.p, v.s[0], v.s[1], size, &c, sl.p, s))
  return done(rc, "kh_rope_store", a[7]);
}
/* q, offsets, out, scale (None: 1 / sqrt(size)), window from a[0] on */
static int attn_rows(PyObject* const* a, kh_attn_rows* r, PyObject** dtype, int* device, int64_t* q_n) {
  Rows q, o, t;
  *device = -1;
  if (storage(a[0], dtype, &r->dtype) || rows(a[0], *dtype, 3, device, "q", &q) || rows(a[1], o_i32, 1, device, "offsets", &o) ||
      rows(a[2], *dtype, 3, device, "out", &t) || i32(a[4], &r->window))
    return -1;
  if (a[3] == Py_None) r->scale = q.n[2] > 0 ? (float)(1.0 / sqrt((double)q.n[2])) : 1.f;
  else if (f32(a[3], &r->scale)) return -1;
  if (fits(q.n[0], &r->n_tokens) || fits(q.n[1], &r->head_num) || fits(q.n[2], &r->head_size) || fits(o.n[0] - 1, &r->n_seqs) ||
      fits(t.n[2], &r->value_size))
    return -1;
  const int64_t on[3] = {q.n[0], q.n[1], t.n[2]};
  if (sizes("out", &t, on)) return -1;
  r->offsets = o.p;
  r->q = q.p;
  r->out = t.p;
  r->q_token = q.s[0], r->q_head = q.s[1], r->o_token = t.s[0], r->o_head = t.s[1];
  for (int i = 0; i < 3; ++i) q_n[i] = q.n[i];
  return 0;
}
/* ..., k, v */
static PyObject* py_attn_packed(PyObject* m, PyObject* const* a, Py_ssize_t n) {
  kh_attn_rows r;
  Rows k, v;
  PyObject* dtype;
  void* s;
  int rc = 0, device;
  int64_t q[3];
  if (count(n, 7) || attn_rows(a, &r, &dtype, &device, q) || rows(a[5], dtype, 3, &device, "k", &k) || rows(a[6], dtype, 3, &device, "v", &v))
    return NULL;
  const int64_t kn[3] = {q[0], k.n[1], q[2]}, vn[3] = {q[0], k.n[1], r.value_size};
  if (sizes("k", &k, kn) || sizes("v", &v, vn) || fits(k.n[1], &r.kv_head_num)) return NULL;
  ON_DEVICE(rc, device, f_attn_packed(&r, k.p, k.s[0], k.s[1], v.p, v.s[0], v.s[1], s))
  return done(rc, "kh_attn_packed", a[2]);
}
/* ..., kcache, vcache, pages, lengths, workspace, max_new */
static PyObject* py_attn_paged(PyObject* m, PyObject* const* a, Py_ssize_t n) {
  kh_attn_rows r;
  kh_page_cache c;
  Rows kc, vc, p, l, w;
  PyObject* dtype;
  void* s;
  int rc = 0, device;
  int64_t q[3];
  int32_t width, most;
  if (count(n, 11) || attn_rows(a, &r, &dtype, &device, q) || page_cache(a[5], a[6], dtype, &device, &c, &kc, &vc) ||
      rows(a[7], o_i32, 2, &device, "pages", &p) || rows(a[8], o_i32, 1, &device, "lengths", &l) || rows(a[9], o_u8, 1, &device, "workspace", &w) ||
      i32(a[10], &most))
    return NULL;
  const int64_t kn[4] = {kc.n[0], kc.n[1], kc.n[2], q[2]}, vn[4] = {kc.n[0], kc.n[1], kc.n[2], r.value_size}, seqs = r.n_seqs, pn[2] = {seqs, p.n[1]};
  if (sizes("kcache", &kc, kn) || sizes("vcache", &vc, vn) || sizes("pages", &p, pn) || sizes("lengths", &l, &seqs) || fits(kc.n[2], &r.kv_head_num) ||
      fits(p.n[1], &width))
    return NULL;
  ON_DEVICE(rc, device, f_attn_paged(&r, &c, p.p, p.s[0], width, l.p, most, w.p, w.n[0], s))
  return done(rc, "kh_attn_paged", a[2]);
}

static void keep(PyObject** at, PyObject* o) {
  Py_INCREF(o);
  Py_XSETREF(*at, o);
}
/* (addresses: add, swiglu, matmul, matmul_q8, rmsnorm, rope, mha, rope_tokens, rope_store, attn_packed, attn_paged), (float32, int32,
 * int8, Tensor, current device, raw stream of a device or None, current stream, check, ctypes.ArgumentError, bfloat16, int64, uint8,
 * set device) */
static PyObject* py_bind(PyObject* m, PyObject* const* a, Py_ssize_t n) {
  enum { CALLS = 11, OBJECTS = 13 };
  void* p[CALLS];
  PyObject** o[OBJECTS] = {&o_f32, &o_i32, &o_i8, &o_tensor, &o_device, &o_raw_stream, &o_stream, &o_check, &o_arg_error,
                           &o_bf16, &o_i64, &o_u8, &o_set_device};
  if (count(n, 2)) return NULL;
  if (!PyTuple_Check(a[0]) || PyTuple_GET_SIZE(a[0]) != CALLS || !PyTuple_Check(a[1]) || PyTuple_GET_SIZE(a[1]) != OBJECTS) {
    PyErr_SetString(PyExc_TypeError, "eleven addresses and thirteen objects are expected");
    return NULL;
  }
  for (int j = 0; j < CALLS; ++j) {
    p[j] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(a[0], j));
    if (!p[j]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "an address is null");
      return NULL;
    }
  }
  f_add = (add_fn)p[0];
  f_swiglu = (add_fn)p[1];
  f_matmul = (matmul_fn)p[2];
  f_matmul_q8 = (matmul_q8_fn)p[3];
  f_rmsnorm = (rmsnorm_fn)p[4];
  f_rope = (rope_fn)p[5];
  f_mha = (mha_fn)p[6];
  f_rope_tokens = (rope_tokens_fn)p[7];
  f_rope_store = (rope_store_fn)p[8];
  f_attn_packed = (attn_packed_fn)p[9];
  f_attn_paged = (attn_paged_fn)p[10];
  for (int j = 0; j < OBJECTS; ++j) keep(o[j], PyTuple_GET_ITEM(a[1], j));
  Py_RETURN_NONE;
}

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))py_##name, METH_FASTCALL, NULL}
static PyMethodDef methods[] = {METHOD(bind), METHOD(add),  METHOD(swiglu), METHOD(matmul), METHOD(matmul_q8),
                                METHOD(rmsnorm), METHOD(rope), METHOD(mha), METHOD(rope_tokens),
                                METHOD(rope_store), METHOD(attn_packed), METHOD(attn_paged), {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "kh_pyops", NULL, -1, methods};
PyMODINIT_FUNC PyInit_kh_pyops(void) {
  s_dtype = PyUnicode_InternFromString("dtype");
  s_is_cuda = PyUnicode_InternFromString("is_cuda");
  s_is_contiguous = PyUnicode_InternFromString("is_contiguous");
  s_data_ptr = PyUnicode_InternFromString("data_ptr");
  s_numel = PyUnicode_InternFromString("numel");
  s_shape = PyUnicode_InternFromString("shape");
  s_stride = PyUnicode_InternFromString("stride");
  s_get_device = PyUnicode_InternFromString("get_device");
  if (!s_dtype || !s_is_cuda || !s_is_contiguous || !s_data_ptr || !s_numel || !s_shape || !s_stride || !s_get_device) return NULL;
  return PyModule_Create(&module);
}

/* The per-layer calls of AttnEngine without ctypes: reads pointers and strides from the tensors and calls the C ABI.
 *
 * A decode step is one call per layer, and while the GPU spends 6 to 10 us on a layer of a short context, ctypes' conversion of
 * 18 arguments, the tensors' accessors as Python calls and the stream object took 7 us of host time before the library
 * was entered.  Here the accessors are vectorcalls on interned names and the arguments plain C values.
 * An integer that does not fit its parameter is refused with the package's PaError (ctypes would wrap it); the GIL is released for the call. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>
#include <stdlib.h>

#include "../../include/pooled_attn.h"

typedef int (*fn_attn_layer)(pa_layer*, uint32_t, uint32_t, uint32_t, int, const void*, uint64_t, uint64_t, const void*, const void*, uint64_t, const void*,
                             uint64_t, uint64_t, const float*, void*, uint64_t, void*);
typedef int (*fn_attn_items)(pa_layer*, const pa_item*, uint32_t, const void*, uint64_t, uint64_t, const void*, const void*, uint64_t, const void*, uint64_t,
                             uint64_t, void*, uint64_t, int, void*);
typedef int (*fn_rope_append)(pa_layer*, uint32_t, uint32_t, uint32_t, const void*, uint64_t, uint64_t, const void*, const void*, uint64_t, const float*, float*,
                              void*);
typedef int (*fn_decode_gather)(pa_layer*, uint32_t, uint32_t, const uint32_t*, uint32_t, const void*, int, uint64_t, uint64_t, const void*, uint64_t,
                                uint64_t, void*, uint64_t, void*);
typedef int (*fn_rotary_apply)(pa_rotary*, const void*, int, uint64_t, uint64_t, uint32_t, const int32_t*, int32_t, uint32_t, void*, int, uint64_t, uint64_t, void*);
typedef int (*fn_rotary_append)(pa_rotary*, pa_layer*, const pa_item*, uint32_t, const uint32_t*, const void*, uint64_t, uint64_t, const void*, const void*, uint64_t,
                                void*, int, uint64_t, void*);
typedef int (*fn_decode_shared)(pa_layer*, pa_layer*, uint32_t, uint32_t, uint32_t, const pa_item*, uint32_t, const void*, int, uint64_t, uint64_t, const void*,
                                uint64_t, uint64_t, void*, uint64_t, void*);
typedef int (*fn_decode_weights)(pa_layer*, const pa_item*, uint32_t, const void*, int, uint64_t, uint64_t, const void*, uint64_t, uint64_t, void*, uint64_t, void*);
typedef int (*fn_evict)(pa_layer*, const pa_evict_item*, uint32_t, uint32_t, uint32_t, uint32_t, uint32_t*, void*);
/* Every call names the entry point (its address in the library the engine loaded) as its first argument: the module keeps
 * nothing of its own. */
static PyObject *s_data_ptr, *s_stride, *s_size, *i_zero;

static int ptr_of(PyObject* t, void** p) {
  if (t == Py_None) { *p = NULL; return 0; }
  PyObject* r = PyObject_VectorcallMethod(s_data_ptr, &t, 1 | PY_VECTORCALL_ARGUMENTS_OFFSET, NULL);
  if (!r) return -1;
  *p = (void*)(uintptr_t)PyLong_AsUnsignedLongLongMask(r);
  Py_DECREF(r);
  return PyErr_Occurred() ? -1 : 0;
}
static int stride0(PyObject* t, uint64_t* s) {
  PyObject* a[2] = {t, i_zero};
  PyObject* r = PyObject_VectorcallMethod(s_stride, a, 2 | PY_VECTORCALL_ARGUMENTS_OFFSET, NULL);
  if (!r) return -1;
  *s = (uint64_t)PyLong_AsUnsignedLongLongMask(r);
  Py_DECREF(r);
  return PyErr_Occurred() ? -1 : 0;
}
/* PaError(-1, ...) of pooled_b200.lib, as a refused call raises */
static int does_not_fit(PyObject* o, const char* what) {
  PyErr_Clear();
  PyObject *lib = PyImport_ImportModule("pooled_b200.lib"), *cls = lib ? PyObject_GetAttrString(lib, "PaError") : NULL;
  PyObject *msg = cls ? PyUnicode_FromFormat("%R is no %s", o, what) : NULL, *err = msg ? PyObject_CallFunction(cls, "iO", -1, msg) : NULL;
  if (err) PyErr_SetObject(cls, err);
  Py_XDECREF(err); Py_XDECREF(msg); Py_XDECREF(cls); Py_XDECREF(lib);
  return -1;
}
/* an integer of [lo, hi] */
static int int_of(PyObject* o, int64_t lo, int64_t hi, const char* what, int64_t* v) {
  int over;
  *v = PyLong_AsLongLongAndOverflow(o, &over);
  if (over || *v < lo || *v > hi) return !over && *v == -1 && PyErr_Occurred() ? -1 : does_not_fit(o, what);
  return *v == -1 && PyErr_Occurred() ? -1 : 0;
}
static int u64_of(PyObject* o, uint64_t* v) {
  int over;
  const long long x = PyLong_AsLongLongAndOverflow(o, &over);
  if (over <= 0 && x < 0) return !over && PyErr_Occurred() ? -1 : does_not_fit(o, "unsigned 64-bit integer");
  *v = over ? PyLong_AsUnsignedLongLong(o) : (uint64_t)x;
  return over && PyErr_Occurred() ? does_not_fit(o, "unsigned 64-bit integer") : 0;
}
static int u32_of(PyObject* o, uint32_t* v) {
  int64_t x;
  if (int_of(o, 0, UINT32_MAX, "unsigned 32-bit integer", &x)) return -1;
  *v = (uint32_t)x;
  return 0;
}
static int i32_of(PyObject* o, int32_t* v) {
  int64_t x;
  if (int_of(o, INT32_MIN, INT32_MAX, "32-bit integer", &x)) return -1;
  *v = (int32_t)x;
  return 0;
}
static int rows_of(PyObject* t, uint32_t* n) {
  PyObject* a[2] = {t, i_zero};
  PyObject* r = PyObject_VectorcallMethod(s_size, a, 2 | PY_VECTORCALL_ARGUMENTS_OFFSET, NULL);
  if (!r) return -1;
  const int bad = u32_of(r, n);
  Py_DECREF(r);
  return bad;
}
static int args_are(Py_ssize_t n, Py_ssize_t want, const char* who) {
  if (n == want) return 0;
  PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", who, want, n);
  return -1;
}

/* attn_layer(entry, layer, seq, pos, mode, q, q_head_stride, k, v, gate, gate_head_stride, cs_table, out, stream) -> status */
static PyObject* attn_layer(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  uint64_t fn, layer, qcs, qhs, kcs, gcs = 0, ghs = 0, ocs, stream;
  uint32_t seq, pos, mode, cols;
  void *q, *k, *v, *g, *cs, *out;
  (void)self;
  if (args_are(n, 14, "attn_layer") || u64_of(a[0], &fn) || u64_of(a[1], &layer) || u32_of(a[2], &seq) || u32_of(a[3], &pos) || u32_of(a[4], &mode) || rows_of(a[5], &cols) ||
      ptr_of(a[5], &q) || stride0(a[5], &qcs) || u64_of(a[6], &qhs) || ptr_of(a[7], &k) || stride0(a[7], &kcs) || ptr_of(a[8], &v) || ptr_of(a[9], &g) ||
      (a[9] != Py_None && (stride0(a[9], &gcs) || u64_of(a[10], &ghs))) || ptr_of(a[11], &cs) || ptr_of(a[12], &out) || stride0(a[12], &ocs) ||
      u64_of(a[13], &stream))
    return NULL;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = ((fn_attn_layer)(uintptr_t)fn)((pa_layer*)(uintptr_t)layer, seq, pos, cols, (int)mode, q, qcs, qhs, k, v, kcs, g, gcs, ghs, (const float*)cs, out, ocs,
                    (void*)(uintptr_t)stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

/* attn_items(entry, layer, [(seq, pos)], q, q_head_stride, k, v, gate, gate_head_stride, out, exchange, stream) -> status */
static PyObject* attn_items(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  uint64_t fn, layer, qcs, qhs, kcs, gcs = 0, ghs = 0, ocs, stream;
  uint32_t exch;
  void *q, *k, *v, *g, *out;
  (void)self;
  if (args_are(n, 12, "attn_items") || u64_of(a[0], &fn) || u64_of(a[1], &layer) || ptr_of(a[3], &q) || stride0(a[3], &qcs) || u64_of(a[4], &qhs) || ptr_of(a[5], &k) ||
      stride0(a[5], &kcs) || ptr_of(a[6], &v) || ptr_of(a[7], &g) || (a[7] != Py_None && (stride0(a[7], &gcs) || u64_of(a[8], &ghs))) || ptr_of(a[9], &out) ||
      stride0(a[9], &ocs) || u32_of(a[10], &exch) || u64_of(a[11], &stream))
    return NULL;
  PyObject* list = PySequence_Fast(a[2], "the items are a sequence of (seq, pos) pairs");
  if (!list) return NULL;
  const Py_ssize_t cnt = PySequence_Fast_GET_SIZE(list);
  pa_item* items = (pa_item*)calloc((size_t)(cnt ? cnt : 1), sizeof(pa_item));
  if (!items) { Py_DECREF(list); return PyErr_NoMemory(); }
  for (Py_ssize_t i = 0; i < cnt; ++i) {
    PyObject* pr = PySequence_Fast(PySequence_Fast_GET_ITEM(list, i), "an item is a (seq, pos) pair");
    int bad = !pr;
    if (pr && PySequence_Fast_GET_SIZE(pr) != 2) { PyErr_SetString(PyExc_ValueError, "an item is a (seq, pos) pair"); bad = 1; }
    bad = bad || u32_of(PySequence_Fast_GET_ITEM(pr, 0), &items[i].seq) || u32_of(PySequence_Fast_GET_ITEM(pr, 1), &items[i].pos);
    Py_XDECREF(pr);
    if (bad) { free(items); Py_DECREF(list); return NULL; }
    items[i].n_cols = 1;
  }
  Py_DECREF(list);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = ((fn_attn_items)(uintptr_t)fn)((pa_layer*)(uintptr_t)layer, items, (uint32_t)cnt, q, qcs, qhs, k, v, kcs, g, gcs, ghs, out, ocs, (int)exch, (void*)(uintptr_t)stream);
  Py_END_ALLOW_THREADS
  free(items);
  return PyLong_FromLong(rc);
}

/* rope_append(entry, layer, seq, pos, q, q_head_stride, k, v, cs_table, q_rot, stream) -> status */
static PyObject* rope_append(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  uint64_t fn, layer, qcs, qhs, kcs, stream;
  uint32_t seq, pos, cols;
  void *q, *k, *v, *cs, *qr;
  (void)self;
  if (args_are(n, 11, "rope_append") || u64_of(a[0], &fn) || u64_of(a[1], &layer) || u32_of(a[2], &seq) || u32_of(a[3], &pos) || rows_of(a[4], &cols) || ptr_of(a[4], &q) ||
      stride0(a[4], &qcs) || u64_of(a[5], &qhs) || ptr_of(a[6], &k) || stride0(a[6], &kcs) || ptr_of(a[7], &v) || ptr_of(a[8], &cs) || ptr_of(a[9], &qr) ||
      u64_of(a[10], &stream))
    return NULL;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = ((fn_rope_append)(uintptr_t)fn)((pa_layer*)(uintptr_t)layer, seq, pos, cols, q, qcs, qhs, k, v, kcs, (const float*)cs, (float*)qr, (void*)(uintptr_t)stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

/* decode_gather(entry, layer, seq, lists, list_stride, q, q_dtype, q_head_stride, gate, gate_head_stride, out, stream) -> status */
static PyObject* decode_gather(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  uint64_t fn, layer, qcs, qhs, gcs = 0, ghs = 0, ocs, stream;
  uint32_t seq, list_stride, cols, qdt;
  void *lists, *q, *g, *out;
  (void)self;
  if (args_are(n, 12, "decode_gather") || u64_of(a[0], &fn) || u64_of(a[1], &layer) || u32_of(a[2], &seq) || ptr_of(a[3], &lists) || u32_of(a[4], &list_stride) ||
      rows_of(a[5], &cols) || ptr_of(a[5], &q) || u32_of(a[6], &qdt) || stride0(a[5], &qcs) || u64_of(a[7], &qhs) || ptr_of(a[8], &g) ||
      (a[8] != Py_None && (stride0(a[8], &gcs) || u64_of(a[9], &ghs))) || ptr_of(a[10], &out) || stride0(a[10], &ocs) || u64_of(a[11], &stream))
    return NULL;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = ((fn_decode_gather)(uintptr_t)fn)((pa_layer*)(uintptr_t)layer, seq, cols, (const uint32_t*)lists, list_stride, q, (int)qdt, qcs, qhs, g, gcs, ghs, out, ocs,
                       (void*)(uintptr_t)stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

/* a sequence of `width`-tuples of integers as `width` words each of a four-word struct, the others `rest`; NULL with an error set.  Freed by the caller. */
static uint32_t* words_of(PyObject* o, Py_ssize_t width, uint32_t rest, const char* what, Py_ssize_t* cnt) {
  PyObject* list = PySequence_Fast(o, what);
  if (!list) return NULL;
  *cnt = PySequence_Fast_GET_SIZE(list);
  uint32_t* w = (uint32_t*)calloc((size_t)(*cnt ? *cnt : 1) * 4, sizeof(uint32_t));
  if (!w) { Py_DECREF(list); PyErr_NoMemory(); return NULL; }
  for (Py_ssize_t i = 0; i < *cnt; ++i) {
    PyObject* t = PySequence_Fast(PySequence_Fast_GET_ITEM(list, i), what);
    int bad = !t;
    if (t && PySequence_Fast_GET_SIZE(t) != width) { PyErr_SetString(PyExc_ValueError, what); bad = 1; }
    for (Py_ssize_t k = 0; !bad && k < width; ++k) bad = u32_of(PySequence_Fast_GET_ITEM(t, k), &w[4 * i + k]);
    Py_XDECREF(t);
    if (bad) { free(w); Py_DECREF(list); return NULL; }
    if (width == 2) w[4 * i + 2] = rest;
  }
  Py_DECREF(list);
  return w;
}
static const char* const kPairs = "the items are a sequence of (seq, pos) pairs";
static const char* const kTriples = "the items are a sequence of triples";

/* rotary_apply(entry, rotary, x, x_dtype, head_stride, n_heads, positions, pos, y, y_dtype, y_head_stride, stream) -> status */
static PyObject* rotary_apply(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  uint64_t fn, rot, xcs, xhs, ycs, yhs, stream;
  uint32_t xdt, ydt, heads, cols;
  int32_t pos;
  void *x, *ps, *y;
  (void)self;
  if (args_are(n, 12, "rotary_apply") || u64_of(a[0], &fn) || u64_of(a[1], &rot) || ptr_of(a[2], &x) || stride0(a[2], &xcs) || rows_of(a[2], &cols) || u32_of(a[3], &xdt) ||
      u64_of(a[4], &xhs) || u32_of(a[5], &heads) || ptr_of(a[6], &ps) || i32_of(a[7], &pos) || ptr_of(a[8], &y) || stride0(a[8], &ycs) || u32_of(a[9], &ydt) ||
      u64_of(a[10], &yhs) || u64_of(a[11], &stream))
    return NULL;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = ((fn_rotary_apply)(uintptr_t)fn)((pa_rotary*)(uintptr_t)rot, x, (int)xdt, xcs, xhs, heads, (const int32_t*)ps, pos, cols, y, (int)ydt, ycs, yhs,
                    (void*)(uintptr_t)stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

/* rotary_append(entry, rotary, layer, [(seq, pos, n_cols)], rows, q, q_head_stride, k, v, q_out, q_out_dtype, stream) -> status */
static PyObject* rotary_append(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  uint64_t fn, rot, layer, qcs = 0, qhs = 0, kcs, ocs = 0, stream;
  uint32_t odt;
  void *q, *k, *v, *o;
  (void)self;
  if (args_are(n, 12, "rotary_append") || u64_of(a[0], &fn) || u64_of(a[1], &rot) || u64_of(a[2], &layer) || ptr_of(a[5], &q) ||
      (a[5] != Py_None && (stride0(a[5], &qcs) || u64_of(a[6], &qhs))) || ptr_of(a[7], &k) || stride0(a[7], &kcs) || ptr_of(a[8], &v) || ptr_of(a[9], &o) ||
      (a[9] != Py_None && stride0(a[9], &ocs)) || u32_of(a[10], &odt) || u64_of(a[11], &stream))
    return NULL;
  Py_ssize_t cnt, nr = 0;
  uint32_t *items = words_of(a[3], 3, 0, kTriples, &cnt), *rows = NULL;
  if (!items) return NULL;
  if (a[4] != Py_None) {
    PyObject* list = PySequence_Fast(a[4], "the rows are a sequence of integers");
    int bad = !list;
    if (list) {
      nr = PySequence_Fast_GET_SIZE(list);
      if (nr != cnt) { PyErr_SetString(PyExc_ValueError, "one row per item"); bad = 1; }
      rows = bad ? NULL : (uint32_t*)calloc((size_t)(nr ? nr : 1), sizeof(uint32_t));
      if (!bad && !rows) { PyErr_NoMemory(); bad = 1; }
      for (Py_ssize_t i = 0; !bad && i < nr; ++i) bad = u32_of(PySequence_Fast_GET_ITEM(list, i), &rows[i]);
      Py_DECREF(list);
    }
    if (bad) { free(rows); free(items); return NULL; }
  }
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = ((fn_rotary_append)(uintptr_t)fn)((pa_rotary*)(uintptr_t)rot, (pa_layer*)(uintptr_t)layer, (const pa_item*)items, (uint32_t)cnt, rows, q, qcs, qhs, k, v, kcs, o,
                    (int)odt, ocs, (void*)(uintptr_t)stream);
  Py_END_ALLOW_THREADS
  free(rows); free(items);
  return PyLong_FromLong(rc);
}

/* decode_shared(entry, layer, prefix_layer, prefix_seq, prefix_len, own_base, [(seq, pos)], q, q_dtype, q_head_stride, gate, gate_head_stride, out, stream) -> status */
static PyObject* decode_shared(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  uint64_t fn, layer, pre, qcs, qhs, gcs = 0, ghs = 0, ocs, stream;
  uint32_t seq, len, base, qdt;
  void *q, *g, *out;
  (void)self;
  if (args_are(n, 14, "decode_shared") || u64_of(a[0], &fn) || u64_of(a[1], &layer) || u64_of(a[2], &pre) || u32_of(a[3], &seq) || u32_of(a[4], &len) || u32_of(a[5], &base) ||
      ptr_of(a[7], &q) || stride0(a[7], &qcs) || u32_of(a[8], &qdt) || u64_of(a[9], &qhs) || ptr_of(a[10], &g) ||
      (a[10] != Py_None && (stride0(a[10], &gcs) || u64_of(a[11], &ghs))) || ptr_of(a[12], &out) || stride0(a[12], &ocs) || u64_of(a[13], &stream))
    return NULL;
  Py_ssize_t cnt;
  uint32_t* items = words_of(a[6], 2, 1, kPairs, &cnt);
  if (!items) return NULL;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = ((fn_decode_shared)(uintptr_t)fn)((pa_layer*)(uintptr_t)layer, (pa_layer*)(uintptr_t)pre, seq, len, base, (const pa_item*)items, (uint32_t)cnt, q, (int)qdt, qcs,
                    qhs, g, gcs, ghs, out, ocs, (void*)(uintptr_t)stream);
  Py_END_ALLOW_THREADS
  free(items);
  return PyLong_FromLong(rc);
}

/* decode_weights(entry, layer, [(seq, pos)], q, q_dtype, q_head_stride, gate, gate_head_stride, out, stream) -> status */
static PyObject* decode_weights(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  uint64_t fn, layer, qcs, qhs, gcs = 0, ghs = 0, ocs, stream;
  uint32_t qdt;
  void *q, *g, *out;
  (void)self;
  if (args_are(n, 10, "decode_weights") || u64_of(a[0], &fn) || u64_of(a[1], &layer) || ptr_of(a[3], &q) || stride0(a[3], &qcs) || u32_of(a[4], &qdt) || u64_of(a[5], &qhs) ||
      ptr_of(a[6], &g) || (a[6] != Py_None && (stride0(a[6], &gcs) || u64_of(a[7], &ghs))) || ptr_of(a[8], &out) || stride0(a[8], &ocs) || u64_of(a[9], &stream))
    return NULL;
  Py_ssize_t cnt;
  uint32_t* items = words_of(a[2], 2, 1, kPairs, &cnt);
  if (!items) return NULL;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = ((fn_decode_weights)(uintptr_t)fn)((pa_layer*)(uintptr_t)layer, (const pa_item*)items, (uint32_t)cnt, q, (int)qdt, qcs, qhs, g, gcs, ghs, out, ocs,
                    (void*)(uintptr_t)stream);
  Py_END_ALLOW_THREADS
  free(items);
  return PyLong_FromLong(rc);
}

/* evict(entry, layer, [(src_seq, dst_seq, n_rows)], n_keep, n_first, n_recent, kept, stream) -> status */
static PyObject* evict(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  uint64_t fn, layer, stream;
  uint32_t keep, first, recent;
  void* kept;
  (void)self;
  if (args_are(n, 8, "evict") || u64_of(a[0], &fn) || u64_of(a[1], &layer) || u32_of(a[3], &keep) || u32_of(a[4], &first) || u32_of(a[5], &recent) || ptr_of(a[6], &kept) ||
      u64_of(a[7], &stream))
    return NULL;
  Py_ssize_t cnt;
  uint32_t* items = words_of(a[2], 3, 0, kTriples, &cnt);
  if (!items) return NULL;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = ((fn_evict)(uintptr_t)fn)((pa_layer*)(uintptr_t)layer, (const pa_evict_item*)items, (uint32_t)cnt, keep, first, recent, (uint32_t*)kept, (void*)(uintptr_t)stream);
  Py_END_ALLOW_THREADS
  free(items);
  return PyLong_FromLong(rc);
}

static PyMethodDef methods[] = {
    {"attn_layer", (PyCFunction)(void (*)(void))attn_layer, METH_FASTCALL, "pa_attn_layer on tensors"},
    {"attn_items", (PyCFunction)(void (*)(void))attn_items, METH_FASTCALL, "pa_attn_items on tensors"},
    {"rope_append", (PyCFunction)(void (*)(void))rope_append, METH_FASTCALL, "pa_rope_append on tensors"},
    {"decode_gather", (PyCFunction)(void (*)(void))decode_gather, METH_FASTCALL, "pa_decode_gather on tensors"},
    {"rotary_apply", (PyCFunction)(void (*)(void))rotary_apply, METH_FASTCALL, "pa_rotary_apply on tensors"},
    {"rotary_append", (PyCFunction)(void (*)(void))rotary_append, METH_FASTCALL, "pa_rotary_append on tensors"},
    {"decode_shared", (PyCFunction)(void (*)(void))decode_shared, METH_FASTCALL, "pa_decode_shared on tensors"},
    {"decode_weights", (PyCFunction)(void (*)(void))decode_weights, METH_FASTCALL, "pa_decode_weights on tensors"},
    {"evict", (PyCFunction)(void (*)(void))evict, METH_FASTCALL, "pa_evict on tensors"},
    {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_pa_call", NULL, -1, methods, NULL, NULL, NULL, NULL};
PyMODINIT_FUNC PyInit__pa_call(void) {
  s_data_ptr = PyUnicode_InternFromString("data_ptr");
  s_stride = PyUnicode_InternFromString("stride");
  s_size = PyUnicode_InternFromString("size");
  i_zero = PyLong_FromLong(0);
  if (!s_data_ptr || !s_stride || !s_size || !i_zero) return NULL;
  return PyModule_Create(&module);
}

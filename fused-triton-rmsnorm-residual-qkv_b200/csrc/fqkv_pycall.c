/* CPython fast path for the hot C-ABI call of the Python package (fqkv_launch).
 *
 * The package binds the library with ctypes; converting fqkv_launch's 22 arguments through
 * ctypes costs a few microseconds per call, more than the C entry point itself (which is
 * mostly the CUDA launch).  This module converts them with the CPython API
 * (METH_FASTCALL) and calls the library's fqkv_launch through a function pointer that the
 * package hands over after loading the library (set_launch), so the library it calls is
 * always the one ctypes loaded.  It has no CUDA or PyTorch dependency of its own.
 *
 * launch(x, residual, rms_weight, rms_weight_dtype, weight, out, residual_out, M, H, N,
 *        ldx, ldr, ldw, ldo, ldro, eps, dtype, schedule, flags, workspace, workspace_bytes,
 *        stream) -> int: the arguments of fqkv_launch in order (pointers and the stream as
 *        Python ints, None for a null pointer); returns its return code.
 *
 * kv4_plan, kv4_append, kv4_gather and kv4_attention do the same for the fqkv_kv4_* calls of
 * those names (set_kv4 hands over their four addresses). */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>

typedef int (*fqkv_launch_fn)(const void*, const void*, const void*, int, const void*, void*, void*, int64_t,
                              int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, float, int, int, int,
                              void*, int64_t, void*);

static fqkv_launch_fn g_launch = NULL;

static void* as_ptr(PyObject* o) { return o == Py_None ? NULL : PyLong_AsVoidPtr(o); }

static PyObject* set_launch(PyObject* self, PyObject* arg) {
  (void)self;
  void* p = PyLong_AsVoidPtr(arg);
  if (p == NULL && PyErr_Occurred()) return NULL;
  g_launch = (fqkv_launch_fn)p;
  Py_RETURN_NONE;
}

static PyObject* launch(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  (void)self;
  if (n != 22) {
    PyErr_Format(PyExc_TypeError, "launch takes 22 arguments (%zd given)", n);
    return NULL;
  }
  if (g_launch == NULL) {
    PyErr_SetString(PyExc_RuntimeError, "launch: the library's fqkv_launch has not been set");
    return NULL;
  }
  const void* x = as_ptr(a[0]);
  const void* r = as_ptr(a[1]);
  const void* g = as_ptr(a[2]);
  const int gdt = (int)PyLong_AsLong(a[3]);
  const void* w = as_ptr(a[4]);
  void* out = as_ptr(a[5]);
  void* rout = as_ptr(a[6]);
  int64_t v[8];
  for (int i = 0; i < 8; ++i) v[i] = (int64_t)PyLong_AsLongLong(a[7 + i]); /* M H N ldx ldr ldw ldo ldro */
  const float eps = (float)PyFloat_AsDouble(a[15]);
  const int dtype = (int)PyLong_AsLong(a[16]);
  const int schedule = (int)PyLong_AsLong(a[17]);
  const int flags = (int)PyLong_AsLong(a[18]);
  void* ws = as_ptr(a[19]);
  const int64_t ws_bytes = (int64_t)PyLong_AsLongLong(a[20]);
  void* stream = as_ptr(a[21]);
  if (PyErr_Occurred()) return NULL;
  const int rc = g_launch(x, r, g, gdt, w, out, rout, v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], eps, dtype,
                          schedule, flags, ws, ws_bytes, stream);
  return PyLong_FromLong(rc);
}

typedef const void* cp;
typedef int64_t i64;
typedef int (*kv4_plan_fn)(cp, cp, i64, cp, i64, i64, cp, i64, cp, i64, i64, cp, cp, cp, cp, cp, cp, i64, cp);
typedef int (*kv4_append_fn)(cp, cp, cp, i64, i64, i64, i64, i64, i64, i64, i64, cp, i64, cp);
typedef int (*kv4_gather_fn)(cp, cp, i64, cp, cp, i64, cp);
typedef int (*kv4_attention_fn)(cp, cp, i64, i64, i64, i64, cp, i64, i64, i64, i64, cp, i64, i64, cp, i64, float, cp,
                                i64, cp, i64, i64, cp);

static kv4_plan_fn g_plan = NULL;
static kv4_append_fn g_append = NULL;
static kv4_gather_fn g_gather = NULL;
static kv4_attention_fn g_attention = NULL;

/* `n` Python ints (None: 0) as 64-bit values, but for index `skip`; 0 on an error. */
static int as_words(const char* name, int set, PyObject* const* a, Py_ssize_t n, Py_ssize_t want, Py_ssize_t skip,
                    i64* v) {
  if (n != want) {
    PyErr_Format(PyExc_TypeError, "%s takes %zd arguments (%zd given)", name, want, n);
    return 0;
  }
  if (!set) {
    PyErr_Format(PyExc_RuntimeError, "%s: the library's address has not been set", name);
    return 0;
  }
  for (Py_ssize_t i = 0; i < n; ++i)
    if (i != skip) v[i] = a[i] == Py_None ? 0 : (i64)PyLong_AsLongLong(a[i]);
  return !PyErr_Occurred();
}
#define P(i) ((cp)(uintptr_t)v[i])

static PyObject* set_kv4(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  (void)self;
  i64 v[4];
  if (!as_words("set_kv4", 1, a, n, 4, -1, v)) return NULL;
  g_plan = (kv4_plan_fn)(uintptr_t)v[0];
  g_append = (kv4_append_fn)(uintptr_t)v[1];
  g_gather = (kv4_gather_fn)(uintptr_t)v[2];
  g_attention = (kv4_attention_fn)(uintptr_t)v[3];
  Py_RETURN_NONE;
}

static PyObject* kv4_plan(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  (void)self;
  i64 v[19];
  if (!as_words("kv4_plan", g_plan != NULL, a, n, 19, -1, v)) return NULL;
  return PyLong_FromLong(g_plan(P(0), P(1), v[2], P(3), v[4], v[5], P(6), v[7], P(8), v[9], v[10], P(11), P(12), P(13),
                                P(14), P(15), P(16), v[17], P(18)));
}

static PyObject* kv4_append(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  (void)self;
  i64 v[14];
  if (!as_words("kv4_append", g_append != NULL, a, n, 14, -1, v)) return NULL;
  return PyLong_FromLong(g_append(P(0), P(1), P(2), v[3], v[4], v[5], v[6], v[7], v[8], v[9], v[10], P(11), v[12], P(13)));
}

static PyObject* kv4_gather(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  (void)self;
  i64 v[7];
  if (!as_words("kv4_gather", g_gather != NULL, a, n, 7, -1, v)) return NULL;
  return PyLong_FromLong(g_gather(P(0), P(1), v[2], P(3), P(4), v[5], P(6)));
}

static PyObject* kv4_attention(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  (void)self;
  i64 v[23];
  if (!as_words("kv4_attention", g_attention != NULL, a, n, 23, 16, v)) return NULL;
  const float scale = (float)PyFloat_AsDouble(a[16]);
  if (PyErr_Occurred()) return NULL;
  return PyLong_FromLong(g_attention(P(0), P(1), v[2], v[3], v[4], v[5], P(6), v[7], v[8], v[9], v[10], P(11), v[12],
                                     v[13], P(14), v[15], scale, P(17), v[18], P(19), v[20], v[21], P(22)));
}

#define FAST(f) (PyCFunction)(void (*)(void))f, METH_FASTCALL
static PyMethodDef kMethods[] = {
    {"set_launch", (PyCFunction)set_launch, METH_O, "Set the address of the library's fqkv_launch."},
    {"launch", (PyCFunction)(void (*)(void))launch, METH_FASTCALL, "Call fqkv_launch with 22 arguments."},
    {"set_kv4", FAST(set_kv4), "Set the addresses of fqkv_kv4_plan, _append, _gather and _attention."},
    {"kv4_plan", FAST(kv4_plan), "Call fqkv_kv4_plan with 19 arguments."},
    {"kv4_append", FAST(kv4_append), "Call fqkv_kv4_append with 14 arguments."},
    {"kv4_gather", FAST(kv4_gather), "Call fqkv_kv4_gather with 7 arguments."},
    {"kv4_attention", FAST(kv4_attention), "Call fqkv_kv4_attention with 23 arguments."},
    {NULL, NULL, 0, NULL}};

static struct PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fqkv_pycall", NULL, -1, kMethods,
                                     NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__fqkv_pycall(void) { return PyModule_Create(&kModule); }

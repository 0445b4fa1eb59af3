/*
 * CPython binding of the GEMM and kv4 entry points for the Python operators
 * (csed499ii_b200.mul_2_4 and friends): the same C ABI as the ctypes table
 * in _ext.py, called with plain integers.  The reference reaches its kernel
 * through a compiled pybind11 extension (marlin_cuda.mul_2_4,
 * kernel_experiments/sparse_marlin/src/marlin/marlin_cuda.cpp:66-99); with
 * ctypes the argument conversion alone cost ~2.5 us per call, as much as a
 * quarter of a decode GEMM, which made an eager decode step host-bound.
 *
 * mul(A, B, meta, C, s, prob_m, prob_n, prob_k, workspace, groupsize, dev,
 *     stream, thread_k, thread_m, sms, max_par, meta_bits, bias, activation)
 * -> int status.  Pointers and the stream are integers (0 = none).
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>

#include "../../include/sm100_marlin.h"

static PyObject* fast_mul(PyObject* self, PyObject* args) {
  unsigned long long a, b, meta, c, s, ws, stream, bias;
  int prob_m, prob_n, prob_k, groupsize, dev, thread_k, thread_m, sms, max_par, meta_bits, act;
  (void)self;
  if (!PyArg_ParseTuple(args, "KKKKKiiiKiiKiiiiiKi", &a, &b, &meta, &c, &s, &prob_m, &prob_n,
                        &prob_k, &ws, &groupsize, &dev, &stream, &thread_k, &thread_m, &sms,
                        &max_par, &meta_bits, &bias, &act))
    return NULL;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  if (bias == 0 && act == 0) {
    if (meta_bits == 4)
      rc = sm100_marlin_mul_2_4((const void*)a, (const void*)b, (const void*)meta, (void*)c,
                                (const void*)s, prob_m, prob_n, prob_k, (void*)ws, groupsize, dev,
                                (void*)stream, thread_k, thread_m, sms, max_par);
    else
      rc = sm100_marlin_mul_2_4_meta3((const void*)a, (const void*)b, (const void*)meta, (void*)c,
                                      (const void*)s, prob_m, prob_n, prob_k, (void*)ws, groupsize,
                                      dev, (void*)stream, thread_k, thread_m, sms, max_par);
  } else {
    rc = sm100_marlin_mul_2_4_epilogue((const void*)a, (const void*)b, (const void*)meta, (void*)c,
                                       (const void*)s, prob_m, prob_n, prob_k, (void*)ws, groupsize,
                                       dev, (void*)stream, thread_k, thread_m, sms, max_par,
                                       meta_bits, (const void*)bias, act);
  }
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

/*
 * The kv4_* entry points: positional integers in the order of the C ABI
 * (pointers, strides and the stream as integers, 0 = none; the softmax scale
 * of kv4_attention is a float) -> int status.
 */
#define MAX_ARGS 25

/* args[0..n) as integers; argument `real` (or -1) as a float. */
static int read_args(PyObject* const* args, Py_ssize_t given, int n, long long* out, int real,
                     double* value) {
  if (given != n) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", n, given);
    return -1;
  }
  for (int i = 0; i < n; ++i) {
    if (i == real) {
      *value = PyFloat_AsDouble(args[i]);
    } else {
      out[i] = PyLong_AsLongLong(args[i]);
    }
  }
  return PyErr_Occurred() ? -1 : 0;
}

static PyObject* fast_kv4_schedule(PyObject* self, PyObject* const* args, Py_ssize_t given) {
  long long a[MAX_ARGS];
  int rc;
  (void)self;
  if (read_args(args, given, 19, a, -1, NULL)) return NULL;
  Py_BEGIN_ALLOW_THREADS
  rc = sm100_marlin_kv4_schedule((const int*)a[0], (const int*)a[1], (int*)a[2], a[3], (int)a[4],
                                 (int)a[5], (int*)a[6], (int)a[7], (const int*)a[8], (int)a[9],
                                 (int)a[10], (int*)a[11], (int*)a[12], (int*)a[13], (int*)a[14],
                                 (int*)a[15], (int*)a[16], (int)a[17], (void*)a[18]);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

static PyObject* fast_kv4_append(PyObject* self, PyObject* const* args, Py_ssize_t given) {
  long long a[MAX_ARGS];
  int rc;
  (void)self;
  if (read_args(args, given, 16, a, -1, NULL)) return NULL;
  Py_BEGIN_ALLOW_THREADS
  rc = sm100_marlin_kv4_append((const void*)a[0], a[1], a[2], (const void*)a[3], a[4], a[5],
                               (void*)a[6], (int)a[7], (int)a[8], (int)a[9], (int)a[10], (int)a[11],
                               (const int*)a[12], (int)a[13], (int)a[14], (void*)a[15]);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

static PyObject* fast_kv4_read(PyObject* self, PyObject* const* args, Py_ssize_t given) {
  long long a[MAX_ARGS];
  int rc;
  (void)self;
  if (read_args(args, given, 12, a, -1, NULL)) return NULL;
  Py_BEGIN_ALLOW_THREADS
  rc = sm100_marlin_kv4_read((const void*)a[0], (int)a[1], (int)a[2], (int)a[3], (int)a[4], (int)a[5],
                             (const int*)a[6], (int)a[7], (void*)a[8], (void*)a[9], (int)a[10],
                             (void*)a[11]);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

static PyObject* fast_kv4_attention(PyObject* self, PyObject* const* args, Py_ssize_t given) {
  long long a[MAX_ARGS];
  double scale = 0;
  int rc;
  (void)self;
  if (read_args(args, given, 25, a, 19, &scale)) return NULL;
  Py_BEGIN_ALLOW_THREADS
  rc = sm100_marlin_kv4_attention(
      (const void*)a[0], a[1], a[2], (const void*)a[3], (int)a[4], (int)a[5], (int)a[6], (int)a[7],
      (int)a[8], (const int*)a[9], a[10], (int)a[11], (const int*)a[12], (const int*)a[13], (int)a[14],
      (int)a[15], (int)a[16], (int)a[17], (int)a[18], (float)scale, (void*)a[20], (void*)a[21],
      (size_t)a[22], (int)a[23], (void*)a[24]);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

#define FAST(name, doc) \
  {#name, (PyCFunction)(void (*)(void))fast_##name, METH_FASTCALL, doc}

static PyMethodDef kMethods[] = {
    {"mul", fast_mul, METH_VARARGS, "2:4 W4A16 GEMM through the C ABI (status code)."},
    FAST(kv4_schedule, "sm100_marlin_kv4_schedule (status code)."),
    FAST(kv4_append, "sm100_marlin_kv4_append (status code)."),
    FAST(kv4_read, "sm100_marlin_kv4_read (status code)."),
    FAST(kv4_attention, "sm100_marlin_kv4_attention (status code)."),
    {NULL, NULL, 0, NULL}};

static struct PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_fastcall", NULL, -1, kMethods,
                                     NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__fastcall(void) { return PyModule_Create(&kModule); }

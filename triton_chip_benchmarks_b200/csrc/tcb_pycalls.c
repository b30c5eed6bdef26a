/* The MX FP4 entry points as Python functions of integers (addresses, sizes; None
 * is a null pointer) that return the status: the operators are called with one
 * token at a time, where what ctypes takes to convert a dozen arguments (2 us) is
 * a good part of a call.  The entry points' addresses come from the libtcb that
 * the ctypes binding has loaded (bind), so both always call the same library. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "tcb.h"

static int (*quantize)(int, const void *, long long, long long, long long, int, void *, void *, void *,
                       void *, tcb_stream_t);
static int (*dequantize)(int, const void *, const void *, long long, long long, void *, long long,
                         tcb_stream_t);
static int (*gemm)(const void *, const void *, const void *, const void *, const void *, int, void *,
                   long long, int, int, int, int *, tcb_stream_t);
static int (*linear)(int, const void *, long long, const void *, const void *, const void *, int, void *,
                     long long, int, int, int, void *, long long, int *, tcb_stream_t);

#define MOST 16

/* Exactly `want` integers or Nones into v; 0 with an exception set otherwise. */
static int integers(PyObject *const *args, Py_ssize_t given, Py_ssize_t want, long long *v) {
  if (given != want) {
    PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", want, given);
    return 0;
  }
  for (Py_ssize_t i = 0; i < want; ++i) {
    v[i] = args[i] == Py_None ? 0 : PyLong_AsLongLong(args[i]);
    if (v[i] == -1 && PyErr_Occurred()) return 0;
  }
  return 1;
}

/* A size that an int parameter takes: past its range it becomes -1, which every
 * entry point refuses. */
static int as_int(long long v) { return v < 0 || v > 2147483647 ? -1 : (int)v; }

#define P(i) ((void *)(intptr_t)v[i])
#define READY(f)                                                         \
  if (f == NULL) {                                                       \
    PyErr_SetString(PyExc_RuntimeError, "libtcb has not been bound yet"); \
    return NULL;                                                         \
  }
#define CALL(expression)             \
  int status;                        \
  Py_BEGIN_ALLOW_THREADS status = expression; \
  Py_END_ALLOW_THREADS return PyLong_FromLong(status)

static PyObject *call_quantize(PyObject *self, PyObject *const *args, Py_ssize_t n) {
  long long v[MOST];
  READY(quantize)
  if (!integers(args, n, 11, v)) return NULL;
  CALL(quantize(as_int(v[0]), P(1), v[2], v[3], v[4], as_int(v[5]), P(6), P(7), P(8), P(9), P(10)));
}

static PyObject *call_dequantize(PyObject *self, PyObject *const *args, Py_ssize_t n) {
  long long v[MOST];
  READY(dequantize)
  if (!integers(args, n, 8, v)) return NULL;
  CALL(dequantize(as_int(v[0]), P(1), P(2), v[3], v[4], P(5), v[6], P(7)));
}

static PyObject *call_gemm(PyObject *self, PyObject *const *args, Py_ssize_t n) {
  long long v[MOST];
  READY(gemm)
  if (!integers(args, n, 13, v)) return NULL;
  CALL(gemm(P(0), P(1), P(2), P(3), P(4), as_int(v[5]), P(6), v[7], as_int(v[8]), as_int(v[9]),
            as_int(v[10]), P(11), P(12)));
}

static PyObject *call_linear(PyObject *self, PyObject *const *args, Py_ssize_t n) {
  long long v[MOST];
  READY(linear)
  if (!integers(args, n, 16, v)) return NULL;
  CALL(linear(as_int(v[0]), P(1), v[2], P(3), P(4), P(5), as_int(v[6]), P(7), v[8], as_int(v[9]),
              as_int(v[10]), as_int(v[11]), P(12), v[13], P(14), P(15)));
}

/* bind(quantize, dequantize, gemm, linear): addresses of the entry points. */
static PyObject *bind(PyObject *self, PyObject *const *args, Py_ssize_t n) {
  long long v[MOST];
  if (!integers(args, n, 4, v)) return NULL;
  *(void **)&quantize = P(0);
  *(void **)&dequantize = P(1);
  *(void **)&gemm = P(2);
  *(void **)&linear = P(3);
  Py_RETURN_NONE;
}

#define METHOD(name, function) {name, (PyCFunction)(void (*)(void))function, METH_FASTCALL, NULL}
static PyMethodDef methods[] = {
    METHOD("bind", bind),
    METHOD("tcb_mx_quantize", call_quantize),
    METHOD("tcb_mx_dequantize", call_dequantize),
    METHOD("tcb_mx_gemm", call_gemm),
    METHOD("tcb_mx_linear", call_linear),
    {NULL, NULL, 0, NULL},
};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tcb_calls", NULL, -1, methods,
                                    NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__tcb_calls(void) { return PyModule_Create(&module); }

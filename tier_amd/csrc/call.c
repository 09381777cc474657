/* call.c -- tier_amd._call: functions of libtiermm.so called from Python with less than ctypes'
 * cost a call, for entry points whose arguments are integers, addresses and at most one float.  A call of
 * 17 arguments takes 0.4 us with its wrapper, 2.1 through ctypes; a small kernel runs 2.3 to 3.5
 * us. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <stddef.h>
#include <stdint.h>
#include <structmember.h>

#define MOST 20

/* x86-64: integer arguments travel as 64-bit words whatever their C type, and a callee ignores
 * those past its own.  A float travels in a vector register, whatever its place among them. */
typedef int (*Fn)(uint64_t, uint64_t, uint64_t, uint64_t, uint64_t, uint64_t, uint64_t, uint64_t, uint64_t, uint64_t,
                  uint64_t, uint64_t, uint64_t, uint64_t, uint64_t, uint64_t, uint64_t, uint64_t, uint64_t, uint64_t,
                  float);

typedef struct {
  PyObject_HEAD
  vectorcallfunc call;
  Fn fn;
  Py_ssize_t n;
  uint32_t numbers; /* bit i: argument i is a number, which None is not */
  unsigned floats;  /* bit i: argument i is a float */
} Call;

static PyObject* call_vector(PyObject* o, PyObject* const* args, size_t nf, PyObject* kw) {
  Call* c = (Call*)o;
  const Py_ssize_t n = PyVectorcall_NARGS(nf);
  if (n != c->n || (kw && PyTuple_GET_SIZE(kw))) {
    PyErr_Format(PyExc_TypeError, "%zd arguments, %zd wanted", n, c->n);
    return NULL;
  }
  uint64_t a[MOST] = {0}, *to = a;
  float f = 0.f;
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (c->floats >> i & 1) {
      const double d = PyFloat_AsDouble(args[i]);
      if (d == -1. && PyErr_Occurred()) return NULL;
      f = (float)d;
      continue;
    }
    if (args[i] == Py_None) { /* a null pointer */
      if (!(c->numbers >> i & 1)) {
        *to++ = 0;
        continue;
      }
      PyErr_Format(PyExc_TypeError, "argument %zd is None, a number is wanted", i + 1);
      return NULL;
    }
    PyObject* v = PyLong_Check(args[i]) ? Py_NewRef(args[i]) : PyNumber_Index(args[i]);
    if (!v) return NULL;
    *to = PyLong_AsUnsignedLongLongMask(v);
    Py_DECREF(v);
    if (*to == (uint64_t)-1 && PyErr_Occurred()) return NULL;
    ++to;
  }
  int code;
  Py_BEGIN_ALLOW_THREADS
  code = c->fn(a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7], a[8], a[9], a[10], a[11], a[12], a[13], a[14], a[15],
               a[16], a[17], a[18], a[19], f);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(code);
}

static PyObject* call_new(PyTypeObject* t, PyObject* args, PyObject* kw) {
  unsigned long long address;
  Py_ssize_t n;
  unsigned numbers = 0, floats = 0;
  if (!PyArg_ParseTuple(args, "Kn|II", &address, &n, &numbers, &floats)) return NULL;
  if (!address || n < 0 || n > MOST || (floats & (floats - 1))) {
    PyErr_SetString(PyExc_ValueError, "Call(address, arguments <= 20, of them one float)");
    return NULL;
  }
  Call* c = (Call*)t->tp_alloc(t, 0);
  if (!c) return NULL;
  c->call = call_vector;
  c->fn = (Fn)(uintptr_t)address;
  c->n = n;
  c->numbers = numbers;
  c->floats = floats;
  return (PyObject*)c;
}

static PyMemberDef call_members[] = {
    {"__vectorcalloffset__", T_PYSSIZET, offsetof(Call, call), READONLY, NULL}, {NULL, 0, 0, 0, NULL}};
static PyType_Slot call_slots[] = {{Py_tp_new, call_new},
                                   {Py_tp_call, PyVectorcall_Call},
                                   {Py_tp_members, call_members},
                                   {Py_tp_doc, "Call(address, n, numbers=0, floats=0): an int function of n integers or addresses; None is a\n"
                                               "null address, refused for the arguments whose bit is set in numbers; the argument\n"
                                               "whose bit is set in floats (one at most) is a float"},
                                   {0, NULL}};
static PyType_Spec call_spec = {"tier_amd._call.Call", sizeof(Call), 0,
                                Py_TPFLAGS_DEFAULT | Py_TPFLAGS_HAVE_VECTORCALL, call_slots};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_call", NULL, -1, NULL, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__call(void) {
  PyObject* m = PyModule_Create(&module);
  if (!m) return NULL;
  PyObject* t = PyType_FromSpec(&call_spec);
  if (!t || PyModule_AddObject(m, "Call", t) < 0) {
    Py_XDECREF(t);
    Py_DECREF(m);
    return NULL;
  }
  return m;
}

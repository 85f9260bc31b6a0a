/* The calls a decode step makes most often, vqm_qmv and those of 8-bit integer passes, from Python without ctypes: with a function that does nothing
 * vqm_qmv takes 1.02 us through ctypes and 0.18 through this (the driver's launch takes 2.2).  Arguments mean what they mean to ctypes and int().
 * Optional: limited API, so that one build serves every CPython from 3.10 on; without it the call goes through ctypes. */
#define PY_SSIZE_T_CLEAN
#define Py_LIMITED_API 0x030A0000
#include <Python.h>

typedef int (*qmv_fn)(void *, const char *, const char *, const char *, int);

/* qmv(function address, handle, weight, x, y, ntok) -> status; the GIL is released during the call */
static PyObject *py_qmv(PyObject *self, PyObject *const *args, Py_ssize_t n) {
    (void)self;
    if (n != 6) {
        PyErr_SetString(PyExc_TypeError, "qmv takes 6 arguments");
        return NULL;
    }
    const qmv_fn fn = (qmv_fn)PyLong_AsVoidPtr(args[0]);
    void *const handle = PyLong_AsVoidPtr(args[1]);
    if (PyErr_Occurred()) return NULL;
    const char *name[3];
    for (int i = 0; i < 3; ++i) {
        PyObject *const s = args[2 + i];
        if (!PyUnicode_Check(s)) {
            PyErr_Format(PyExc_AttributeError, "%R object has no attribute 'encode'", (PyObject *)Py_TYPE(s));
            return NULL;
        }
        name[i] = PyUnicode_AsUTF8AndSize(s, NULL);
        if (name[i] == NULL) return NULL;
    }
    PyObject *const whole = PyNumber_Long(args[5]);
    if (whole == NULL) return NULL;
    const int ntok = (int)PyLong_AsUnsignedLongMask(whole);
    Py_DECREF(whole);
    if (PyErr_Occurred()) return NULL;
    if (fn == NULL || handle == NULL) {
        PyErr_SetString(PyExc_ValueError, "the runtime is closed");
        return NULL;
    }
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = fn(handle, name[0], name[1], name[2], ntok);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(status);
}

/* What every call below begins with: the function's address, the runtime's handle. */
static int begin(PyObject *const *args, Py_ssize_t n, Py_ssize_t want, const char *call, void **fn, void **handle) {
    if (n != want) {
        PyErr_Format(PyExc_TypeError, "%s takes %zd arguments", call, want);
        return -1;
    }
    *fn = PyLong_AsVoidPtr(args[0]);
    *handle = PyLong_AsVoidPtr(args[1]);
    if (PyErr_Occurred()) return -1;
    if (*fn == NULL || *handle == NULL) {
        PyErr_SetString(PyExc_ValueError, "the runtime is closed");
        return -1;
    }
    return 0;
}
/* A str, or None where that is allowed. */
static int name_of(PyObject *s, int optional, const char **out) {
    *out = NULL;
    if (optional && s == Py_None) return 0;
    if (!PyUnicode_Check(s)) {
        PyErr_Format(PyExc_AttributeError, "%R object has no attribute 'encode'", (PyObject *)Py_TYPE(s));
        return -1;
    }
    *out = PyUnicode_AsUTF8AndSize(s, NULL);
    return *out == NULL ? -1 : 0;
}
static int int_of(PyObject *v, int *out) {
    PyObject *const whole = PyNumber_Long(v);
    if (whole == NULL) return -1;
    *out = (int)PyLong_AsUnsignedLongMask(whole);
    Py_DECREF(whole);
    return PyErr_Occurred() ? -1 : 0;
}

typedef int (*rows_fn)(void *, const char *, const char *, const char *, int, int, int, const char *, const char *, const char *, const char *, float);

/* rows_i8(address, handle, x, q, scales, cols, ntok, flags, x2, residual, total, norm, eps) */
static PyObject *py_rows_i8(PyObject *self, PyObject *const *args, Py_ssize_t n) {
    (void)self;
    void *fn, *handle;
    const char *name[7];
    int whole[3], status;
    if (begin(args, n, 13, "rows_i8", &fn, &handle) < 0) return NULL;
    for (int i = 0; i < 3; ++i)
        if (name_of(args[2 + i], 0, &name[i]) < 0 || int_of(args[5 + i], &whole[i]) < 0) return NULL;
    for (int i = 0; i < 4; ++i)
        if (name_of(args[8 + i], 1, &name[3 + i]) < 0) return NULL;
    const double eps = PyFloat_AsDouble(args[12]);
    if (PyErr_Occurred()) return NULL;
    Py_BEGIN_ALLOW_THREADS
    status = ((rows_fn)fn)(handle, name[0], name[1], name[2], whole[0], whole[1], whole[2], name[3], name[4], name[5], name[6], (float)eps);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(status);
}

typedef int (*qmm_fn)(void *, const char *, const char *, const char *, const char *, int, int);

/* qmm_i8(address, handle, weight, q, scales, y, ntok, flags) */
static PyObject *py_qmm_i8(PyObject *self, PyObject *const *args, Py_ssize_t n) {
    (void)self;
    void *fn, *handle;
    const char *name[4];
    int whole[2], status;
    if (begin(args, n, 8, "qmm_i8", &fn, &handle) < 0) return NULL;
    for (int i = 0; i < 4; ++i)
        if (name_of(args[2 + i], 0, &name[i]) < 0) return NULL;
    for (int i = 0; i < 2; ++i)
        if (int_of(args[6 + i], &whole[i]) < 0) return NULL;
    Py_BEGIN_ALLOW_THREADS
    status = ((qmm_fn)fn)(handle, name[0], name[1], name[2], name[3], whole[0], whole[1]);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(status);
}

typedef int (*verify_fn)(void *, const char *, const char *, const char *, const char *, const char *, const char *, int, int, int, const char *, int *);

/* verify(address, handle, target, draft, tokens, lens, uniforms, temperature, vocab, seqs, drafts, out, address of the answer or 0) */
static PyObject *py_verify(PyObject *self, PyObject *const *args, Py_ssize_t n) {
    (void)self;
    void *fn, *handle;
    const char *name[6], *out;
    int whole[3], status;
    if (begin(args, n, 13, "verify", &fn, &handle) < 0) return NULL;
    for (int i = 0; i < 6; ++i)
        if (name_of(args[2 + i], i == 1 || i == 2 || i == 3 || i == 5, &name[i]) < 0) return NULL;
    for (int i = 0; i < 3; ++i)
        if (int_of(args[8 + i], &whole[i]) < 0) return NULL;
    if (name_of(args[11], 0, &out) < 0) return NULL;
    int *const answer = (int *)PyLong_AsVoidPtr(args[12]);
    if (PyErr_Occurred()) return NULL;
    Py_BEGIN_ALLOW_THREADS
    status = ((verify_fn)fn)(handle, name[0], name[1], name[2], name[3], name[4], name[5], whole[0], whole[1], whole[2], out, answer);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(status);
}

#define METHOD(name, text) {#name, (PyCFunction)(void (*)(void))py_##name, METH_FASTCALL, text}
static PyMethodDef methods[] = {METHOD(qmv, "vqm_qmv"), METHOD(rows_i8, "vqm_rows_i8"), METHOD(qmm_i8, "vqm_qmm_i8"), METHOD(verify, "vqm_verify"), {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_vqm_pycall", NULL, -1, methods, NULL, NULL, NULL, NULL};
PyMODINIT_FUNC PyInit__vqm_pycall(void) { return PyModule_Create(&module); }

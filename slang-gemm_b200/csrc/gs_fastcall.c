/* gs_fastcall.c -- CPython binding of the FP8 and routed-expert calls.
 *
 * These calls are issued many times a step on small problems, where the host's
 * time per call is what counts: converting their two dozen arguments through
 * ctypes took 3.5 us of 6, here it takes 0.4. gemm_sm100.py wraps each function
 * and turns a status into an exception; the argument checks are the library's.
 * A pointer argument is None, an int, or an object with data_ptr() (a tensor).
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <limits.h>
#include <string.h>

#include "gemm_sm100.h"

static PyObject *data_ptr_name;

typedef union {
    void *p;
    long long q;
    int i;
    float f;
} value;

/* Converts args by `kinds`: p pointer, i int, q long long, f float. Returns 0, or -1 with an exception set. */
static int convert(const char *name, PyObject *const *args, Py_ssize_t n, const char *kinds, value *out) {
    const Py_ssize_t want = (Py_ssize_t)strlen(kinds);
    if (n != want) {
        PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", name, want, n);
        return -1;
    }
    for (Py_ssize_t k = 0; k < n; ++k) {
        PyObject *a = args[k];
        switch (kinds[k]) {
        case 'i':
        case 'q': {
            const long long v = PyLong_AsLongLong(a);
            if (v == -1 && PyErr_Occurred()) return -1;
            if (kinds[k] == 'q') {
                out[k].q = v;
            } else {
                if (v < INT_MIN || v > INT_MAX) {
                    PyErr_Format(PyExc_OverflowError, "argument %zd of %s does not fit a C int", k, name);
                    return -1;
                }
                out[k].i = (int)v;
            }
            break;
        }
        case 'f': {
            const double v = PyFloat_AsDouble(a);
            if (v == -1.0 && PyErr_Occurred()) return -1;
            out[k].f = (float)v;
            break;
        }
        default:
            if (a == Py_None) {
                out[k].p = NULL;
            } else if (PyLong_Check(a)) {
                out[k].p = PyLong_AsVoidPtr(a);
                if (out[k].p == NULL && PyErr_Occurred()) return -1;
            } else {
                PyObject *r = PyObject_CallMethodNoArgs(a, data_ptr_name);
                if (r == NULL) return -1;
                out[k].p = PyLong_AsVoidPtr(r);
                Py_DECREF(r);
                if (out[k].p == NULL && PyErr_Occurred()) return -1;
            }
        }
    }
    return 0;
}

/* The call, without the interpreter's lock (a full launch queue waits). */
#define CALL(expr)                         \
    do {                                   \
        gs_status s_;                      \
        Py_BEGIN_ALLOW_THREADS             \
        s_ = (expr);                       \
        Py_END_ALLOW_THREADS               \
        return PyLong_FromLong((long)s_);  \
    } while (0)

#define ARGS(kinds)                                                            \
    value v[sizeof(kinds) - 1];                                                \
    (void)self;                                                                \
    if (convert(__func__, args, n, kinds, v) != 0) return NULL

static PyObject *set_stream(PyObject *self, PyObject *const *args, Py_ssize_t n) {
    ARGS("pp");
    return PyLong_FromLong((long)gs_set_stream((gs_handle)v[0].p, v[1].p));
}

static PyObject *fp8_quantize(PyObject *self, PyObject *const *args, Py_ssize_t n) {
    ARGS("piiiipiipiipiipi");
    CALL(gs_fp8_quantize((gs_handle)v[0].p, v[1].i, v[2].i, v[3].i, v[4].i, v[5].p, v[6].i, v[7].i, (const int32_t *)v[8].p,
                         v[9].i, v[10].i, v[11].p, v[12].i, v[13].i, (float *)v[14].p, v[15].i));
}

static PyObject *gemm_fp8(PyObject *self, PyObject *const *args, Py_ssize_t n) {
    ARGS("piiiiifpiipiipiipiifpii");
    CALL(gs_gemm_fp8((gs_handle)v[0].p, v[1].i, v[2].i, v[3].i, v[4].i, v[5].i, &v[6].f, v[7].p, v[8].i, v[9].i,
                     (const float *)v[10].p, v[11].i, v[12].i, v[13].p, v[14].i, v[15].i, (const float *)v[16].p, v[17].i,
                     v[18].i, &v[19].f, v[20].p, v[21].i, v[22].i));
}

static PyObject *gemm_fp8_grouped(PyObject *self, PyObject *const *args, Py_ssize_t n) {
    ARGS("piiiiiiipfpiiqpiiqpiipiifpiiq");
    CALL(gs_gemm_fp8_grouped((gs_handle)v[0].p, v[1].i, v[2].i, v[3].i, v[4].i, v[5].i, v[6].i, v[7].i, (const int32_t *)v[8].p,
                             &v[9].f, v[10].p, v[11].i, v[12].i, v[13].q, (const float *)v[14].p, v[15].i, v[16].i, v[17].q,
                             v[18].p, v[19].i, v[20].i, (const float *)v[21].p, v[22].i, v[23].i, &v[24].f, v[25].p, v[26].i,
                             v[27].i, v[28].q));
}

/* gs_route_desc's fields in its order. */
#define ROUTE_KINDS "iiipiipiiiifpippppp" "ipq"
static gs_route_desc route_desc(const value *v) {
    gs_route_desc d = {v[0].i, v[1].i, v[2].i, v[3].p, v[4].i, v[5].i, (const float *)v[6].p, v[7].i, v[8].i, v[9].i, v[10].i,
                       v[11].f, (const int32_t *)v[12].p, v[13].i, (int32_t *)v[14].p, (float *)v[15].p, (int32_t *)v[16].p,
                       (int32_t *)v[17].p, (int32_t *)v[18].p, v[19].i, v[20].p, (size_t)v[21].q};
    return d;
}

static PyObject *moe_route(PyObject *self, PyObject *const *args, Py_ssize_t n) {
    ARGS("p" ROUTE_KINDS);
    const gs_route_desc d = route_desc(v + 1);
    CALL(gs_moe_route((gs_handle)v[0].p, &d));
}

static PyObject *moe_route_backward(PyObject *self, PyObject *const *args, Py_ssize_t n) {
    ARGS("p" ROUTE_KINDS "ppii");
    const gs_route_desc d = route_desc(v + 1);
    CALL(gs_moe_route_backward((gs_handle)v[0].p, &d, (const float *)v[23].p, v[24].p, v[25].i, v[26].i));
}

static PyObject *moe_combine(PyObject *self, PyObject *const *args, Py_ssize_t n) {
    ARGS("piiipiiipppii");
    CALL(gs_moe_combine((gs_handle)v[0].p, v[1].i, v[2].i, v[3].i, v[4].p, v[5].i, v[6].i, v[7].i, (const int32_t *)v[8].p,
                        (const float *)v[9].p, v[10].p, v[11].i, v[12].i));
}

static PyObject *moe_combine_backward(PyObject *self, PyObject *const *args, Py_ssize_t n) {
    ARGS("piiipiiippppipip");
    CALL(gs_moe_combine_backward((gs_handle)v[0].p, v[1].i, v[2].i, v[3].i, v[4].p, v[5].i, v[6].i, v[7].i,
                                 (const int32_t *)v[8].p, (const int32_t *)v[9].p, (const float *)v[10].p, v[11].p, v[12].i,
                                 v[13].p, v[14].i, (float *)v[15].p));
}

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, NULL}
static PyMethodDef methods[] = {METHOD(set_stream),         METHOD(fp8_quantize),         METHOD(gemm_fp8),
                                METHOD(gemm_fp8_grouped),   METHOD(moe_route),            METHOD(moe_route_backward),
                                METHOD(moe_combine),        METHOD(moe_combine_backward), {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_gs_fastcall", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__gs_fastcall(void) {
    data_ptr_name = PyUnicode_InternFromString("data_ptr");
    return data_ptr_name == NULL ? NULL : PyModule_Create(&module);
}

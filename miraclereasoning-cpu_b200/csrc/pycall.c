/* _pycall: the array operators' calls from Python.
 *
 * The operators on arrays of any owner (include/miracle_cuda.h: mr_array) take
 * up to eleven of them, each described by five accessors of a Python object.
 * Read in Python and passed through ctypes, that is most of a small call's time
 * (a one-token attention took the host 17.7 microseconds so, 13.3 through this
 * module); here the accessors are read into the structs and the library's
 * function is called directly.  Everything
 * else of the binding stays in ctypes (_native.py), which also hands over the
 * functions' addresses, so that this module links to no library.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <stdint.h>
#include <string.h>

#include "../../include/miracle_cuda.h"

#define MOST 11

enum { APPEND, PAGED, WINDOW, EVICT, ROTATED, READ, SCORE, CALLS };  /* arrays.py has the same order */
static const struct {
    int arrays, scalars;
    const char *names[MOST];
} calls[CALLS] = {
    {7, 0, {"keys", "values", "key_pages", "value_pages", "page_table", "lengths", "offsets"}},
    {7, 3, {"query", "key_pages", "value_pages", "page_table", "lengths", "weights", "out"}},
    {6, 3, {"query", "keys", "values", "query_offsets", "key_offsets", "out"}},
    {11, 3, {"key_pages", "value_pages", "page_table", "lengths", "weights", "target_keys", "target_values",
             "target_table", "kept", "new_lengths", "new_weights"}},
    {11, 1, {"query", "keys", "values", "key_pages", "value_pages", "page_table", "lengths", "offsets", "frequencies",
             "positions", "out"}},
    {7, 0, {"key_pages", "value_pages", "page_table", "lengths", "offsets", "keys", "values"}},
    {6, 0, {"logits", "tokens", "logprobs", "entropy", "top_tokens", "top_logprobs"}},
};
static void *functions[CALLS];
static PyObject *codes;      /* dtype -> enum mr_dtype, of the types met */
static PyObject *slow;       /* arrays.described: what is wrong with an array, or its bytes */
static PyObject *get_device, *shape, *stride, *dtype, *data_ptr;

/* A tuple's whole numbers; their count, or -1. */
static int numbers(PyObject *tuple, int64_t *to) {
    if (!tuple || !PyTuple_Check(tuple)) return -1;
    const Py_ssize_t n = PyTuple_GET_SIZE(tuple);
    if (n < 1 || n > 4) return -1;
    for (Py_ssize_t i = 0; i < n; ++i) {
        to[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(tuple, i));
        if (to[i] == -1 && PyErr_Occurred()) return -1;
    }
    return (int)n;
}

/* 1 if the object describes an array on the device in the usual way. */
static int read_array(PyObject *array, long device, mr_array *to) {
    int ok = 0;
    PyObject *where = PyObject_CallMethodNoArgs(array, get_device), *dims = NULL, *steps = NULL, *kind = NULL, *at = NULL;
    memset(to, 0, sizeof(*to));
    if (where && PyLong_AsLong(where) == device && (dims = PyObject_GetAttr(array, shape)) &&
        (steps = PyObject_CallMethodNoArgs(array, stride)) && (kind = PyObject_GetAttr(array, dtype)) &&
        (at = PyObject_CallMethodNoArgs(array, data_ptr))) {
        PyObject *code = PyDict_GetItemWithError(codes, kind);
        to->ndim = numbers(dims, to->shape);
        to->data = PyLong_AsVoidPtr(at);
        if (code && to->ndim > 0 && numbers(steps, to->stride) == to->ndim && !PyErr_Occurred()) {
            to->dtype = (int32_t)PyLong_AsLong(code);
            ok = 1;
        }
    }
    Py_XDECREF(where);
    Py_XDECREF(dims);
    Py_XDECREF(steps);
    Py_XDECREF(kind);
    Py_XDECREF(at);
    PyErr_Clear();
    return ok;
}

static int describe_into(PyObject *array, const char *name, long device, mr_array *to) {
    if (read_array(array, device, to)) return 1;
    PyObject *bytes = PyObject_CallFunction(slow, "Osl", array, name, device);
    if (!bytes) return 0;
    const int ok = PyBytes_Check(bytes) && PyBytes_GET_SIZE(bytes) == (Py_ssize_t)sizeof(*to);
    if (ok) memcpy(to, PyBytes_AS_STRING(bytes), sizeof(*to));
    else PyErr_Format(PyExc_ValueError, "%s is not described as an array", name);
    Py_DECREF(bytes);
    return ok;
}

/* describe(array, name, device) -> the mr_array's bytes */
static PyObject *describe(PyObject *self, PyObject *const *args, Py_ssize_t n) {
    (void)self;
    mr_array array;
    if (n != 3) return PyErr_Format(PyExc_TypeError, "describe takes 3 arguments, not %zd", n);
    const char *name = PyUnicode_AsUTF8(args[1]);
    const long device = PyLong_AsLong(args[2]);
    if (!name || PyErr_Occurred() || !describe_into(args[0], name, device, &array)) return NULL;
    return PyBytes_FromStringAndSize((const char *)&array, sizeof(array));
}

/* call(which, context, device, *arrays, *scalars) -> the status; an optional array may be None */
static PyObject *call(PyObject *self, PyObject *const *args, Py_ssize_t n) {
    (void)self;
    mr_array arrays[MOST];
    const mr_array *a[MOST];
    const long which = n > 0 ? PyLong_AsLong(args[0]) : -1;
    if (which < 0 || which >= CALLS || n != 3 + calls[which].arrays + calls[which].scalars)
        return PyErr_Occurred() ? NULL : PyErr_Format(PyExc_TypeError, "no such call");
    mr_context *ctx = PyLong_AsVoidPtr(args[1]);
    const long device = PyLong_AsLong(args[2]);
    if (PyErr_Occurred()) return NULL;
    for (int i = 0; i < calls[which].arrays; ++i) {
        a[i] = args[3 + i] == Py_None ? NULL : &arrays[i];
        if (a[i] && !describe_into(args[3 + i], calls[which].names[i], device, &arrays[i])) return NULL;
    }
    PyObject *const *s = args + 3 + calls[which].arrays;
    int x[3] = {0, 0, 0};
    float scale = 0.f;
    for (int i = 0; i < calls[which].scalars; ++i) {
        if (i == 2 && which != EVICT) scale = (float)PyFloat_AsDouble(s[i]);
        else x[i] = (int)PyLong_AsLong(s[i]);  /* counted in 31 bits by the caller */
        if (PyErr_Occurred()) return NULL;
    }
    typedef const mr_array *A;
    void *f = functions[which];
    int status;
    Py_BEGIN_ALLOW_THREADS
    if (which == APPEND)
        status = ((int (*)(mr_context *, A, A, A, A, A, A, A))f)(ctx, a[0], a[1], a[2], a[3], a[4], a[5], a[6]);
    else if (which == PAGED)
        status = ((int (*)(mr_context *, A, A, A, A, A, A, A, int, int, float))f)(ctx, a[0], a[1], a[2], a[3], a[4], a[5],
                                                                                a[6], x[0], x[1], scale);
    else if (which == WINDOW)
        status = ((int (*)(mr_context *, A, A, A, A, A, A, int, int, float))f)(ctx, a[0], a[1], a[2], a[3], a[4], a[5], x[0],
                                                                             x[1], scale);
    else if (which == EVICT)
        status = ((int (*)(mr_context *, A, A, A, A, A, A, A, A, A, A, A, int, int, int))f)(
            ctx, a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7], a[8], a[9], a[10], x[0], x[1], x[2]);
    else if (which == ROTATED)
        status = ((int (*)(mr_context *, A, A, A, A, A, A, A, A, A, A, A, int))f)(
            ctx, a[0], a[1], a[2], a[3], a[4], a[5], a[6], a[7], a[8], a[9], a[10], x[0]);
    else if (which == READ)
        status = ((int (*)(mr_context *, A, A, A, A, A, A, A))f)(ctx, a[0], a[1], a[2], a[3], a[4], a[5], a[6]);
    else
        status = ((int (*)(mr_context *, A, A, A, A, A, A))f)(ctx, a[0], a[1], a[2], a[3], a[4], a[5]);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(status);
}

/* bind(addresses): of the library's functions, in that order */
static PyObject *bind(PyObject *self, PyObject *const *args, Py_ssize_t n) {
    (void)self;
    if (n != CALLS) return PyErr_Format(PyExc_TypeError, "bind takes %d addresses, not %zd", CALLS, n);
    for (int i = 0; i < CALLS; ++i) functions[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return NULL;
    Py_RETURN_NONE;
}

/* types(codes, slow): the dictionary of the types met, and what to call for the others */
static PyObject *types(PyObject *self, PyObject *const *args, Py_ssize_t n) {
    (void)self;
    if (n != 2 || !PyDict_Check(args[0])) return PyErr_Format(PyExc_TypeError, "types takes a dictionary and a function");
    Py_XSETREF(codes, Py_NewRef(args[0]));
    Py_XSETREF(slow, Py_NewRef(args[1]));
    Py_RETURN_NONE;
}

static PyMethodDef methods[] = {
    {"describe", (PyCFunction)(void (*)(void))describe, METH_FASTCALL, "describe(array, name, device) -> bytes of mr_array"},
    {"call", (PyCFunction)(void (*)(void))call, METH_FASTCALL, "call(which, context, device, *arrays, *scalars) -> status"},
    {"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, "bind(*addresses) of the library's functions"},
    {"types", (PyCFunction)(void (*)(void))types, METH_FASTCALL, "types(codes, slow)"},
    {NULL, NULL, 0, NULL},
};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_pycall", "The array operators' calls from Python.", -1, methods,
                                    NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__pycall(void) {
    PyObject *m = PyModule_Create(&module);
    get_device = PyUnicode_InternFromString("get_device");
    shape = PyUnicode_InternFromString("shape");
    stride = PyUnicode_InternFromString("stride");
    dtype = PyUnicode_InternFromString("dtype");
    data_ptr = PyUnicode_InternFromString("data_ptr");
    if (m && get_device && shape && stride && dtype && data_ptr) return m;
    Py_XDECREF(m);
    return NULL;
}

/* _pycall: the array operators' calls from Python.
 *
 * The operators on arrays of any owner (include/miracle_cuda.h: mr_array) take
 * up to eleven of them, each described by five accessors of a Python object.
 * Read in Python and passed through ctypes, that is most of a small call's time
 * (a one-token attention took the host 17.7 microseconds so, 13.3 through this
 * module); here the accessors are read into the structs and the library's
 * function is called directly.  A type of arrays that offers DLPack's exchange of
 * descriptions in C (version 1, __dlpack_c_exchange_api__, as torch's tensors do)
 * is read by that, one call an array instead of five (an append of 64 rows with
 * their rotation, ten arrays, 11.8 microseconds without and 9.0 so).
 * Everything else of the binding stays in ctypes (_native.py), which also hands over the
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

/* Of DLPack 1: a description of an array, and the table of functions of which one fills it in (0: done). */
typedef struct {
    void *data;
    int32_t device_type, device;
    int32_t ndim;
    uint8_t code, bits;
    uint16_t lanes;
    int64_t *shape, *strides;
    uint64_t byte_offset;
} dl_array;
typedef struct {
    uint32_t major, minor;
    void *earlier, *allocate, *from_object, *to_object;
    int (*describe)(void *object, dl_array *to);
    void *stream;
} dl_functions;
enum { DL_CUDA = 2 };
static PyTypeObject *met;                  /* the type of arrays met last, and its function or NULL */
static int (*met_describe)(void *, dl_array *);
static PyObject *exchange;

/* The type's own function: an heir's accessors may say something else. */
static void meet(PyTypeObject *type) {
    PyObject *capsule = type->tp_dict ? PyDict_GetItemWithError(type->tp_dict, exchange) : NULL;
    const dl_functions *f = NULL;
    if (capsule && PyCapsule_IsValid(capsule, "dlpack_exchange_api")) f = PyCapsule_GetPointer(capsule, "dlpack_exchange_api");
    met_describe = f && f->major == 1 ? f->describe : NULL;
    Py_INCREF(type);
    Py_XSETREF(met, type);
    PyErr_Clear();
}

/* 1 if the object's type describes it as an array on the device by the exchange. */
static int read_exchanged(PyObject *array, long device, mr_array *to) {
    dl_array x;
    if (Py_TYPE(array) != met) meet(Py_TYPE(array));
    if (!met_describe) return 0;
    if (met_describe(array, &x)) {
        PyErr_Clear();
        return 0;
    }
    const int bits = x.lanes == 1 ? x.code << 8 | x.bits : 0;
    const int type = bits == (2 << 8 | 32)   ? MR_DTYPE_F32
                     : bits == (2 << 8 | 16) ? MR_DTYPE_F16
                     : bits == (4 << 8 | 16) ? MR_DTYPE_BF16
                     : bits == (0 << 8 | 32) ? MR_DTYPE_I32
                     : bits == (1 << 8 | 8)  ? MR_DTYPE_U8
                                             : -1;
    if (x.device_type != DL_CUDA || x.device != device || x.ndim < 1 || x.ndim > 4 || !x.strides || type < 0) return 0;
    memset(to, 0, sizeof(*to));
    to->data = x.data ? (char *)x.data + x.byte_offset : NULL;
    to->dtype = type;
    to->ndim = x.ndim;
    memcpy(to->shape, x.shape, sizeof(int64_t) * (size_t)x.ndim);
    memcpy(to->stride, x.strides, sizeof(int64_t) * (size_t)x.ndim);
    return 1;
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
    if (read_exchanged(array, device, to) || read_array(array, device, to)) return 1;
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
    exchange = PyUnicode_InternFromString("__dlpack_c_exchange_api__");
    if (m && exchange && get_device && shape && stride && dtype && data_ptr) return m;
    Py_XDECREF(m);
    return NULL;
}

/*
 * emmyrt._calls: an operator's call from Python, after its first one.
 *
 * Small operators are bound by the host: reading the kind (element type, shape, strides, device) and the address of each
 * operand, comparing the spans that must not overlap and filling in the argument block took 7 us of a 14 us call of nine
 * operands in Python, about as long as the launch itself and torch's own look-up of the stream.  Here a call's kind is
 * looked up in the operator's plans as a tuple; what a plan holds is prepared in Python (emmyrt/operands.py).
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stdint.h>

#define MAX_OPERANDS 16
#define MAX_ARGS 512

typedef int (*entry_fn)(const void *args, int device, uint64_t stream);

typedef struct {
    int i, j;                   /* places: operands, then the operator's own arrays */
    uint64_t span_i, span_j;
    PyObject *meets;            /* called with both addresses where the spans overlap: raises, or allows it */
} Check;

typedef struct {
    PyObject_HEAD
    entry_fn entry;
    Py_ssize_t bytes, operands, own, checks;
    Py_ssize_t offset[MAX_OPERANDS];        /* of the operands' addresses in the argument block */
    uint64_t own_at[MAX_OPERANDS];
    Check *check;
    unsigned char args[MAX_ARGS] __attribute__((aligned(16)));
} Plan;

static PyObject *s_dtype, *s_shape, *s_strides, *s_stride, *s_device, *s_ptr, *s_data_ptr, *array_type;

static void plan_dealloc(PyObject *self) {
    Plan *p = (Plan *)self;
    for (Py_ssize_t k = 0; k < p->checks; ++k) Py_XDECREF(p->check[k].meets);
    PyMem_Free(p->check);
    Py_TYPE(self)->tp_free(self);
}

/* Plan(entry's address, argument block, offsets of the operands' addresses, addresses of the own arrays, checks) */
static PyObject *plan_new(PyTypeObject *type, PyObject *args, PyObject *kw) {
    unsigned long long entry;
    const char *block;
    Py_ssize_t bytes;
    PyObject *offsets, *own, *checks;
    if (kw && PyDict_GET_SIZE(kw)) {
        PyErr_SetString(PyExc_TypeError, "Plan takes no keywords");
        return NULL;
    }
    if (!PyArg_ParseTuple(args, "Ky#O!O!O!", &entry, &block, &bytes, &PyTuple_Type, &offsets, &PyTuple_Type, &own, &PyList_Type, &checks))
        return NULL;
    const Py_ssize_t n = PyTuple_GET_SIZE(offsets), m = PyTuple_GET_SIZE(own), c = PyList_GET_SIZE(checks);
    if (!entry || bytes > MAX_ARGS || n + m > MAX_OPERANDS) {
        PyErr_SetString(PyExc_ValueError, "a plan of too many operands, or without an entry");
        return NULL;
    }
    Plan *p = (Plan *)type->tp_alloc(type, 0);      /* zeroed */
    if (!p) return NULL;
    p->entry = (entry_fn)(uintptr_t)entry;
    p->bytes = bytes, p->operands = n, p->own = m;
    memcpy(p->args, block, (size_t)bytes);
    for (Py_ssize_t k = 0; k < n; ++k) {
        p->offset[k] = PyLong_AsSsize_t(PyTuple_GET_ITEM(offsets, k));
        if (p->offset[k] < 0 || p->offset[k] + 8 > bytes) {
            if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "an offset outside the argument block");
            goto fail;
        }
    }
    for (Py_ssize_t k = 0; k < m; ++k) {
        p->own_at[k] = PyLong_AsUnsignedLongLong(PyTuple_GET_ITEM(own, k));
        if (PyErr_Occurred()) goto fail;
    }
    p->check = PyMem_Calloc((size_t)(c ? c : 1), sizeof(Check));
    if (!p->check) {
        PyErr_NoMemory();
        goto fail;
    }
    for (Py_ssize_t k = 0; k < c; ++k) {
        Check *to = &p->check[k];
        unsigned long long span_i, span_j;
        PyObject *meets;
        if (!PyArg_ParseTuple(PyList_GET_ITEM(checks, k), "iiKKO", &to->i, &to->j, &span_i, &span_j, &meets)) goto fail;
        if (to->i < 0 || to->i >= n + m || to->j < 0 || to->j >= n + m) {
            PyErr_SetString(PyExc_ValueError, "a check of no operand");
            goto fail;
        }
        to->span_i = span_i, to->span_j = span_j;
        to->meets = Py_NewRef(meets);
        p->checks = k + 1;
    }
    return (PyObject *)p;
fail:
    Py_DECREF(p);
    return NULL;
}

static PyTypeObject PlanType = {
    PyVarObject_HEAD_INIT(NULL, 0).tp_name = "emmyrt._calls.Plan",
    .tp_basicsize = sizeof(Plan),
    .tp_dealloc = plan_dealloc,
    .tp_flags = Py_TPFLAGS_DEFAULT,
    .tp_doc = "What calls with operands of one kind have in common.",
    .tp_new = plan_new,
};

static int address(PyObject *number, uint64_t *at) {
    if (!number) return -1;
    *at = PyLong_AsUnsignedLongLong(number);
    Py_DECREF(number);
    return PyErr_Occurred() ? -1 : 0;
}

/* an operand's address, and the four parts of its kind (new references); -1 with an exception */
static int describe(PyObject *x, PyObject **kind, uint64_t *at) {
    const int own = (PyObject *)Py_TYPE(x) == array_type;
    if (!(kind[0] = PyObject_GetAttr(x, s_dtype))) return -1;
    if (!(kind[1] = PyObject_GetAttr(x, s_shape))) return -1;
    if (!(kind[2] = own ? PyObject_GetAttr(x, s_strides) : PyObject_CallMethodNoArgs(x, s_stride))) return -1;
    if (!(kind[3] = PyObject_GetAttr(x, s_device))) return -1;
    return address(own ? PyObject_GetAttr(x, s_ptr) : PyObject_CallMethodNoArgs(x, s_data_ptr), at);
}

/* call(plans, operands, options, device, stream): the entry's status, the call's kind where the plans do not have it, or None where an
 * operand is nothing that has a kind */
static PyObject *call(PyObject *self, PyObject *const *arg, Py_ssize_t nargs) {
    (void)self;
    if (nargs != 5 || !PyDict_Check(arg[0]) || !PyTuple_Check(arg[1])) {
        PyErr_SetString(PyExc_TypeError, "call(plans, operands, options, device, stream)");
        return NULL;
    }
    const Py_ssize_t n = PyTuple_GET_SIZE(arg[1]);
    if (n > MAX_OPERANDS) {
        PyErr_SetString(PyExc_ValueError, "too many operands");
        return NULL;
    }
    const long device = PyLong_AsLong(arg[3]);
    if (device == -1 && PyErr_Occurred()) return NULL;
    const uint64_t stream = PyLong_AsUnsignedLongLong(arg[4]);
    if (stream == (uint64_t)-1 && PyErr_Occurred()) return NULL;

    uint64_t at[2 * MAX_OPERANDS];
    PyObject *key = PyTuple_New(1 + 4 * n);
    if (!key) return NULL;
    PyTuple_SET_ITEM(key, 0, Py_NewRef(arg[2]));
    for (Py_ssize_t k = 0; k < n; ++k) {
        PyObject *x = PyTuple_GET_ITEM(arg[1], k), *kind[4] = {NULL, NULL, NULL, NULL};
        int failed = 0;
        at[k] = 0;
        if (x != Py_None) failed = describe(x, kind, &at[k]);
        for (int i = 0; i < 4; ++i) PyTuple_SET_ITEM(key, 1 + 4 * k + i, kind[i] ? kind[i] : Py_NewRef(Py_None));
        if (failed) {
            Py_DECREF(key);
            if (!PyErr_ExceptionMatches(PyExc_AttributeError) && !PyErr_ExceptionMatches(PyExc_TypeError)) return NULL;
            PyErr_Clear();
            Py_RETURN_NONE;
        }
    }
    PyObject *found = PyDict_GetItemWithError(arg[0], key);
    if (!found) {
        if (!PyErr_Occurred()) return key;
        Py_DECREF(key);
        return NULL;
    }
    Py_DECREF(key);
    if (Py_TYPE(found) != &PlanType || ((Plan *)found)->operands != n) {
        PyErr_SetString(PyExc_TypeError, "not a plan of this call");
        return NULL;
    }
    Plan *p = (Plan *)Py_NewRef(found);
    for (Py_ssize_t k = 0; k < p->own; ++k) at[n + k] = p->own_at[k];
    for (Py_ssize_t k = 0; k < p->checks; ++k) {
        const Check *c = &p->check[k];
        const uint64_t a = at[c->i], b = at[c->j];
        if (a < b + c->span_j && b < a + c->span_i) {
            PyObject *r = PyObject_CallFunction(c->meets, "KK", (unsigned long long)a, (unsigned long long)b);
            if (!r) {
                Py_DECREF(p);
                return NULL;
            }
            Py_DECREF(r);
        }
    }
    unsigned char args[MAX_ARGS] __attribute__((aligned(16)));
    memcpy(args, p->args, (size_t)p->bytes);
    for (Py_ssize_t k = 0; k < n; ++k) memcpy(args + p->offset[k], &at[k], 8);
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = p->entry(args, (int)device, stream);
    Py_END_ALLOW_THREADS
    Py_DECREF(p);
    return PyLong_FromLong(status);
}

/* set_array(type): operands of this type have `strides` and `ptr`, others `stride()` and `data_ptr()` */
static PyObject *set_array(PyObject *self, PyObject *type) {
    (void)self;
    Py_XSETREF(array_type, Py_NewRef(type));
    Py_RETURN_NONE;
}

static PyMethodDef methods[] = {{"call", (PyCFunction)(void (*)(void))call, METH_FASTCALL, NULL},
                                {"set_array", set_array, METH_O, NULL},
                                {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, .m_name = "_calls", .m_size = -1, .m_methods = methods};

PyMODINIT_FUNC PyInit__calls(void) {
    if (PyType_Ready(&PlanType) < 0) return NULL;
    const struct { PyObject **to; const char *text; } names[] = {{&s_dtype, "dtype"}, {&s_shape, "shape"}, {&s_strides, "strides"},
        {&s_stride, "stride"}, {&s_device, "device"}, {&s_ptr, "ptr"}, {&s_data_ptr, "data_ptr"}};
    for (size_t i = 0; i < sizeof names / sizeof *names; ++i)
        if (!(*names[i].to = PyUnicode_InternFromString(names[i].text))) return NULL;
    PyObject *m = PyModule_Create(&module);
    if (m && PyModule_AddObjectRef(m, "Plan", (PyObject *)&PlanType) < 0) Py_CLEAR(m);
    return m;
}

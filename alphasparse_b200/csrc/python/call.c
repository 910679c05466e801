/* The calls of asp_spmv and of block-sparse matrices (asp_b200_block8.h) from Python (the module alphasparse_b200._call).
 *
 * A small SpMV takes the GPU less time than its launch takes the host (2.0 us on the measured machine), and ctypes spends 0.7 us more on
 * converting six arguments. This binding is made once per plan group and converts two: 0.1 us. It holds addresses of what the
 * group and its context hold themselves (the context's handle, the array of plans) and reads them at every call, so a context or a
 * group that has been closed is NULL to asp_spmv, as it is through ctypes. The GIL is released meanwhile: a launch waits where the
 * stream's queue is full. asp_block8_apply, of ten arguments, is bound the same way (1.2 us by ctypes), and the other calls of asp_b200_block8.h that launch
 * something. */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stddef.h>
#include <string.h>

typedef int (*spmv_fn)(void *ctx, void *const *plans, int n_plans, const void *d_x, void *d_y, int zero_y);

typedef struct
{
    PyObject_HEAD
    vectorcallfunc vectorcall;
    spmv_fn fn;
    void **ctx; /* where the handle is */
    void **plans;
    int n;
} Spmv;

/* (d_x, d_y, zero_y as asp_spmv takes it) -> status; TypeError where a pointer is no int */
static PyObject *spmv_call(PyObject *self, PyObject *const *args, size_t nargsf, PyObject *kwnames)
{
    Spmv *s = (Spmv *)self;
    if (PyVectorcall_NARGS(nargsf) != 3 || (kwnames && PyTuple_GET_SIZE(kwnames)) || !PyLong_Check(args[0]) || !PyLong_Check(args[1]) || !PyLong_Check(args[2]))
    {
        PyErr_SetString(PyExc_TypeError, "three ints are wanted");
        return NULL;
    }
    /* as ctypes takes ints for pointers: modulo 2^64 */
    const unsigned long long x = PyLong_AsUnsignedLongLongMask(args[0]), y = PyLong_AsUnsignedLongLongMask(args[1]);
    const long zero_y = PyLong_AsLong(args[2]);
    if (PyErr_Occurred()) return NULL;
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = s->fn(*s->ctx, s->plans, s->n, (const void *)(size_t)x, (void *)(size_t)y, (int)zero_y);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(status);
}

static PyObject *spmv_new(PyTypeObject *type, PyObject *args, PyObject *kw)
{
    unsigned long long fn, ctx, plans;
    int n;
    (void)kw;
    if (!PyArg_ParseTuple(args, "KKKi", &fn, &ctx, &plans, &n)) return NULL;
    Spmv *s = (Spmv *)type->tp_alloc(type, 0);
    if (!s) return NULL;
    s->vectorcall = spmv_call;
    s->fn = (spmv_fn)(size_t)fn;
    s->ctx = (void **)(size_t)ctx;
    s->plans = (void **)(size_t)plans;
    s->n = n;
    return (PyObject *)s;
}

static PyTypeObject SpmvType = {
    PyVarObject_HEAD_INIT(NULL, 0).tp_name = "alphasparse_b200._call.Spmv",
    .tp_doc = "Spmv(address of asp_spmv, address of the context's handle, address of the plans, number of plans)",
    .tp_basicsize = sizeof(Spmv),
    .tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_HAVE_VECTORCALL,
    .tp_new = spmv_new,
    .tp_call = PyVectorcall_Call,
    .tp_vectorcall_offset = offsetof(Spmv, vectorcall),
};

typedef int (*apply_fn)(void *ctx, const void *m, int transposed, const void *d_x, int x_dtype, unsigned long long n, unsigned long long ldx, void *d_y, int y_dtype, unsigned long long ldy);

typedef struct
{
    PyObject_HEAD
    vectorcallfunc vectorcall;
    apply_fn fn;
    void **ctx, **matrix; /* where the handles are */
} Apply;

/* (transposed, d_x, x_dtype, n, ldx, d_y, y_dtype, ldy) -> status; TypeError where one is no int */
static PyObject *apply_call(PyObject *self, PyObject *const *args, size_t nargsf, PyObject *kwnames)
{
    Apply *s = (Apply *)self;
    int ints = PyVectorcall_NARGS(nargsf) == 8 && !(kwnames && PyTuple_GET_SIZE(kwnames));
    for (int i = 0; ints && i < 8; i++) ints = PyLong_Check(args[i]);
    if (!ints)
    {
        PyErr_SetString(PyExc_TypeError, "eight ints are wanted");
        return NULL;
    }
    unsigned long long v[8];
    for (int i = 0; i < 8; i++) v[i] = PyLong_AsUnsignedLongLongMask(args[i]);
    if (PyErr_Occurred()) return NULL;
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = s->fn(*s->ctx, *s->matrix, (int)v[0], (const void *)(size_t)v[1], (int)v[2], v[3], v[4], (void *)(size_t)v[5], (int)v[6], v[7]);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(status);
}

static PyObject *apply_new(PyTypeObject *type, PyObject *args, PyObject *kw)
{
    unsigned long long fn, ctx, matrix;
    (void)kw;
    if (!PyArg_ParseTuple(args, "KKK", &fn, &ctx, &matrix)) return NULL;
    Apply *s = (Apply *)type->tp_alloc(type, 0);
    if (!s) return NULL;
    s->vectorcall = apply_call;
    s->fn = (apply_fn)(size_t)fn;
    s->ctx = (void **)(size_t)ctx;
    s->matrix = (void **)(size_t)matrix;
    return (PyObject *)s;
}

static PyTypeObject ApplyType = {
    PyVarObject_HEAD_INIT(NULL, 0).tp_name = "alphasparse_b200._call.Apply",
    .tp_doc = "Apply(address of asp_block8_apply, address of the context's handle, address of the matrix's handle)",
    .tp_basicsize = sizeof(Apply),
    .tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_HAVE_VECTORCALL,
    .tp_new = apply_new,
    .tp_call = PyVectorcall_Call,
    .tp_vectorcall_offset = offsetof(Apply, vectorcall),
};

/* the others: (ctx, handle, ...), by their arguments behind the two */
enum
{
    ROWS8_QUANTIZE,
    ROWS8_RESTORE,
    BLOCK8_SET_VALUES,
    BLOCK8_GET_VALUES,
    BLOCK8_PRODUCT,
    BLOCK8_GRADIENT,
    N_CALLS
};
static const char *const call_names[N_CALLS] = {"asp_rows8_quantize", "asp_rows8_restore", "asp_block8_set_values", "asp_block8_get_values", "asp_block8_product", "asp_block8_gradient"};
static const int call_args[N_CALLS] = {4, 3, 2, 1, 5, 6};

typedef struct
{
    PyObject_HEAD
    vectorcallfunc vectorcall;
    int which;
    void *fn;
    void **ctx, **handle; /* where the handles are */
} Bound;

static int bound_run(const Bound *b, const unsigned long long *v)
{
    typedef unsigned long long u64;
    void *ctx = *b->ctx, *h = *b->handle;
#define P(i) ((void *)(size_t)v[i])
    switch (b->which)
    {
    case ROWS8_QUANTIZE: return ((int (*)(void *, void *, const void *, int, u64, u64))b->fn)(ctx, h, P(0), (int)v[1], v[2], v[3]);
    case ROWS8_RESTORE: return ((int (*)(void *, const void *, void *, int, u64))b->fn)(ctx, h, P(0), (int)v[1], v[2]);
    case BLOCK8_SET_VALUES: return ((int (*)(void *, void *, const void *, int))b->fn)(ctx, h, P(0), (int)v[1]);
    case BLOCK8_GET_VALUES: return ((int (*)(void *, const void *, float *))b->fn)(ctx, h, (float *)P(0));
    case BLOCK8_PRODUCT: return ((int (*)(void *, const void *, int, const void *, void *, int, u64))b->fn)(ctx, h, (int)v[0], P(1), P(2), (int)v[3], v[4]);
    default: return ((int (*)(void *, const void *, const void *, const void *, int, u64, float *, int))b->fn)(ctx, h, P(0), P(1), (int)v[2], v[3], (float *)P(4), (int)v[5]);
    }
#undef P
}

/* (the arguments behind the handles) -> status; TypeError where one is no int */
static PyObject *bound_call(PyObject *self, PyObject *const *args, size_t nargsf, PyObject *kwnames)
{
    Bound *b = (Bound *)self;
    const int n = call_args[b->which];
    int ints = PyVectorcall_NARGS(nargsf) == n && !(kwnames && PyTuple_GET_SIZE(kwnames));
    for (int i = 0; ints && i < n; i++) ints = PyLong_Check(args[i]);
    if (!ints)
    {
        PyErr_Format(PyExc_TypeError, "%d ints are wanted", n);
        return NULL;
    }
    unsigned long long v[8];
    for (int i = 0; i < n; i++) v[i] = PyLong_AsUnsignedLongLongMask(args[i]);
    if (PyErr_Occurred()) return NULL;
    int status;
    Py_BEGIN_ALLOW_THREADS
    status = bound_run(b, v);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(status);
}

static PyObject *bound_new(PyTypeObject *type, PyObject *args, PyObject *kw)
{
    const char *name;
    unsigned long long fn, ctx, handle;
    int which = 0;
    (void)kw;
    if (!PyArg_ParseTuple(args, "sKKK", &name, &fn, &ctx, &handle)) return NULL;
    while (which < N_CALLS && strcmp(call_names[which], name)) which++;
    if (which == N_CALLS) return PyErr_Format(PyExc_ValueError, "no call %s", name);
    Bound *b = (Bound *)type->tp_alloc(type, 0);
    if (!b) return NULL;
    b->vectorcall = bound_call;
    b->which = which;
    b->fn = (void *)(size_t)fn;
    b->ctx = (void **)(size_t)ctx;
    b->handle = (void **)(size_t)handle;
    return (PyObject *)b;
}

static PyTypeObject BoundType = {
    PyVarObject_HEAD_INIT(NULL, 0).tp_name = "alphasparse_b200._call.Bound",
    .tp_doc = "Bound(name of a call, its address, address of the context's handle, address of the handle it is for)",
    .tp_basicsize = sizeof(Bound),
    .tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_HAVE_VECTORCALL,
    .tp_new = bound_new,
    .tp_call = PyVectorcall_Call,
    .tp_vectorcall_offset = offsetof(Bound, vectorcall),
};

static PyModuleDef module = {PyModuleDef_HEAD_INIT, .m_name = "_call", .m_doc = "asp_spmv and the calls of asp_b200_block8.h without ctypes", .m_size = -1};

PyMODINIT_FUNC PyInit__call(void)
{
    if (PyType_Ready(&SpmvType) < 0 || PyType_Ready(&ApplyType) < 0 || PyType_Ready(&BoundType) < 0) return NULL;
    PyObject *m = PyModule_Create(&module);
    if (m && (PyModule_AddObjectRef(m, "Spmv", (PyObject *)&SpmvType) < 0 || PyModule_AddObjectRef(m, "Apply", (PyObject *)&ApplyType) < 0 ||
              PyModule_AddObjectRef(m, "Bound", (PyObject *)&BoundType) < 0))
    {
        Py_DECREF(m);
        return NULL;
    }
    return m;
}

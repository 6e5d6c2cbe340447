/*
 * ckq_tensors.cpp - the calls that parity.py's fp8 and experts' front-ends make when nothing is wrong with their tensors, as a CPython module: it
 * reads types, shapes, strides and devices from the tensors themselves, where Python pays 0.06 us for each, and calls ckq_call_dev on the current
 * stream.  A call it does not take (NOT_TAKEN) has changed nothing; parity.py then looks at the same tensors and says why.  Every check here is made
 * there too, and in the library behind both. `built_for` names the torch and the Python it was compiled for (CKQ_BUILT_FOR, from the Makefile):
 * parity.py uses it with no others.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>
#include <c10/hip/HIPStream.h>
#include <cstdint>
#include <initializer_list>

namespace {

constexpr long NOT_TAKEN = -1000;
int (*g_call)(const void *) = nullptr;      /* ckq_call_dev of the library that the process has loaded */

/* The numbers of ckq_call_dev (ckernel_quant_hip.h). */
enum { QUANTIZE, DEQUANTIZE, SWIGLU, GEMM, EXPERTS, SORT, GATHER, GATHER_F8, COMBINE, BACKWARD };

struct Call {
    PyObject *const *args;
    Py_ssize_t n;
    int dev;
    bool ok = true;

    /* The i-th argument as a tensor on the current device; not one: the call is not taken. */
    const at::Tensor *tensor(Py_ssize_t i)
    {
        if (i >= n || !THPVariable_Check(args[i])) { ok = false; return nullptr; }
        const at::Tensor &t = THPVariable_Unpack(args[i]);
        if (!t.is_cuda() || t.get_device() != dev || t.layout() != at::kStrided) { ok = false; return nullptr; }
        return &t;
    }
};

/* Whether the i-th argument is None. */
bool args_none(const Call &c, Py_ssize_t i) { return i < c.n && c.args[i] == Py_None; }

int64_t address(const at::Tensor *t) { return (int64_t)(uintptr_t)t->data_ptr(); }

/* CKDataType of a tensor of floats; -1: none. */
int kind(const at::Tensor *t)
{
    switch (t->scalar_type()) {
    case at::kFloat:    return 0;
    case at::kBFloat16: return 1;
    case at::kHalf:     return 2;
    default:            return -1;
    }
}

struct Rows { int64_t n = 0, k = 0, ld = 0; bool ok = false; };

/* Rows whose elements lie side by side, sizes within 31 bits; a single row's pitch is its length. */
Rows rows(const at::Tensor *t, int from = 0)
{
    Rows r;
    if (!t || t->dim() != from + 2) return r;
    r.n = t->size(from);
    r.k = t->size(from + 1);
    r.ld = r.n > 1 ? t->stride(from) : r.k;
    r.ok = ((r.n | r.k) >> 31) == 0 && (r.k <= 1 || t->stride(from + 1) == 1);
    return r;
}
bool same(const Rows &a, const Rows &b) { return a.ok && b.ok && a.n == b.n && a.k == b.k; }
bool f8(const at::Tensor *t) { return t && t->scalar_type() == at::kFloat8_e4m3fn; }
int64_t groups(int64_t k) { return (k + 127) / 128; }

/* The pitch of scales [rows, groups], the first index fastest; 0: not such. */
int64_t side(const at::Tensor *t, int64_t n, int64_t g)
{
    if (!t || t->scalar_type() != at::kFloat || t->dim() != 2 || t->size(0) != n || t->size(1) != g) return 0;
    const int64_t ld = g == 1 ? n : t->stride(1);
    return (n == 1 || t->stride(0) == 1) && ld >= n ? ld : 0;
}
bool whole(const at::Tensor *t, at::ScalarType type, std::initializer_list<int64_t> shape)
{
    if (!t || t->scalar_type() != type || !t->is_contiguous() || t->dim() != (int64_t)shape.size()) return false;
    int64_t i = 0;
    for (int64_t s : shape)
        if (t->size(i++) != s) return false;
    return true;
}
int64_t sixteen(int64_t k) { return (k + 15) / 16 * 16; }

/* position [tokens, choices]; false: not such. */
bool places(const at::Tensor *t, int64_t &tokens, int64_t &choices)
{
    if (!t || t->dim() != 2 || t->scalar_type() != at::kInt || !t->is_contiguous()) return false;
    tokens = t->size(0);
    choices = t->size(1);
    return ((tokens | choices) >> 31) == 0;
}

template <class F>
PyObject *guarded(PyObject *const *args, Py_ssize_t n, F &&fill)
{
    long rc = NOT_TAKEN;
    try {
        if (g_call) {
            Call c{args, n, (int)c10::hip::current_device()};
            int64_t a[21] = {0};
            if (fill(c, a) && c.ok) {
                void *stream = (void *)c10::hip::getCurrentHIPStream((c10::DeviceIndex)c.dev).stream();
                static const unsigned char arguments[] = {10, 10, 11, 16, 20, 8, 11, 13, 12, 15};
                a[arguments[a[0]]] = (int64_t)(uintptr_t)stream;      /* the last argument of each */
                Py_BEGIN_ALLOW_THREADS
                rc = g_call(a);
                Py_END_ALLOW_THREADS
            }
        }
    } catch (...) {
        PyErr_Clear();
        rc = NOT_TAKEN;
    }
    return PyLong_FromLong(rc);
}

#define CALL(name) PyObject *name(PyObject *, PyObject *const *args, Py_ssize_t nargs)
#define PUT(...)                                                                                     \
    do {                                                                                             \
        const int64_t v[] = {__VA_ARGS__};                                                           \
        for (size_t i = 0; i < sizeof v / sizeof v[0]; ++i) a[i] = v[i];                             \
    } while (0)

CALL(quantize)                              /* x, q, scale */
{
    return guarded(args, nargs, [](Call &c, int64_t *a) {
        const at::Tensor *x = c.tensor(0), *q = c.tensor(1), *s = c.tensor(2);
        if (!c.ok) return false;
        const Rows rx = rows(x), rq = rows(q);
        const int64_t lds = side(s, rx.n, groups(rx.k));
        if (!same(rx, rq) || !f8(q) || kind(x) < 0 || !lds) return false;
        PUT(QUANTIZE, kind(x), address(x), rx.ld, address(q), rq.ld, address(s), lds, rx.n, rx.k);
        return true;
    });
}

CALL(dequantize)                            /* q, scale, y */
{
    return guarded(args, nargs, [](Call &c, int64_t *a) {
        const at::Tensor *q = c.tensor(0), *s = c.tensor(1), *y = c.tensor(2);
        if (!c.ok) return false;
        const Rows rq = rows(q), ry = rows(y);
        const int64_t lds = side(s, rq.n, groups(rq.k));
        if (!same(rq, ry) || !f8(q) || kind(y) < 0 || !lds) return false;
        PUT(DEQUANTIZE, address(q), rq.ld, address(s), lds, kind(y), address(y), ry.ld, rq.n, rq.k);
        return true;
    });
}

CALL(swiglu)                                /* gate, up, q, scale */
{
    return guarded(args, nargs, [](Call &c, int64_t *a) {
        const at::Tensor *g = c.tensor(0), *u = c.tensor(1), *q = c.tensor(2), *s = c.tensor(3);
        if (!c.ok) return false;
        const Rows rg = rows(g), ru = rows(u), rq = rows(q);
        const int64_t lds = side(s, rg.n, groups(rg.k));
        if (!same(rg, ru) || !same(rg, rq) || rg.ld != ru.ld || !f8(q) || kind(g) < 0 || g->scalar_type() != u->scalar_type() || !lds) return false;
        PUT(SWIGLU, kind(g), address(g), address(u), rg.ld, address(q), rq.ld, address(s), lds, rg.n, rg.k);
        return true;
    });
}

CALL(gemm)                                  /* a, sa, b, sb, bias or None, c */
{
    return guarded(args, nargs, [](Call &c, int64_t *a) {
        const at::Tensor *x = c.tensor(0), *sa = c.tensor(1), *w = c.tensor(2), *sb = c.tensor(3), *o = c.tensor(5);
        const at::Tensor *bias = args_none(c, 4) ? nullptr : c.tensor(4);
        if (!c.ok) return false;
        const Rows rx = rows(x), rw = rows(w), ro = rows(o);
        if (!rx.ok || !rw.ok || !ro.ok || rx.k != rw.k || ro.n != rx.n || ro.k != rw.n || !f8(x) || !f8(w) || kind(o) < 0) return false;
        const int64_t G = groups(rx.k), ldsa = side(sa, rx.n, G);
        if (!ldsa || !whole(sb, at::kFloat, {groups(rw.n), G}) || (bias && !whole(bias, at::kFloat, {rw.n}))) return false;
        PUT(GEMM, address(x), rx.n > 1 ? rx.ld : sixteen(rx.k), address(sa), ldsa, address(w), rw.n > 1 ? rw.ld : sixteen(rw.k), address(sb), G, bias ? address(bias) : 0, kind(o), address(o), ro.ld, rx.n,
            rw.n, rx.k);
        return true;
    });
}

CALL(experts)                               /* a, sa, b, sb, offsets, bias or None, c */
{
    return guarded(args, nargs, [](Call &c, int64_t *a) {
        const at::Tensor *x = c.tensor(0), *sa = c.tensor(1), *w = c.tensor(2), *sb = c.tensor(3), *offsets = c.tensor(4), *o = c.tensor(6);
        const at::Tensor *bias = args_none(c, 5) ? nullptr : c.tensor(5);
        if (!c.ok) return false;
        const Rows rx = rows(x), rw = rows(w, 1), ro = rows(o);
        if (!rx.ok || !rw.ok || !ro.ok || rx.k != rw.k || ro.n != rx.n || ro.k != rw.n || !f8(x) || !f8(w) || kind(o) < 0) return false;
        const int64_t E = w->size(0), G = groups(rx.k), blocks = groups(rw.n), ldsa = side(sa, rx.n, G);
        if (E >> 31 || !ldsa || !whole(sb, at::kFloat, {E, blocks, G}) || !whole(offsets, at::kInt, {E + 1}) || (bias && !whole(bias, at::kFloat, {E, rw.n}))) return false;
        PUT(EXPERTS, address(x), rx.n > 1 ? rx.ld : sixteen(rx.k), address(sa), ldsa, address(w), rw.n > 1 ? rw.ld : sixteen(rw.k), E > 1 ? w->stride(0) : 0, address(sb), G, blocks * G,
            bias ? address(bias) : 0, address(offsets), E, kind(o), address(o), ro.ld, rx.n, rw.n, rx.k);
        return true;
    });
}

CALL(sort)                                  /* ids, experts, offsets, order, position */
{
    return guarded(args, nargs, [](Call &c, int64_t *a) {
        const at::Tensor *ids = c.tensor(0), *offsets = c.tensor(2), *order = c.tensor(3), *position = c.tensor(4);
        if (!c.ok || !PyLong_CheckExact(c.args[1])) return false;
        int beyond = 0;
        const int64_t E = PyLong_AsLongLongAndOverflow(c.args[1], &beyond);
        int64_t T, n;
        if (beyond || E < 1 || E >> 31 || !places(ids, T, n) || !whole(offsets, at::kInt, {E + 1}) || !whole(order, at::kInt, {T * n}) || !whole(position, at::kInt, {T, n})) return false;
        PUT(SORT, address(ids), T, n, E, address(offsets), address(order), address(position));
        return true;
    });
}

CALL(gather)                                /* x, position, y */
{
    return guarded(args, nargs, [](Call &c, int64_t *a) {
        const at::Tensor *x = c.tensor(0), *p = c.tensor(1), *y = c.tensor(2);
        if (!c.ok) return false;
        const Rows rx = rows(x), ry = rows(y);
        int64_t T, n;
        if (!rx.ok || !ry.ok || !places(p, T, n) || rx.n != T || ry.k != rx.k || kind(x) < 0 || x->scalar_type() != y->scalar_type()) return false;
        PUT(GATHER, kind(x), address(x), rx.ld, address(p), address(y), ry.ld, T, n, ry.n, rx.k);
        return true;
    });
}

CALL(gather_f8)                             /* x, position, q, scale */
{
    return guarded(args, nargs, [](Call &c, int64_t *a) {
        const at::Tensor *x = c.tensor(0), *p = c.tensor(1), *q = c.tensor(2), *s = c.tensor(3);
        if (!c.ok) return false;
        const Rows rx = rows(x), rq = rows(q);
        int64_t T, n;
        if (!rx.ok || !rq.ok || !places(p, T, n) || rx.n != T || rq.k != rx.k || kind(x) < 0 || !f8(q)) return false;
        const int64_t lds = side(s, rq.n, groups(rx.k));
        if (!lds) return false;
        PUT(GATHER_F8, kind(x), address(x), rx.ld, address(p), address(q), rq.ld, address(s), lds, T, n, rq.n, rx.k);
        return true;
    });
}

CALL(combine)                               /* y, position, weights or None, out */
{
    return guarded(args, nargs, [](Call &c, int64_t *a) {
        const at::Tensor *y = c.tensor(0), *p = c.tensor(1), *o = c.tensor(3);
        const at::Tensor *w = args_none(c, 2) ? nullptr : c.tensor(2);
        if (!c.ok) return false;
        const Rows ry = rows(y), ro = rows(o);
        int64_t T, n;
        if (!ry.ok || !ro.ok || !places(p, T, n) || ro.n != T || ro.k != ry.k || kind(y) < 0 || y->scalar_type() != o->scalar_type() || (w && !whole(w, at::kFloat, {T, n}))) return false;
        PUT(COMBINE, kind(y), address(y), ry.ld, address(p), w ? address(w) : 0, address(o), ro.ld, T, n, ry.n, ry.k);
        return true;
    });
}

CALL(backward)                              /* dout, y, position, weights, dy, dweights */
{
    return guarded(args, nargs, [](Call &c, int64_t *a) {
        const at::Tensor *d = c.tensor(0), *y = c.tensor(1), *p = c.tensor(2), *w = c.tensor(3), *dy = c.tensor(4), *dw = c.tensor(5);
        if (!c.ok) return false;
        const Rows rd = rows(d), ry = rows(y), rg = rows(dy);
        int64_t T, n;
        if (!rd.ok || !same(ry, rg) || !places(p, T, n) || rd.n != T || rd.k != ry.k || kind(d) < 0 || d->scalar_type() != y->scalar_type() || d->scalar_type() != dy->scalar_type() ||
            !whole(w, at::kFloat, {T, n}) || !whole(dw, at::kFloat, {T, n})) return false;
        PUT(BACKWARD, kind(d), address(d), rd.ld, address(y), ry.ld, address(p), address(w), address(dy), rg.ld, address(dw), T, n, ry.n, ry.k);
        return true;
    });
}

/* The address of ckq_call_dev; 0: calls are not taken. */
PyObject *bind(PyObject *, PyObject *address)
{
    const unsigned long long p = PyLong_AsUnsignedLongLong(address);
    if (PyErr_Occurred()) return nullptr;
    g_call = (int (*)(const void *))(uintptr_t)p;
    Py_RETURN_NONE;
}

#define METHOD(name) {#name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(quantize), METHOD(dequantize), METHOD(swiglu), METHOD(gemm), METHOD(experts), METHOD(sort), METHOD(gather), METHOD(gather_f8), METHOD(combine), METHOD(backward),
                         {"bind", bind, METH_O, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "ckq_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_ckq_tensors(void)
{
    PyObject *m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "built_for", CKQ_BUILT_FOR) < 0) Py_CLEAR(m);
    return m;
}

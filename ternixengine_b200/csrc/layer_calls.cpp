// The Python entry points of the layer operators for the case that a decode loop repeats: every operand given, on the
// current device, well formed.  Then a call is one pass over the operands' attributes and the C ABI entry, in 4 to 5 us
// instead of 7 (the launch itself takes 2.4).  Anything else -- an output to allocate, another device, any operand that
// does not check -- returns None and is left to the Python code of the package, which allocates, guards or raises; this
// file raises nothing itself and knows no error messages.
//
// Plain CPython API; tensors are read through the methods that Python code would use, torch's objects come in through
// setup(), the library's entry points as addresses, so nothing is linked but Python.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cstdint>
#include <cstring>

#include "ternix_b200.h"

namespace {

PyObject *s_dtype, *s_shape, *s_data_ptr, *s_get_device, *s_is_contiguous, *s_stride, *s_dim, *s_numel;
PyObject* g_types[5] = {};                 // float32, bfloat16, float16, int8, uint8: index = dtype code for the first three
PyObject *g_current_device = nullptr, *g_raw_stream = nullptr, *g_tensor = nullptr;
decltype(&ternix_b200_rmsnorm_quantize) g_norm = nullptr;
decltype(&ternix_b200_glu_quantize) g_glu = nullptr;
decltype(&ternix_b200_matmul_fused) g_mm = nullptr;
constexpr int kI8 = 3, kU8 = 4;

// A new reference that is dropped at the end of the scope.
struct Ref {
    PyObject* o;
    explicit Ref(PyObject* p) : o(p) {}
    ~Ref() { Py_XDECREF(o); }
    Ref(const Ref&) = delete;
    Ref& operator=(const Ref&) = delete;
};

bool as_ll(PyObject* o, long long* v) {
    if (!o || !PyLong_Check(o)) return false;
    *v = PyLong_AsLongLong(o);
    return !(*v == -1 && PyErr_Occurred());
}
bool call_ll(PyObject* t, PyObject* name, long long* v) {
    Ref r(PyObject_CallMethodNoArgs(t, name));
    return as_ll(r.o, v);
}
bool call_true(PyObject* t, PyObject* name) {
    Ref r(PyObject_CallMethodNoArgs(t, name));
    return r.o == Py_True;
}
int type_of(PyObject* t) {
    Ref r(PyObject_GetAttr(t, s_dtype));
    for (int i = 0; r.o && i < 5; ++i)
        if (r.o == g_types[i]) return i;
    return -1;
}
bool pair_of(PyObject* tuple, long long* a, long long* b) {
    return tuple && PyTuple_Check(tuple) && PyTuple_GET_SIZE(tuple) == 2 && as_ll(PyTuple_GET_ITEM(tuple, 0), a) &&
           as_ll(PyTuple_GET_ITEM(tuple, 1), b);
}
bool on(PyObject* t, long long dev) {
    long long d;
    return call_ll(t, s_get_device, &d) && d == dev;
}
bool address(PyObject* t, void** p) {
    Ref r(PyObject_CallMethodNoArgs(t, s_data_ptr));
    if (!r.o || !PyLong_Check(r.o)) return false;
    *p = PyLong_AsVoidPtr(r.o);
    return !PyErr_Occurred();
}

struct Rows {
    void* p = nullptr;
    long long ld = 0;
};
// A row-major operand of the given type and sizes with unit column stride.
bool rows(PyObject* t, int type, long long dev, long long M, long long K, Rows* out) {
    if (type_of(t) != type || !on(t, dev)) return false;
    long long m, k;
    {
        Ref shape(PyObject_GetAttr(t, s_shape));
        if (!pair_of(shape.o, &m, &k) || m != M || k != K) return false;
    }
    out->ld = K;
    if (!call_true(t, s_is_contiguous)) {
        if (PyErr_Occurred()) return false;
        long long ld, inner;
        Ref stride(PyObject_CallMethodNoArgs(t, s_stride));
        if (!pair_of(stride.o, &ld, &inner) || (inner != 1 && K > 1)) return false;
        if (M > 1) {
            if (ld < K) return false;
            out->ld = ld;
        }
    }
    return address(t, &out->p);
}
// A contiguous vector; its type has to be `type` or float32 (type < 0: float32, bfloat16 or float16).
bool vec(PyObject* t, int type, long long dev, long long n, void** p, int* got) {
    const int ty = type_of(t);
    if (ty < 0 || ty > 2 || (type >= 0 && ty != type && ty != 0)) return false;
    long long d, c;
    if (!on(t, dev) || !call_ll(t, s_dim, &d) || d != 1 || !call_ll(t, s_numel, &c) || c != n || !call_true(t, s_is_contiguous)) return false;
    *got = ty;
    return address(t, p);
}
bool shape_of(PyObject* t, long long* M, long long* K) {
    Ref shape(PyObject_GetAttr(t, s_shape));
    return pair_of(shape.o, M, K);
}
// The device's current stream, if the device is the current one.
bool stream_of(PyObject* dev_obj, long long dev, void** st) {
    Ref cur(PyObject_CallNoArgs(g_current_device));
    long long c;
    if (!as_ll(cur.o, &c) || c != dev) return false;
    Ref s(PyObject_CallOneArg(g_raw_stream, dev_obj));
    if (!s.o || !PyLong_Check(s.o)) return false;
    *st = PyLong_AsVoidPtr(s.o);
    return !PyErr_Occurred();
}
// None, with whatever went wrong forgotten: the caller's Python code finds out for itself.
PyObject* leave() {
    PyErr_Clear();
    Py_RETURN_NONE;
}
bool fits(long long a, long long b) { return a <= 0x7fffffff && b <= 0x7fffffff; }
bool quantized(PyObject* out, PyObject* scale, long long dev, long long M, long long K, void** q, void** s) {
    Rows r;
    int ty;
    if (!rows(out, kI8, dev, M, K, &r) || r.ld != K || !call_true(out, s_is_contiguous)) return false;
    *q = r.p;
    return vec(scale, 0, dev, M, s, &ty);
}

// rmsnorm_quantize(x, weight, residual, eps, out, row_scale, residual_out) -> status or None
PyObject* norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 7 || !g_norm) return leave();
    PyObject *x = a[0], *weight = a[1], *residual = a[2], *h = a[6];
    if (!PyFloat_Check(a[3]) || (residual == Py_None) != (h == Py_None)) return leave();
    const int type = type_of(x);
    if (type < 0 || type > 2) return leave();
    Ref dev_obj(PyObject_CallMethodNoArgs(x, s_get_device));
    long long dev, M, K;
    if (!as_ll(dev_obj.o, &dev) || dev < 0 || !shape_of(x, &M, &K) || !fits(M, K)) return leave();
    Rows rx, rr, rh;
    void *w = nullptr, *q, *s, *st;
    int w_type = 0;
    if (!rows(x, type, dev, M, K, &rx) || !quantized(a[4], a[5], dev, M, K, &q, &s)) return leave();
    if (weight != Py_None && !vec(weight, type, dev, K, &w, &w_type)) return leave();
    if (residual != Py_None && (!rows(residual, type, dev, M, K, &rr) || !rows(h, type, dev, M, K, &rh))) return leave();
    if (!stream_of(dev_obj.o, dev, &st)) return leave();
    const float eps = static_cast<float>(PyFloat_AS_DOUBLE(a[3]));
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = g_norm(rx.p, rx.ld, rr.p, rr.ld, type, w, w_type, eps, rh.p, rh.ld, static_cast<int8_t*>(q), static_cast<float*>(s),
                static_cast<int>(M), static_cast<int>(K), st);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

// glu_quantize(gate, up, activation code, weight, eps or None, out, row_scale) -> status or None
PyObject* glu(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 7 || !g_glu) return leave();
    PyObject *gate = a[0], *weight = a[3];
    long long act, dev, M, K;
    const bool normed = a[4] != Py_None;
    if (!as_ll(a[2], &act) || (normed && !PyFloat_Check(a[4])) || (weight != Py_None && !normed)) return leave();
    const int type = type_of(gate);
    if (type < 0 || type > 2) return leave();
    Ref dev_obj(PyObject_CallMethodNoArgs(gate, s_get_device));
    if (!as_ll(dev_obj.o, &dev) || dev < 0 || !shape_of(gate, &M, &K) || !fits(M, K)) return leave();
    Rows rg, ru;
    void *w = nullptr, *q, *s, *st;
    int w_type = 0;
    if (!rows(gate, type, dev, M, K, &rg) || !rows(a[1], type, dev, M, K, &ru) || !quantized(a[5], a[6], dev, M, K, &q, &s)) return leave();
    if (weight != Py_None && !vec(weight, type, dev, K, &w, &w_type)) return leave();
    if (!stream_of(dev_obj.o, dev, &st)) return leave();
    const float eps = normed ? static_cast<float>(PyFloat_AS_DOUBLE(a[4])) : 0.0f;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = g_glu(rg.p, rg.ld, ru.p, ru.ld, type, static_cast<int>(act), normed, w, w_type, eps, static_cast<int8_t*>(q),
               static_cast<float*>(s), static_cast<int>(M), static_cast<int>(K), st);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

// matmul_fused(a, w_packed, row_scale, w_scale, bias, activation code, residual, out, kernel code) -> status or None
PyObject* mm(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 9 || !g_mm) return leave();
    long long act, kernel, dev, M, K, K2, N4;
    if (!as_ll(a[5], &act) || !as_ll(a[8], &kernel)) return leave();
    Ref dev_obj(PyObject_CallMethodNoArgs(a[0], s_get_device));
    if (!as_ll(dev_obj.o, &dev) || dev < 0 || !shape_of(a[0], &M, &K) || !shape_of(a[1], &K2, &N4) || K2 != K || !fits(M, K) || !fits(4 * N4, 0))
        return leave();
    const long long N = 4 * N4;
    const int type = type_of(a[7]);
    if (type < 0 || type > 2) return leave();
    Rows ra, rw, ry, rr;
    ternix_b200_epilogue ep;
    std::memset(&ep, 0, sizeof ep);
    void *scale, *st, *col = nullptr, *bias = nullptr;
    int ty, b_type = 0;
    if (!rows(a[0], kI8, dev, M, K, &ra) || !call_true(a[0], s_is_contiguous) || !rows(a[1], kU8, dev, K, N4, &rw) ||
        !call_true(a[1], s_is_contiguous) || !rows(a[7], type, dev, M, N, &ry) || !vec(a[2], 0, dev, M, &scale, &ty))
        return leave();
    if (PyFloat_Check(a[3])) ep.w_scale = static_cast<float>(PyFloat_AS_DOUBLE(a[3]));
    else if (PyObject_TypeCheck(a[3], reinterpret_cast<PyTypeObject*>(g_tensor))) {
        if (!vec(a[3], 0, dev, N, &col, &ty)) return leave();
    } else return leave();
    if (a[4] != Py_None && !vec(a[4], -1, dev, N, &bias, &b_type)) return leave();
    if (a[6] != Py_None && !rows(a[6], type, dev, M, N, &rr)) return leave();
    if (!stream_of(dev_obj.o, dev, &st)) return leave();
    ep.row_scale = static_cast<const float*>(scale);
    ep.col_scale = static_cast<const float*>(col);
    ep.activation = static_cast<int>(act);
    ep.bias = bias;
    ep.bias_dtype = b_type;
    ep.out_dtype = type;
    ep.residual = rr.p;
    ep.ldr = rr.ld;
    int rc;
    Py_BEGIN_ALLOW_THREADS
    rc = g_mm(static_cast<const int8_t*>(ra.p), static_cast<const uint8_t*>(rw.p), &ep, ry.p, ry.ld, static_cast<int>(M), static_cast<int>(K),
              static_cast<int>(N), static_cast<int>(kernel), nullptr, st);
    Py_END_ALLOW_THREADS
    return PyLong_FromLong(rc);
}

// setup((float32, bfloat16, float16, int8, uint8), Tensor, current_device, raw_stream, address, address, address)
PyObject* setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (n != 7 || !PyTuple_Check(a[0]) || PyTuple_GET_SIZE(a[0]) != 5 || !PyType_Check(a[1])) {
        PyErr_SetString(PyExc_TypeError, "setup(types, Tensor, current_device, raw_stream, norm, glu, product)");
        return nullptr;
    }
    void* f[3];
    for (int i = 0; i < 3; ++i) {
        f[i] = PyLong_AsVoidPtr(a[4 + i]);
        if (PyErr_Occurred()) return nullptr;
    }
    for (int i = 0; i < 5; ++i) Py_XSETREF(g_types[i], Py_NewRef(PyTuple_GET_ITEM(a[0], i)));
    Py_XSETREF(g_tensor, Py_NewRef(a[1]));
    Py_XSETREF(g_current_device, Py_NewRef(a[2]));
    Py_XSETREF(g_raw_stream, Py_NewRef(a[3]));
    g_norm = reinterpret_cast<decltype(g_norm)>(f[0]);
    g_glu = reinterpret_cast<decltype(g_glu)>(f[1]);
    g_mm = reinterpret_cast<decltype(g_mm)>(f[2]);
    Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}
PyMethodDef g_methods[] = {method<setup>("setup"), method<norm>("rmsnorm_quantize"), method<glu>("glu_quantize"),
                           method<mm>("matmul_fused"), {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_layer_calls", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__layer_calls(void) {
    struct { PyObject** at; const char* name; } const names[] = {
        {&s_dtype, "dtype"}, {&s_shape, "shape"}, {&s_data_ptr, "data_ptr"}, {&s_get_device, "get_device"},
        {&s_is_contiguous, "is_contiguous"}, {&s_stride, "stride"}, {&s_dim, "dim"}, {&s_numel, "numel"}};
    for (const auto& x : names)
        if (!(*x.at = PyUnicode_InternFromString(x.name))) return nullptr;
    return PyModule_Create(&g_module);
}

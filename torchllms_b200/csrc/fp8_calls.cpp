// Calls of the 8-bit rows' operators from Python: the arguments' check, the outputs, the launch (as fp4_calls.cpp has them for the
// 4-bit cache's).  A step of few tokens takes the device 2 to 20 us for one of these, and a front end in Python 13 to 17 us a launch.
//
// What stays in Python is their signature, their documentation, and what they say when arguments do not fit: a call that finds
// something wrong, or nothing to do, returns None and does nothing, and the Python side takes the arguments apart.  The kernels'
// entry points come as addresses (bind), so this module is linked against none of their libraries.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

namespace {

// (the entry points' declarations are those of rows_fp8.cu, gemm_fp8.cu and moe.cu)
struct Entries {
    int (*rows)(const void*, int, void*, void*, int, int, int, int, float, float, float, void*);
    int (*norm)(float*, const void*, int, int, long long, const float*, void*, void*, int, int, float, void*);
    int (*product)(const void*, const void*, const void*, const void*, void*, int, int, int, int, int, int*, void*);
    int (*act_product)(const void*, const void*, const void*, const void*, void*, void*, int, int, int, int, int, float, float, float, int, const int*, int,
                       int, int*, void*);
    int (*tile_rows)(int, int);
    int (*plan)(const int*, int, int, int, int*, int*, int*, int, void*);
    int (*placed)(const void*, int, void*, void*, int, int, const int*, int, void*);
    int (*experts)(const void*, const void*, const void*, const void*, void*, int, int, int, int, int, const int*, int, int, int*, void*);
    int (*combine)(const void*, int, int, const int*, const float*, const void*, int, int, long long, const float*, void*, int, int, int, void*);
} entry;
constexpr int ENTRIES = 9;

constexpr int ALIGN = 16, MAX_NORM_WIDTH = 32768;

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }
bool whole(PyObject* o, int& v) {
    if (!PyLong_Check(o)) return false;
    int over = 0;
    const long long x = PyLong_AsLongLongAndOverflow(o, &over);
    v = (int)x;
    return over == 0 && x == (long long)v;
}
bool number(PyObject* o, double& v) {
    if (!PyFloat_Check(o) && !PyLong_Check(o)) return false;
    v = PyFloat_AsDouble(o);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}
int code_of(const at::Tensor& t) { return t.scalar_type() == at::kFloat ? 0 : t.scalar_type() == at::kBFloat16 ? 1 : -1; }
bool aligned(const at::Tensor& t) { return (uintptr_t)t.data_ptr() % 16 == 0; }
// a tensor of this type in one piece on the current device
bool here(const at::Tensor* t, int device) { return t != nullptr && t->is_cuda() && t->get_device() == device && t->is_contiguous(); }
long long pitch(long long width) { return 4 * ((width + 511) / 512); }
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
    return at::Tensor(at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt));
}
// What lives in one call only comes in one piece (an allocation takes the host some 0.6 us): parts of it, each on 256 bytes
struct Pieces {
    long long bytes = 0;
    at::Tensor memory;
    long long add(long long n) {
        const long long at = bytes;
        bytes += (n + 255) / 256 * 256;
        return at;
    }
    char* take(const at::Tensor& like) {
        memory = fresh({bytes}, at::kByte, like);
        return (char*)memory.data_ptr();
    }
};
void* stream_of(int device) { return (void*)c10::cuda::getCurrentCUDAStream(device).stream(); }
// float32/bfloat16 rows whose width is `parts` times a multiple of 16
bool plain_rows(const at::Tensor* x, int device, int parts) {
    return here(x, device) && code_of(*x) >= 0 && x->dim() == 2 && x->size(0) > 0 && x->size(0) <= INT32_MAX && x->size(1) > 0 &&
           x->size(1) % (parts * ALIGN) == 0 && x->size(1) <= (1 << 26) && aligned(*x);
}
// 8-bit rows, [rows, width], or those of experts, [experts, rows, width]
bool held_rows(const at::Tensor* c, const at::Tensor* s, int device, int dims = 2) {
    if (!here(c, device) || !here(s, device) || c->scalar_type() != at::kFloat8_e4m3fn || s->scalar_type() != at::kFloat8_e8m0fnu || c->dim() != dims ||
        s->dim() != dims)
        return false;
    const long long width = c->size(-1);
    for (int i = 0; i + 1 < dims; ++i)
        if (c->size(i) != s->size(i) || c->size(i) < 1 || c->size(i) > INT32_MAX) return false;
    return width > 0 && width % ALIGN == 0 && width <= (1 << 26) && s->size(-1) == pitch(width) && aligned(*c) && (uintptr_t)s->data_ptr() % 4 == 0;
}
PyObject* both(at::Tensor&& a, at::Tensor&& b) {
    PyObject *x = THPVariable_Wrap(std::move(a)), *y = THPVariable_Wrap(std::move(b));
    PyObject* t = x != nullptr && y != nullptr ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return t;
}

PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != ENTRIES) {
        PyErr_SetString(PyExc_TypeError, "bind takes nine addresses");
        return nullptr;
    }
    void* at[ENTRIES];
    for (int i = 0; i < ENTRIES; ++i) at[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return nullptr;
    entry.rows = (decltype(entry.rows))at[0];
    entry.norm = (decltype(entry.norm))at[1];
    entry.product = (decltype(entry.product))at[2];
    entry.act_product = (decltype(entry.act_product))at[3];
    entry.tile_rows = (decltype(entry.tile_rows))at[4];
    entry.plan = (decltype(entry.plan))at[5];
    entry.placed = (decltype(entry.placed))at[6];
    entry.experts = (decltype(entry.experts))at[7];
    entry.combine = (decltype(entry.combine))at[8];
    Py_RETURN_NONE;
}

// x, form (0 the rows, 1 act, 2 gated act of the halves), act, limit, alpha, up_offset -> (codes, scales), an error code, or None
PyObject* rows(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    int form, act, device = c10::cuda::current_device();
    double limit, alpha, offset;
    if (n != 6) Py_RETURN_NONE;
    const at::Tensor* x = tensor(args[0]);
    if (!whole(args[1], form) || !whole(args[2], act) || !number(args[3], limit) || !number(args[4], alpha) || !number(args[5], offset) ||
        !plain_rows(x, device, form == 2 ? 2 : 1))
        Py_RETURN_NONE;
    const long long T = x->size(0), K = x->size(1) / (form == 2 ? 2 : 1);
    at::Tensor codes = fresh({T, K}, at::kFloat8_e4m3fn, *x), scales = fresh({T, pitch(K)}, at::kFloat8_e8m0fnu, *x);
    const int rc = entry.rows(x->data_ptr(), code_of(*x), codes.data_ptr(), scales.data_ptr(), (int)T, (int)K, form, act, (float)limit, (float)alpha,
                              (float)offset, stream_of(device));
    if (rc != 0) return PyLong_FromLong(rc);
    return both(std::move(codes), std::move(scales));
    END_HANDLE_TH_ERRORS
}

// h, delta or None, weight, eps -> (codes, scales), an error code, or None
PyObject* norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4) Py_RETURN_NONE;
    const int device = c10::cuda::current_device();
    const at::Tensor *h = tensor(args[0]), *delta = tensor(args[1]), *weight = tensor(args[2]);
    double eps;
    if (!plain_rows(h, device, 1) || code_of(*h) != 0 || h->size(1) > MAX_NORM_WIDTH || !here(weight, device) || weight->scalar_type() != at::kFloat ||
        weight->numel() != h->size(1) || !aligned(*weight) || !number(args[3], eps) || (delta == nullptr && args[1] != Py_None))
        Py_RETURN_NONE;
    const long long T = h->size(0), K = h->size(1);
    long long splits = 1, plane = 0;
    if (delta != nullptr) {
        const long long d = delta->dim();
        if (!here(delta, device) || code_of(*delta) < 0 || !aligned(*delta) || d < 2 || d > 3 || delta->size(-1) != K || delta->size(-2) != T ||
            (d == 3 && code_of(*delta) != 0))
            Py_RETURN_NONE;
        if (d == 3) splits = delta->size(0), plane = T * K;
        if (splits < 1 || splits > INT32_MAX) Py_RETURN_NONE;
    }
    at::Tensor codes = fresh({T, K}, at::kFloat8_e4m3fn, *h), scales = fresh({T, pitch(K)}, at::kFloat8_e8m0fnu, *h);
    const int rc = entry.norm(h->data_ptr<float>(), delta == nullptr ? nullptr : delta->data_ptr(), delta == nullptr ? 0 : code_of(*delta), (int)splits,
                              plane, weight->data_ptr<float>(), codes.data_ptr(), scales.data_ptr(), (int)T, (int)K, (float)eps, stream_of(device));
    if (rc != 0) return PyLong_FromLong(rc);
    return both(std::move(codes), std::move(scales));
    END_HANDLE_TH_ERRORS
}

// x (codes, or rows to be brought to 8 bits first), its scales or None, w's codes, w's scales, out's type (0 float32, 1 bfloat16), form,
// the caller's status word (its address) -> out, an error code, or None
PyObject* product(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 7) Py_RETURN_NONE;
    const int device = c10::cuda::current_device();
    const at::Tensor *x = tensor(args[0]), *xs = tensor(args[1]), *w = tensor(args[2]), *ws = tensor(args[3]);
    int type, form;
    if (!whole(args[4], type) || type < 0 || type > 1 || !whole(args[5], form) || !held_rows(w, ws, device) || x == nullptr ||
        (xs == nullptr ? args[1] != Py_None || !plain_rows(x, device, 1) : !held_rows(x, xs, device)) || x->size(1) != w->size(1))
        Py_RETURN_NONE;
    int* status = PyLong_Check(args[6]) ? (int*)PyLong_AsVoidPtr(args[6]) : nullptr;
    if (status == nullptr) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    const long long M = x->size(0), N = w->size(0), K = x->size(1);
    void* stream = stream_of(device);
    Pieces held;
    void *codes, *scales;
    if (xs == nullptr) {
        const long long codes_at = held.add(M * K), scales_at = held.add(M * pitch(K));
        char* memory = held.take(*x);
        codes = memory + codes_at, scales = memory + scales_at;
        const int rc = entry.rows(x->data_ptr(), code_of(*x), codes, scales, (int)M, (int)K, 0, 0, 0.f, 0.f, 0.f, stream);
        if (rc != 0) return PyLong_FromLong(rc);
    } else {
        codes = x->data_ptr(), scales = xs->data_ptr();
    }
    at::Tensor out = fresh({M, N}, type == 0 ? at::kFloat : at::kBFloat16, *x);
    const int rc = entry.product(codes, scales, w->data_ptr(), ws->data_ptr(), out.data_ptr(), type == 0 ? 1 : 0, (int)M, (int)N, (int)K, form, status, stream);
    if (rc != 0) return PyLong_FromLong(rc);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// x (codes, or rows to be brought to 8 bits first), its scales or None, w's codes, w's scales, act, gated, limit, alpha, up_offset, form, the
// caller's status word -> (codes, scales) of act(x . w^T), an error code, or None
PyObject* act_product(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 11) Py_RETURN_NONE;
    const int device = c10::cuda::current_device();
    const at::Tensor *x = tensor(args[0]), *xs = tensor(args[1]), *w = tensor(args[2]), *ws = tensor(args[3]);
    int act, gated, form;
    double limit, alpha, offset;
    if (!whole(args[4], act) || !whole(args[5], gated) || !number(args[6], limit) || !number(args[7], alpha) || !number(args[8], offset) ||
        !whole(args[9], form) || !held_rows(w, ws, device) || x == nullptr ||
        (xs == nullptr ? args[1] != Py_None || !plain_rows(x, device, 1) : !held_rows(x, xs, device)) || x->size(1) != w->size(1))
        Py_RETURN_NONE;
    const long long M = x->size(0), K = x->size(1), hidden = gated ? w->size(0) / 2 : w->size(0);
    int* status = PyLong_Check(args[10]) ? (int*)PyLong_AsVoidPtr(args[10]) : nullptr;
    if (status == nullptr || hidden % ALIGN != 0 || (gated && w->size(0) % 2 != 0)) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    void* stream = stream_of(device);
    Pieces held;
    void *codes, *scales;
    if (xs == nullptr) {
        const long long codes_at = held.add(M * K), scales_at = held.add(M * pitch(K));
        char* memory = held.take(*x);
        codes = memory + codes_at, scales = memory + scales_at;
        const int rc = entry.rows(x->data_ptr(), code_of(*x), codes, scales, (int)M, (int)K, 0, 0, 0.f, 0.f, 0.f, stream);
        if (rc != 0) return PyLong_FromLong(rc);
    } else {
        codes = x->data_ptr(), scales = xs->data_ptr();
    }
    at::Tensor out = fresh({M, hidden}, at::kFloat8_e4m3fn, *x), out_scales = fresh({M, pitch(hidden)}, at::kFloat8_e8m0fnu, *x);
    const int rc = entry.act_product(codes, scales, w->data_ptr(), ws->data_ptr(), out.data_ptr(), out_scales.data_ptr(), (int)M, (int)hidden, (int)K, gated, act, (float)limit,
                                     (float)alpha, (float)offset, 1, nullptr, 0, form, status, stream);
    if (rc != 0) return PyLong_FromLong(rc);
    return both(std::move(out), std::move(out_scales));
    END_HANDLE_TH_ERRORS
}

// x, chosen, weights, up's codes and scales, down's codes and scales, act, gated, limit, alpha, up_offset, shared, shared_gate, form, the caller's
// status word -> out, an error code, or None
PyObject* experts(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 16) Py_RETURN_NONE;
    const int device = c10::cuda::current_device();
    const at::Tensor *x = tensor(args[0]), *chosen = tensor(args[1]), *weights = tensor(args[2]), *up = tensor(args[3]), *up_s = tensor(args[4]),
                     *down = tensor(args[5]), *down_s = tensor(args[6]), *shared = tensor(args[12]), *gate = tensor(args[13]);
    int act, gated, form;
    double limit, alpha, offset;
    if (!whole(args[7], act) || !whole(args[8], gated) || !number(args[9], limit) || !number(args[10], alpha) || !number(args[11], offset) ||
        !whole(args[14], form) || !plain_rows(x, device, 1) || !held_rows(up, up_s, device, 3) || !held_rows(down, down_s, device, 3) ||
        !here(chosen, device) || chosen->scalar_type() != at::kInt || chosen->dim() != 2 || !here(weights, device) || weights->scalar_type() != at::kFloat ||
        weights->sizes() != chosen->sizes() || (shared == nullptr && args[12] != Py_None) || (gate == nullptr && args[13] != Py_None))
        Py_RETURN_NONE;
    const long long T = x->size(0), dim = x->size(1), top = chosen->size(1), E = up->size(0), hidden = gated ? up->size(1) / 2 : up->size(1), pairs = T * top;
    if (chosen->size(0) != T || top < 1 || top > 64 || pairs > INT32_MAX / 4 || E > 4096 || (gated && up->size(1) % 2 != 0) || up->size(2) != dim ||
        down->size(0) != E || down->size(1) != dim || down->size(2) != hidden)
        Py_RETURN_NONE;
    long long splits = 1, plane = 0;
    const int code = code_of(*x);
    if (shared != nullptr) {
        const long long d = shared->dim();
        if (!here(shared, device) || d < 2 || d > 3 || shared->size(-1) != dim || shared->size(-2) != T ||
            (code_of(*shared) != 0 && (d == 3 || code_of(*shared) != code)))
            Py_RETURN_NONE;
        if (d == 3) splits = shared->size(0), plane = T * dim;
        if (splits < 1 || splits > INT32_MAX) Py_RETURN_NONE;
    }
    if (gate != nullptr && (!here(gate, device) || gate->scalar_type() != at::kFloat || gate->numel() != T || shared == nullptr)) Py_RETURN_NONE;
    int* status = PyLong_Check(args[15]) ? (int*)PyLong_AsVoidPtr(args[15]) : nullptr;
    if (status == nullptr) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    void* stream = stream_of(device);
    const int P = (int)pairs, width = entry.tile_rows(P, (int)E);
    const long long tiles_most = (pairs + width - 1) / width + E, most = tiles_most < pairs ? tiles_most : pairs;
    Pieces held;
    const long long index_at = held.add(4 * (2 * pairs + 1 + 3 * most)), rows_at = held.add(pairs * dim), rows_s_at = held.add(pairs * pitch(dim)),
                    hid_at = held.add(pairs * hidden), hid_s_at = held.add(pairs * pitch(hidden)), y_at = held.add(4 * pairs * dim);
    at::Tensor out = fresh({T, dim}, x->scalar_type(), *x);
    char* memory = held.take(*x);
    int *order = (int*)(memory + index_at), *place = order + pairs, *tiles = place + pairs;
    void *rows = memory + rows_at, *rows_s = memory + rows_s_at, *hid = memory + hid_at, *hid_s = memory + hid_s_at, *y = memory + y_at;
    int rc = entry.plan(chosen->data_ptr<int>(), P, (int)E, width, order, place, tiles, (int)most, stream);
    if (rc == 0) rc = entry.placed(x->data_ptr(), code, rows, rows_s, (int)T, (int)dim, place, (int)top, stream);
    if (rc == 0)
        rc = entry.act_product(rows, rows_s, up->data_ptr(), up_s->data_ptr(), hid, hid_s, P, (int)hidden, (int)dim,
                               gated, act, (float)limit, (float)alpha, (float)offset, (int)E, tiles, (int)most, gated ? 0 : form, status, stream);
    // (an expert's result stays in float32 until the choices have been added up: rounded to bfloat16 on its way, a token's error against 64 bits
    // was 0.0024 of its size, for the 0.0017 that the sum's own rounding makes)
    if (rc == 0)
        rc = entry.experts(hid, hid_s, down->data_ptr(), down_s->data_ptr(), y, 1, P, (int)dim, (int)hidden,
                           (int)E, tiles, (int)most, form, status, stream);
    if (rc == 0)
        rc = entry.combine(y, 0, code, place, weights->data_ptr<float>(), shared == nullptr ? nullptr : shared->data_ptr(),
                           shared == nullptr ? 0 : code_of(*shared), (int)splits, plane, gate == nullptr ? nullptr : gate->data_ptr<float>(), out.data_ptr(),
                           (int)T, (int)dim, (int)top, stream);
    if (rc != 0) return PyLong_FromLong(rc);
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void*)bind, METH_FASTCALL, "the kernels' entry points, as addresses"},
    {"rows", (PyCFunction)(void*)rows, METH_FASTCALL, "rows, or an activation of them, into 8 bits"},
    {"norm", (PyCFunction)(void*)norm, METH_FASTCALL, "residual sum, RMS norm, rows into 8 bits"},
    {"product", (PyCFunction)(void*)product, METH_FASTCALL, "8-bit rows times an 8-bit weight"},
    {"act_product", (PyCFunction)(void*)act_product, METH_FASTCALL, "8-bit rows of an activation of that"},
    {"experts", (PyCFunction)(void*)experts, METH_FASTCALL, "routed experts with 8-bit weights"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "fp8_calls", "Calls of the 8-bit rows' operators.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_fp8_calls() { return PyModule_Create(&module); }

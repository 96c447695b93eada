// Calls of the 4-bit cache's operators from Python: the arguments' check, the outputs, the launch.
//
// A step of few tokens takes the device 3 to 10 us for one of these, and a front end in Python 13 to 16 us (one decoded token: 16.2 us a
// call of the attention through ctypes; the launch itself is 3 of them).  So for these operators the front end is this module.  What
// stays in Python is their signature, their documentation, and what they say when arguments do not fit: a call that finds
// something wrong returns None and does nothing, and the Python side takes the arguments apart.
//
// The kernels' entry points come as addresses (bind), so this module is linked against none of their libraries.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <vector>

namespace {

// (the entry points' declarations are those of kv_fp4.cu, attention_fp4.cu, attention_fp4_decode.cu and attention_fp4_prefill.cu)
struct Entries {
    int (*write)(const void*, int, int, const int*, const float*, const int*, void*, void*, void*, int, int, int, int, int, int, int, long long, int,
                 int, const float*, int, float, float, void*);
    int (*read)(const void*, const void*, const int*, void*, void*, int, int, long long, int, int, int, void*);
    int (*general)(const void*, const void*, const void*, void*, const int*, int, int, const int*, const int*, int, int, int, int, int, int, long long,
                   int, int, float, void*);
    int (*decode)(const void*, const void*, const void*, void*, const int*, int, int, const int*, const int*, float*, int*, int*, int, int, int, int, int,
                  int, long long, int, int, int, float, void*);
    int (*decode_plan)(int, int, int, int, int, int, int, int, long long*, long long*);
    int (*prefill)(const void*, const void*, const void*, void*, const int*, int, int, const int*, const int*, float*, int*, long long, int, int, int, int,
                   int, long long, int, int, float, int, void*);
    int (*prefill_plan)(long long, int, int, int, int, int, int, int, int*, long long*);
} entry;

constexpr int GROUP = 16, RECORD = 16, MAX_HEAD_DIM = 256;

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }
// an int that fits 32 bits
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
bool ints(const at::Tensor* t) { return t != nullptr && t->is_cuda() && t->scalar_type() == at::kInt && t->is_contiguous(); }
bool pages_fit(const at::Tensor* k, const at::Tensor* v, long long kv_heads, int head_dim, int page_size) {
    return k != nullptr && v != nullptr && k->is_cuda() && v->is_cuda() && k->scalar_type() == at::kByte && v->scalar_type() == at::kByte &&
           k->dim() == 4 && k->sizes() == v->sizes() && k->size(0) > 0 && k->size(1) == kv_heads && head_dim > 0 && head_dim % GROUP == 0 &&
           head_dim <= MAX_HEAD_DIM && page_size > 0 && k->size(2) * RECORD == page_size && k->size(3) == 9 * head_dim && k->is_contiguous() &&
           v->is_contiguous();
}
// (straight from the allocator: by way of the dispatcher a decoded token's attention has the host for 6.3 us instead of 5.4)
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
    return at::Tensor(at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt));
}
void* stream_of(const at::Tensor& t) { return (void*)c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// Ints that are zero between launches and that no other stream's work uses.  A graph may be replayed on any stream, beside whatever its
// capture's stream does then: a capture has counters of its own, and setting them to zero is the first thing it records of them.
struct Counts {
    int device;
    void* stream;
    bool capturing;
    unsigned long long capture;
    at::Tensor buffer;
};
std::vector<Counts>& all_counts() {
    static auto* counts = new std::vector<Counts>;        // (never destroyed: the device may be gone when the process ends)
    return *counts;
}
int* counters(const at::Tensor& like, void* stream, long long n) {
    cudaStreamCaptureStatus state = cudaStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (cudaStreamGetCaptureInfo((cudaStream_t)stream, &state, &id) != cudaSuccess) {
        cudaGetLastError();
        return nullptr;
    }
    const bool capturing = state == cudaStreamCaptureStatusActive;
    if (!capturing) id = 0;
    Counts* found = nullptr;
    for (Counts& c : all_counts())
        if (c.device == like.get_device() && c.stream == stream && c.capturing == capturing) found = &c;
    if (found == nullptr) {
        all_counts().push_back({(int)like.get_device(), stream, capturing, id, at::Tensor()});
        found = &all_counts().back();
    }
    if (!found->buffer.defined() || found->capture != id || found->buffer.numel() < n) {
        // (what is replaced goes back to the allocator, which hands it out again behind this stream's work)
        found->buffer = at::zeros({n > 4096 ? n : 4096}, like.options().dtype(at::kInt));
        found->capture = id;
    }
    return found->buffer.data_ptr<int>();
}

PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != 7) {
        PyErr_SetString(PyExc_TypeError, "bind takes seven addresses");
        return nullptr;
    }
    void* at[7];
    for (int i = 0; i < 7; ++i) at[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return nullptr;
    entry.write = (decltype(entry.write))at[0];
    entry.read = (decltype(entry.read))at[1];
    entry.general = (decltype(entry.general))at[2];
    entry.decode = (decltype(entry.decode))at[3];
    entry.decode_plan = (decltype(entry.decode_plan))at[4];
    entry.prefill = (decltype(entry.prefill))at[5];
    entry.prefill_plan = (decltype(entry.prefill_plan))at[6];
    Py_RETURN_NONE;
}

// After a kernel gave up: the next call counts from zero.
PyObject* reset(PyObject*, PyObject*) {
    HANDLE_TH_ERRORS
    for (Counts& c : all_counts())
        if (!c.capturing && c.buffer.defined()) c.buffer.zero_();
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

// qkv, positions, table, n_heads, n_kv_heads, head_dim, interleaved, k_pages, v_pages, slot_mapping, page_size, out_dtype (0, 1, or -1: qkv's),
// ssq, inv_dim, eps -> q, an error code, or None where something does not fit
PyObject* write(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 15) Py_RETURN_NONE;
    const at::Tensor *qkv = tensor(args[0]), *positions = tensor(args[1]), *table = tensor(args[2]), *k = tensor(args[7]), *v = tensor(args[8]),
                     *slots = tensor(args[9]), *ssq = tensor(args[12]);
    int heads, kv_heads, head_dim, page_size, out_code;
    double inv_dim, eps;
    if (qkv == nullptr || !whole(args[3], heads) || !whole(args[4], kv_heads) || !whole(args[5], head_dim) || !whole(args[10], page_size) ||
        !whole(args[11], out_code) || !number(args[13], inv_dim) || !number(args[14], eps))
        Py_RETURN_NONE;
    const int in_code = code_of(*qkv), interleaved = PyObject_IsTrue(args[6]);
    if (interleaved < 0) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    if (out_code < 0) out_code = in_code;
    const long long dims = qkv->dim(), splits = dims == 3 ? qkv->size(0) : 1;
    if (!qkv->is_cuda() || in_code < 0 || out_code > 1 || dims < 2 || dims > 3 || !qkv->is_contiguous() || heads <= 0 || kv_heads <= 0 || head_dim <= 0 ||
        head_dim % GROUP != 0 || (in_code == 1 && (out_code == 0 || splits != 1)) || qkv->size(-1) != ((long long)heads + 2ll * kv_heads) * head_dim)
        Py_RETURN_NONE;
    const long long T = qkv->size(-2);
    if (!ints(positions) || positions->numel() != T || T > INT32_MAX || table == nullptr || !table->is_cuda() || table->scalar_type() != at::kFloat ||
        !table->is_contiguous() || table->dim() != 3 || table->size(1) < 1 || table->size(1) > head_dim / 2 || table->size(2) != 2)
        Py_RETURN_NONE;
    const bool writes = k != nullptr;
    if (writes ? (!pages_fit(k, v, kv_heads, head_dim, page_size) || !ints(slots) || slots->numel() != T) : (v != nullptr || args[7] != Py_None)) Py_RETURN_NONE;
    at::Tensor q = fresh({T, heads, head_dim}, out_code == 0 ? at::kFloat : at::kBFloat16, *qkv);
    const int rc = entry.write(qkv->data_ptr(), in_code, (int)splits, positions->data_ptr<int>(), table->data_ptr<float>(),
                               writes ? slots->data_ptr<int>() : nullptr, q.data_ptr(), writes ? k->data_ptr() : nullptr, writes ? v->data_ptr() : nullptr,
                               out_code, (int)T, heads, kv_heads, head_dim, 2 * (int)table->size(1), writes ? page_size : RECORD, writes ? k->size(0) : 0,
                               (int)table->size(0), interleaved, ssq == nullptr ? nullptr : ssq->data_ptr<float>(), ssq == nullptr ? 0 : (int)ssq->size(1),
                               (float)inv_dim, (float)eps, stream_of(*qkv));
    if (rc != 0) return PyLong_FromLong(rc);
    return THPVariable_Wrap(std::move(q));
    END_HANDLE_TH_ERRORS
}

// k_pages, v_pages, slots, head_dim, page_size, out_dtype (0, 1) -> (k, v), an error code, or None
PyObject* read(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 6) Py_RETURN_NONE;
    const at::Tensor *k = tensor(args[0]), *v = tensor(args[1]), *slots = tensor(args[2]);
    int head_dim, page_size, code;
    if (k == nullptr || k->dim() != 4 || !whole(args[3], head_dim) || !whole(args[4], page_size) || !whole(args[5], code) || code < 0 || code > 1 ||
        !pages_fit(k, v, k->size(1), head_dim, page_size) || !ints(slots) || slots->dim() != 1 || slots->numel() > INT32_MAX)
        Py_RETURN_NONE;
    const long long count = slots->numel();
    const at::ScalarType type = code == 0 ? at::kFloat : at::kBFloat16;
    at::Tensor k_out = fresh({count, k->size(1), head_dim}, type, *k), v_out = fresh({count, k->size(1), head_dim}, type, *k);
    const int rc = entry.read(k->data_ptr(), v->data_ptr(), slots->data_ptr<int>(), k_out.data_ptr(), v_out.data_ptr(), code, (int)count, k->size(0),
                              (int)k->size(1), head_dim, page_size, stream_of(*k));
    if (rc != 0) return PyLong_FromLong(rc);
    PyObject *a = THPVariable_Wrap(std::move(k_out)), *b = THPVariable_Wrap(std::move(v_out));
    PyObject* both = PyTuple_Pack(2, a, b);
    Py_DECREF(a);
    Py_DECREF(b);
    return both;
    END_HANDLE_TH_ERRORS
}

// Whether a step is one for the tcgen05 kernel, whose CTA has 256 rows and an SM to itself, and not for the mma.sync kernel, which unpacks keys and
// values again for every 16 rows.  `rows`: tokens x query heads of a key head; `units`: requests x key heads.  Measured (us, the mma.sync
// kernel and the other; contexts of 200, 2,000 and 12,000 tokens):
//   1 request, 32 / 8 heads of 128, 16 rows:  9.5 10.3   14.5 15.5   26.7 22.0     64: 10.2 10.7   16.2 16.5   35.0 23.7     256: 14.8 14.7   27.2 23.8    80  33
//   8 requests                      16 rows: 10.2 11.0   19.2 22.9   49.4 96.6     64: 11.4 11.5   39.4 24.2   147  99       256: 40.3 15.5   118  36     537 117
//   1 request,           of 64      32 rows:  7.8  8.6   11.0 15.2   17.6 21.4     64:  8.0  8.6   11.9 15.7   24.1 22.2     256: 11.1 12.3   19.0 19.2    58  28
//   8 requests                      32 rows:  8.8  9.4   19.0 20.6   57.5 71.0     64:  8.8  9.4   28.2 21.0   105  72       256: 27.5 13.0   80   30     374  91
// So it is one from `least` rows on, and with heads of 128 from 17 on where the context is long (beyond 1,024: the engine's steps plan for a power of two
// that is no less, so that all shorter contexts come as 1,024) and there are no more than 1,024 tiles of 128 keys
// (32 rows: one request of 12,000 tokens 25.9 and 22.7, 8 of 2,000 27.0 and 23.7; but 8 of 12,000 82 and 98, one of 200 9.6 and 10.4).
// The rule is one line for rows and one for tiles, and takes the slower side here and there: the tcgen05 kernel for one request and heads of 64 (64 rows behind 2,000 a
// third slower, 256 up to a tenth), the other for 16 rows of heads of 128 behind 12,000 (a fifth).
// Those are times with keys that the tcgen05 kernel may cut into pieces.  Where it may not (`cut`), a CTA walks all keys of its rows, and more than two tiles of
// them are for it only where rows are many: the mma.sync kernel, which cuts them as it likes, and the tcgen05 kernel without pieces, contexts of 2,000 and 12,000:
//   rows x units     512 (1 request, 64 rows):  of 64: 11.6  27.8   24.4 131   of 128: 16.1  33.5   36.0 149       2,048 (4 requests): 19.4 28.3  59.8 163   27.7 34.1  86 192
//                  4,096 (2 requests, 256 rows):       28.6  37.0    107 168           41.7  43.9    155 201       8,192 (4 requests): 47.9 37.2   204 174   70.6 44.2 294 208
bool many_rows(long long rows, int head_dim, long long units, int max_kv, int least, bool cut) {
    if (!cut && max_kv > 256) return rows >= least && rows * units >= 8192;
    return rows >= least || (head_dim == 128 && rows > 16 && max_kv > 1024 && units * ((max_kv + 127) / 128) <= 1024);
}

// q, k_pages, v_pages, block_table, q_start, kv_len, n_seqs, max_q_len, max_kv_len, scale, window, page_size, allow_split, impl (0 the kernel that fits,
// 1 general, 2 decode, 3 prefill), n_tokens, out, rows of a request from which 3 fits, the caller's status word (its address) -> (out, launches), an
// error code, or None
PyObject* attend(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 18) Py_RETURN_NONE;
    const at::Tensor *q = tensor(args[0]), *k = tensor(args[1]), *v = tensor(args[2]), *table = tensor(args[3]), *q_start = tensor(args[4]),
                     *kv_len = tensor(args[5]), *given = tensor(args[15]);
    int n_seqs, max_q, max_kv, page_size, split, impl, min_rows, window = 0, n_tokens = 1;
    double scale;
    if (q == nullptr || k == nullptr || table == nullptr || q->dim() != 3 || k->dim() != 4 || !whole(args[6], n_seqs) || !whole(args[7], max_q) ||
        !whole(args[8], max_kv) || !number(args[9], scale) || !std::isfinite((float)scale) || (args[10] != Py_None && (!whole(args[10], window) || window <= 0)) ||
        !whole(args[11], page_size) || !whole(args[12], split) || !whole(args[13], impl) || (args[14] != Py_None && !whole(args[14], n_tokens)) ||
        !whole(args[16], min_rows))
        Py_RETURN_NONE;
    int* status = PyLong_Check(args[17]) ? (int*)PyLong_AsVoidPtr(args[17]) : nullptr;
    if (status == nullptr) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
    const int code = code_of(*q);
    const long long heads = q->size(1), head_dim = q->size(2), kv_heads = k->size(1), n_pages = k->size(0);
    if (!q->is_cuda() || code < 0 || !q->is_contiguous() || heads <= 0 || heads > INT32_MAX || kv_heads <= 0 || heads % kv_heads != 0 ||
        head_dim > MAX_HEAD_DIM || !pages_fit(k, v, kv_heads, (int)head_dim, page_size) || !ints(q_start) || !ints(kv_len) || !table->is_cuda() ||
        table->scalar_type() != at::kInt || table->dim() != 2 || (table->size(1) > 1 && table->stride(1) != 1) || table->size(0) < n_seqs ||
        table->size(1) * page_size < max_kv || table->size(1) * page_size > INT32_MAX || table->stride(0) > INT32_MAX || q_start->numel() <= n_seqs ||
        kv_len->numel() < n_seqs || n_tokens <= 0 || (args[14] != Py_None && n_tokens > q->size(0)))
        Py_RETURN_NONE;
    const bool tensor_cores = head_dim == 64 || head_dim == 128;
    if (impl < 0 || impl > 3 || (impl >= 2 && !tensor_cores) || (impl == 3 && code != 1)) Py_RETURN_NONE;
    if (given != nullptr ? (!given->is_cuda() || given->scalar_type() != q->scalar_type() || !given->is_contiguous() || given->sizes() != q->sizes())
                         : args[15] != Py_None)
        Py_RETURN_NONE;
    at::Tensor out = given != nullptr ? *given : fresh(q->sizes(), q->scalar_type(), *q);
    if (impl == 0) {        // (the tcgen05 kernel stores 32 bytes at a time)
        const bool many = code == 1 && (uintptr_t)out.data_ptr() % 32 == 0 &&
                          many_rows(max_q * (heads / kv_heads), (int)head_dim, n_seqs * kv_heads, max_kv, min_rows, split != 0);
        impl = !tensor_cores ? 1 : many ? 3 : 2;
    }
    void* stream = stream_of(*q);
    const int* bt = table->data_ptr<int>();
    const int stride = (int)table->stride(0), columns = (int)table->size(1);
    int rc = 0, launches = 1;
    if (n_seqs > 0 && max_q > 0) {
        if (impl == 2) {
            long long floats = 0, count = 0;
            rc = entry.decode_plan(code, n_seqs, (int)heads, (int)kv_heads, (int)head_dim, page_size, max_q, max_kv, &floats, &count);
            if (rc == 0) {
                at::Tensor scratch = fresh({floats}, at::kFloat, *q);
                int* counts = counters(*q, stream, count);
                rc = entry.decode(q->data_ptr(), k->data_ptr(), v->data_ptr(), out.data_ptr(), bt, stride, columns, q_start->data_ptr<int>(),
                                  kv_len->data_ptr<int>(), scratch.data_ptr<float>(), counts, status, code, n_seqs, (int)heads, (int)kv_heads,
                                  (int)head_dim, page_size, n_pages, max_q, max_kv, window, (float)scale, stream);
            }
        } else if (impl == 3) {
            int pieces = 1;
            long long floats = 0;
            rc = entry.prefill_plan(q->size(0), n_seqs, (int)heads, (int)kv_heads, (int)head_dim, max_q, max_kv, split, &pieces, &floats);
            if (rc == 0) {
                at::Tensor scratch;
                if (floats > 0) scratch = fresh({floats}, at::kFloat, *q);
                rc = entry.prefill(q->data_ptr(), k->data_ptr(), v->data_ptr(), out.data_ptr(), bt, stride, columns, q_start->data_ptr<int>(),
                                   kv_len->data_ptr<int>(), floats > 0 ? scratch.data_ptr<float>() : nullptr, status, q->size(0), n_seqs,
                                   (int)heads, (int)kv_heads, (int)head_dim, page_size, n_pages, max_q, window, (float)scale, pieces, stream);
                if (pieces > 1) launches = 2;
            }
        } else {
            rc = entry.general(q->data_ptr(), k->data_ptr(), v->data_ptr(), out.data_ptr(), bt, stride, columns, q_start->data_ptr<int>(),
                               kv_len->data_ptr<int>(), code, n_seqs, (int)heads, (int)kv_heads, (int)head_dim, page_size, n_pages, max_q, window,
                               (float)scale, stream);
        }
    }
    if (rc != 0) return PyLong_FromLong(rc);
    PyObject *a = THPVariable_Wrap(std::move(out)), *b = PyLong_FromLong(launches);
    PyObject* both = PyTuple_Pack(2, a, b);
    Py_DECREF(a);
    Py_DECREF(b);
    return both;
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void*)bind, METH_FASTCALL, "the kernels' entry points, as addresses"},
    {"reset", reset, METH_NOARGS, "counters back to zero"},
    {"write", (PyCFunction)(void*)write, METH_FASTCALL, "rows rotated, keys and values into a 4-bit cache"},
    {"read", (PyCFunction)(void*)read, METH_FASTCALL, "keys and values of a 4-bit cache"},
    {"attend", (PyCFunction)(void*)attend, METH_FASTCALL, "attention over a 4-bit cache"},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "fp4_calls", "Calls of the 4-bit cache's operators.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_fp4_calls() { return PyModule_Create(&module); }

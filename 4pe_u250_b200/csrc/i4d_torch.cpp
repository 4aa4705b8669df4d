// i4d_torch.cpp -- torch binding of the long-context serving operators.
//
// Checks tensors, takes outputs and workspaces from torch's allocator and
// calls the C ABI on torch's current stream of the context's GPU.  Plain
// CPython calls with positional arguments: a decode step makes several such
// calls of a few microseconds of GPU work each, so their host side counts
// (about 2 us a call here, 15 to 20 us for the same checks in Python).
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <Python.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <string>

#include "i4d.h"

namespace {

PyObject* g_error = nullptr;  // the package's I4DError

struct OpError {
    int status;
    std::string message;
};

[[noreturn]] void refuse(const char* fmt, ...) __attribute__((format(printf, 1, 2)));
void refuse(const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    throw OpError{I4D_ERR_ARG, buf};
}

void raise(const OpError& e) {
    if (!g_error) {
        PyErr_SetString(PyExc_RuntimeError, e.message.c_str());
        return;
    }
    PyObject* x = PyObject_CallFunction(g_error, "is", e.status, e.message.c_str());
    if (x) {
        PyErr_SetObject(g_error, x);
        Py_DECREF(x);
    }
}

struct PyRaised {};  // a Python exception is set

// The arguments of a call, taken in order.
class Args {
  public:
    Args(PyObject* const* v, Py_ssize_t n, Py_ssize_t want) : v_(v) {
        if (n != want) refuse("%zd arguments, not %zd", n, want);
        ctx_ = reinterpret_cast<i4d_ctx*>(PyLong_AsVoidPtr(v_[0]));
        if (PyErr_Occurred()) throw PyRaised{};
        at_ = 1;
        device_ = static_cast<int>(integer("device"));
    }
    i4d_ctx* ctx() const { return ctx_; }
    int device() const { return device_; }
    cudaStream_t stream() const {
        const cudaStream_t s = at::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device_)).stream();
        return s ? s : cudaStreamLegacy;
    }
    int64_t integer(const char* what) {
        const int64_t x = PyLong_AsLongLong(v_[at_++]);
        if (x == -1 && PyErr_Occurred()) throw PyRaised{};
        (void)what;
        return x;
    }
    int small(const char* what) {
        const int64_t x = integer(what);
        if (x < INT32_MIN || x > INT32_MAX) refuse("%s %lld does not fit 32 bits", what, static_cast<long long>(x));
        return static_cast<int>(x);
    }
    double real() {
        const double x = PyFloat_AsDouble(v_[at_++]);
        if (x == -1.0 && PyErr_Occurred()) throw PyRaised{};
        return x;
    }
    bool truth() {
        const int x = PyObject_IsTrue(v_[at_++]);
        if (x < 0) throw PyRaised{};
        return x != 0;
    }
    PyObject* object() { return v_[at_++]; }
    bool next_is_none() const { return v_[at_] == Py_None; }
    void skip() { ++at_; }
    // A tensor on the context's GPU whose last dimension is contiguous; null for None where that is allowed.
    const at::Tensor* tensor(const char* what, int dims, bool none_ok = false) {
        PyObject* o = v_[at_++];
        if (o == Py_None && none_ok) return nullptr;
        if (!THPVariable_Check(o)) refuse("%s is not a tensor", what);
        const at::Tensor& t = THPVariable_Unpack(o);
        if (t.requires_grad() && c10::GradMode::is_enabled()) refuse("%s requires a gradient, which the operators do not give: call them under torch.no_grad()", what);
        if (!t.is_cuda() || t.get_device() != device_) refuse("%s is not on GPU %d", what, device_);
        if (t.dim() != dims) refuse("%s has %lld dimensions, not %d", what, static_cast<long long>(t.dim()), dims);
        if (dims && t.size(-1) > 1 && t.stride(-1) != 1) refuse("%s is not contiguous in its last dimension", what);
        return &t;
    }
    const at::Tensor* typed(const char* what, at::ScalarType type, int dims, bool none_ok = false) {
        const at::Tensor* t = tensor(what, dims, none_ok);
        if (t && t->scalar_type() != type) refuse("%s has type %s, not %s", what, c10::toString(t->scalar_type()), c10::toString(type));
        return t;
    }
    i4d_kv8 cache() {
        PyObject* o = v_[at_++];
        if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 10) refuse("not a KV8Cache");
        int64_t x[10];
        for (int i = 0; i < 10; ++i) x[i] = static_cast<int64_t>(PyLong_AsUnsignedLongLong(PyTuple_GET_ITEM(o, i)));
        if (PyErr_Occurred()) throw PyRaised{};
        if (x[9] != device_) refuse("the cache is not on GPU %d", device_);
        i4d_kv8 c;
        c.k = reinterpret_cast<void*>(x[0]);
        c.v = reinterpret_cast<void*>(x[1]);
        c.k_scale = reinterpret_cast<float*>(x[2]);
        c.v_scale = reinterpret_cast<float*>(x[3]);
        c.blocks = static_cast<int>(x[4]);
        c.heads = static_cast<int>(x[5]);
        c.block_tokens = static_cast<int>(x[6]);
        c.dim = static_cast<int>(x[7]);
        c.code = static_cast<int>(x[8]);
        return c;
    }

  private:
    PyObject* const* v_;
    Py_ssize_t at_ = 0;
    i4d_ctx* ctx_ = nullptr;
    int device_ = 0;
};

void check(i4d_ctx* ctx, i4d_status st) {
    if (st != I4D_OK) throw OpError{st, i4d_last_error(ctx)};
}

int dtype_of(const at::Tensor& t, const char* what) {
    switch (t.scalar_type()) {
        case at::kFloat: return I4D_F32;
        case at::kBFloat16: return I4D_BF16;
        case at::kHalf: return I4D_F16;
        default: refuse("%s has type %s (float32, bfloat16 or float16)", what, c10::toString(t.scalar_type()));
    }
}

int count(int64_t n, const char* what) {
    if (n > INT32_MAX) refuse("%s: %lld is too many", what, static_cast<long long>(n));
    return static_cast<int>(n);
}

template <typename T>
T* ptr(const at::Tensor* t) {
    return t ? static_cast<T*>(t->data_ptr()) : nullptr;
}

PyObject* give(const at::Tensor& t) { return THPVariable_Wrap(t); }

struct Batch {
    const int32_t *q_start, *lengths, *table;
    int64_t table_stride;
    int table_blocks, batch;
};

// Strides count only where there are several rows; 0 shares one row among all.
int64_t row_stride(const at::Tensor& t) { return t.size(0) <= 1 ? t.size(1) : t.stride(0); }

Batch batch_of(Args& a) {
    const at::Tensor* q = a.typed("q_start", at::kInt, 1);
    const at::Tensor* l = a.typed("lengths", at::kInt, 1);
    const at::Tensor* t = a.typed("block_table", at::kInt, 2);
    if (q->size(0) != l->size(0) + 1 || t->size(0) != l->size(0)) refuse("q_start has batch + 1 entries, lengths and block_table batch");
    return {ptr<int32_t>(q), ptr<int32_t>(l), ptr<int32_t>(t), row_stride(*t), count(t->size(1), "block_table"), count(l->size(0), "batch")};
}

// ------------------------------------------------------------------ calls

PyObject* rope(Args& a) {
    const at::Tensor* q = a.tensor("q", 3);
    const at::Tensor* k = a.tensor("k", 3, true);
    const at::Tensor* pos = a.typed("positions", at::kInt, 1);
    const at::Tensor* turns = a.typed("table", at::kLong, 1);
    i4d_rope_args r = {};
    r.rot_dim = a.small("rot_dim");
    r.magnitude = static_cast<float>(a.real());
    r.interleaved = a.truth();
    r.inverse = a.truth();
    r.dtype = dtype_of(*q, "q");
    if (turns->size(0) != r.rot_dim / 2) refuse("table has %lld frequencies, not %d", static_cast<long long>(turns->size(0)), r.rot_dim / 2);
    if (pos->size(0) != q->size(0)) refuse("positions is [tokens]");
    if (k && (k->scalar_type() != q->scalar_type() || k->size(0) != q->size(0) || k->size(2) != q->size(2))) refuse("k is [tokens, heads, dim] like q");
    at::Tensor qo, ko;
    if (a.next_is_none()) {
        qo = at::empty(q->sizes(), q->options());
        a.skip();
    } else {
        qo = *a.typed("q_out", q->scalar_type(), 3);
    }
    if (!k || a.next_is_none()) {
        if (k) ko = at::empty(k->sizes(), k->options());
        a.skip();
    } else {
        ko = *a.typed("k_out", q->scalar_type(), 3);
    }
    if (qo.sizes() != q->sizes() || (k && ko.sizes() != k->sizes())) refuse("outputs have the inputs' shapes");
    r.q = q->data_ptr();
    r.q_out = qo.data_ptr();
    r.positions = ptr<int32_t>(pos);
    r.turns = static_cast<const uint64_t*>(turns->data_ptr());
    r.tokens = count(q->size(0), "tokens");
    r.q_heads = count(q->size(1), "heads");
    r.dim = count(q->size(2), "dim");
    r.q_stride = q->stride(0);
    r.q_head_stride = q->stride(1);
    r.q_out_stride = qo.stride(0);
    r.q_out_head_stride = qo.stride(1);
    if (k) {
        r.k = k->data_ptr();
        r.k_out = ko.data_ptr();
        r.k_heads = count(k->size(1), "heads");
        r.k_stride = k->stride(0);
        r.k_head_stride = k->stride(1);
        r.k_out_stride = ko.stride(0);
        r.k_out_head_stride = ko.stride(1);
    }
    r.stream = a.stream();
    check(a.ctx(), i4d_rope(a.ctx(), &r));
    PyObject* pair = PyTuple_New(2);
    if (!pair) throw PyRaised{};
    PyTuple_SET_ITEM(pair, 0, give(qo));
    if (k) {
        PyTuple_SET_ITEM(pair, 1, give(ko));
    } else {
        Py_INCREF(Py_None);
        PyTuple_SET_ITEM(pair, 1, Py_None);
    }
    return pair;
}

PyObject* kv8_append(Args& a) {
    i4d_kv8_append_args r = {};
    r.cache = a.cache();
    const at::Tensor* k = a.tensor("k", 3);
    const at::Tensor* v = a.typed("v", k->scalar_type(), 3);
    r.dtype = dtype_of(*k, "k");
    if (k->sizes() != v->sizes() || k->size(1) != r.cache.heads || k->size(2) != r.cache.dim) refuse("k and v are [tokens, cache heads, dim]");
    const Batch b = batch_of(a);
    r.k = k->data_ptr();
    r.v = v->data_ptr();
    r.k_stride = k->stride(0);
    r.k_head_stride = k->stride(1);
    r.v_stride = v->stride(0);
    r.v_head_stride = v->stride(1);
    r.q_start = b.q_start;
    r.lengths = b.lengths;
    r.block_table = b.table;
    r.table_stride = b.table_stride;
    r.table_blocks = b.table_blocks;
    r.batch = b.batch;
    r.tokens = count(k->size(0), "tokens");
    r.max_q = a.small("max_q");
    r.stream = a.stream();
    check(a.ctx(), i4d_kv8_append(a.ctx(), &r));
    Py_RETURN_NONE;
}

PyObject* kv8_read(Args& a) {
    i4d_kv8_read_args r = {};
    r.cache = a.cache();
    const Batch b = batch_of(a);
    r.max_q = a.small("max_q");
    r.tokens = a.small("tokens");
    if (r.tokens < 0) refuse("%d tokens", r.tokens);
    at::Tensor out[2];
    const int64_t shape[3] = {r.tokens, r.cache.heads, r.cache.dim};
    for (int i = 0; i < 2; ++i) {
        if (a.next_is_none()) {
            out[i] = at::empty(shape, at::TensorOptions().dtype(at::kBFloat16).device(at::kCUDA, static_cast<c10::DeviceIndex>(a.device())));
            a.skip();
        } else {
            out[i] = *a.typed(i ? "v_out" : "k_out", at::kBFloat16, 3);
            if (out[i].sizes() != at::IntArrayRef(shape, 3) || !out[i].is_contiguous()) refuse("k_out and v_out are contiguous [tokens, cache heads, dim]");
        }
    }
    r.k_out = out[0].data_ptr();
    r.v_out = out[1].data_ptr();
    r.q_start = b.q_start;
    r.lengths = b.lengths;
    r.block_table = b.table;
    r.table_stride = b.table_stride;
    r.table_blocks = b.table_blocks;
    r.batch = b.batch;
    r.stream = a.stream();
    check(a.ctx(), i4d_kv8_read(a.ctx(), &r));
    PyObject* pair = PyTuple_New(2);
    if (!pair) throw PyRaised{};
    for (int i = 0; i < 2; ++i) PyTuple_SET_ITEM(pair, i, give(out[i]));
    return pair;
}

// The caller's workspace, or one of the size the call needs.
at::Tensor workspace(Args& a, size_t need) {
    if (!a.next_is_none()) return *a.typed("workspace", at::kByte, 1);
    a.skip();
    if (!need) return {};
    return at::empty({static_cast<int64_t>(need)}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, static_cast<c10::DeviceIndex>(a.device())));
}

void weights_shape(const at::Tensor& w, const char* what, int64_t batch, int64_t heads, int64_t length) {
    if (w.size(0) != batch || w.size(1) != heads || w.size(2) < length) refuse("%s is [batch, cache heads, >= max_length]", what);
    if (batch > 1 && heads > 1 && w.stride(0) != heads * w.stride(1)) refuse("%s has gaps between its sequences", what);
    if ((heads > 1 && w.stride(1) < w.size(2)) || (batch > 1 && w.stride(0) < w.size(2))) refuse("rows of %s overlap", what);
}

PyObject* kv8_attention(Args& a) {
    i4d_kv8_attention_args r = {};
    r.cache = a.cache();
    const at::Tensor* q = a.tensor("q", 3);
    r.dtype = dtype_of(*q, "q");
    if (q->size(2) != r.cache.dim) refuse("q has %lld values a head, the cache %d", static_cast<long long>(q->size(2)), r.cache.dim);
    const Batch b = batch_of(a);
    r.max_q = a.small("max_q");
    r.max_length = a.small("max_length");
    if (a.next_is_none()) {
        r.scale = static_cast<float>(1.0 / std::sqrt(static_cast<double>(r.cache.dim)));
        a.skip();
    } else {
        r.scale = static_cast<float>(a.real());
    }
    r.window = a.small("window");
    at::Tensor out;
    if (a.next_is_none()) {
        out = at::empty(q->sizes(), q->options());
        a.skip();
    } else {
        out = *a.typed("out", q->scalar_type(), 3);
        if (out.sizes() != q->sizes()) refuse("out has q's shape");
    }
    const at::Tensor* lse = a.typed("lse", at::kFloat, 2, true);
    if (lse && (lse->size(0) != q->size(0) || lse->size(1) != q->size(1) || !lse->is_contiguous())) refuse("lse is contiguous [tokens, heads]");
    const at::Tensor* w = a.typed("weights", at::kFloat, 3, true);
    if (w) {
        weights_shape(*w, "weights", b.batch, r.cache.heads, r.max_length);
        r.weights_stride = w->size(1) > 1 ? w->stride(1) : w->size(0) > 1 ? w->stride(0) : w->size(2);
    }
    r.q = q->data_ptr();
    r.out = out.data_ptr();
    r.lse = ptr<float>(lse);
    r.weights = ptr<float>(w);
    r.q_stride = q->stride(0);
    r.q_head_stride = q->stride(1);
    r.out_stride = out.stride(0);
    r.out_head_stride = out.stride(1);
    r.q_start = b.q_start;
    r.lengths = b.lengths;
    r.block_table = b.table;
    r.table_stride = b.table_stride;
    r.table_blocks = b.table_blocks;
    r.batch = b.batch;
    r.tokens = count(q->size(0), "tokens");
    r.heads = count(q->size(1), "heads");
    r.stream = a.stream();
    size_t need = 0;
    if (a.next_is_none()) check(a.ctx(), i4d_kv8_attention_workspace(a.ctx(), &r, &need));
    const at::Tensor ws = workspace(a, need);
    if (ws.defined()) {
        r.workspace = ws.data_ptr();
        r.workspace_bytes = static_cast<size_t>(ws.numel());
    }
    check(a.ctx(), i4d_kv8_attention(a.ctx(), &r));
    return give(out);
}

PyObject* kv8_evict(Args& a) {
    i4d_kv8_evict_args r = {};
    r.cache = a.cache();
    const at::Tensor* l = a.typed("lengths", at::kInt, 1);
    const at::Tensor* t = a.typed("block_table", at::kInt, 2);
    const at::Tensor* w = a.typed("weights", at::kFloat, 3);
    r.budget = a.small("budget");
    r.recent = a.small("recent");
    r.max_length = a.small("max_length");
    r.batch = count(l->size(0), "batch");
    if (t->size(0) != r.batch) refuse("block_table is [batch, blocks]");
    if (r.budget < 0) refuse("budget %d", r.budget);
    weights_shape(*w, "weights", r.batch, r.cache.heads, r.max_length);
    at::Tensor lengths_out, keep, weights_out;
    const int64_t shape[3] = {r.batch, r.cache.heads, r.budget};
    if (a.next_is_none()) {
        lengths_out = at::empty(l->sizes(), l->options());
        a.skip();
    } else {
        lengths_out = *a.typed("lengths_out", at::kInt, 1);
        if (lengths_out.sizes() != l->sizes()) refuse("lengths_out is [batch]");
    }
    if (a.next_is_none()) {
        keep = at::empty(shape, l->options());
        a.skip();
    } else {
        keep = *a.typed("keep", at::kInt, 3);
        if (keep.sizes() != at::IntArrayRef(shape, 3) || !keep.is_contiguous()) refuse("keep is contiguous [batch, cache heads, budget]");
    }
    if (a.next_is_none()) {
        weights_out = *w;
        a.skip();
    } else {
        weights_out = *a.typed("weights_out", at::kFloat, 3);
        weights_shape(weights_out, "weights_out", r.batch, r.cache.heads, r.max_length);
    }
    const auto stride = [](const at::Tensor& x) { return x.size(1) > 1 ? x.stride(1) : x.size(0) > 1 ? x.stride(0) : x.size(2); };
    r.weights = ptr<float>(w);
    r.weights_out = ptr<float>(&weights_out);
    r.weights_stride = stride(*w);
    r.weights_out_stride = stride(weights_out);
    r.lengths = ptr<int32_t>(l);
    r.lengths_out = ptr<int32_t>(&lengths_out);
    r.keep = ptr<int32_t>(&keep);
    r.block_table = ptr<int32_t>(t);
    r.table_stride = row_stride(*t);
    r.table_blocks = count(t->size(1), "block_table");
    r.stream = a.stream();
    size_t need = 0;
    if (a.next_is_none()) check(a.ctx(), i4d_kv8_evict_workspace(a.ctx(), &r, &need));
    const at::Tensor ws = workspace(a, need);
    if (ws.defined()) {
        r.workspace = ws.data_ptr();
        r.workspace_bytes = static_cast<size_t>(ws.numel());
    }
    check(a.ctx(), i4d_kv8_evict(a.ctx(), &r));
    PyObject* triple = PyTuple_New(3);
    if (!triple) throw PyRaised{};
    PyTuple_SET_ITEM(triple, 0, give(lengths_out));
    PyTuple_SET_ITEM(triple, 1, give(keep));
    PyTuple_SET_ITEM(triple, 2, give(weights_out));
    return triple;
}

const at::Tensor* per_row(Args& a, const char* what, at::ScalarType type, int64_t rows) {
    const at::Tensor* t = a.typed(what, type, 1, true);
    if (t && t->size(0) != rows) refuse("%s has %lld entries, not one a row", what, static_cast<long long>(t->size(0)));
    return t;
}

const at::Tensor* table_of(Args& a, const char* what, at::ScalarType type, int64_t rows) {
    const at::Tensor* t = a.typed(what, type, 2, true);
    if (t && t->size(0) != rows) refuse("%s has %lld rows, not %lld", what, static_cast<long long>(t->size(0)), static_cast<long long>(rows));
    return t;
}

PyObject* logits_process(Args& a) {
    i4d_logits_args r = {};
    const at::Tensor* x = a.tensor("logits", 2);
    r.dtype = dtype_of(*x, "logits");
    const int64_t rows = x->size(0);
    at::Tensor out;
    if (a.next_is_none()) {
        out = at::empty(x->sizes(), x->options());
        a.skip();
    } else {
        out = *a.typed("out", x->scalar_type(), 2);
        if (out.sizes() != x->sizes()) refuse("out has the logits' shape");
    }
    r.best = ptr<int32_t>(per_row(a, "best", at::kInt, rows));
    const at::Tensor* hist = table_of(a, "history", at::kInt, rows);
    r.history_len = ptr<int32_t>(per_row(a, "history_len", at::kInt, rows));
    r.prompt_len = ptr<int32_t>(per_row(a, "prompt_len", at::kInt, rows));
    r.repetition = ptr<float>(per_row(a, "repetition", at::kFloat, rows));
    r.frequency = ptr<float>(per_row(a, "frequency", at::kFloat, rows));
    r.presence = ptr<float>(per_row(a, "presence", at::kFloat, rows));
    const at::Tensor* ids = table_of(a, "bias_ids", at::kInt, rows);
    const at::Tensor* values = table_of(a, "bias_values", at::kFloat, rows);
    r.bias_len = ptr<int32_t>(per_row(a, "bias_len", at::kInt, rows));
    const at::Tensor* mask = table_of(a, "mask", at::kInt, rows);
    if (hist) {
        r.history_stride = row_stride(*hist);
        r.history_max = count(hist->size(1), "history");
    }
    if (ids) {
        r.bias_stride = row_stride(*ids);
        r.bias_max = count(ids->size(1), "bias_ids");
        if (!values || values->sizes() != ids->sizes() || row_stride(*values) != r.bias_stride) refuse("bias_values has bias_ids' shape and strides");
    }
    if (mask) {
        if (mask->size(1) * 32 < x->size(1)) refuse("mask has fewer than vocab bits a row");
        r.mask_stride = row_stride(*mask);
    }
    r.logits = x->data_ptr();
    r.out = out.data_ptr();
    r.history = ptr<int32_t>(hist);
    r.bias_ids = ptr<int32_t>(ids);
    r.bias_values = ptr<float>(values);
    r.mask = static_cast<const uint32_t*>(mask ? mask->data_ptr() : nullptr);
    r.stride = x->stride(0);
    r.out_stride = out.stride(0);
    r.rows = count(rows, "rows");
    r.vocab = count(x->size(1), "vocab");
    r.stream = a.stream();
    check(a.ctx(), i4d_logits_process(a.ctx(), &r));
    return give(out);
}

// Waits for the stream without Python's lock, which what the stream waits for
// may need; what follows then waits for nothing of it, and the context and its
// message are touched with the lock held.
PyObject* ops_check(Args& a) {
    const cudaStream_t s = a.stream();
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(a.device()));
    cudaError_t e;
    Py_BEGIN_ALLOW_THREADS;
    e = cudaStreamSynchronize(s);
    Py_END_ALLOW_THREADS;
    if (e != cudaSuccess) throw OpError{I4D_ERR_CUDA, cudaGetErrorString(e)};
    check(a.ctx(), i4d_ops_check(a.ctx(), a.stream()));
    Py_RETURN_NONE;
}

// ------------------------------------------------------------------ module

template <PyObject* (*F)(Args&), int N>
PyObject* entry(PyObject*, PyObject* const* v, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    try {
        Args a(v, n, N);
        return F(a);
    } catch (const OpError& e) {
        raise(e);
    } catch (const PyRaised&) {
    }
    return nullptr;
    END_HANDLE_TH_ERRORS
}

PyObject* set_error(PyObject*, PyObject* cls) {
    Py_XINCREF(cls);
    Py_XDECREF(g_error);
    g_error = cls;
    Py_RETURN_NONE;
}

template <PyObject* (*F)(Args&), int N>
PyMethodDef method(const char* name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, N>)), METH_FASTCALL, nullptr};
}

PyMethodDef g_methods[] = {
    {"set_error", set_error, METH_O, nullptr},
    method<rope, 12>("rope"),
    method<kv8_append, 9>("kv8_append"),
    method<kv8_read, 10>("kv8_read"),
    method<kv8_attention, 15>("kv8_attention"),
    method<kv8_evict, 13>("kv8_evict"),
    method<logits_process, 15>("logits_process"),
    method<ops_check, 2>("ops_check"),
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_i4d_torch", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__i4d_torch() { return PyModule_Create(&g_module); }

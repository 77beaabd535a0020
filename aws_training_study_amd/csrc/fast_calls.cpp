// Per-call host path of the Python entry points, as a CPython extension over
// torch's C++ tensors.
//
// A small launch takes less time on the GPU than Python spends on checking
// its tensors and converting its arguments: 12 us of host work for a call of
// two kernels and 14 us more than here for an append of two, of which each
// launch itself takes 2.3 us (the C caller's figure).  Each object here is
// one entry point's call for a fixed configuration: it takes the common form
// of the arguments (plain GPU tensors of the expected shapes and types on the
// current device, Python floats and ints), checks exactly what the Python
// entry checks, allocates the outputs and calls the C ABI on the current
// stream.  For anything else it returns None, with nothing launched, and the
// Python entry goes on with its general path, conversions and error messages.
// A status of the C call other than PCPA_OK comes back as an int for the
// Python entry to raise: kernels may be queued by then, so the call is not made
// again.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <initializer_list>
#include <new>
#include <vector>

#include "pcp_attention_hip.h"

namespace {

// What the calls take and return, checked when the module is loaded (as is
// PCPA_TORCH_VERSION, the torch that the build line names).
constexpr int kVersion = 3;

PyObject* g_raw_stream = nullptr;  // torch._C._cuda_getCurrentRawStream
PyObject* g_device = nullptr;      // torch._C._cuda_getDevice
PyObject* g_capturing = nullptr;   // torch._C._cuda_isCurrentStreamCapturing

// A plain torch.Tensor (no subclass), or nullptr.
const at::Tensor* plain(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

bool shaped(const at::Tensor& t, std::initializer_list<int64_t> shape) {
    return t.sizes() == at::IntArrayRef(shape.begin(), shape.size());
}

// A contiguous strided tensor of `type` on GPU `dev`.
bool on_gpu(const at::Tensor& t, at::ScalarType type, int dev) {
    return t.is_cuda() && t.get_device() == dev && t.scalar_type() == type && t.layout() == at::kStrided &&
           t.is_contiguous();
}

bool table_on(const at::Tensor& t, int dev) {
    return on_gpu(t, at::kInt, dev) || on_gpu(t, at::kLong, dev);
}

// The current device if it is `dev`, and its current stream; false otherwise
// (with any Python error cleared).
bool current_stream(int dev, void*& stream) {
    PyObject* d = PyObject_CallNoArgs(g_device);
    const long cur = d ? PyLong_AsLong(d) : -1;
    Py_XDECREF(d);
    if (cur != dev) {
        PyErr_Clear();
        return false;
    }
    PyObject* index = PyLong_FromLong(dev);
    PyObject* s = index ? PyObject_CallOneArg(g_raw_stream, index) : nullptr;
    Py_XDECREF(index);
    if (!s) {
        PyErr_Clear();
        return false;
    }
    stream = PyLong_AsVoidPtr(s);
    Py_DECREF(s);
    if (PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}

bool real(PyObject* o, float& x) {
    if (!PyFloat_CheckExact(o)) return false;
    x = (float)PyFloat_AS_DOUBLE(o);
    return true;
}

bool whole(PyObject* o, int64_t& x) {
    if (!PyLong_CheckExact(o)) return false;
    int overflow = 0;
    x = PyLong_AsLongLongAndOverflow(o, &overflow);
    return !overflow;
}

// One entry point's call.
struct Call {
    PyObject_HEAD
    vectorcallfunc call;
    pcpa_params p;
    at::ScalarType kv_type;
    int32_t interleave;
    int dev;
    void* fn;
    // history
    int n_split;
    bool workspace;        // the split entry, with a workspace of ws_bytes
    int64_t ws_bytes;
    PyObject* ws_maker;    // f(bytes, stream) -> uint8 tensor
    struct Space {
        void* stream;
        at::Tensor tensor;
        unsigned long thread = 0;  // (attention of a chunk)
    };
    std::vector<Space>* spaces;
    // rotation
    pcpa_rotary rotary;    // without its device pointers
    // attention of a chunk: the entry that says how large its workspace is
    void* size_fn;
};

#define GIVE_UP Py_RETURN_NONE

using HistoryLse = decltype(&pcpa_history_attention_lse);
using HistorySplit = decltype(&pcpa_history_attention_split);
using Current = decltype(&pcpa_current_attention);
using Write = decltype(&pcpa_kv_cache_write);
using Alloc = decltype(&pcpa_page_alloc);

template <class F>
int32_t launch(F&& f) {
    int32_t status;
    Py_BEGIN_ALLOW_THREADS
    status = f();
    Py_END_ALLOW_THREADS
    return status;
}

PyObject* tensors(const at::Tensor& out, const at::Tensor& lse) {
    if (!lse.defined()) return THPVariable_Wrap(out);
    PyObject* a = THPVariable_Wrap(out);
    PyObject* b = THPVariable_Wrap(lse);
    PyObject* t = a && b ? PyTuple_Pack(2, a, b) : nullptr;
    Py_XDECREF(a);
    Py_XDECREF(b);
    return t;
}

// Forget the remembered workspaces.  Freeing a tensor can release the GIL, and
// another thread's call then looks through the same vector: it must find it
// whole, so the tensors are freed after they have left it.
void forget(Call* c) {
    std::vector<Call::Space> old;
    old.swap(*c->spaces);
}

// The workspace kept for `stream`: the Python object's (ws_maker), remembered
// here until it is told to forget.
void* workspace_for(Call* c, void* stream, at::Tensor& hold) {
    for (const Call::Space& s : *c->spaces)
        if (s.stream == stream) {
            hold = s.tensor;
            return hold.data_ptr();
        }
    PyObject* t = PyObject_CallFunction(c->ws_maker, "Ln", (long long)c->ws_bytes, (Py_ssize_t)(intptr_t)stream);
    if (!t) {
        // an interrupt is the caller's; errors are the general path's to meet
        if (PyErr_ExceptionMatches(PyExc_Exception)) PyErr_Clear();
        return nullptr;
    }
    hold = THPVariable_Unpack(t);
    Py_DECREF(t);
    if (c->spaces->size() >= 16) forget(c);
    c->spaces->push_back({stream, hold});
    return hold.data_ptr();
}

// (q, kv_pages, block_table, page_valid_len, k_scale, v_scale, out, return_lse) -> outputs or a status
PyObject* history(Call* c, PyObject* const* a) {
    const at::Tensor *q = plain(a[0]), *kv = plain(a[1]), *table = plain(a[2]), *valid = plain(a[3]);
    const at::Tensor* given = a[6] == Py_None ? nullptr : plain(a[6]);
    if (!q || !kv || !table || !valid || (a[6] != Py_None && !given)) GIVE_UP;
    pcpa_params p = c->p;
    if (!real(a[4], p.k_scale) || !real(a[5], p.v_scale) || !PyBool_Check(a[7])) GIVE_UP;
    const int dev = c->dev;
    const int64_t page = 2 * (int64_t)p.num_kv_heads * p.block_size * p.head_dim;
    if (!on_gpu(*q, at::kBFloat16, dev) || !shaped(*q, {p.pcp_size, p.num_q_heads, p.local_q_len, p.head_dim}) ||
        !on_gpu(*kv, c->kv_type, dev) || kv->dim() != 2 || kv->size(1) != page || kv->size(0) > INT32_MAX ||
        !table_on(*table, dev) || !shaped(*table, {p.pcp_size, p.max_local_blocks}) ||
        !on_gpu(*valid, at::kInt, dev) || !shaped(*valid, {p.pcp_size, p.max_local_blocks}))
        GIVE_UP;
    if (given && (!on_gpu(*given, at::kBFloat16, dev) || given->sizes() != q->sizes())) GIVE_UP;
    void* stream = nullptr;
    if (!current_stream(dev, stream)) GIVE_UP;
    p.num_pages = (int32_t)kv->size(0);
    if (table->scalar_type() == at::kLong) p.flags |= PCPA_FLAG_TABLE_INT64;
    const at::Tensor out = given ? *given : at::empty(q->sizes(), q->options().requires_grad(false));
    at::Tensor lse, ws;
    if (a[7] == Py_True)
        lse = at::empty({p.pcp_size, p.num_q_heads, p.local_q_len}, q->options().dtype(at::kFloat).requires_grad(false));
    float* const lse_ptr = lse.defined() ? (float*)lse.data_ptr() : nullptr;
    const void *qp = q->data_ptr(), *kp = kv->data_ptr(), *tp = table->data_ptr();
    const int32_t* const vp = (const int32_t*)valid->data_ptr();
    void* const op = out.data_ptr();
    int32_t status;
    if (c->workspace) {
        void* const w = workspace_for(c, stream, ws);
        if (!w) {
            if (PyErr_Occurred()) return nullptr;
            GIVE_UP;
        }
        status = launch([&] {
            return ((HistorySplit)c->fn)(&p, c->n_split, qp, kp, tp, vp, op, lse_ptr, w, c->ws_bytes, stream);
        });
    } else {
        status = launch([&] { return ((HistoryLse)c->fn)(&p, qp, kp, tp, vp, op, lse_ptr, stream); });
    }
    if (status) return PyLong_FromLong(status);
    return tensors(out, lse);
}

// (q, kv_current, hist_out, hist_lse, out, return_lse) -> outputs or a status
PyObject* current(Call* c, PyObject* const* a) {
    const at::Tensor *q = plain(a[0]), *kv = plain(a[1]);
    const at::Tensor* hist = a[2] == Py_None ? nullptr : plain(a[2]);
    const at::Tensor* hlse = a[3] == Py_None ? nullptr : plain(a[3]);
    const at::Tensor* given = a[4] == Py_None ? nullptr : plain(a[4]);
    if (!q || !kv || (a[2] != Py_None && !hist) || (a[3] != Py_None && !hlse) || (a[4] != Py_None && !given) ||
        !hist != !hlse || !PyBool_Check(a[5]) || !q->is_cuda())
        GIVE_UP;
    const pcpa_params& p = c->p;
    const int dev = q->get_device();
    const int64_t len = (int64_t)p.pcp_size * p.local_q_len;
    if (!on_gpu(*q, at::kBFloat16, dev) || !shaped(*q, {p.pcp_size, p.num_q_heads, p.local_q_len, p.head_dim}) ||
        !on_gpu(*kv, at::kBFloat16, dev) || !shaped(*kv, {2, p.num_kv_heads, len, p.head_dim}))
        GIVE_UP;
    if (hist && (!on_gpu(*hist, at::kBFloat16, dev) || hist->sizes() != q->sizes() ||
                 !on_gpu(*hlse, at::kFloat, dev) || !shaped(*hlse, {p.pcp_size, p.num_q_heads, p.local_q_len})))
        GIVE_UP;
    if (given && (!on_gpu(*given, at::kBFloat16, dev) || given->sizes() != q->sizes())) GIVE_UP;
    void* stream = nullptr;
    if (!current_stream(dev, stream)) GIVE_UP;
    const at::Tensor out = given ? *given : at::empty(q->sizes(), q->options().requires_grad(false));
    at::Tensor lse;
    if (a[5] == Py_True)
        lse = at::empty({p.pcp_size, p.num_q_heads, p.local_q_len}, q->options().dtype(at::kFloat).requires_grad(false));
    const void *qp = q->data_ptr(), *kp = kv->data_ptr(), *hp = hist ? hist->data_ptr() : nullptr;
    const float* const hl = hlse ? (const float*)hlse->data_ptr() : nullptr;
    void* const op = out.data_ptr();
    float* const lp = lse.defined() ? (float*)lse.data_ptr() : nullptr;
    const int32_t status =
        launch([&] { return ((Current)c->fn)(&p, c->interleave, qp, kp, hp, hl, op, lp, stream); });
    if (status) return PyLong_FromLong(status);
    return tensors(out, lse);
}

// (k, v, kv_pages, block_table, first_pos, k_scale, v_scale, page_valid_len) -> status
PyObject* write(Call* c, PyObject* const* a) {
    const at::Tensor *k = plain(a[0]), *v = plain(a[1]), *kv = plain(a[2]), *table = plain(a[3]);
    const at::Tensor* valid = a[7] == Py_None ? nullptr : plain(a[7]);
    pcpa_params p = c->p;
    int64_t first;
    if (!k || !v || !kv || !table || (a[7] != Py_None && !valid) || !whole(a[4], first) || first < 0 ||
        !real(a[5], p.k_scale) || !real(a[6], p.v_scale) || !k->is_cuda() || k->dim() != 3)
        GIVE_UP;
    const int dev = k->get_device();
    const int64_t page = 2 * (int64_t)p.num_kv_heads * p.block_size * p.head_dim, n = k->size(1);
    if (n > INT32_MAX || !on_gpu(*k, at::kBFloat16, dev) || !shaped(*k, {p.num_kv_heads, n, p.head_dim}) ||
        !on_gpu(*v, at::kBFloat16, dev) || v->sizes() != k->sizes() || !on_gpu(*kv, c->kv_type, dev) ||
        kv->dim() != 2 || kv->size(1) != page || kv->size(0) > INT32_MAX || !table_on(*table, dev) ||
        !shaped(*table, {p.pcp_size, p.max_local_blocks}) ||
        (valid && (!on_gpu(*valid, at::kInt, dev) || valid->sizes() != table->sizes())))
        GIVE_UP;
    void* stream = nullptr;
    if (!current_stream(dev, stream)) GIVE_UP;
    p.num_pages = (int32_t)kv->size(0);
    if (table->scalar_type() == at::kLong) p.flags |= PCPA_FLAG_TABLE_INT64;
    const void *kp = k->data_ptr(), *vp = v->data_ptr(), *tp = table->data_ptr();
    void* const pages = kv->data_ptr();
    int32_t* const lens = valid ? (int32_t*)valid->data_ptr() : nullptr;
    const int32_t status = launch([&] {
        return ((Write)c->fn)(&p, c->interleave, first, (int32_t)n, kp, vp, tp, pages, lens, stream);
    });
    return PyLong_FromLong(status);
}

// (first_pos, num_tokens, block_table, free_pages, free_count) -> status
PyObject* alloc(Call* c, PyObject* const* a) {
    const at::Tensor *table = plain(a[2]), *pages = plain(a[3]), *count = plain(a[4]);
    int64_t first, n;
    if (!table || !pages || !count || !whole(a[0], first) || !whole(a[1], n) || n < 0 || n > INT32_MAX ||
        !pages->is_cuda())
        GIVE_UP;
    pcpa_params p = c->p;
    const int dev = pages->get_device();
    if (!table_on(*table, dev) || !shaped(*table, {p.pcp_size, p.max_local_blocks})) GIVE_UP;
    void* stream = nullptr;
    if (!current_stream(dev, stream)) GIVE_UP;
    if (table->scalar_type() == at::kLong) p.flags |= PCPA_FLAG_TABLE_INT64;
    void* const tp = table->data_ptr();
    const int32_t* const pp = (const int32_t*)pages->data_ptr();
    int32_t* const cp = (int32_t*)count->data_ptr();
    const int32_t status =
        launch([&] { return ((Alloc)c->fn)(&p, c->interleave, first, (int32_t)n, tp, pp, cp, stream); });
    return PyLong_FromLong(status);
}

// ---- chunks of new tokens over paged caches -----------------------------------

// An argument that may be None: false for anything but None and a plain tensor.
bool optional(PyObject* o, const at::Tensor*& t) {
    t = o == Py_None ? nullptr : plain(o);
    return t || o == Py_None;
}

// [n, heads, head_dim] bf16 rows on GPU `dev` that the kernels can address.
bool rows_on(const at::Tensor& t, int64_t n, int64_t heads, int64_t d, int dev) {
    return t.is_cuda() && t.scalar_type() == at::kBFloat16 && t.get_device() == dev && t.layout() == at::kStrided &&
           shaped(t, {n, heads, d}) && t.stride(2) == 1 && (n == 1 || t.stride(0) % 8 == 0) &&
           (heads == 1 || t.stride(1) % 8 == 0) && ((uintptr_t)t.data_ptr() & 15u) == 0;
}
pcpa_rows view_of(const at::Tensor& t) {
    return pcpa_rows{t.data_ptr(), t.size(0) > 1 ? t.stride(0) : 0, t.size(1) > 1 ? t.stride(1) : 0};
}

// Whether the memory that the rows of a and b lie in meets (what is in between is
// the general path's to look at).
bool meet(const at::Tensor& a, const at::Tensor& b) {
    auto end = [](const at::Tensor& t) {
        int64_t last = 0;
        for (int i = 0; i < 3; ++i) last += (t.size(i) - 1) * t.stride(i);
        return (const char*)t.data_ptr() + 2 * (last + 1);
    };
    return (const char*)a.data_ptr() < end(b) && (const char*)b.data_ptr() < end(a);
}
// Whether a given output is its own input, or apart from it.
bool in_place_or_apart(const at::Tensor& out, const at::Tensor& in) {
    return (out.data_ptr() == in.data_ptr() && out.strides() == in.strides()) || !meet(out, in);
}

// The chunk of `n` rows that lengths and starts describe.
bool chunk_of(const Call* c, const at::Tensor& lengths, const at::Tensor* starts, int64_t n, int dev, pcpa_chunk& out) {
    if (!on_gpu(lengths, at::kInt, dev) || lengths.dim() != 1 || lengths.size(0) < 1 || lengths.size(0) >= INT32_MAX)
        return false;
    const int64_t batch = lengths.size(0);
    if (starts ? !on_gpu(*starts, at::kInt, dev) || !shaped(*starts, {batch + 1}) : n % batch != 0) return false;
    out = pcpa_chunk{c->interleave,  (int32_t)batch,
                     (int32_t)n,     0,
                     (const int32_t*)lengths.data_ptr(), starts ? (const int32_t*)starts->data_ptr() : nullptr};
    return true;
}

// The cache of a call: its pages, table of `batch` sequences and scales, into p.
bool cache_of(const Call* c, const at::Tensor& kv, const at::Tensor& table, const at::Tensor* scales, PyObject* k_scale,
              PyObject* v_scale, int64_t batch, int dev, pcpa_params& p) {
    const int64_t page = 2 * (int64_t)p.num_kv_heads * p.block_size * p.head_dim;
    if (!real(k_scale, p.k_scale) || !real(v_scale, p.v_scale) || !on_gpu(kv, c->kv_type, dev) || kv.dim() != 2 ||
        kv.size(1) != page || kv.size(0) < 1 || kv.size(0) > INT32_MAX || !table_on(table, dev))
        return false;
    if (!shaped(table, {batch, p.pcp_size, p.max_local_blocks}) &&
        !(batch == 1 && shaped(table, {p.pcp_size, p.max_local_blocks})))
        return false;
    if (scales && (c->kv_type != at::kFloat8_e4m3fn || !on_gpu(*scales, at::kFloat, dev) ||
                   !shaped(*scales, {kv.size(0), 2, p.num_kv_heads, p.block_size}) || p.k_scale != 1.f ||
                   p.v_scale != 1.f))
        return false;
    p.num_pages = (int32_t)kv.size(0);
    if (table.scalar_type() == at::kLong) p.flags |= PCPA_FLAG_TABLE_INT64;
    return true;
}

// The rotation with this device's frequencies and these weights.
bool rotary_of(const Call* c, const at::Tensor& turns, const at::Tensor* qw, const at::Tensor* kw, int dev,
               pcpa_rotary& r) {
    r = c->rotary;
    if (!on_gpu(turns, at::kDouble, dev) || turns.numel() != r.rotary_dim / 2) return false;
    r.turns = (const double*)turns.data_ptr();
    for (const at::Tensor* w : {qw, kw}) {
        if (!w) continue;
        const bool f32 = w->scalar_type() == at::kFloat;
        if (!on_gpu(*w, f32 ? at::kFloat : at::kBFloat16, dev) || !shaped(*w, {c->p.head_dim})) return false;
        if ((uintptr_t)w->data_ptr() & (f32 ? 15u : 7u)) return false;
        r.weight_dtype = f32 ? PCPA_DTYPE_FP32 : PCPA_DTYPE_BF16;
    }
    if (qw && kw && qw->scalar_type() != kw->scalar_type()) return false;
    r.q_weight = qw ? qw->data_ptr() : nullptr;
    r.k_weight = kw ? kw->data_ptr() : nullptr;
    return true;
}

// An output that was given (contiguous; other layouts are the general path's) or is made.
bool output(PyObject* o, const at::Tensor& like, at::IntArrayRef shape, int dev, at::Tensor& out) {
    const at::Tensor* given;
    if (!optional(o, given)) return false;
    if (given && (!on_gpu(*given, at::kBFloat16, dev) || given->sizes() != shape || ((uintptr_t)given->data_ptr() & 15u)))
        return false;
    out = given ? *given : at::empty(shape, like.options().requires_grad(false));
    return true;
}

using Rotate = decltype(&pcpa_rotate);
using ChunkWrite = decltype(&pcpa_chunk_write);
using ChunkPrepare = decltype(&pcpa_chunk_prepare);
using CacheRead = decltype(&pcpa_cache_read);
using ChunkAttention = decltype(&pcpa_chunk_attention);
using ChunkBytes = decltype(&pcpa_chunk_workspace_bytes);

// (q, k, positions, lengths, chunk_starts, q_weight, k_weight, q_out, k_out, turns) -> outputs or a status
PyObject* rotate(Call* c, PyObject* const* a) {
    const at::Tensor *q = plain(a[0]), *k = plain(a[1]), *positions, *lengths, *starts, *qw, *kw, *turns = plain(a[9]);
    if (!q || !k || !turns || !optional(a[2], positions) || !optional(a[3], lengths) || !optional(a[4], starts) ||
        !optional(a[5], qw) || !optional(a[6], kw) || !positions == !lengths || (positions && starts) || !q->is_cuda() ||
        q->dim() != 3 || q->size(0) < 1 || q->size(0) > INT32_MAX)
        GIVE_UP;
    const pcpa_params& p = c->p;
    const int dev = q->get_device();
    const int64_t n = q->size(0);
    pcpa_chunk chunk{c->interleave, 1, (int32_t)n, 0, nullptr, nullptr};
    pcpa_rotary r;
    at::Tensor q_out, k_out;
    int32_t bits = 0;
    if (!rows_on(*q, n, p.num_q_heads, p.head_dim, dev) || !rows_on(*k, n, p.num_kv_heads, p.head_dim, dev)) GIVE_UP;
    if (positions) {
        if (!table_on(*positions, dev) || !shaped(*positions, {n})) GIVE_UP;
        bits = positions->scalar_type() == at::kLong ? 64 : 32;
    } else if (!chunk_of(c, *lengths, starts, n, dev, chunk)) {
        GIVE_UP;
    }
    if (!rotary_of(c, *turns, qw, kw, dev, r) || !output(a[7], *q, {n, p.num_q_heads, p.head_dim}, dev, q_out) ||
        !output(a[8], *q, {n, p.num_kv_heads, p.head_dim}, dev, k_out))
        GIVE_UP;
    if (a[7] != Py_None && (!in_place_or_apart(q_out, *q) || meet(q_out, *k) || meet(q_out, k_out))) GIVE_UP;
    if (a[8] != Py_None && (!in_place_or_apart(k_out, *k) || meet(k_out, *q) || meet(k_out, q_out))) GIVE_UP;
    void* stream = nullptr;
    if (!current_stream(dev, stream)) GIVE_UP;
    const pcpa_rows qi = view_of(*q), ki = view_of(*k), qo = view_of(q_out), ko = view_of(k_out);
    const void* const pp = positions ? positions->data_ptr() : nullptr;
    const int32_t status = launch([&] {
        return ((Rotate)c->fn)(&p, &chunk, &r, pp, bits, 0, &qi, &ki, nullptr, &qo, &ko, nullptr, 0, stream);
    });
    if (status) return PyLong_FromLong(status);
    return tensors(q_out, k_out);
}

// (q, k, v, first_pos, q_weight, k_weight, turns) -> (q_stacked, kv_current) or a status
PyObject* rotate_prefill(Call* c, PyObject* const* a) {
    const at::Tensor *q = plain(a[0]), *k = plain(a[1]), *v = plain(a[2]), *qw, *kw, *turns = plain(a[6]);
    int64_t first;
    if (!q || !k || !v || !turns || !whole(a[3], first) || first < 0 || first >= (1ll << 62) || !optional(a[4], qw) ||
        !optional(a[5], kw) || !q->is_cuda())
        GIVE_UP;
    const pcpa_params& p = c->p;
    const int dev = q->get_device();
    const int64_t n = (int64_t)p.pcp_size * p.local_q_len;
    pcpa_rotary r;
    if (n > INT32_MAX || !rows_on(*q, n, p.num_q_heads, p.head_dim, dev) ||
        !rows_on(*k, n, p.num_kv_heads, p.head_dim, dev) || !rows_on(*v, n, p.num_kv_heads, p.head_dim, dev) ||
        !rotary_of(c, *turns, qw, kw, dev, r))
        GIVE_UP;
    void* stream = nullptr;
    if (!current_stream(dev, stream)) GIVE_UP;
    const auto options = q->options().requires_grad(false);
    const at::Tensor stacked = at::empty({p.pcp_size, p.num_q_heads, p.local_q_len, p.head_dim}, options);
    const at::Tensor kv = at::empty({2, p.num_kv_heads, n, p.head_dim}, options);
    const pcpa_chunk chunk{c->interleave, 1, (int32_t)n, 0, nullptr, nullptr};
    const pcpa_rows qi = view_of(*q), ki = view_of(*k), vi = view_of(*v), qo{stacked.data_ptr(), 0, 0};
    const pcpa_rows ko{kv.data_ptr(), p.head_dim, n * p.head_dim};
    const pcpa_rows vo{(char*)kv.data_ptr() + (int64_t)p.num_kv_heads * n * p.head_dim * 2, ko.token_stride,
                       ko.head_stride};
    const int32_t status = launch([&] {
        return ((Rotate)c->fn)(&p, &chunk, &r, nullptr, -1, first, &qi, &ki, &vi, &qo, &ko, &vo, 1, stream);
    });
    if (status) return PyLong_FromLong(status);
    return tensors(stacked, kv);
}

// (k, v, kv_pages, block_table, lengths, chunk_starts, k_scale, v_scale, token_scales) -> status
PyObject* chunk_write(Call* c, PyObject* const* a) {
    const at::Tensor *k = plain(a[0]), *v = plain(a[1]), *kv = plain(a[2]), *table = plain(a[3]), *lengths = plain(a[4]);
    const at::Tensor *starts, *scales;
    if (!k || !v || !kv || !table || !lengths || !optional(a[5], starts) || !optional(a[8], scales) || !k->is_cuda() ||
        k->dim() != 3 || k->size(0) < 1 || k->size(0) > INT32_MAX)
        GIVE_UP;
    pcpa_params p = c->p;
    const int dev = k->get_device();
    const int64_t n = k->size(0);
    pcpa_chunk chunk;
    if (!rows_on(*k, n, p.num_kv_heads, p.head_dim, dev) || !rows_on(*v, n, p.num_kv_heads, p.head_dim, dev) ||
        !chunk_of(c, *lengths, starts, n, dev, chunk) ||
        !cache_of(c, *kv, *table, scales, a[6], a[7], chunk.batch, dev, p))
        GIVE_UP;
    void* stream = nullptr;
    if (!current_stream(dev, stream)) GIVE_UP;
    const pcpa_rows ki = view_of(*k), vi = view_of(*v);
    void *tp = table->data_ptr(), *pages = kv->data_ptr();
    float* const sp = scales ? (float*)scales->data_ptr() : nullptr;
    return PyLong_FromLong(
        launch([&] { return ((ChunkWrite)c->fn)(&p, &chunk, &ki, &vi, tp, pages, sp, stream); }));
}

// (q, k, v, kv_pages, block_table, lengths, chunk_starts, q_weight, k_weight, k_scale, v_scale, token_scales, q_out,
// turns) -> q_out or a status
PyObject* chunk_prepare(Call* c, PyObject* const* a) {
    const at::Tensor *q = plain(a[0]), *k = plain(a[1]), *v = plain(a[2]), *kv = plain(a[3]), *table = plain(a[4]);
    const at::Tensor *lengths = plain(a[5]), *turns = plain(a[13]), *starts, *qw, *kw, *scales;
    if (!q || !k || !v || !kv || !table || !lengths || !turns || !optional(a[6], starts) || !optional(a[7], qw) ||
        !optional(a[8], kw) || !optional(a[11], scales) || !q->is_cuda() || q->dim() != 3 || q->size(0) < 1 ||
        q->size(0) > INT32_MAX)
        GIVE_UP;
    pcpa_params p = c->p;
    const int dev = q->get_device();
    const int64_t n = q->size(0);
    pcpa_chunk chunk;
    pcpa_rotary r;
    at::Tensor q_out;
    if (!rows_on(*q, n, p.num_q_heads, p.head_dim, dev) || !rows_on(*k, n, p.num_kv_heads, p.head_dim, dev) ||
        !rows_on(*v, n, p.num_kv_heads, p.head_dim, dev) || !chunk_of(c, *lengths, starts, n, dev, chunk) ||
        !cache_of(c, *kv, *table, scales, a[9], a[10], chunk.batch, dev, p) || !rotary_of(c, *turns, qw, kw, dev, r) ||
        !output(a[12], *q, {n, p.num_q_heads, p.head_dim}, dev, q_out))
        GIVE_UP;
    if (a[12] != Py_None && (!in_place_or_apart(q_out, *q) || meet(q_out, *k) || meet(q_out, *v))) GIVE_UP;
    void* stream = nullptr;
    if (!current_stream(dev, stream)) GIVE_UP;
    const pcpa_rows qi = view_of(*q), ki = view_of(*k), vi = view_of(*v), qo = view_of(q_out);
    void *tp = table->data_ptr(), *pages = kv->data_ptr();
    float* const sp = scales ? (float*)scales->data_ptr() : nullptr;
    const int32_t status = launch(
        [&] { return ((ChunkPrepare)c->fn)(&p, &chunk, &r, &qi, &ki, &vi, &qo, tp, pages, sp, stream); });
    if (status) return PyLong_FromLong(status);
    return THPVariable_Wrap(q_out);
}

// (kv_pages, block_table, first_pos, num_tokens, k_scale, v_scale, token_scales) -> (k, v) or a status
PyObject* cache_read(Call* c, PyObject* const* a) {
    const at::Tensor *kv = plain(a[0]), *table = plain(a[1]), *scales;
    int64_t first, n;
    if (!kv || !table || !whole(a[2], first) || !whole(a[3], n) || first < 0 || first >= (1ll << 62) || n < 1 ||
        n > INT32_MAX || !optional(a[6], scales) || !kv->is_cuda())
        GIVE_UP;
    pcpa_params p = c->p;
    const int dev = kv->get_device();
    if (!cache_of(c, *kv, *table, scales, a[4], a[5], 1, dev, p)) GIVE_UP;
    void* stream = nullptr;
    if (!current_stream(dev, stream)) GIVE_UP;
    const auto options = kv->options().dtype(at::kBFloat16).requires_grad(false);
    const at::Tensor k = at::empty({p.num_kv_heads, n, p.head_dim}, options), v = at::empty(k.sizes(), options);
    const void *tp = table->data_ptr(), *pages = kv->data_ptr();
    const float* const sp = scales ? (const float*)scales->data_ptr() : nullptr;
    void *kp = k.data_ptr(), *vp = v.data_ptr();
    const int32_t status = launch(
        [&] { return ((CacheRead)c->fn)(&p, c->interleave, first, (int32_t)n, tp, pages, sp, kp, vp, stream); });
    if (status) return PyLong_FromLong(status);
    return tensors(k, v);
}

// The workspace of `bytes` kept for this thread's calls on `stream` (another
// thread's launches may come between a call's two); one of the graph's own under
// capture.
bool chunk_workspace(Call* c, int64_t bytes, void* stream, const at::Tensor& q, at::Tensor& hold) {
    PyObject* capturing = PyObject_CallNoArgs(g_capturing);
    const int is = capturing ? PyObject_IsTrue(capturing) : -1;
    Py_XDECREF(capturing);
    if (is < 0) return false;
    if (is) {
        hold = at::empty({bytes}, q.options().dtype(at::kByte).requires_grad(false));
        return true;
    }
    const unsigned long thread = PyThread_get_thread_ident();
    for (const Call::Space& s : *c->spaces)
        if (s.stream == stream && s.thread == thread && s.tensor.get_device() == q.get_device()) {
            if (s.tensor.numel() >= bytes) {
                hold = s.tensor;
                return true;
            }
            break;
        }
    // (the Python object keeps it and forgets here what it drops)
    PyObject* t = PyObject_CallFunction(c->ws_maker, "Lin", (long long)bytes, (int)q.get_device(),
                                        (Py_ssize_t)(intptr_t)stream);
    if (!t) return false;
    hold = THPVariable_Unpack(t);
    Py_DECREF(t);
    c->spaces->push_back({stream, hold, thread});
    return true;
}

// (q, kv_pages, block_table, lengths, chunk_starts, k_scale, v_scale, token_scales, out, return_lse, workspace)
// -> outputs or a status
PyObject* chunk_attention(Call* c, PyObject* const* a) {
    const at::Tensor *q = plain(a[0]), *kv = plain(a[1]), *table = plain(a[2]), *lengths = plain(a[3]);
    const at::Tensor *starts, *scales, *given_ws;
    if (!q || !kv || !table || !lengths || !optional(a[4], starts) || !optional(a[7], scales) || !PyBool_Check(a[9]) ||
        !optional(a[10], given_ws) || !q->is_cuda() || q->dim() != 3 || q->size(0) < 1 || q->size(0) > INT32_MAX)
        GIVE_UP;
    pcpa_params p = c->p;
    const int dev = q->get_device();
    const int64_t n = q->size(0);
    pcpa_chunk chunk;
    at::Tensor out, lse, ws;
    if (!on_gpu(*q, at::kBFloat16, dev) || !shaped(*q, {n, p.num_q_heads, p.head_dim}) ||
        ((uintptr_t)q->data_ptr() & 15u) || !chunk_of(c, *lengths, starts, n, dev, chunk) ||
        !cache_of(c, *kv, *table, scales, a[5], a[6], chunk.batch, dev, p) ||
        (given_ws && !on_gpu(*given_ws, at::kByte, dev)) || !output(a[8], *q, q->sizes(), dev, out) || (a[8] != Py_None && !in_place_or_apart(out, *q)))
        GIVE_UP;
    void* stream = nullptr;
    if (!current_stream(dev, stream)) GIVE_UP;
    const int64_t bytes = ((ChunkBytes)c->size_fn)(&p, &chunk);
    if (bytes < 0) return PyLong_FromLong((long)bytes);
    if (given_ws) {
        ws = *given_ws;
    } else if (bytes > 0 && !chunk_workspace(c, bytes, stream, *q, ws)) {
        // an interrupt is the caller's; errors are the general path's to meet
        if (PyErr_Occurred() && !PyErr_ExceptionMatches(PyExc_Exception)) return nullptr;
        PyErr_Clear();
        GIVE_UP;
    }
    if (a[9] == Py_True) lse = at::empty({n, p.num_q_heads}, q->options().dtype(at::kFloat).requires_grad(false));
    const void *qp = q->data_ptr(), *pages = kv->data_ptr(), *tp = table->data_ptr();
    const float* const sp = scales ? (const float*)scales->data_ptr() : nullptr;
    void *op = out.data_ptr(), *wp = ws.defined() ? ws.data_ptr() : nullptr;
    float* const lp = lse.defined() ? (float*)lse.data_ptr() : nullptr;
    const int64_t have = ws.defined() ? ws.numel() : 0;
    const int32_t status = launch(
        [&] { return ((ChunkAttention)c->fn)(&p, &chunk, qp, pages, sp, tp, op, lp, wp, have, stream); });
    if (status) return PyLong_FromLong(status);
    return tensors(out, lse);
}

template <PyObject* (*F)(Call*, PyObject* const*), Py_ssize_t N>
PyObject* vector(PyObject* self, PyObject* const* args, size_t nargsf, PyObject* kwnames) {
    if (PyVectorcall_NARGS(nargsf) != N || kwnames) {
        PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
        return nullptr;
    }
    try {
        return F((Call*)self, args);
    } catch (...) {
        // e.g. a tensor without storage: the general path says so
        PyErr_Clear();
        Py_RETURN_NONE;
    }
}

void call_dealloc(PyObject* self) {
    Call* c = (Call*)self;
    PyObject_GC_UnTrack(self);
    Py_CLEAR(c->ws_maker);
    delete c->spaces;
    Py_TYPE(self)->tp_free(self);
}
int call_traverse(PyObject* self, visitproc visit, void* arg) {
    Py_VISIT(((Call*)self)->ws_maker);
    return 0;
}
int call_clear(PyObject* self) {
    Py_CLEAR(((Call*)self)->ws_maker);
    return 0;
}
PyObject* call_forget(PyObject* self, PyObject*) {
    forget((Call*)self);
    Py_RETURN_NONE;
}
PyMethodDef call_methods[] = {
    {"forget", call_forget, METH_NOARGS, "Drop the workspaces remembered for streams."},
    {nullptr, nullptr, 0, nullptr},
};
PyTypeObject CallType = {PyVarObject_HEAD_INIT(nullptr, 0)};

Call* new_call(vectorcallfunc f, const char* params, Py_ssize_t size, int fp8, int interleave, unsigned long long fn) {
    if (size != (Py_ssize_t)sizeof(pcpa_params)) {
        PyErr_SetString(PyExc_ValueError, "launch parameters of another size");
        return nullptr;
    }
    Call* c = PyObject_GC_New(Call, &CallType);
    if (!c) return nullptr;
    c->call = f;
    memcpy(&c->p, params, sizeof(pcpa_params));
    c->kv_type = fp8 ? at::kFloat8_e4m3fn : at::kBFloat16;
    c->interleave = interleave;
    c->dev = -1;
    c->fn = (void*)(uintptr_t)fn;
    c->n_split = 1;
    c->workspace = false;
    c->ws_bytes = 0;
    c->ws_maker = nullptr;
    c->rotary = pcpa_rotary{};
    c->size_fn = nullptr;
    c->spaces = new (std::nothrow) std::vector<Call::Space>();
    PyObject_GC_Track((PyObject*)c);
    if (!c->spaces) {
        Py_DECREF(c);
        PyErr_NoMemory();
        return nullptr;
    }
    return c;
}

// make(kind, params bytes, fp8 cache, interleave, C function address)
PyObject* make(PyObject*, PyObject* args) {
    const char *kind, *params;
    Py_ssize_t size;
    int fp8, interleave;
    unsigned long long fn;
    if (!PyArg_ParseTuple(args, "sy#piK", &kind, &params, &size, &fp8, &interleave, &fn)) return nullptr;
    vectorcallfunc f = !strcmp(kind, "current") ? vector<current, 6>
                       : !strcmp(kind, "write") ? vector<write, 8>
                       : !strcmp(kind, "alloc") ? vector<alloc, 5>
                       : !strcmp(kind, "chunk_write") ? vector<chunk_write, 9>
                       : !strcmp(kind, "cache_read")  ? vector<cache_read, 7>
                                                      : nullptr;
    if (!f) {
        PyErr_SetString(PyExc_ValueError, "unknown call");
        return nullptr;
    }
    return (PyObject*)new_call(f, params, size, fp8, interleave, fn);
}

// make_history(params bytes, fp8 cache, C function address, device index, splits, workspace bytes or -1, maker)
PyObject* make_history(PyObject*, PyObject* args) {
    const char* params;
    Py_ssize_t size;
    int fp8, dev, splits;
    unsigned long long fn;
    long long ws;
    PyObject* maker;
    if (!PyArg_ParseTuple(args, "y#pKiiLO", &params, &size, &fp8, &fn, &dev, &splits, &ws, &maker)) return nullptr;
    Call* c = new_call(vector<history, 8>, params, size, fp8, 0, fn);
    if (!c) return nullptr;
    c->dev = dev;
    c->n_split = splits;
    c->workspace = ws >= 0;
    c->ws_bytes = ws;
    Py_INCREF(maker);
    c->ws_maker = maker;
    return (PyObject*)c;
}

// make_rotation(kind, params bytes, fp8 cache, interleave, C function address, rotary bytes)
PyObject* make_rotation(PyObject*, PyObject* args) {
    const char *kind, *params, *rotary;
    Py_ssize_t size, rotary_size;
    int fp8, interleave;
    unsigned long long fn;
    if (!PyArg_ParseTuple(args, "sy#piKy#", &kind, &params, &size, &fp8, &interleave, &fn, &rotary, &rotary_size))
        return nullptr;
    vectorcallfunc f = !strcmp(kind, "rotate")           ? vector<rotate, 10>
                       : !strcmp(kind, "rotate_prefill") ? vector<rotate_prefill, 7>
                       : !strcmp(kind, "chunk_prepare")  ? vector<chunk_prepare, 14>
                                                         : nullptr;
    if (!f || rotary_size != (Py_ssize_t)sizeof(pcpa_rotary)) {
        PyErr_SetString(PyExc_ValueError, "unknown call, or a rotation of another size");
        return nullptr;
    }
    Call* c = new_call(f, params, size, fp8, interleave, fn);
    if (c) memcpy(&c->rotary, rotary, sizeof(pcpa_rotary));
    return (PyObject*)c;
}

// make_attention(params bytes, fp8 cache, interleave, C function address, that of its workspace's size, maker)
PyObject* make_attention(PyObject*, PyObject* args) {
    const char* params;
    Py_ssize_t size;
    int fp8, interleave;
    unsigned long long fn, size_fn;
    PyObject* maker;
    if (!PyArg_ParseTuple(args, "y#piKKO", &params, &size, &fp8, &interleave, &fn, &size_fn, &maker)) return nullptr;
    Call* c = new_call(vector<chunk_attention, 11>, params, size, fp8, interleave, fn);
    if (!c) return nullptr;
    c->size_fn = (void*)(uintptr_t)size_fn;
    Py_INCREF(maker);
    c->ws_maker = maker;
    return (PyObject*)c;
}

PyMethodDef methods[] = {
    {"make_rotation", make_rotation, METH_VARARGS, "A call that rotates Q and K."},
    {"make_attention", make_attention, METH_VARARGS, "A call of the attention of a chunk."},
    {"make", make, METH_VARARGS, "A call of the current step, a cache writer or reader or the page allocator."},
    {"make_history", make_history, METH_VARARGS, "A call of the history attention."},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_pcpa_fast_calls", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__pcpa_fast_calls(void) {
    CallType.tp_name = "_pcpa_fast_calls.Call";
    CallType.tp_basicsize = sizeof(Call);
    CallType.tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_HAVE_VECTORCALL | Py_TPFLAGS_HAVE_GC;
    CallType.tp_vectorcall_offset = offsetof(Call, call);
    CallType.tp_call = PyVectorcall_Call;
    CallType.tp_dealloc = call_dealloc;
    CallType.tp_traverse = call_traverse;
    CallType.tp_clear = call_clear;
    CallType.tp_methods = call_methods;
    if (PyType_Ready(&CallType) < 0) return nullptr;
    PyObject* c = PyImport_ImportModule("torch._C");
    if (!c) return nullptr;
    g_raw_stream = PyObject_GetAttrString(c, "_cuda_getCurrentRawStream");
    g_device = PyObject_GetAttrString(c, "_cuda_getDevice");
    g_capturing = PyObject_GetAttrString(c, "_cuda_isCurrentStreamCapturing");
    Py_DECREF(c);
    if (!g_raw_stream || !g_device || !g_capturing) return nullptr;
    PyObject* const m = PyModule_Create(&module);
    if (!m) return nullptr;
    if (PyModule_AddIntConstant(m, "version", kVersion) < 0 ||
        PyModule_AddStringConstant(m, "torch_version", PCPA_TORCH_VERSION) < 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}

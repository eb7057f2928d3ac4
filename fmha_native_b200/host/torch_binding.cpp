// torch_binding.cpp -- the torch side of the serving operators: checks of the
// tensors, output and workspace allocation, and the calls of the C ABI in
// include/fmha_paged.h.  fmha_native_b200/paged.py wraps these functions with
// their keyword forms and documentation.
//
// A decode step runs kernels of a few microseconds; in Python the same checks
// take longer than that.  The C entries are called through pointers that
// bind() receives, so this module follows whichever library Python loaded.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <string>

#include "fmha_paged.h"

namespace {

struct Bad {
    int status;
    std::string what;
};
struct PythonError {};  // already set

[[noreturn]] void bad(std::string what) { throw Bad{FMHA_ERR_ARG, std::move(what)}; }

using RopeFn = int (*)(const FmhaRopeParams*, CUstream_st*);
using PagedFn = int (*)(const FmhaPagedParams*, CUstream_st*);
using BytesFn = size_t (*)(int, int, int, int, int, int);
RopeFn g_rope = nullptr, g_append = nullptr;
PagedFn g_paged = nullptr, g_prefix = nullptr;
BytesFn g_bytes = nullptr;
PyObject* g_error = nullptr;  // FmhaError(status, what)

const at::Tensor& tensor(PyObject* o, const char* what) {
    if (!THPVariable_Check(o)) bad(std::string(what) + " must be a tensor");
    return THPVariable_Unpack(o);
}
const at::Tensor* optional(PyObject* o, const char* what) { return o == Py_None ? nullptr : &tensor(o, what); }

long long integer(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw PythonError{};
    return v;
}
bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw PythonError{};
    return v != 0;
}
int narrow(long long v, const char* what) {
    if (v < 0 || v > 0x7fffffffll) bad(std::string(what) + " is out of range");
    return (int)v;
}

// Layout codes of paged.py: thd, htd, bshd, bhsd.
struct Axes {
    int token, head;
    bool dense;
};
Axes axes_of(PyObject* layout) {
    switch (integer(layout)) {
        case 0: return {0, 1, false};
        case 1: return {1, 0, false};
        case 2: return {1, 2, true};
        case 3: return {2, 1, true};
        default: bad("unknown layout");
    }
}

struct Heads {
    uint16_t* p;
    long long token, head, batch;  // strides
    long long tokens, heads, batches;
};
Heads heads(const at::Tensor& x, const char* what, Axes ax, int device) {
    if (!x.is_cuda() || x.scalar_type() != at::kBFloat16 || x.dim() != (ax.dense ? 4 : 3) || x.size(-1) != 64)
        bad(std::string(what) + " must be a CUDA bf16 tensor with head_dim 64 and the layout's dimensions");
    if (x.stride(-1) != 1) bad(std::string(what) + ": the head dimension must be contiguous");
    if (x.get_device() != device) bad(std::string(what) + " must be on the same device as the others");
    return {static_cast<uint16_t*>(x.data_ptr()), x.stride(ax.token), x.stride(ax.head),
            ax.dense ? x.stride(0) : 0, x.size(ax.token), x.size(ax.head), ax.dense ? x.size(0) : 1};
}
bool same_tokens(const Heads& a, const Heads& b) { return a.tokens == b.tokens && a.batches == b.batches; }
bool same_shape(const Heads& a, const Heads& b) { return same_tokens(a, b) && a.heads == b.heads; }

const int32_t* ints(const at::Tensor& x, const char* what, int dims, int device) {
    if (!x.is_cuda() || x.scalar_type() != at::kInt || x.dim() != dims || x.get_device() != device ||
        (x.size(-1) > 1 && x.stride(-1) != 1))
        bad(std::string(what) + " must be an int32 tensor of " + std::to_string(dims) +
            " dimension(s) on the same device, its last dimension contiguous");
    return static_cast<const int32_t*>(x.data_ptr());
}

// The angle table and the axis of every pair, from `sections` (pairs of each
// axis in order) or `axis_of` (axis of each pair).  Returns the axes named.
int angles(FmhaRopeParams& p, const at::Tensor& t, PyObject* sections, PyObject* axis_of, int device) {
    if (!t.is_cuda() || t.scalar_type() != at::kFloat || t.dim() != 2 || !t.is_contiguous() || t.get_device() != device)
        bad("cos_sin must be a contiguous fp32 [max_pos, rot_dim] tensor on the same device");
    const long long rot = t.size(1);
    if (rot != 16 && rot != 32 && rot != 48 && rot != 64)
        bad("cos_sin must be [max_pos, rot_dim] with rot_dim 16, 32, 48 or 64");
    p.cos_sin = static_cast<const float*>(t.data_ptr());
    p.max_pos = narrow(t.size(0), "max_pos");
    if (p.max_pos == 0) bad("cos_sin has no rows");
    p.n_pairs = (int)rot / 2;
    int filled = 0, most = 0;
    auto put = [&](long long axis, long long count) {
        if (axis < 0 || axis > 3 || count < 0 || filled + count > p.n_pairs)
            bad("sections / axis_of must assign every pair to one of at most 4 axes");
        for (long long i = 0; i < count; ++i) p.axis_of[filled++] = (uint8_t)axis;
        if (count > 0 && axis > most) most = (int)axis;
    };
    PyObject* given = axis_of != Py_None ? axis_of : sections;
    if (given == Py_None) {
        put(0, p.n_pairs);
    } else {
        PyObject* seq = PySequence_Fast(given, "sections and axis_of are sequences of integers");
        if (!seq) throw PythonError{};
        struct Hold {
            PyObject* o;
            ~Hold() { Py_DECREF(o); }
        } hold{seq};
        const Py_ssize_t n = PySequence_Fast_GET_SIZE(seq);
        for (Py_ssize_t i = 0; i < n; ++i) {
            const long long v = integer(PySequence_Fast_GET_ITEM(seq, i));
            if (axis_of != Py_None) put(v, 1);
            else put(i, v);
        }
    }
    if (filled != p.n_pairs) bad("sections / axis_of must assign every pair to one of at most 4 axes");
    return most + 1;
}

// Positions: the token dimensions, or [axes, token dimensions].
void positions(FmhaRopeParams& p, const at::Tensor& t, const Heads& x, Axes ax, int axes, int device) {
    const int lead = ax.dense ? 2 : 1;
    const bool many = t.dim() == lead + 1;
    if (t.dim() != lead && !many) bad("positions must have the token dimensions, or [axes] and those");
    p.positions = ints(t, "positions", (int)t.dim(), device);
    const int d = many ? 1 : 0;
    const long long have = many ? t.size(0) : 1;
    if (t.size(d + lead - 1) != x.tokens || (ax.dense && t.size(d) != x.batches) || have < axes ||
        (ax.dense && x.batches > 1 && t.stride(d) != x.tokens))
        bad("positions must have a row for every axis, contiguous over the tokens");
    p.axis_stride = many ? t.stride(0) : 0;
}

struct Cache {
    Heads k, v;
    int page, heads, pages;
};
Cache cache(const at::Tensor& k, const at::Tensor& v, int device) {
    const Axes ax{1, 2, true};  // [pages, tokens, heads, 64]
    if (k.sizes() != v.sizes()) bad("k_cache and v_cache must have the same shape");
    Cache c{heads(k, "k_cache", ax, device), heads(v, "v_cache", ax, device), 0, 0, 0};
    c.page = narrow(c.k.tokens, "page_size");
    c.heads = narrow(c.k.heads, "heads");
    c.pages = narrow(c.k.batches, "num_pages");
    return c;
}

struct Batch {
    const int32_t *table, *lengths, *starts;
    long long table_stride;
    int batch, max_pages;
};
Batch batch_of(const at::Tensor& table, const at::Tensor& lengths, const at::Tensor* starts, const Heads& x, Axes ax,
               int device) {
    Batch b{ints(table, "page_table", 2, device), ints(lengths, "seqlens_k", 1, device), nullptr, table.stride(0),
            narrow(lengths.size(0), "batch"), narrow(table.size(1), "max_pages")};
    if (table.size(0) != b.batch) bad("page_table must be [batch, max_pages] and seqlens_k [batch]");
    if (ax.dense) {
        if (starts || x.batches != b.batch)
            bad("dense tokens are [batch, seqlen_q, ...] with page_table's batch and no cu_seqlens_q");
    } else {
        if (!starts) bad("packed tokens need cu_seqlens_q");
        b.starts = ints(*starts, "cu_seqlens_q", 1, device);
        if (starts->size(0) != b.batch + 1) bad("cu_seqlens_q must be [batch + 1]");
    }
    return b;
}

// The stream of a call: the current one, or the one that the caller names.  A
// named stream is the current one while a CallStream lives, so that the scratch
// and the results come from memory that is this stream's to use: the allocator
// hands a block that was freed on one stream to that stream's next request at
// once, whatever other streams still do with it.  given(): a result goes back to
// a caller on another stream, who may drop it while that stream still reads it.
class CallStream {
public:
    CallStream(PyObject* o, int device) : outer_(c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device)) {
        cudaStream_t named = outer_.stream();
        if (o != Py_None) named = reinterpret_cast<cudaStream_t>(static_cast<uintptr_t>(integer(o)));
        if (named == cudaStreamLegacy) named = nullptr;  // two names of the default stream
        stream_ = named;
        other_ = named != outer_.stream();
        if (other_)
            c10::cuda::setCurrentCUDAStream(c10::cuda::getStreamFromExternal(named, (c10::DeviceIndex)device));
    }
    ~CallStream() {
        if (other_) c10::cuda::setCurrentCUDAStream(outer_);
    }
    CallStream(const CallStream&) = delete;
    CallStream& operator=(const CallStream&) = delete;
    CUstream_st* get() const { return stream_; }
    const at::Tensor& given(const at::Tensor& t) const {
        if (other_) t.record_stream(outer_);
        return t;
    }

private:
    c10::cuda::CUDAStream outer_;
    cudaStream_t stream_ = nullptr;
    bool other_ = false;
};

// A given tensor was written: autograd, which this module runs below, must not
// take it for what it saved.  (Inference tensors have no version.)
void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

void done(int status, const char* what) {
    if (status != FMHA_OK) throw Bad{status, what};
}

PyObject* none() { Py_RETURN_NONE; }
PyObject* wrapped(PyObject* given, const at::Tensor& t) {
    if (given != Py_None) return Py_NewRef(given);
    return THPVariable_Wrap(t);
}

// q, k, cos_sin, positions, sections, axis_of, interleaved, inverse, layout, q_out, k_out, stream
PyObject* rope(PyObject* const* a) {
    const Axes ax = axes_of(a[8]);
    const at::Tensor& q = tensor(a[0], "q");
    const at::Tensor* k = optional(a[1], "k");
    const int dev = q.is_cuda() ? q.get_device() : -1;
    const Heads x = heads(q, "q", ax, dev);
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
    const at::AutoDispatchBelowADInplaceOrView below;
    const CallStream stream(a[11], dev);
    FmhaRopeParams p{};
    at::Tensor qo = a[9] == Py_None ? stream.given(at::empty_like(q)) : tensor(a[9], "out");
    const Heads xo = heads(qo, "out", ax, dev);
    if (!same_shape(x, xo)) bad("out must have q's and k's shapes");
    at::Tensor ko;
    if (k) {
        const Heads y = heads(*k, "k", ax, dev);
        if (!same_tokens(x, y)) bad("k must have q's tokens");
        ko = a[10] == Py_None ? stream.given(at::empty_like(*k)) : tensor(a[10], "out");
        const Heads yo = heads(ko, "out", ax, dev);
        if (!same_shape(y, yo)) bad("out must have q's and k's shapes");
        p.k = y.p, p.k_out = yo.p;
        p.stride_k = y.token, p.nhead_stride_k = y.head, p.batch_stride_k = y.batch;
        p.stride_ko = yo.token, p.nhead_stride_ko = yo.head, p.batch_stride_ko = yo.batch;
        p.nhead_k = narrow(y.heads, "heads");
    }
    const int axes = angles(p, tensor(a[2], "cos_sin"), a[4], a[5], dev);
    positions(p, tensor(a[3], "positions"), x, ax, axes, dev);
    p.q = x.p, p.q_out = xo.p;
    p.stride_q = x.token, p.nhead_stride_q = x.head, p.batch_stride_q = x.batch;
    p.stride_qo = xo.token, p.nhead_stride_qo = xo.head, p.batch_stride_qo = xo.batch;
    p.batch = narrow(x.batches, "batch"), p.seqlen_q = narrow(x.tokens, "tokens");
    p.nhead_q = narrow(x.heads, "heads");
    p.interleaved = truth(a[6]), p.inverse = truth(a[7]);
    if (q.numel() == 0) p.q = p.q_out = nullptr;
    if (k && k->numel() == 0) p.k = p.k_out = nullptr;
    if (p.q || p.k) done(g_rope(&p, stream.get()), "rope");
    if (a[9] != Py_None) written(qo);
    if (k && a[10] != Py_None) written(ko);
    PyObject* first = wrapped(a[9], qo);
    PyObject* second = k ? wrapped(a[10], ko) : none();
    PyObject* both = first && second ? PyTuple_Pack(2, first, second) : nullptr;
    Py_XDECREF(first);
    Py_XDECREF(second);
    return both;
}

// k, v, k_cache, v_cache, page_table, seqlens_k, q, cos_sin, positions, sections, axis_of, interleaved,
// cu_seqlens_q, layout, q_out, stream
PyObject* append(PyObject* const* a) {
    const Axes ax = axes_of(a[13]);
    const at::Tensor& k = tensor(a[0], "k");
    const int dev = k.is_cuda() ? k.get_device() : -1;
    const Heads x = heads(k, "k", ax, dev), y = heads(tensor(a[1], "v"), "v", ax, dev);
    if (!same_shape(x, y)) bad("v must have k's shape");
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
    const at::AutoDispatchBelowADInplaceOrView below;
    const CallStream stream(a[15], dev);
    const Cache c = cache(tensor(a[2], "k_cache"), tensor(a[3], "v_cache"), dev);
    if (x.heads != c.heads) bad("k must have the cache's heads");
    const Batch b = batch_of(tensor(a[4], "page_table"), tensor(a[5], "seqlens_k"), optional(a[12], "cu_seqlens_q"), x,
                             ax, dev);
    FmhaRopeParams p{};
    at::Tensor qo;
    const at::Tensor* q = optional(a[6], "q");
    if (q) {
        const Heads z = heads(*q, "q", ax, dev);
        if (!same_tokens(x, z)) bad("q must have k's tokens");
        qo = a[14] == Py_None ? stream.given(at::empty_like(*q)) : tensor(a[14], "q_out");
        const Heads zo = heads(qo, "q_out", ax, dev);
        if (!same_shape(z, zo)) bad("q_out must have q's shape");
        p.q = z.p, p.q_out = zo.p;
        p.stride_q = z.token, p.nhead_stride_q = z.head, p.batch_stride_q = z.batch;
        p.stride_qo = zo.token, p.nhead_stride_qo = zo.head, p.batch_stride_qo = zo.batch;
        p.nhead_q = narrow(z.heads, "heads");
        if (q->numel() == 0) p.q = p.q_out = nullptr;
    }
    const at::Tensor* table = optional(a[7], "cos_sin");
    const at::Tensor* pos = optional(a[8], "positions");
    if (table) {
        const int axes = angles(p, *table, a[9], a[10], dev);
        if (pos) positions(p, *pos, x, ax, axes, dev);
    } else if (pos) {
        bad("positions need cos_sin");
    }
    p.k = x.p, p.v = y.p, p.k_out = c.k.p, p.v_out = c.v.p;
    p.seqstart_q = b.starts, p.page_table = b.table, p.seqlens_k = b.lengths;
    p.stride_k = x.token, p.nhead_stride_k = x.head, p.batch_stride_k = x.batch;
    p.stride_v = y.token, p.nhead_stride_v = y.head, p.batch_stride_v = y.batch;
    p.stride_ko = c.k.token, p.nhead_stride_ko = c.k.head, p.batch_stride_ko = c.k.batch;
    p.stride_vo = c.v.token, p.nhead_stride_vo = c.v.head, p.batch_stride_vo = c.v.batch;
    p.table_stride = b.table_stride;
    p.batch = b.batch, p.seqlen_q = narrow(x.tokens, "tokens");
    p.total_q = ax.dense ? 0 : p.seqlen_q;
    p.nhead_k = c.heads, p.page_size = c.page, p.num_pages = c.pages, p.max_pages = b.max_pages;
    p.interleaved = truth(a[11]);
    if (x.tokens > 0 && x.batches > 0) {
        done(g_append(&p, stream.get()), "paged_append");
        written(tensor(a[2], "k_cache"));
        written(tensor(a[3], "v_cache"));
        if (q && a[14] != Py_None) written(qo);
    }
    return q ? wrapped(a[14], qo) : none();
}

// q, k_cache, v_cache, page_table, seqlens_k, prefix_pages, prefix_len, causal, cu_seqlens_q, max_seqlen_q,
// scale, return_lse, layout, out, lse_out, workspace, stream
PyObject* attend(PyObject* const* a) {
    const Axes ax = axes_of(a[12]);
    const at::Tensor& q = tensor(a[0], "q");
    const int dev = q.is_cuda() ? q.get_device() : -1;
    const Heads x = heads(q, "q", ax, dev);
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)dev);
    const at::AutoDispatchBelowADInplaceOrView below;
    const CallStream stream(a[16], dev);
    const Cache c = cache(tensor(a[1], "k_cache"), tensor(a[2], "v_cache"), dev);
    const Batch b = batch_of(tensor(a[3], "page_table"), tensor(a[4], "seqlens_k"), optional(a[8], "cu_seqlens_q"), x,
                             ax, dev);
    if (c.heads == 0 || x.heads % c.heads) bad("q's heads must be a multiple of the cache's");
    FmhaPagedParams p{};
    const at::Tensor* prefix = optional(a[5], "prefix_pages");
    if (prefix) {
        p.prefix_pages = ints(*prefix, "prefix_pages", 1, dev);
        const long long len = integer(a[6]);
        if (len < 1 || len > prefix->size(0) * c.page || len > 0x7fffffffll)
            bad("prefix_pages must be [pages] with room for prefix_len >= 1 keys");
        p.prefix_len = (int)len;
    }
    at::Tensor out = a[13] == Py_None ? stream.given(at::empty_like(q)) : tensor(a[13], "out");
    const Heads xo = heads(out, "out", ax, dev);
    if (!same_shape(x, xo)) bad("out must have q's shape");
    at::Tensor lse;
    const bool with_lse = truth(a[11]);
    if (with_lse) {
        const std::array<int64_t, 3> want{b.batch, x.heads, x.tokens};
        const at::IntArrayRef shape(want.data() + (ax.dense ? 0 : 1), ax.dense ? 3 : 2);
        if (a[14] == Py_None) {
            lse = stream.given(at::empty(shape, q.options().dtype(at::kFloat)));
        } else {
            lse = tensor(a[14], "lse_out");
            if (lse.sizes() != shape || lse.scalar_type() != at::kFloat || !lse.is_contiguous() || !lse.is_cuda() ||
                lse.get_device() != dev)
                bad("lse_out must be a contiguous fp32 tensor [batch, heads, seqlen_q] or [heads, total] on q's device");
        }
        p.lse = static_cast<float*>(lse.data_ptr());
    }
    if (q.numel() > 0) {
        p.total_q = ax.dense ? 0 : narrow(x.tokens, "tokens");
        p.seqlen_q = a[9] == Py_None || ax.dense ? narrow(x.tokens, "tokens") : narrow(integer(a[9]), "max_seqlen_q");
        p.nhead_q = narrow(x.heads, "heads"), p.nhead_k = c.heads;
        const size_t need = g_bytes(b.batch, p.seqlen_q, p.total_q, p.nhead_q, p.nhead_k, p.prefix_len);
        if (need == 0) bad("sizes out of range (max_seqlen_q must be positive)");
        at::Tensor space;
        if (a[15] == Py_None) {
            space = at::empty({(int64_t)need}, q.options().dtype(at::kByte));
        } else {
            space = tensor(a[15], "workspace");
            if (!space.is_cuda() || space.get_device() != dev || !space.is_contiguous() || space.nbytes() < need)
                bad("workspace must be a contiguous tensor of " + std::to_string(need) + " bytes on q's device");
        }
        p.workspace = space.data_ptr();
        p.workspace_bytes = (long long)space.nbytes();
        p.q = x.p, p.k_cache = c.k.p, p.v_cache = c.v.p, p.o = xo.p;
        p.seqstart_q = b.starts, p.page_table = b.table, p.seqlens_k = b.lengths;
        p.stride_q = x.token, p.nhead_stride_q = x.head, p.batch_stride_q = x.batch;
        p.stride_o = xo.token, p.nhead_stride_o = xo.head, p.batch_stride_o = xo.batch;
        p.stride_k = c.k.token, p.nhead_stride_k = c.k.head, p.page_stride_k = c.k.batch;
        p.stride_v = c.v.token, p.nhead_stride_v = c.v.head, p.page_stride_v = c.v.batch;
        p.table_stride = b.table_stride;
        p.batch = b.batch, p.page_size = c.page, p.num_pages = c.pages, p.max_pages = b.max_pages;
        p.causal = truth(a[7]);
        double scale = 0.125;
        if (a[10] != Py_None) {
            scale = PyFloat_AsDouble(a[10]);
            if (scale == -1.0 && PyErr_Occurred()) throw PythonError{};
        }
        p.scale = (float)(scale * 1.4426950408889634);
        done((prefix ? g_prefix : g_paged)(&p, stream.get()), prefix ? "prefix_fwd" : "paged_fwd");
        if (a[13] != Py_None) written(out);
        if (with_lse && a[14] != Py_None) written(lse);
    }
    PyObject* first = wrapped(a[13], out);
    if (!with_lse) return first;
    PyObject* second = wrapped(a[14], lse);
    PyObject* both = first && second ? PyTuple_Pack(2, first, second) : nullptr;
    Py_XDECREF(first);
    Py_XDECREF(second);
    return both;
}

// Addresses of the five C entries, then the error class.
PyObject* bind(PyObject* const* a) {
    g_rope = reinterpret_cast<RopeFn>(static_cast<uintptr_t>(integer(a[0])));
    g_append = reinterpret_cast<RopeFn>(static_cast<uintptr_t>(integer(a[1])));
    g_paged = reinterpret_cast<PagedFn>(static_cast<uintptr_t>(integer(a[2])));
    g_prefix = reinterpret_cast<PagedFn>(static_cast<uintptr_t>(integer(a[3])));
    g_bytes = reinterpret_cast<BytesFn>(static_cast<uintptr_t>(integer(a[4])));
    Py_XSETREF(g_error, Py_NewRef(a[5]));
    return none();
}

// Argument count, C++ exceptions -> Python errors.
template <PyObject* (*F)(PyObject* const*), int N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
    if (n != N) {
        PyErr_Format(PyExc_TypeError, "takes %d arguments, got %zd", N, n);
        return nullptr;
    }
    try {
        if (F != bind && g_error == nullptr) {
            PyErr_SetString(PyExc_RuntimeError, "bind() first");
            return nullptr;
        }
        return F(args);
    } catch (const Bad& e) {
        PyObject* v = Py_BuildValue("(is)", e.status, e.what.c_str());
        if (v) {
            PyErr_SetObject(g_error, v);
            Py_DECREF(v);
        }
    } catch (const PythonError&) {
    } catch (const c10::OutOfMemoryError& e) {
        PyObject* torch = PyImport_ImportModule("torch");
        PyObject* cls = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
        if (cls) PyErr_SetString(cls, e.what_without_backtrace());
        Py_XDECREF(cls);
        Py_XDECREF(torch);
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

#define ENTRY(name, n) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<name, n>)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {ENTRY(bind, 6), ENTRY(rope, 12), ENTRY(append, 16), ENTRY(attend, 17),
                          {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_torch_binding", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_binding() { return PyModule_Create(&kModule); }

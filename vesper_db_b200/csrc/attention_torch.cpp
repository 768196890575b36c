// The attention operators on torch tensors (vesper_db_b200/attention.py): checks of the
// tensors, outputs and workspaces from torch's allocator, and the call of the C entry point
// on the tensors' device and its current stream.  Written against the CPython interface:
// done in Python, a call of one token took 11 to 17 us of the host, most of it here.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <string>

#include "../../include/vesper_b200.h"

namespace {

PyObject* g_error = nullptr;  // vesper_db_b200.index.VesperError

struct Refused {
    vesper_status_t status;
    std::string why;
};
[[noreturn]] void refuse(const std::string& why) { throw Refused{VESPER_ERROR_INVALID_PARAM, why}; }

// Runs f and turns what it throws into a Python exception.
template <class F>
PyObject* entry(F&& f) {
    try {
        return f();
    } catch (const Refused& r) {
        PyObject* e = PyObject_CallFunction(g_error, "is", (int)r.status, r.why.c_str());
        if (e) {
            PyErr_SetObject(g_error, e);
            Py_DECREF(e);
        }
    } catch (const std::exception& x) {
        PyErr_SetString(PyExc_RuntimeError, x.what());
    } catch (...) {
        PyErr_SetString(PyExc_RuntimeError, "unknown error");
    }
    return nullptr;
}

void check(vesper_status_t status) {
    if (status != VESPER_OK) throw Refused{status, vesper_get_last_error()};
}

// ---- arguments ------------------------------------------------------------------------
void arguments(Py_ssize_t n, Py_ssize_t want) {
    if (n != want) refuse("wrong number of arguments");
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
    return THPVariable_Unpack(o);
}

const at::Tensor& cuda_tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o) || !THPVariable_Unpack(o).is_cuda()) refuse(std::string(name) + " must be a CUDA tensor");
    return THPVariable_Unpack(o);
}

long long whole(PyObject* o, const char* name) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse(std::string(name) + " must be a whole number");
    }
    return v;
}

size_t count(PyObject* o, const char* name) {
    const long long v = whole(o, name);
    if (v < 0) refuse(std::string(name) + " must not be negative");
    return (size_t)v;
}

double number(PyObject* o, const char* name) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) {
        PyErr_Clear();
        refuse(std::string(name) + " must be a number");
    }
    return v;
}

bool truth(PyObject* o, const char* name) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) {
        PyErr_Clear();
        refuse(std::string(name) + " must be true or false");
    }
    return v != 0;
}

std::string shape_of(const at::Tensor& t) {
    std::string s = "[";
    for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
    return s + "]";
}

// There is no backward pass: a result outside the graph of its inputs would go unnoticed.
void untracked(const at::Tensor& t, const char* name) {
    if (t.requires_grad() && c10::GradMode::is_enabled())
        refuse(std::string(name) + " requires a gradient, and the operator has none: call it under torch.no_grad() or detach");
}

void same(const at::Tensor& t, c10::Device dev, at::ScalarType type, const char* name) {
    if (t.device() != dev) refuse(std::string(name) + " is on " + t.device().str() + ", not on " + dev.str());
    if (t.scalar_type() != type)
        refuse(std::string(name) + " is " + c10::toString(t.scalar_type()) + ", " + c10::toString(type) + " expected");
    untracked(t, name);
}

// Address of a contiguous vector.
template <class T>
T* vector(const at::Tensor& t, c10::Device dev, at::ScalarType type, const char* name, int64_t n = -1) {
    same(t, dev, type, name);
    if (t.dim() != 1 || (n >= 0 && t.size(0) != n) || !t.is_contiguous())
        refuse(std::string(name) + " must be a contiguous vector" + (n >= 0 ? " of " + std::to_string(n) : ""));
    return static_cast<T*>(t.data_ptr());
}

// Stride of dimension i; that of a single element does not matter.
size_t step(const at::Tensor& t, int64_t i) { return t.size(i) > 1 ? (size_t)t.stride(i) : 8; }

void inner(const at::Tensor& t, const char* name) {
    if (t.size(-1) > 1 && t.stride(-1) != 1) refuse(std::string(name) + ": the last dimension must be contiguous");
}

size_t dtype_of(const at::Tensor& q) {
    if (q.scalar_type() == at::kBFloat16) return VESPER_BF16;
    if (q.scalar_type() == at::kHalf) return VESPER_F16;
    refuse("q must be bf16 or f16, [tokens, heads, head_dim]");
}

const at::Tensor& queries(PyObject* o) {
    const at::Tensor& q = cuda_tensor(o, "q");
    dtype_of(q);
    if (q.dim() != 3) refuse("q must be bf16 or f16, [tokens, heads, head_dim]");
    inner(q, "q");
    untracked(q, "q");
    return q;
}

// A [tokens, heads, head_dim] tensor beside q; -1: any number.
const at::Tensor& beside(PyObject* o, const at::Tensor& q, const char* name, int64_t tokens, int64_t heads) {
    const at::Tensor& t = tensor(o, name);
    same(t, q.device(), q.scalar_type(), name);
    if (t.dim() != 3 || t.size(2) != q.size(2) || (tokens >= 0 && t.size(0) != tokens) || (heads >= 0 && t.size(1) != heads))
        refuse(std::string(name) + " has shape " + shape_of(t) + ": [tokens, heads, head_dim] in line with q expected");
    inner(t, name);
    return t;
}

// Both caches: [pages, page_size, kv_heads, head_dim].
template <class P>
void caches(P& p, PyObject* ko, PyObject* vo, const at::Tensor& q, int64_t kv_heads) {
    const at::Tensor &k = tensor(ko, "k_cache"), &v = tensor(vo, "v_cache");
    same(k, q.device(), q.scalar_type(), "k_cache");
    same(v, q.device(), q.scalar_type(), "v_cache");
    if (k.dim() != 4 || k.sizes() != v.sizes() || k.size(3) != q.size(2) || (kv_heads >= 0 && k.size(2) != kv_heads))
        refuse("k_cache " + shape_of(k) + " and v_cache " + shape_of(v) +
               ": [pages, page_size, kv_heads, head_dim] in line with q expected");
    inner(k, "k_cache");
    inner(v, "v_cache");
    p.d_k_cache = k.data_ptr();
    p.k_page_stride = step(k, 0);
    p.k_slot_stride = step(k, 1);
    p.k_cache_head_stride = step(k, 2);
    p.d_v_cache = v.data_ptr();
    p.v_page_stride = step(v, 0);
    p.v_slot_stride = step(v, 1);
    p.v_cache_head_stride = step(v, 2);
    p.n_pages = (size_t)k.size(0);
    p.page_size = (size_t)k.size(1);
}

const at::Tensor& page_table(PyObject* o, c10::Device dev, int64_t n, size_t& width, size_t& row_stride) {
    const at::Tensor& t = tensor(o, "table");
    same(t, dev, at::kInt, "table");
    if (t.dim() != 2 || t.size(0) != n || (t.size(1) > 1 && t.stride(1) != 1))
        refuse("table must be [requests, width] with contiguous rows");
    width = (size_t)t.size(1);
    row_stride = n > 1 ? (size_t)t.stride(0) : width;
    return t;
}

// The library launches on the calling thread's device; the stream is that device's current one.
struct OnDevice {
    c10::cuda::CUDAGuard guard;
    void* stream;
    explicit OnDevice(c10::Device dev) : guard(dev), stream(c10::cuda::getCurrentCUDAStream(dev.index()).stream()) {}
};

// A tensor that a call has written in place counts the write, as torch's own calls do.
void written(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

at::Tensor empty(at::IntArrayRef sizes, const at::Tensor& like) { return at::empty(sizes, like.options()); }
at::Tensor empty(at::IntArrayRef sizes, const at::Tensor& like, at::ScalarType type) {
    return at::empty(sizes, like.options().dtype(type));
}

PyObject* none() { Py_RETURN_NONE; }

// (a, b), taking both references.
PyObject* two(PyObject* a, PyObject* b) {
    PyObject* t = PyTuple_New(2);
    PyTuple_SET_ITEM(t, 0, a);
    PyTuple_SET_ITEM(t, 1, b);
    return t;
}

// ---- operators ------------------------------------------------------------------------
// (cached, fresh, free, table, page_size, total, base) -> (lengths, starts, positions, slots, used)
PyObject* page_tables(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return entry([&] {
        arguments(n_args, 7);
        const at::Tensor& cached = cuda_tensor(a[0], "cached");
        const c10::Device dev = cached.device();
        vesper_page_tables_params_t p{};
        p.struct_size = sizeof(p);
        p.d_cached = vector<int32_t>(cached, dev, at::kInt, "cached");
        const int64_t n = cached.size(0);
        p.n_requests = (size_t)n;
        p.d_fresh = vector<int32_t>(tensor(a[1], "fresh"), dev, at::kInt, "fresh", n);
        const at::Tensor& free = tensor(a[2], "free");
        p.d_free = vector<int32_t>(free, dev, at::kInt, "free");
        p.n_free = (size_t)free.size(0);
        p.d_table = static_cast<int32_t*>(page_table(a[3], dev, n, p.table_width, p.table_stride).data_ptr());
        p.page_size = count(a[4], "page_size");
        p.n_tokens = count(a[5], "total");
        if (p.n_tokens > 0x7fffffff) refuse("sizes must be below 2^31");
        p.base = whole(a[6], "base");
        OnDevice on(dev);
        const int64_t total = (int64_t)p.n_tokens;
        at::Tensor lengths = empty({n}, cached), starts = empty({n + 1}, cached), positions = empty({total}, cached);
        at::Tensor slots = empty({total}, cached, at::kLong), used = empty({1}, cached);
        p.d_lengths = static_cast<int32_t*>(lengths.data_ptr());
        p.d_starts = static_cast<int32_t*>(starts.data_ptr());
        p.d_positions = static_cast<int32_t*>(positions.data_ptr());
        p.d_slots = static_cast<int64_t*>(slots.data_ptr());
        p.d_used = static_cast<int32_t*>(used.data_ptr());
        check(vesper_page_tables_device(&p, on.stream));
        written(tensor(a[3], "table"));
        PyObject* t = PyTuple_New(5);
        PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::move(lengths)));
        PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::move(starts)));
        PyTuple_SET_ITEM(t, 2, THPVariable_Wrap(std::move(positions)));
        PyTuple_SET_ITEM(t, 3, THPVariable_Wrap(std::move(slots)));
        PyTuple_SET_ITEM(t, 4, THPVariable_Wrap(std::move(used)));
        return t;
    });
}

// (q, k, v, positions, turns, q_weight, k_weight, eps, pairs, slots, k_cache, v_cache, keep_k) -> (q, k or None)
PyObject* norm_rotate(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return entry([&] {
        arguments(n_args, 13);
        const at::Tensor& q = queries(a[0]);
        const c10::Device dev = q.device();
        const int64_t t = q.size(0), heads = q.size(1), dim = q.size(2);
        const at::Tensor& k = beside(a[1], q, "k", t, -1);
        const int64_t kv = k.size(1);
        vesper_norm_rotate_params_t p{};
        p.struct_size = sizeof(p);
        p.dtype = dtype_of(q);
        p.n_tokens = (size_t)t;
        p.heads = (size_t)heads;
        p.kv_heads = (size_t)kv;
        p.head_dim = (size_t)dim;
        p.d_q = q.data_ptr();
        p.q_token_stride = step(q, 0);
        p.q_head_stride = step(q, 1);
        p.d_k = k.data_ptr();
        p.k_token_stride = step(k, 0);
        p.k_head_stride = step(k, 1);
        p.d_positions = vector<int32_t>(tensor(a[3], "positions"), dev, at::kInt, "positions", t);
        const at::Tensor& turns = tensor(a[4], "turns");
        same(turns, dev, at::kFloat, "turns");
        if (turns.dim() != 2 || !turns.is_contiguous()) refuse("turns must be [positions, turned], contiguous");
        p.d_turns = static_cast<const float*>(turns.data_ptr());
        p.n_positions = (size_t)turns.size(0);
        p.turned = (size_t)turns.size(1);
        if (a[5] != Py_None) p.d_q_weight = vector<void>(tensor(a[5], "q_weight"), dev, q.scalar_type(), "q_weight", dim);
        if (a[6] != Py_None) p.d_k_weight = vector<void>(tensor(a[6], "k_weight"), dev, q.scalar_type(), "k_weight", dim);
        p.eps = number(a[7], "eps");
        p.pairs = truth(a[8], "pairs");
        if (a[9] != Py_None) {
            if (a[2] == Py_None || a[10] == Py_None || a[11] == Py_None) refuse("slots need v, k_cache and v_cache");
            p.d_slots = vector<int64_t>(tensor(a[9], "slots"), dev, at::kLong, "slots", t);
            const at::Tensor& v = beside(a[2], q, "v", t, kv);
            p.d_v = v.data_ptr();
            p.v_token_stride = step(v, 0);
            p.v_head_stride = step(v, 1);
            caches(p, a[10], a[11], q, kv);
        }
        OnDevice on(dev);
        at::Tensor out_q = empty({t, heads, dim}, q), out_k;
        p.d_out_q = out_q.data_ptr();
        if (truth(a[12], "keep_k")) {
            out_k = empty({t, kv, dim}, q);
            p.d_out_k = out_k.data_ptr();
        }
        check(vesper_norm_rotate_device(&p, on.stream));
        if (p.d_slots) {
            written(tensor(a[10], "k_cache"));
            written(tensor(a[11], "v_cache"));
        }
        PyObject* second = out_k.defined() ? THPVariable_Wrap(std::move(out_k)) : none();
        return two(THPVariable_Wrap(std::move(out_q)), second);
    });
}

// (q, k, v, starts, starts_k, causal, scale, stats) -> out or (out, lse)
PyObject* prompt_attention(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return entry([&] {
        arguments(n_args, 8);
        const at::Tensor& q = queries(a[0]);
        const c10::Device dev = q.device();
        const int64_t t = q.size(0), heads = q.size(1), dim = q.size(2);
        const at::Tensor& k = beside(a[1], q, "k", -1, -1);
        const at::Tensor& v = beside(a[2], q, "v", k.size(0), k.size(1));
        vesper_prompt_attention_params_t p{};
        p.struct_size = sizeof(p);
        p.dtype = dtype_of(q);
        p.n_q = (size_t)t;
        p.n_k = (size_t)k.size(0);
        p.heads = (size_t)heads;
        p.kv_heads = (size_t)k.size(1);
        p.head_dim = (size_t)dim;
        p.d_q = q.data_ptr();
        p.q_token_stride = step(q, 0);
        p.q_head_stride = step(q, 1);
        p.d_k = k.data_ptr();
        p.k_token_stride = step(k, 0);
        p.k_head_stride = step(k, 1);
        p.d_v = v.data_ptr();
        p.v_token_stride = step(v, 0);
        p.v_head_stride = step(v, 1);
        const at::Tensor& starts = tensor(a[3], "starts");
        p.d_starts = vector<int32_t>(starts, dev, at::kInt, "starts");
        if (starts.size(0) == 0) refuse("starts must hold at least one entry");
        p.n_requests = (size_t)starts.size(0) - 1;
        if (a[4] != Py_None)
            p.d_starts_k = vector<int32_t>(tensor(a[4], "starts_k"), dev, at::kInt, "starts_k", starts.size(0));
        p.causal = truth(a[5], "causal");
        p.scale = a[6] == Py_None ? 1.0 / std::sqrt((double)dim) : number(a[6], "scale");
        const bool stats = truth(a[7], "stats");
        OnDevice on(dev);
        at::Tensor out = empty({t, heads, dim}, q), lse, space;
        p.d_out = out.data_ptr();
        if (stats) {
            lse = empty({t, heads}, q, at::kFloat);
            p.d_lse = static_cast<float*>(lse.data_ptr());
        }
        p.workspace_bytes = vesper_prompt_attention_workspace(&p);
        if (p.workspace_bytes) {
            space = empty({(int64_t)p.workspace_bytes}, q, at::kByte);
            p.d_workspace = space.data_ptr();
        }
        check(vesper_prompt_attention_device(&p, on.stream));
        PyObject* o = THPVariable_Wrap(std::move(out));
        return stats ? two(o, THPVariable_Wrap(std::move(lse))) : o;
    });
}

// (q, k_cache, v_cache, prefix_pages, prefix_len, table, lengths, scale, stats) -> out or (out, lse)
PyObject* shared_prefix_attention(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
    return entry([&] {
        arguments(n_args, 9);
        const at::Tensor& q = queries(a[0]);
        const c10::Device dev = q.device();
        const int64_t b = q.size(0), heads = q.size(1), dim = q.size(2);
        vesper_shared_prefix_attention_params_t p{};
        p.struct_size = sizeof(p);
        p.dtype = dtype_of(q);
        p.n_requests = (size_t)b;
        p.heads = (size_t)heads;
        p.head_dim = (size_t)dim;
        p.d_q = q.data_ptr();
        p.q_token_stride = step(q, 0);
        p.q_head_stride = step(q, 1);
        caches(p, a[1], a[2], q, -1);
        p.kv_heads = (size_t)THPVariable_Unpack(a[1]).size(2);
        const at::Tensor& pages = tensor(a[3], "prefix_pages");
        p.d_prefix_pages = vector<int32_t>(pages, dev, at::kInt, "prefix_pages");
        p.prefix_len = count(a[4], "prefix_len");
        if ((size_t)pages.size(0) * p.page_size < p.prefix_len) refuse("prefix_pages do not hold prefix_len tokens");
        p.d_table = static_cast<const int32_t*>(page_table(a[5], dev, b, p.table_width, p.table_stride).data_ptr());
        p.d_lengths = vector<int32_t>(tensor(a[6], "lengths"), dev, at::kInt, "lengths", b);
        p.scale = a[7] == Py_None ? 1.0 / std::sqrt((double)dim) : number(a[7], "scale");
        const bool stats = truth(a[8], "stats");
        OnDevice on(dev);
        at::Tensor out = empty({b, heads, dim}, q), lse, space;
        p.d_out = out.data_ptr();
        if (stats) {
            lse = empty({b, heads}, q, at::kFloat);
            p.d_lse = static_cast<float*>(lse.data_ptr());
        }
        p.workspace_bytes = vesper_shared_prefix_attention_workspace(&p);
        if (p.workspace_bytes) {
            space = empty({(int64_t)p.workspace_bytes}, q, at::kByte);
            p.d_workspace = space.data_ptr();
        }
        check(vesper_shared_prefix_attention_device(&p, on.stream));
        PyObject* o = THPVariable_Wrap(std::move(out));
        return stats ? two(o, THPVariable_Wrap(std::move(lse))) : o;
    });
}

PyMethodDef methods[] = {
    {"page_tables", (PyCFunction)(void*)page_tables, METH_FASTCALL, nullptr},
    {"norm_rotate", (PyCFunction)(void*)norm_rotate, METH_FASTCALL, nullptr},
    {"prompt_attention", (PyCFunction)(void*)prompt_attention, METH_FASTCALL, nullptr},
    {"shared_prefix_attention", (PyCFunction)(void*)shared_prefix_attention, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_attention", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__attention() {
    PyObject* index = PyImport_ImportModule("vesper_db_b200.index");
    if (!index) return nullptr;
    g_error = PyObject_GetAttrString(index, "VesperError");
    Py_DECREF(index);
    return g_error ? PyModule_Create(&module) : nullptr;
}

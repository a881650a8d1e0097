// paged_ext.cpp -- the serving calls for torch tensors, as a CPython module.
//
// A call of the smallest sizes is a few microseconds of GPU work, less than a
// Python function needs to read the attributes of a dozen tensors and fill a
// structure.  This module reads them from the tensors themselves, checks them
// (types, shapes, devices, contiguity), allocates what is returned from
// torch's allocator, and calls the C ABI on torch's current stream.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <string>

#include "b200exec.h"

namespace {

struct Raise {
    PyObject* type;
    std::string msg;
};
PyObject* g_status_error = nullptr;   // CudaRuntimeError(code, message)
int g_device = -1;

[[noreturn]] void value_error(std::string m) { throw Raise{PyExc_ValueError, std::move(m)}; }
[[noreturn]] void type_error(std::string m) { throw Raise{PyExc_TypeError, std::move(m)}; }
void need(bool ok, const char* m) {
    if (!ok) value_error(m);
}

struct Status {
    int code;
};
void check(int code) {
    if (code) throw Status{code};
}

std::string text_of(at::IntArrayRef x) {
    std::string s = "[";
    for (size_t i = 0; i < x.size(); i++) s += (i ? ", " : "") + std::to_string(x[i]);
    return s + "]";
}
std::string shape_of(const at::Tensor& t) { return text_of(t.sizes()); }

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) type_error(std::string(name) + " must be a tensor");
    return THPVariable_Unpack(o);
}
const at::Tensor* optional(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }
int64_t integer(PyObject* o, const char* name) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        type_error(std::string(name) + " must be an integer");
    }
    return v;
}
bool truth(PyObject* o, const char* name) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) {   // an array of several, say
        PyErr_Clear();
        type_error(std::string(name) + " must be true or false");
    }
    return v;
}
int narrow(int64_t v, const char* name) {
    if (v < INT32_MIN || v > INT32_MAX) value_error(std::string(name) + " does not fit 32 bits");
    return (int)v;
}

int act_code(const at::Tensor& t, const char* name) {
    if (t.scalar_type() == at::kFloat) return RT_F32;
    if (t.scalar_type() == at::kBFloat16) return RT_BF16;
    type_error(std::string(name) + " must be float32 or bfloat16, got " + toString(t.scalar_type()));
}

// The library on this device (chosen by the first call, of the process or after
// rt_destroy; does nothing where it runs there already).
void use_device(int device) {
    check(rt_init(device));
    g_device = device;
}
void use_device(const at::Tensor& t, const char* name) {
    if (!t.is_cuda()) value_error(std::string(name) + " must be a CUDA tensor");
    use_device(t.get_device());
}
void on_device(const at::Tensor& t, const char* name) {
    if (!t.is_cuda() || t.get_device() != g_device)
        value_error(std::string(name) + " is on " + t.device().str() + ", expected cuda:" + std::to_string(g_device));
}
void* stream() { return c10::cuda::getCurrentCUDAStream(g_device).stream(); }
at::Tensor empty(at::IntArrayRef shape, at::ScalarType type) {
    return at::empty(shape, at::TensorOptions().dtype(type).device(at::kCUDA, g_device));
}
void* index(const at::Tensor& t, const char* name, at::IntArrayRef shape, at::ScalarType type) {
    if (t.scalar_type() != type) type_error(std::string(name) + " must be " + toString(type) + ", got " + toString(t.scalar_type()));
    on_device(t, name);
    if (t.sizes() != shape || !t.is_contiguous())
        value_error(std::string(name) + " must be contiguous " + text_of(shape) + ", got " + (t.sizes() == shape ? "strided " : "") + text_of(t.sizes()));
    return t.data_ptr();
}
// A dense [a, b, c] operand with contiguous innermost dimension.
void rows(const at::Tensor& t, const char* name, int64_t a, int64_t b, int64_t c, int64_t (&stride)[2]) {
    on_device(t, name);
    if (t.dim() != 3 || t.size(0) != a || t.size(1) != b || t.size(2) != c)
        value_error(std::string(name) + " must be [" + std::to_string(a) + ", " + std::to_string(b) + ", " + std::to_string(c) +
                    "], got " + shape_of(t));
    if (t.stride(2) != 1 && c > 1) value_error(std::string(name) + " needs contiguous features");
    stride[0] = t.stride(0);
    stride[1] = t.stride(1);
}
void same_type(const at::Tensor& t, const char* name, const at::Tensor& as) {
    if (t.scalar_type() != as.scalar_type())
        type_error(std::string(name) + " must be " + toString(as.scalar_type()) + ", got " + toString(t.scalar_type()));
}

void cache(RtKvCache& c, const at::Tensor& k, const at::Tensor& v, const at::Tensor* ks, const at::Tensor* vs) {
    switch (k.scalar_type()) {
        case at::kFloat: c.dtype = RT_F32; break;
        case at::kBFloat16: c.dtype = RT_BF16; break;
        case at::kFloat8_e4m3fn: c.dtype = RT_F8E4M3; break;
        case at::kChar: c.dtype = RT_I8; break;
        default: type_error(std::string("a cache holds float32, bfloat16, float8_e4m3fn or int8, got ") + toString(k.scalar_type()));
    }
    same_type(v, "v_pages", k);
    use_device(k, "k_pages");
    on_device(v, "v_pages");
    if (k.dim() != 4 || v.sizes() != k.sizes())
        value_error("cache pages must be [pages, page_size, heads, head_dim], got " + shape_of(k) + " / " + shape_of(v));
    need(k.strides() == v.strides() && k.stride(3) == 1, "k_pages and v_pages need the same strides and contiguous features");
    c.k = k.data_ptr();
    c.v = v.data_ptr();
    for (int i = 0; i < 3; i++) c.stride[i] = k.stride(i);
    c.n_pages = narrow(k.size(0), "pages");
    c.page_size = narrow(k.size(1), "page_size");
    c.n_heads = narrow(k.size(2), "heads");
    c.head_dim = narrow(k.size(3), "head_dim");
    c.flags = RT_POINTERS_CHECKED;
    if (c.dtype >= RT_F8E4M3) {
        need(ks && vs, "an 8-bit cache needs k_scale and v_scale");
        if (ks->scalar_type() != at::kFloat || vs->scalar_type() != at::kFloat) type_error("scales must be float32");
        on_device(*ks, "k_scale");
        on_device(*vs, "v_scale");
        need(ks->dim() == 3 && ks->sizes() == k.sizes().slice(0, 3) && vs->sizes() == ks->sizes() && ks->strides() == vs->strides(),
             "scales must be [pages, page_size, heads] beside their pages, with the same strides");
        c.k_scale = ks->data_ptr<float>();
        c.v_scale = vs->data_ptr<float>();
        for (int i = 0; i < 3; i++) c.scale_stride[i] = ks->stride(i);
    } else {
        need(!ks && !vs, "only an 8-bit cache has scales");
    }
}
template <class T>
void page_table(T& x, const at::Tensor& t, int64_t n) {
    if (t.scalar_type() != at::kInt) type_error(std::string("page_table must be int32, got ") + toString(t.scalar_type()));
    on_device(t, "page_table");
    if (t.dim() != 2 || t.size(0) != n || (t.size(1) > 1 && t.stride(1) != 1))
        value_error("page_table must be [" + std::to_string(n) + ", pages] with contiguous rows, got " + shape_of(t));
    x.page_table = static_cast<const int*>(t.data_ptr());
    x.table_stride = t.stride(0);
    x.table_width = narrow(t.size(1), "page_table");
}

// Runs f and turns what it throws into a Python exception.
template <class F>
PyObject* guarded(F&& f) {
    try {
        return f();
    } catch (const Raise& e) {
        PyErr_SetString(e.type, e.msg.c_str());
    } catch (const Status& e) {
        PyObject* args = Py_BuildValue("(is)", e.code, rt_last_error_message());
        PyObject* err = args && g_status_error ? PyObject_CallObject(g_status_error, args) : nullptr;
        if (err) PyErr_SetObject(g_status_error, err);
        else if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, rt_last_error_message());
        Py_XDECREF(err);
        Py_XDECREF(args);
    } catch (const std::exception& e) {   // torch's allocator, among others
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}
bool count(Py_ssize_t n, Py_ssize_t want) {
    if (n == want) return true;
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
    return false;
}
PyObject* pair(const at::Tensor& a, const at::Tensor& b) {
    PyObject* x = THPVariable_Wrap(a);
    PyObject* y = THPVariable_Wrap(b);
    PyObject* t = PyTuple_Pack(2, x, y);
    Py_DECREF(x);
    Py_DECREF(y);
    return t;
}

PyObject* kv_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!count(n, 7)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor &k = tensor(a[0], "k"), &v = tensor(a[1], "v"), &slots = tensor(a[4], "slots");
        RtKvWrite w{};
        cache(w.cache, tensor(a[2], "k_pages"), tensor(a[3], "v_pages"), optional(a[5], "k_scale"), optional(a[6], "v_scale"));
        w.dtype = act_code(k, "k");
        same_type(v, "v", k);
        const int64_t tokens = k.dim() ? k.size(0) : 0;
        rows(k, "k", tokens, w.cache.n_heads, w.cache.head_dim, w.k_stride);
        rows(v, "v", tokens, w.cache.n_heads, w.cache.head_dim, w.v_stride);
        w.k = k.data_ptr();
        w.v = v.data_ptr();
        w.n_tokens = narrow(tokens, "tokens");
        w.slots = static_cast<const int64_t*>(index(slots, "slots", {tokens}, at::kLong));
        check(rt_kv_write(&w, stream()));
        Py_RETURN_NONE;
    });
}

PyObject* kv_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!count(n, 11)) return nullptr;
    return guarded([&]() -> PyObject* {
        RtKvRead r{};
        cache(r.cache, tensor(a[0], "k_pages"), tensor(a[1], "v_pages"), optional(a[6], "k_scale"), optional(a[7], "v_scale"));
        const at::Tensor& cu = tensor(a[4], "cu");
        const int64_t total = integer(a[5], "total"), seqs = cu.numel() - 1;
        need(total >= 0, "total must not be negative");
        need(seqs >= 0, "cu needs at least one element");
        at::Tensor k, v;
        if (a[9] == Py_None) {
            const at::ScalarType t = integer(a[8], "dtype") == RT_BF16 ? at::kBFloat16 : at::kFloat;
            k = empty({total, r.cache.n_heads, r.cache.head_dim}, t);
            v = empty({total, r.cache.n_heads, r.cache.head_dim}, t);
        } else {
            k = tensor(a[9], "k out");
            v = tensor(a[10], "v out");
        }
        r.dtype = act_code(k, "k out");
        same_type(v, "v out", k);
        rows(k, "k out", total, r.cache.n_heads, r.cache.head_dim, r.k_stride);
        rows(v, "v out", total, r.cache.n_heads, r.cache.head_dim, r.v_stride);
        r.k_out = k.data_ptr();
        r.v_out = v.data_ptr();
        r.n_rows = narrow(total, "total");
        r.n_seqs = narrow(seqs, "cu");
        page_table(r, tensor(a[2], "page_table"), seqs);
        if (const at::Tensor* start = optional(a[3], "start")) r.start = static_cast<const int*>(index(*start, "start", {seqs}, at::kInt));
        r.cu = static_cast<const int*>(index(cu, "cu", {seqs + 1}, at::kInt));
        check(rt_kv_read(&r, stream()));
        return pair(k, v);
    });
}

PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!count(n, 15)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor &q = tensor(a[0], "q"), &lens = tensor(a[4], "kv_lens");
        RtPagedAttention p{};
        cache(p.cache, tensor(a[1], "k_pages"), tensor(a[2], "v_pages"), optional(a[6], "k_scale"), optional(a[7], "v_scale"));
        if (q.dim() != 3) value_error("q must be [tokens, heads, head_dim], got " + shape_of(q));
        const int64_t tokens = q.size(0), heads = q.size(1), dim = p.cache.head_dim;
        p.dtype = act_code(q, "q");
        rows(q, "q", tokens, heads, dim, p.q_stride);
        const bool own = a[13] == Py_None;
        const at::Tensor out = own ? empty({tokens, heads, dim}, q.scalar_type()) : tensor(a[13], "out");
        same_type(out, "out", q);
        rows(out, "out", tokens, heads, dim, p.out_stride);
        p.q = q.data_ptr();
        p.out = out.data_ptr();
        p.total_new = narrow(tokens, "tokens");
        p.n_q_heads = narrow(heads, "heads");
        if (const at::Tensor* lse = optional(a[14], "lse")) p.lse = static_cast<float*>(index(*lse, "lse", {tokens, heads}, at::kFloat));
        p.n_seqs = narrow(lens.numel(), "kv_lens");
        page_table(p, tensor(a[3], "page_table"), p.n_seqs);
        p.kv_lens = static_cast<const int*>(index(lens, "kv_lens", {p.n_seqs}, at::kInt));
        p.cu_new = static_cast<const int*>(index(tensor(a[5], "cu_new"), "cu_new", {p.n_seqs + 1}, at::kInt));
        if (a[8] == Py_None) {
            p.scale = 1.0f / sqrtf((float)dim);
        } else {
            p.scale = (float)PyFloat_AsDouble(a[8]);
            if (PyErr_Occurred()) {
                PyErr_Clear();
                type_error("scale must be a number");
            }
        }
        p.causal = truth(a[9], "causal");
        p.window = narrow(integer(a[10], "window"), "window");
        p.max_new = a[11] == Py_None ? p.total_new : narrow(integer(a[11], "max_new"), "max_new");
        const int64_t width = (int64_t)p.table_width * p.cache.page_size;
        p.max_kv = a[12] == Py_None ? (int)std::min<int64_t>(width, INT32_MAX) : narrow(integer(a[12], "max_kv"), "max_kv");
        at::Tensor ws;
        const size_t bytes = rt_paged_attention_workspace(&p);
        if (bytes) ws = empty({(int64_t)bytes}, at::kByte);
        check(rt_paged_attention(&p, bytes ? ws.data_ptr() : nullptr, bytes, stream()));
        if (own) return THPVariable_Wrap(out);
        Py_INCREF(a[13]);
        return a[13];
    });
}

PyObject* verify_draft(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!count(n, 6)) return nullptr;
    return guarded([&]() -> PyObject* {
        const at::Tensor& target = tensor(a[0], "target");
        use_device(target, "target");
        if (target.dim() != 3 || target.size(1) < 1) value_error("target must be [sequences, drafts + 1, vocab], got " + shape_of(target));
        RtVerifyDraft v{};
        const int64_t B = target.size(0), N = target.size(1) - 1, V = target.size(2);
        v.dtype = act_code(target, "target");
        rows(target, "target", B, N + 1, V, v.target_stride);
        v.target = target.data_ptr();
        if (const at::Tensor* draft = optional(a[1], "draft")) {
            same_type(*draft, "draft", target);
            rows(*draft, "draft", B, N, V, v.draft_stride);
            v.draft = draft->data_ptr();
        }
        v.draft_tokens = static_cast<const int*>(index(tensor(a[2], "draft_tokens"), "draft_tokens", {B, N}, at::kInt));
        v.accept_u = static_cast<const float*>(index(tensor(a[3], "accept_u"), "accept_u", {B, N}, at::kFloat));
        v.sample_u = static_cast<const float*>(index(tensor(a[4], "sample_u"), "sample_u", {B}, at::kFloat));
        if (const at::Tensor* lens = optional(a[5], "draft_lens")) v.draft_lens = static_cast<const int*>(index(*lens, "draft_lens", {B}, at::kInt));
        const at::Tensor tokens = empty({B, N + 1}, at::kInt), accepted = empty({B}, at::kInt);
        v.tokens = static_cast<int*>(tokens.data_ptr());
        v.accepted = static_cast<int*>(accepted.data_ptr());
        v.n_seqs = narrow(B, "sequences");
        v.n_drafts = narrow(N, "drafts");
        v.vocab = narrow(V, "vocab");
        v.flags = RT_POINTERS_CHECKED;
        check(rt_verify_draft(&v, stream()));
        return pair(tokens, accepted);
    });
}

PyObject* check_stream(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!count(n, 1)) return nullptr;
    return guarded([&]() -> PyObject* {
        use_device(narrow(integer(a[0], "device"), "device"));
        int code;
        void* st = stream();
        Py_BEGIN_ALLOW_THREADS;
        code = rt_check_stream(st);
        Py_END_ALLOW_THREADS;
        check(code);
        Py_RETURN_NONE;
    });
}

PyObject* set_status_error(PyObject*, PyObject* const* a, Py_ssize_t n) {
    if (!count(n, 1)) return nullptr;
    Py_INCREF(a[0]);
    Py_XSETREF(g_status_error, a[0]);
    Py_RETURN_NONE;
}

#define FN(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(name)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {FN(kv_write), FN(kv_read), FN(paged_attention), FN(verify_draft), FN(check_stream), FN(set_status_error),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "b200paged", "Serving calls of libb200exec for torch tensors", -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_b200paged(void) { return PyModule_Create(&g_module); }

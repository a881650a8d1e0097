// serving.cu -- entry points of the serving calls (paged key/value cache,
// attention over it, verification of drafted tokens): argument checks, then
// the launches of k_kvcache.cu, k_paged_attention.cu and k_verify.cu on the
// caller's stream.  Everything a host can see is checked here; what lies in
// device memory (slots, page numbers, lengths) the kernels bounds-check.
#include <exception>

#include "rt_internal.h"

namespace rt {
namespace {

Status bad(const std::string& m) { return Status::err(RT_ERR_ARGUMENT, m); }

// The library's device, for the length of one call.
struct DeviceGuard {
    int before = -1;
    DeviceGuard() {
        int now = -1;
        if (cudaGetDevice(&now) == cudaSuccess && now != runtime_device()) {
            before = now;
            cudaSetDevice(runtime_device());
        }
    }
    ~DeviceGuard() {
        if (before >= 0) cudaSetDevice(before);
    }
};

thread_local bool t_checked = false;   // the call's pointers need no query
Status check_pointer(const void* p, size_t bytes, const char* what) {
    if (t_checked) return p || !bytes ? Status::ok() : Status::err(RT_ERR_NULL_POINTER, std::string(what) + " is NULL");
    return check_device_pointer(p, bytes, what);
}

#define CHECK(expr)                \
    do {                           \
        Status _s = (expr);        \
        if (!_s.good()) return _s; \
    } while (0)

Status check_act(int dtype) {
    return dtype == RT_F32 || dtype == RT_BF16 ? Status::ok()
                                               : Status::err(RT_ERR_UNSUPPORTED, "dtype must be RT_F32 or RT_BF16");
}

// Elements spanned by `n` counts at `stride` strides (non-negative strides).
int64_t span(int64_t a, int64_t sa, int64_t b, int64_t sb, int64_t tail) {
    return (a > 0 ? (a - 1) * sa : 0) + (b > 0 ? (b - 1) * sb : 0) + tail;
}

Status check_cache(const RtKvCache& c) {
    if (c.dtype < RT_F32 || c.dtype > RT_I8) return Status::err(RT_ERR_UNSUPPORTED, "cache: unknown dtype");
    if (c.n_pages < 1 || c.page_size < 1 || c.n_heads < 1) return bad("cache: n_pages, page_size and n_heads must be positive");
    if (c.head_dim < 16 || c.head_dim > 128 || c.head_dim % 16)
        return Status::err(RT_ERR_UNSUPPORTED, "cache: head_dim must be a multiple of 16 up to 128");
    const int e = dtype_bytes(c.dtype);
    if (!aligned16(c.k) || !aligned16(c.v)) return bad("cache: k and v must be 16-byte aligned");
    for (int i = 0; i < 3; i++)
        if (c.stride[i] < 0 || (c.stride[i] * e) % 16) return bad("cache: strides must be non-negative multiples of 16 bytes");
    if (c.page_size > 1 && c.stride[1] < c.head_dim) return bad("cache: slots overlap");
    if (c.n_heads > 1 && c.stride[2] < c.head_dim) return bad("cache: heads overlap");
    if (c.n_pages > 1 && c.stride[0] < c.head_dim) return bad("cache: pages overlap");
    const int64_t elems = span(c.n_pages, c.stride[0], c.page_size, c.stride[1], (c.n_heads - 1) * c.stride[2] + c.head_dim);
    // kernels keep a row's place in units of 16 bytes in 32 bits
    if (elems * e / 16 >= 0xffffffffll) return Status::err(RT_ERR_UNSUPPORTED, "cache: k and v must span less than 64 GiB each");
    if ((int64_t)c.n_pages * c.page_size > 0x7fffffffll) return Status::err(RT_ERR_UNSUPPORTED, "cache: more than 2^31 - 1 slots");
    CHECK(check_pointer(c.k, (size_t)elems * e, "cache k"));
    CHECK(check_pointer(c.v, (size_t)elems * e, "cache v"));
    if (e == 1) {
        int64_t s = 0;
        for (int i = 0; i < 3; i++)
            if (c.scale_stride[i] < 0) return bad("cache: negative scale stride");
        s = span(c.n_pages, c.scale_stride[0], c.page_size, c.scale_stride[1], (c.n_heads - 1) * c.scale_stride[2] + 1);
        if (s > 0x7fffffffll) return Status::err(RT_ERR_UNSUPPORTED, "cache: scales span more than 2^31 - 1 elements");
        if (!c.k_scale || !c.v_scale) return Status::err(RT_ERR_NULL_POINTER, "cache: an 8-bit cache needs k_scale and v_scale");
        CHECK(check_pointer(c.k_scale, (size_t)s * 4, "cache k_scale"));
        CHECK(check_pointer(c.v_scale, (size_t)s * 4, "cache v_scale"));
    }
    return Status::ok();
}

Status check_rows(const void* p, const int64_t st[2], int64_t rows, int heads, int dim, int dtype, const char* what) {
    if (st[0] < 0 || st[1] < 0) return bad(std::string(what) + ": negative stride");
    const int e = dtype_bytes(dtype);
    if (reinterpret_cast<uintptr_t>(p) % e) return bad(std::string(what) + ": not aligned to its element size");
    return check_pointer(p, (size_t)span(rows, st[0], heads, st[1], dim) * e, what);
}

// What a call writes: rows that would fall on one another are refused.
Status check_out(const void* p, const int64_t st[2], int64_t rows, int heads, int dim, int dtype, const char* what) {
    CHECK(check_rows(p, st, rows, heads, dim, dtype, what));
    if ((heads > 1 && st[1] < dim) || (rows > 1 && st[0] < dim)) return bad(std::string(what) + ": rows overlap");
    return Status::ok();
}

Status check_table(const int* table, int64_t stride, int width, int n_seqs) {
    if (width < 0 || stride < 0) return bad("page_table: negative width or stride");
    if (width == 0 || n_seqs == 0) return Status::ok();
    return check_pointer(table, (size_t)((n_seqs - 1) * stride + width) * 4, "page_table");
}

Status do_write(const RtKvWrite& w, void* stream) {
    t_checked = w.cache.flags & RT_POINTERS_CHECKED;
    CHECK(check_act(w.dtype));
    CHECK(check_cache(w.cache));
    if (w.n_tokens < 0) return bad("kv_write: negative n_tokens");
    if (w.n_tokens == 0) return Status::ok();
    CHECK(check_rows(w.k, w.k_stride, w.n_tokens, w.cache.n_heads, w.cache.head_dim, w.dtype, "kv_write k"));
    CHECK(check_rows(w.v, w.v_stride, w.n_tokens, w.cache.n_heads, w.cache.head_dim, w.dtype, "kv_write v"));
    CHECK(check_pointer(w.slots, (size_t)w.n_tokens * 8, "kv_write slots"));
    DeviceGuard g;
    return launch_kv_write(w, static_cast<cudaStream_t>(stream));
}

Status do_read(const RtKvRead& r, void* stream) {
    t_checked = r.cache.flags & RT_POINTERS_CHECKED;
    CHECK(check_act(r.dtype));
    CHECK(check_cache(r.cache));
    if (r.n_rows < 0 || r.n_seqs < 0) return bad("kv_read: negative n_rows or n_seqs");
    if (r.n_rows == 0) return Status::ok();   // (without sequences every row is written as zeros)
    CHECK(check_out(r.k_out, r.k_stride, r.n_rows, r.cache.n_heads, r.cache.head_dim, r.dtype, "kv_read k_out"));
    CHECK(check_out(r.v_out, r.v_stride, r.n_rows, r.cache.n_heads, r.cache.head_dim, r.dtype, "kv_read v_out"));
    CHECK(check_table(r.page_table, r.table_stride, r.table_width, r.n_seqs));
    if (r.start && r.n_seqs) CHECK(check_pointer(r.start, (size_t)r.n_seqs * 4, "kv_read start"));
    CHECK(check_pointer(r.cu, (size_t)(r.n_seqs + 1) * 4, "kv_read cu"));
    DeviceGuard g;
    return launch_kv_read(r, static_cast<cudaStream_t>(stream));
}

Status check_attention_sizes(const RtPagedAttention& p) {
    CHECK(check_act(p.dtype));
    if (p.n_seqs < 0 || p.total_new < 0 || p.max_new < 0 || p.max_kv < 0 || p.window < 0)
        return bad("paged_attention: negative count");
    if (p.n_seqs > 16384) return Status::err(RT_ERR_UNSUPPORTED, "paged_attention: more than 16384 sequences");
    if (p.n_q_heads < 1 || p.cache.n_heads < 1 || p.n_q_heads % p.cache.n_heads)
        return bad("paged_attention: n_q_heads must be a multiple of the cache's n_heads");
    if (!(p.scale > 0.0f) || p.scale > 1e30f) return bad("paged_attention: scale must be positive and finite");
    return Status::ok();
}

Status do_attention(const RtPagedAttention& p, void* ws, size_t ws_bytes, void* stream) {
    t_checked = p.cache.flags & RT_POINTERS_CHECKED;
    CHECK(check_attention_sizes(p));
    CHECK(check_cache(p.cache));
    if (p.total_new == 0) return Status::ok();   // (without sequences every row is written as zeros)
    const int D = p.cache.head_dim;
    CHECK(check_rows(p.q, p.q_stride, p.total_new, p.n_q_heads, D, p.dtype, "paged_attention q"));
    CHECK(check_out(p.out, p.out_stride, p.total_new, p.n_q_heads, D, p.dtype, "paged_attention out"));
    if (p.lse) CHECK(check_pointer(p.lse, (size_t)p.total_new * p.n_q_heads * 4, "paged_attention lse"));
    CHECK(check_table(p.page_table, p.table_stride, p.table_width, p.n_seqs));
    if (p.n_seqs) CHECK(check_pointer(p.kv_lens, (size_t)p.n_seqs * 4, "paged_attention kv_lens"));
    CHECK(check_pointer(p.cu_new, (size_t)(p.n_seqs + 1) * 4, "paged_attention cu_new"));
    const size_t need = paged_attention_workspace(p);
    if (ws_bytes < need) return bad("paged_attention: workspace of " + std::to_string(ws_bytes) + " bytes, needs " + std::to_string(need));
    if (need) {
        if (!aligned16(ws)) return bad("paged_attention: workspace must be 16-byte aligned");
        CHECK(check_pointer(ws, need, "paged_attention workspace"));
    }
    DeviceGuard g;
    return launch_paged_attention(p, ws, static_cast<cudaStream_t>(stream));
}

Status do_verify(const RtVerifyDraft& v, void* stream) {
    t_checked = v.flags & RT_POINTERS_CHECKED;
    CHECK(check_act(v.dtype));
    if (v.n_seqs < 0 || v.n_drafts < 0) return bad("verify_draft: negative count");
    if (v.n_drafts > 1024) return Status::err(RT_ERR_UNSUPPORTED, "verify_draft: more than 1024 drafts");
    if (v.vocab < 1 || v.vocab > (1 << 22)) return Status::err(RT_ERR_UNSUPPORTED, "verify_draft: vocab must be 1 .. 2^22");
    if (v.n_seqs > 65535) return Status::err(RT_ERR_UNSUPPORTED, "verify_draft: more than 65535 sequences");
    if (v.n_seqs == 0) return Status::ok();
    CHECK(check_rows(v.target, v.target_stride, v.n_seqs, v.n_drafts + 1, v.vocab, v.dtype, "verify_draft target"));
    if (v.n_drafts) {
        if (v.draft) CHECK(check_rows(v.draft, v.draft_stride, v.n_seqs, v.n_drafts, v.vocab, v.dtype, "verify_draft draft"));
        CHECK(check_pointer(v.draft_tokens, (size_t)v.n_seqs * v.n_drafts * 4, "verify_draft draft_tokens"));
        CHECK(check_pointer(v.accept_u, (size_t)v.n_seqs * v.n_drafts * 4, "verify_draft accept_u"));
    }
    if (v.draft_lens) CHECK(check_pointer(v.draft_lens, (size_t)v.n_seqs * 4, "verify_draft draft_lens"));
    CHECK(check_pointer(v.sample_u, (size_t)v.n_seqs * 4, "verify_draft sample_u"));
    CHECK(check_pointer(v.tokens, (size_t)v.n_seqs * (v.n_drafts + 1) * 4, "verify_draft tokens"));
    CHECK(check_pointer(v.accepted, (size_t)v.n_seqs * 4, "verify_draft accepted"));
    DeviceGuard g;
    return launch_verify_draft(v, static_cast<cudaStream_t>(stream));
}

// No exception leaves a C entry point.
template <class F>
int guarded(F&& f) {
    try {
        if (!runtime_ready()) return report(Status::err(RT_ERR_NOT_INITIALIZED, "rt_init not called"));
        Status s = f();
        return s.good() ? RT_OK : report(s);
    } catch (const std::exception&) {
        return RT_ERR_OOM;   // only host allocations throw here
    }
}

}  // namespace
}  // namespace rt

using namespace rt;

extern "C" {

int rt_kv_write(const RtKvWrite* w, void* stream) {
    return guarded([&] { return w ? do_write(*w, stream) : Status::err(RT_ERR_NULL_POINTER, "rt_kv_write: NULL"); });
}
int rt_kv_read(const RtKvRead* r, void* stream) {
    return guarded([&] { return r ? do_read(*r, stream) : Status::err(RT_ERR_NULL_POINTER, "rt_kv_read: NULL"); });
}
size_t rt_paged_attention_workspace(const RtPagedAttention* p) {
    if (!p) return 0;
    try {
        return check_attention_sizes(*p).good() ? paged_attention_workspace(*p) : 0;
    } catch (const std::exception&) {
        return 0;
    }
}
int rt_paged_attention(const RtPagedAttention* p, void* ws, size_t ws_bytes, void* stream) {
    return guarded([&] {
        return p ? do_attention(*p, ws, ws_bytes, stream) : Status::err(RT_ERR_NULL_POINTER, "rt_paged_attention: NULL");
    });
}
int rt_verify_draft(const RtVerifyDraft* v, void* stream) {
    return guarded([&] { return v ? do_verify(*v, stream) : Status::err(RT_ERR_NULL_POINTER, "rt_verify_draft: NULL"); });
}
int rt_check_stream(void* stream) {
    return guarded([&] {
        cudaError_t e = cudaStreamSynchronize(static_cast<cudaStream_t>(stream));
        if (e != cudaSuccess) return Status::err(RT_ERR_CUDA, std::string("stream: ") + cudaGetErrorString(e));
        return serving_status();
    });
}

}  // extern "C"

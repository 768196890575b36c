// C entry points of the operators that answer from retrieved passages: every refusal is
// made here, before anything is queued; nothing throws across the C boundary.
#include <exception>
#include <new>
#include <string>

#include "attention.cuh"
#include "c_error.hpp"
#include "../../include/vesper_b200.h"

using vesper_c::clear_error;
using vesper_c::set_error;

namespace {

// A refusal: the message becomes the last error.
struct Refused {
    std::string why;
};
void need(bool ok, const char* why) {
    if (!ok) throw Refused{why};
}

template <class P, class F>
vesper_status_t entry(const P* p, F&& f) {
    clear_error();
    if (!p) {
        set_error("params is NULL");
        return VESPER_ERROR_INVALID_PARAM;
    }
    try {
        need(p->struct_size == sizeof(P), "struct_size is not that of the params struct");
        f();
        return VESPER_OK;
    } catch (const Refused& r) {
        set_error(r.why);
        return VESPER_ERROR_INVALID_PARAM;
    } catch (const std::bad_alloc&) {
        set_error("allocation failure");
        return VESPER_ERROR_INTERNAL;
    } catch (const std::exception& e) {
        set_error(e.what());
        return VESPER_ERROR_INTERNAL;
    } catch (...) {
        set_error("unknown error");
        return VESPER_ERROR_UNKNOWN;
    }
}

constexpr size_t kMaxInt = 0x7fffffff;
constexpr size_t kMaxStride = (size_t)1 << 38;

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool stride_ok(size_t s) { return s > 0 && s % 8 == 0 && s < kMaxStride; }

int page_shift_of(size_t page_size) {
    int s = 4;
    while (s < 9 && ((size_t)1 << s) != page_size) ++s;
    need(s < 9, "page_size must be a power of two from 16 to 256");
    return s;
}

void check_heads(size_t dtype, size_t heads, size_t kv_heads, size_t head_dim, size_t max_dim) {
    need(dtype == VESPER_BF16 || dtype == VESPER_F16, "dtype must be bf16 or f16");
    need(kv_heads > 0 && heads > 0 && heads % kv_heads == 0, "heads must be a multiple of kv_heads");
    need(heads / kv_heads <= 128 && heads <= 65535, "at most 128 query heads a key head and 65535 heads");
    need(head_dim >= 8 && head_dim % 8 == 0 && head_dim <= max_dim,
         max_dim == 128 ? "head_dim must be a multiple of 8, 8 to 128" : "head_dim must be a multiple of 8, 8 to 256");
}

vgpu::HeadsView view(const void* p, size_t tok, size_t head, const char* what) {
    need(p != nullptr, what);
    need(aligned16(p) && stride_ok(tok) && stride_ok(head),
         "tensors must be 16-byte aligned with strides that are multiples of 8 elements");
    return {p, (long long)tok, (long long)head};
}

vgpu::PagedView paged(const void* p, size_t page, size_t slot, size_t head, const char* what) {
    need(p != nullptr, what);
    need(aligned16(p) && stride_ok(page) && stride_ok(slot) && stride_ok(head),
         "caches must be 16-byte aligned with strides that are multiples of 8 elements");
    return {const_cast<void*>(p), (long long)page, (long long)slot, (long long)head};
}

// In 32 bits, where the kernels multiply it by log2(e) once more: 2e38 leaves room for that.
float scale_of(double scale) {
    need(scale > 0 && scale <= 2e38 && (float)scale > 0, "scale must be positive and at most 2e38");
    return (float)scale;
}

vgpu::PromptArgs prompt_args(const vesper_prompt_attention_params_t& p) {
    check_heads(p.dtype, p.heads, p.kv_heads, p.head_dim, 128);
    // Rows, keys and pieces are numbered in 32 bits, and counted in whole tiles past their ends.
    need(p.n_q < kMaxInt - 256 && p.n_k < kMaxInt - 256 && p.n_requests < kMaxInt - 256,
         "tokens and requests must be below 2^31 - 257");
    vgpu::PromptArgs a{};
    a.f16 = p.dtype == VESPER_F16;
    a.heads = (int)p.heads;
    a.kv_heads = (int)p.kv_heads;
    a.dim = (int)p.head_dim;
    a.n_q = (long long)p.n_q;
    a.n_k = (long long)p.n_k;
    a.n_requests = (int)p.n_requests;
    a.causal = p.causal != 0;
    a.scale = scale_of(p.scale);
    a.lse = p.d_lse;
    return a;
}

vgpu::SharedArgs shared_args(const vesper_shared_prefix_attention_params_t& p) {
    check_heads(p.dtype, p.heads, p.kv_heads, p.head_dim, 128);
    need(p.n_requests <= kMaxInt && p.n_requests * p.heads <= kMaxInt, "n_requests * heads must be below 2^31");
    need(p.prefix_len <= kMaxInt - 256, "prefix_len must be below 2^31 - 256");
    vgpu::SharedArgs a{};
    a.f16 = p.dtype == VESPER_F16;
    a.heads = (int)p.heads;
    a.kv_heads = (int)p.kv_heads;
    a.dim = (int)p.head_dim;
    a.n_requests = (int)p.n_requests;
    a.page_shift = page_shift_of(p.page_size);
    need(p.n_pages <= kMaxInt, "at most 2^31 - 1 pages");
    need(p.table_width <= (kMaxInt >> a.page_shift), "table_width * page_size must be below 2^31");
    need((p.n_requests * ((p.heads / p.kv_heads + 7) / 8) * p.table_width) <= (((size_t)1 << 34) >> a.page_shift),
         "n_requests * table_width * page_size must be at most 2^34 for eight query heads a key head");
    a.n_pages = (long long)p.n_pages;
    a.prefix_len = (long long)p.prefix_len;
    a.table_width = (int)p.table_width;
    a.table_stride = (long long)p.table_stride;
    a.scale = scale_of(p.scale);
    a.lse = p.d_lse;
    return a;
}

}  // namespace

extern "C" {

VESPER_C_API vesper_status_t vesper_page_tables_device(const vesper_page_tables_params_t* params, void* cuda_stream) {
    return entry(params, [&] {
        const vesper_page_tables_params_t& p = *params;
        need(p.n_requests <= (size_t)vgpu::kMaxTableRequests, "at most 16384 requests");
        need(p.n_tokens <= kMaxInt && p.n_free <= kMaxInt && p.table_width <= kMaxInt, "sizes must be below 2^31");
        need(p.base >= 0 && p.base <= (int64_t)kMaxInt, "base must be 0 to 2^31 - 1");
        vgpu::PageTablesArgs a{};
        a.page_shift = page_shift_of(p.page_size);
        need(p.d_starts && p.d_used, "d_starts and d_used must not be NULL");
        if (p.n_requests) {
            need(p.d_cached && p.d_fresh && p.d_lengths, "d_cached, d_fresh and d_lengths must not be NULL");
            need(p.d_table || p.table_width == 0, "d_table must not be NULL");
            need(p.table_stride >= p.table_width && p.table_stride < kMaxStride, "table_stride is below table_width");
        }
        need(p.d_free || p.n_free == 0, "d_free must not be NULL");
        need(p.n_tokens == 0 || (p.d_positions && p.d_slots), "d_positions and d_slots must not be NULL");
        a.cached = p.d_cached;
        a.fresh = p.d_fresh;
        a.n_requests = (int)p.n_requests;
        a.free_pages = p.d_free;
        a.n_free = (long long)p.n_free;
        a.table = p.d_table;
        a.table_width = (int)p.table_width;
        a.table_stride = (long long)p.table_stride;
        a.n_tokens = (int)p.n_tokens;
        a.base = (int)p.base;
        a.lengths = p.d_lengths;
        a.starts = p.d_starts;
        a.positions = p.d_positions;
        a.slots = p.d_slots;
        a.used = p.d_used;
        a.wide = aligned16(p.d_positions) && aligned16(p.d_slots);
        vgpu::launch_page_tables(a, static_cast<cudaStream_t>(cuda_stream));
    });
}

VESPER_C_API vesper_status_t vesper_norm_rotate_device(const vesper_norm_rotate_params_t* params, void* cuda_stream) {
    return entry(params, [&] {
        const vesper_norm_rotate_params_t& p = *params;
        check_heads(p.dtype, p.heads, p.kv_heads, p.head_dim, 256);
        need(p.turned % 16 == 0 && p.turned <= p.head_dim, "turned must be a multiple of 16, at most head_dim");
        need(p.n_tokens <= kMaxInt && p.n_positions <= kMaxInt, "sizes must be below 2^31");
        need(p.eps >= 0 && p.eps <= 3e38, "eps must be 0 to 3e38");
        if (p.n_tokens == 0) return;
        vgpu::NormRotateArgs a{};
        a.f16 = p.dtype == VESPER_F16;
        a.n_tokens = (int)p.n_tokens;
        a.heads = (int)p.heads;
        a.kv_heads = (int)p.kv_heads;
        a.dim = (int)p.head_dim;
        a.turned = (int)p.turned;
        a.pairs = p.pairs != 0;
        a.eps = (float)p.eps;
        a.q = view(p.d_q, p.q_token_stride, p.q_head_stride, "d_q must not be NULL");
        a.k = view(p.d_k, p.k_token_stride, p.k_head_stride, "d_k must not be NULL");
        need(p.d_positions != nullptr, "d_positions must not be NULL");
        need(p.turned == 0 || p.d_turns, "d_turns must not be NULL");
        need(aligned16(p.d_turns), "d_turns must be 16-byte aligned");
        need(aligned16(p.d_q_weight) && aligned16(p.d_k_weight), "weights must be 16-byte aligned");
        need(p.d_out_q != nullptr && aligned16(p.d_out_q) && aligned16(p.d_out_k),
             "d_out_q must not be NULL and outputs must be 16-byte aligned");
        a.positions = p.d_positions;
        a.turns = p.d_turns;
        a.n_positions = (int)p.n_positions;
        a.q_weight = p.d_q_weight;
        a.k_weight = p.d_k_weight;
        a.out_q = p.d_out_q;
        a.out_k = p.d_out_k;
        if (p.d_slots) {
            a.slots = p.d_slots;
            a.page_shift = page_shift_of(p.page_size);
            need(p.n_pages <= kMaxInt, "at most 2^31 - 1 pages");
            a.n_pages = (long long)p.n_pages;
            a.v = view(p.d_v, p.v_token_stride, p.v_head_stride, "d_v must not be NULL with d_slots");
            a.k_cache = paged(p.d_k_cache, p.k_page_stride, p.k_slot_stride, p.k_cache_head_stride,
                              "d_k_cache must not be NULL with d_slots");
            a.v_cache = paged(p.d_v_cache, p.v_page_stride, p.v_slot_stride, p.v_cache_head_stride,
                              "d_v_cache must not be NULL with d_slots");
        }
        vgpu::launch_norm_rotate(a, static_cast<cudaStream_t>(cuda_stream));
    });
}

VESPER_C_API size_t vesper_prompt_attention_workspace(const vesper_prompt_attention_params_t* params) {
    size_t bytes = 0;
    entry(params, [&] { bytes = vgpu::prompt_attention_workspace(prompt_args(*params)); });
    return bytes;
}

VESPER_C_API vesper_status_t vesper_prompt_attention_device(const vesper_prompt_attention_params_t* params,
                                                            void* cuda_stream) {
    return entry(params, [&] {
        const vesper_prompt_attention_params_t& p = *params;
        vgpu::PromptArgs a = prompt_args(p);
        if (p.n_q == 0) return;
        a.q = view(p.d_q, p.q_token_stride, p.q_head_stride, "d_q must not be NULL");
        if (p.n_k) {
            a.k = view(p.d_k, p.k_token_stride, p.k_head_stride, "d_k must not be NULL");
            a.v = view(p.d_v, p.v_token_stride, p.v_head_stride, "d_v must not be NULL");
        }
        need(p.d_starts != nullptr, "d_starts must not be NULL");
        need(p.d_starts_k || p.n_q == p.n_k, "q and k have different lengths: d_starts_k is needed");
        need(p.d_out != nullptr && aligned16(p.d_out), "d_out must not be NULL and must be 16-byte aligned");
        a.starts = p.d_starts;
        a.starts_k = p.d_starts_k ? p.d_starts_k : p.d_starts;
        a.out = p.d_out;
        const size_t bytes = vgpu::prompt_attention_workspace(a);
        need(bytes == 0 || (p.d_workspace && aligned16(p.d_workspace) && p.workspace_bytes >= bytes),
             "d_workspace is smaller than vesper_prompt_attention_workspace says");
        a.workspace = p.d_workspace;
        a.workspace_bytes = p.workspace_bytes;
        vgpu::launch_prompt_attention(a, static_cast<cudaStream_t>(cuda_stream));
    });
}

VESPER_C_API size_t vesper_shared_prefix_attention_workspace(const vesper_shared_prefix_attention_params_t* params) {
    size_t bytes = 0;
    entry(params, [&] { bytes = vgpu::shared_attention_workspace(shared_args(*params)); });
    return bytes;
}

VESPER_C_API vesper_status_t vesper_shared_prefix_attention_device(
    const vesper_shared_prefix_attention_params_t* params, void* cuda_stream) {
    return entry(params, [&] {
        const vesper_shared_prefix_attention_params_t& p = *params;
        vgpu::SharedArgs a = shared_args(p);
        if (p.n_requests == 0) return;
        a.q = view(p.d_q, p.q_token_stride, p.q_head_stride, "d_q must not be NULL");
        a.k_cache = paged(p.d_k_cache, p.k_page_stride, p.k_slot_stride, p.k_cache_head_stride,
                          "d_k_cache must not be NULL");
        a.v_cache = paged(p.d_v_cache, p.v_page_stride, p.v_slot_stride, p.v_cache_head_stride,
                          "d_v_cache must not be NULL");
        need(p.n_pages > 0, "the cache has no pages");
        need(p.prefix_len == 0 || p.d_prefix_pages, "d_prefix_pages must not be NULL");
        need(p.table_width == 0 || p.d_table, "d_table must not be NULL");
        need(p.n_requests == 1 || p.table_stride >= p.table_width, "table_stride is below table_width");
        need(p.table_stride < kMaxStride, "table_stride is too large");
        need(p.d_lengths != nullptr, "d_lengths must not be NULL");
        need(p.d_out != nullptr && aligned16(p.d_out), "d_out must not be NULL and must be 16-byte aligned");
        a.prefix_pages = p.d_prefix_pages;
        a.table = p.d_table;
        a.lengths = p.d_lengths;
        a.out = p.d_out;
        const size_t bytes = vgpu::shared_attention_workspace(a);
        need(bytes == 0 || (p.d_workspace && aligned16(p.d_workspace) && p.workspace_bytes >= bytes),
             "d_workspace is smaller than vesper_shared_prefix_attention_workspace says");
        a.workspace = p.d_workspace;
        a.workspace_bytes = p.workspace_bytes;
        vgpu::launch_shared_attention(a, static_cast<cudaStream_t>(cuda_stream));
    });
}

}  // extern "C"

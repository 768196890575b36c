// Operators that answer from retrieved passages: page tables of a paged key/value cache,
// norm and rotation of queries and keys, attention over packed prompts, and attention of
// single tokens over a shared prefix.  Host-side argument blocks and launchers; the
// entry points (argument checks, error codes) are in attention_c_api.cpp.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "common.cuh"

namespace vgpu {

constexpr int kMaxTableRequests = 16384;  // of one page_tables call

// Address and strides (elements) of a [tokens, heads, dim] view; dim is contiguous.
struct HeadsView {
    const void* p;
    long long tok, head;
};

// A paged cache [pages, page_size, heads, dim]; strides in elements, dim contiguous.
struct PagedView {
    void* p;
    long long page, tok, head;
};

struct PageTablesArgs {
    const int32_t* cached;
    const int32_t* fresh;
    int n_requests;
    const int32_t* free_pages;
    long long n_free;
    int32_t* table;
    int table_width;
    long long table_stride;
    int page_shift;
    int n_tokens;
    int base;
    int32_t* lengths;
    int32_t* starts;
    int32_t* positions;
    int64_t* slots;
    int32_t* used;
    bool wide;  // positions and slots are 16-byte aligned
};

struct NormRotateArgs {
    bool f16;
    int n_tokens, heads, kv_heads, dim, turned;
    bool pairs;
    float eps;
    HeadsView q, k, v;
    const int32_t* positions;
    const float* turns;
    int n_positions;
    const void* q_weight;
    const void* k_weight;
    const int64_t* slots;  // null: no cache
    PagedView k_cache, v_cache;
    long long n_pages;
    int page_shift;
    void* out_q;  // contiguous
    void* out_k;  // contiguous, may be null
};

struct PromptArgs {
    bool f16;
    int heads, kv_heads, dim;
    long long n_q, n_k;
    HeadsView q, k, v;
    const int32_t* starts;
    const int32_t* starts_k;
    int n_requests;
    bool causal;
    float scale;
    void* out;   // [n_q, heads, dim] contiguous
    float* lse;  // [n_q, heads] or null
    void* workspace;
    size_t workspace_bytes;
};

struct SharedArgs {
    bool f16;
    int heads, kv_heads, dim;
    int n_requests;
    HeadsView q;
    PagedView k_cache, v_cache;
    long long n_pages;
    int page_shift;
    const int32_t* prefix_pages;
    long long prefix_len;
    const int32_t* table;
    int table_width;
    long long table_stride;
    const int32_t* lengths;
    float scale;
    void* out;   // [n_requests, heads, dim] contiguous
    float* lse;  // [n_requests, heads] or null
    void* workspace;
    size_t workspace_bytes;
};

void launch_page_tables(const PageTablesArgs& a, cudaStream_t st);
void launch_norm_rotate(const NormRotateArgs& a, cudaStream_t st);
size_t prompt_attention_workspace(const PromptArgs& a);
void launch_prompt_attention(const PromptArgs& a, cudaStream_t st);
size_t shared_attention_workspace(const SharedArgs& a);
void launch_shared_attention(const SharedArgs& a, cudaStream_t st);

// Opts a kernel in to its dynamic shared memory, once a device; `more` runs with it.
template <class K, class F>
void opt_in(std::atomic<uint64_t>& devices, K* kernel, int smem, F&& more) {
    int dev = 0;
    VGPU_CHECK(cudaGetDevice(&dev));
    const uint64_t bit = 1ull << (dev & 63);
    if (devices.load(std::memory_order_relaxed) & bit) return;
    VGPU_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    more();
    devices.fetch_or(bit, std::memory_order_relaxed);
}

}  // namespace vgpu

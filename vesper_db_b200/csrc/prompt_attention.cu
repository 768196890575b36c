// Attention over packed prompts and over a shared prefix: one warp a query row.
//
//   s_j = scale * q . k_j over the row's visible keys, out = sum_j softmax(s)_j v_j,
//   lse = log sum_j exp(s_j); a row without visible keys gives zeros and -inf.
//
// One pass over the keys with the running maximum m and sum l of the softmax: when a key
// raises m, what was summed so far is scaled by exp(m_old - m_new).  Sums in 32 bits.
#include <algorithm>

#include "attention.cuh"
#include "common.cuh"
#include "half_types.cuh"

namespace vgpu {

namespace {

constexpr int kWarps = 4;
constexpr float kLog2e = 1.4426950408889634f;

// A lane holds values lane * 4 .. lane * 4 + 3 of a row of up to 128.
template <class H>
__device__ __forceinline__ float4 load4(const void* p, long long at, bool live) {
    if (!live) return make_float4(0, 0, 0, 0);
    const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const typename H::type*>(p) + at);
    const float2 a = H::unpack(u.x), b = H::unpack(u.y);
    return make_float4(a.x, a.y, b.x, b.y);
}

struct RowState {
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0, 0, 0, 0);
};

template <class H>
__device__ __forceinline__ void visit(RowState& r, float4 q, const void* kp, const void* vp, long long ka, long long va,
                                      bool live) {
    const float4 k = load4<H>(kp, ka, live);
    float s = q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float4 v = load4<H>(vp, va, live);
    const float m = fmaxf(r.m, s), c = exp2f(r.m - m), p = exp2f(s - m);
    r.m = m;
    r.l = r.l * c + p;
    r.o.x = r.o.x * c + p * v.x;
    r.o.y = r.o.y * c + p * v.y;
    r.o.z = r.o.z * c + p * v.z;
    r.o.w = r.o.w * c + p * v.w;
}

template <class H>
__device__ __forceinline__ void finish(const RowState& r, void* out, long long at, float* lse, long long lse_at, int lane,
                                       bool live) {
    const float inv = r.l > 0.0f ? 1.0f / r.l : (r.l == 0.0f ? 0.0f : r.l);
    if (live)
        *reinterpret_cast<uint2*>(static_cast<typename H::type*>(out) + at) =
            make_uint2(H::pack(r.o.x * inv, r.o.y * inv), H::pack(r.o.z * inv, r.o.w * inv));
    if (lse && lane == 0) lse[lse_at] = (r.m + log2f(r.l)) / kLog2e;
}

template <class H>
__global__ void __launch_bounds__(kWarps * 32) prompt_rows_kernel(const __grid_constant__ PromptArgs a) {
    const int lane = threadIdx.x & 31;
    const long long row = blockIdx.x * (long long)kWarps + (threadIdx.x >> 5);
    if (row >= a.n_q * a.heads) return;
    const long long t = row / a.heads;
    const int h = (int)(row % a.heads), kh = h / (a.heads / a.kv_heads);
    int lo = 0, hi = a.n_requests;  // the last request whose start is <= t
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.starts[mid] <= t) lo = mid; else hi = mid;
    }
    const long long q0 = max(a.starts[lo], 0), q1 = a.n_requests ? min((long long)a.starts[lo + 1], a.n_q) : 0;
    long long k0 = 0, k1 = 0;
    if (t >= q0 && t < q1) {
        k0 = min(max((long long)a.starts_k[lo], 0LL), a.n_k);
        k1 = min(max((long long)a.starts_k[lo + 1], k0), a.n_k);
        if (a.causal) k1 = min(k1, k1 - (q1 - t) + 1);
    }
    const bool live = lane * 4 < a.dim;
    float4 q = load4<H>(a.q.p, t * a.q.tok + h * a.q.head + lane * 4, live);
    const float f = a.scale * kLog2e;
    q = make_float4(q.x * f, q.y * f, q.z * f, q.w * f);
    RowState r;
    for (long long j = k0; j < k1; ++j)
        visit<H>(r, q, a.k.p, a.v.p, j * a.k.tok + kh * a.k.head + lane * 4, j * a.v.tok + kh * a.v.head + lane * 4, live);
    finish<H>(r, a.out, row * a.dim + lane * 4, a.lse, row, lane, live);
}

template <class H>
__global__ void __launch_bounds__(kWarps * 32) shared_rows_kernel(const __grid_constant__ SharedArgs a) {
    const int lane = threadIdx.x & 31;
    const long long row = blockIdx.x * (long long)kWarps + (threadIdx.x >> 5);
    if (row >= (long long)a.n_requests * a.heads) return;
    const int b = (int)(row / a.heads), h = (int)(row % a.heads), kh = h / (a.heads / a.kv_heads);
    const bool live = lane * 4 < a.dim;
    float4 q = load4<H>(a.q.p, b * a.q.tok + h * a.q.head + lane * 4, live);
    const float f = a.scale * kLog2e;
    q = make_float4(q.x * f, q.y * f, q.z * f, q.w * f);
    RowState r;
    const int mask = (1 << a.page_shift) - 1;
    auto run = [&](const int32_t* pages, long long n) {
        for (long long j = 0; j < n; ++j) {
            const long long p = pages[j >> a.page_shift];
            const bool ok = live && p >= 0 && p < a.n_pages;
            visit<H>(r, q, a.k_cache.p, a.v_cache.p,
                     p * a.k_cache.page + (j & mask) * a.k_cache.tok + kh * a.k_cache.head + lane * 4,
                     p * a.v_cache.page + (j & mask) * a.v_cache.tok + kh * a.v_cache.head + lane * 4, ok);
        }
    };
    run(a.prefix_pages, a.prefix_len);
    run(a.table + (long long)b * a.table_stride,
        min((long long)max(a.lengths[b], 0), (long long)a.table_width << a.page_shift));
    finish<H>(r, a.out, row * a.dim + lane * 4, a.lse, row, lane, live);
}

}  // namespace

size_t prompt_attention_workspace(const PromptArgs&) { return 0; }
size_t shared_attention_workspace(const SharedArgs&) { return 0; }

void launch_prompt_attention(const PromptArgs& a, cudaStream_t st) {
    const int blocks = ceil_div(a.n_q * a.heads, kWarps);
    if (a.f16) prompt_rows_kernel<F16><<<blocks, kWarps * 32, 0, st>>>(a);
    else prompt_rows_kernel<Bf16><<<blocks, kWarps * 32, 0, st>>>(a);
    VGPU_LAUNCH("prompt_rows_kernel");
}

void launch_shared_attention(const SharedArgs& a, cudaStream_t st) {
    const int blocks = ceil_div((long long)a.n_requests * a.heads, kWarps);
    if (a.f16) shared_rows_kernel<F16><<<blocks, kWarps * 32, 0, st>>>(a);
    else shared_rows_kernel<Bf16><<<blocks, kWarps * 32, 0, st>>>(a);
    VGPU_LAUNCH("shared_rows_kernel");
}

}  // namespace vgpu

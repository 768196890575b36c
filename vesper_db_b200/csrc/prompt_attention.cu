// Attention over packed prompts, and over a shared prefix joined with each request's own
// pages: launchers, the kernel of the own pages, and the join of partial results.
#include <algorithm>

#include "attention.cuh"
#include "attn_tile.cuh"
#include "common.cuh"
#include "half_types.cuh"

namespace vgpu {

namespace {

using attn::kKeys;
using attn::kRows;
using attn::kThreads;
using attn::TileParams;

constexpr int kSms = 148;
constexpr float kLog2e = 1.4426950408889634f;

// ---------------------------------------------------------------------------------
// Tensor maps (through the driver entry point: no libcuda link dependency).
// ---------------------------------------------------------------------------------
using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_fn() {
    static const EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        check(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q), "cudaGetDriverEntryPoint");
        if (!p || q != cudaDriverEntryPointSuccess) throw CudaError("cuTensorMapEncodeTiled unavailable");
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

// 4-D map of 16-bit values, boxes of 64 values of the innermost dimension, 128-byte
// swizzle; what lies outside the tensor reads as zero.  Strides in elements.
CUtensorMap make_map(bool f16, const void* base, const long long (&dims)[4], const long long (&strides)[3],
                     const int (&box)[4]) {
    CUtensorMap m;
    cuuint64_t gd[4], gs[3];
    cuuint32_t bx[4];
    const cuuint32_t es[4] = {1, 1, 1, 1};
    for (int i = 0; i < 4; ++i) {
        gd[i] = (cuuint64_t)std::max<long long>(dims[i], 1);
        bx[i] = (cuuint32_t)box[i];
    }
    for (int i = 0; i < 3; ++i) gs[i] = (cuuint64_t)strides[i] * 2;
    const CUresult r = encode_fn()(&m, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                                   const_cast<void*>(base), gd, gs, bx, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) throw CudaError("attention: the driver refused a tensor map of these strides");
    return m;
}

void fill_queries(TileParams& p, bool f16, const HeadsView& q, int heads, int kv_heads, int dim, long long n_q) {
    p.heads = heads;
    p.kv_heads = kv_heads;
    p.group = heads / kv_heads;
    p.dim = dim;
    p.tile_tokens = kRows / p.group;
    p.n_q = (int)n_q;
    p.q = q;
    p.mq = make_map(f16, q.p, {dim, p.group, kv_heads, n_q}, {q.head, q.head * p.group, q.tok},
                    {64, p.group, 1, p.tile_tokens});
}

template <class H, int D, bool PAGED>
void launch_tiles_as(const TileParams& p, long long blocks, cudaStream_t st) {
    auto* kernel = attn::attn_tile_kernel<H, D, PAGED>;
    constexpr int smem = attn::smem_bytes<D>();
    static const bool ready = [&] {
        VGPU_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        cudaFuncAttributes fa;
        VGPU_CHECK(cudaFuncGetAttributes(&fa, kernel));
        // the softmax warps' registers come out of what the block is launched with
        if (fa.numRegs * kThreads < 256 * attn::kSoftmaxRegs + 128 * attn::kServiceRegs)
            throw CudaError("attn_tile_kernel: launched with too few registers for its split");
        return true;
    }();
    (void)ready;
    kernel<<<(unsigned)blocks, kThreads, smem, st>>>(p);
    VGPU_LAUNCH("attn_tile_kernel");
}

template <bool PAGED>
void launch_tiles(const TileParams& p, bool f16, long long blocks, cudaStream_t st) {
    if (blocks <= 0) return;
    if (blocks > 0x7fffffffLL) throw CudaError("attention: too many tiles for one launch");
    if (f16) {
        if (p.dim <= 64) launch_tiles_as<F16, 64, PAGED>(p, blocks, st);
        else launch_tiles_as<F16, 128, PAGED>(p, blocks, st);
    } else {
        if (p.dim <= 64) launch_tiles_as<Bf16, 64, PAGED>(p, blocks, st);
        else launch_tiles_as<Bf16, 128, PAGED>(p, blocks, st);
    }
}

// ---------------------------------------------------------------------------------
// Own pages of each request: one warp a query row.
// ---------------------------------------------------------------------------------
constexpr int kWarps = 4;

// A lane holds values lane * 4 .. lane * 4 + 3 of a row of up to 128.
template <class H>
__device__ __forceinline__ float4 load4(const void* p, long long at, bool live) {
    if (!live) return make_float4(0, 0, 0, 0);
    const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const typename H::type*>(p) + at);
    const float2 a = H::unpack(u.x), b = H::unpack(u.y);
    return make_float4(a.x, a.y, b.x, b.y);
}

template <class H>
__global__ void __launch_bounds__(kWarps * 32) own_rows_kernel(const __grid_constant__ SharedArgs a, float* part_o,
                                                               float* part_lse) {
    const int lane = threadIdx.x & 31;
    const long long row = blockIdx.x * (long long)kWarps + (threadIdx.x >> 5);
    if (row >= (long long)a.n_requests * a.heads) return;
    const int b = (int)(row / a.heads), h = (int)(row % a.heads), kh = h / (a.heads / a.kv_heads);
    const bool live = lane * 4 < a.dim;
    float4 q = load4<H>(a.q.p, b * a.q.tok + h * a.q.head + lane * 4, live);
    const float f = a.scale * kLog2e;
    q = make_float4(q.x * f, q.y * f, q.z * f, q.w * f);
    float m = -INFINITY, l = 0.0f;
    float4 o = make_float4(0, 0, 0, 0);
    const int mask = (1 << a.page_shift) - 1;
    const int32_t* pages = a.table + (long long)b * a.table_stride;
    const long long n = min((long long)max(a.lengths[b], 0), (long long)a.table_width << a.page_shift);
    for (long long j = 0; j < n; ++j) {
        const long long p = pages[j >> a.page_shift];
        const bool ok = live && p >= 0 && p < a.n_pages;
        const float4 k = load4<H>(
            a.k_cache.p, p * a.k_cache.page + (j & mask) * a.k_cache.tok + kh * a.k_cache.head + lane * 4, ok);
        float s = q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w;
#pragma unroll
        for (int e = 16; e > 0; e >>= 1) s += __shfl_xor_sync(0xffffffffu, s, e);
        const float4 v = load4<H>(
            a.v_cache.p, p * a.v_cache.page + (j & mask) * a.v_cache.tok + kh * a.v_cache.head + lane * 4, ok);
        const float up = fmaxf(m, s), c = exp2f(m - up), x = exp2f(s - up);
        m = up;
        l = l * c + x;
        o = make_float4(o.x * c + x * v.x, o.y * c + x * v.y, o.z * c + x * v.z, o.w * c + x * v.w);
    }
    const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
    if (live) *reinterpret_cast<float4*>(part_o + row * a.dim + lane * 4) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    if (lane == 0) part_lse[row] = m + log2f(l);
}

// ---------------------------------------------------------------------------------
// Join of partial results: with L_i their log2-sum-exp and M = max L_i, the weights are
// 2^(L_i - M) and out = sum w_i O_i / sum w_i.  One warp a row.
// ---------------------------------------------------------------------------------
template <class H>
__global__ void __launch_bounds__(128) join_kernel(int parts, long long rows, int dim, const float* __restrict__ part_o,
                                                   const float* __restrict__ part_lse, void* out, float* lse) {
    const int lane = threadIdx.x & 31;
    const long long row = blockIdx.x * 4LL + (threadIdx.x >> 5);
    if (row >= rows) return;
    float m = -INFINITY;
    bool nan = false;
    for (int i = 0; i < parts; ++i) {
        const float x = part_lse[i * rows + row];
        nan |= isnan(x);
        m = fmaxf(m, x);
    }
    float total = 0.0f;
    float4 o = make_float4(0, 0, 0, 0);
    const bool live = lane * 4 < dim;
    for (int i = 0; i < parts; ++i) {
        const float x = part_lse[i * rows + row];
        if (x == -INFINITY) continue;
        const float w = exp2f(x - m);
        total += w;
        if (live) {
            const float4 v = *reinterpret_cast<const float4*>(part_o + (i * rows + row) * dim + lane * 4);
            o = make_float4(o.x + w * v.x, o.y + w * v.y, o.z + w * v.z, o.w + w * v.w);
        }
    }
    const float inv = total > 0.0f ? 1.0f / total : (total == 0.0f && !nan ? 0.0f : __int_as_float(0x7fc00000));
    if (live)
        *reinterpret_cast<uint2*>(static_cast<typename H::type*>(out) + row * dim + lane * 4) =
            make_uint2(H::pack(o.x * inv, o.y * inv), H::pack(o.z * inv, o.w * inv));
    if (lse && lane == 0) lse[row] = nan ? __int_as_float(0x7fc00000) : (m + log2f(total)) / kLog2e;
}

void launch_join(bool f16, int parts, long long rows, int dim, const float* part_o, const float* part_lse, void* out,
                 float* lse, cudaStream_t st) {
    const int blocks = ceil_div(rows, 4);
    if (f16) join_kernel<F16><<<blocks, 128, 0, st>>>(parts, rows, dim, part_o, part_lse, out, lse);
    else join_kernel<Bf16><<<blocks, 128, 0, st>>>(parts, rows, dim, part_o, part_lse, out, lse);
    VGPU_LAUNCH("join_kernel");
}

size_t part_bytes(long long parts, long long rows, int dim) { return (size_t)(parts * rows * (dim + 1)) * sizeof(float); }

// How many ways to split the keys: as many as give each SM a block, but at least four key
// tiles a split.
int splits_for(long long blocks, long long key_tiles) {
    const long long by_sms = kSms / std::max<long long>(blocks, 1), by_keys = key_tiles / 4;
    return (int)std::max<long long>(1, std::min<long long>({by_sms, by_keys, 64}));
}

struct PromptPlan {
    long long tiles;  // upper bound of block tiles: the requests' lengths are on the device
    int splits;
};
PromptPlan prompt_plan(const PromptArgs& a) {
    const int span = 2 * (kRows / (a.heads / a.kv_heads));
    PromptPlan pl;
    pl.tiles = a.n_q / span + std::min<long long>(a.n_requests + 2, a.n_q);
    const long long likely = (a.n_q + span - 1) / span + std::max(a.n_requests - 1, 0);
    pl.splits = splits_for(likely * a.kv_heads, a.n_k / kKeys / std::max(a.n_requests, 1));
    return pl;
}

int shared_splits(const SharedArgs& a) {
    const int span = 2 * (kRows / (a.heads / a.kv_heads));
    return splits_for((long long)ceil_div(a.n_requests, span) * a.kv_heads, a.prefix_len / kKeys);
}

}  // namespace

size_t prompt_attention_workspace(const PromptArgs& a) {
    if (a.n_q == 0) return 0;
    const PromptPlan pl = prompt_plan(a);
    return pl.splits > 1 ? part_bytes(pl.splits, a.n_q * a.heads, a.dim) : 0;
}

void launch_prompt_attention(const PromptArgs& a, cudaStream_t st) {
    const PromptPlan pl = prompt_plan(a);
    const long long rows = a.n_q * a.heads;
    TileParams p{};
    fill_queries(p, a.f16, a.q, a.heads, a.kv_heads, a.dim, a.n_q);
    p.n_k = (int)a.n_k;
    if (a.n_k) {
        p.mk = make_map(a.f16, a.k.p, {a.dim, a.kv_heads, a.n_k, 1}, {a.k.head, a.k.tok, a.k.tok}, {64, 1, kKeys, 1});
        p.mv = make_map(a.f16, a.v.p, {a.dim, a.kv_heads, a.n_k, 1}, {a.v.head, a.v.tok, a.v.tok}, {64, 1, kKeys, 1});
    }
    p.k = a.k;
    p.v = a.v;
    p.starts = a.starts;
    p.starts_k = a.starts_k;
    p.n_requests = a.n_requests;
    p.causal = a.causal;
    p.scale_log2 = a.scale * kLog2e;
    p.splits = pl.splits;
    p.part = pl.splits > 1;
    p.out = a.out;
    p.lse = a.lse;
    p.part_o = static_cast<float*>(a.workspace);
    p.part_lse = p.part_o + pl.splits * rows * a.dim;
    launch_tiles<false>(p, a.f16, pl.tiles * a.kv_heads * pl.splits, st);
    if (p.part) launch_join(a.f16, pl.splits, rows, a.dim, p.part_o, p.part_lse, a.out, a.lse, st);
}

size_t shared_attention_workspace(const SharedArgs& a) {
    if (a.n_requests == 0) return 0;
    return part_bytes(1 + (a.prefix_len ? shared_splits(a) : 0), (long long)a.n_requests * a.heads, a.dim);
}

void launch_shared_attention(const SharedArgs& a, cudaStream_t st) {
    const long long rows = (long long)a.n_requests * a.heads;
    const int splits = a.prefix_len ? shared_splits(a) : 0;
    float* part_o = static_cast<float*>(a.workspace);
    float* part_lse = part_o + (splits + 1) * rows * a.dim;
    if (splits) {
        TileParams p{};
        fill_queries(p, a.f16, a.q, a.heads, a.kv_heads, a.dim, a.n_requests);
        const int page = 1 << a.page_shift, box = std::min(page, kKeys);
        const PagedView &k = a.k_cache, &v = a.v_cache;
        p.mk = make_map(a.f16, k.p, {a.dim, a.kv_heads, page, a.n_pages}, {k.head, k.tok, k.page}, {64, 1, box, 1});
        p.mv = make_map(a.f16, v.p, {a.dim, a.kv_heads, page, a.n_pages}, {v.head, v.tok, v.page}, {64, 1, box, 1});
        p.n_k = (int)a.prefix_len;
        p.pages = a.prefix_pages;
        p.page_shift = a.page_shift;
        p.scale_log2 = a.scale * kLog2e;
        p.splits = splits;
        p.part = true;
        p.part_o = part_o;
        p.part_lse = part_lse;
        launch_tiles<true>(p, a.f16, (long long)ceil_div(a.n_requests, 2 * p.tile_tokens) * a.kv_heads * splits, st);
    }
    const int blocks = ceil_div(rows, kWarps);
    float* own_o = part_o + splits * rows * a.dim;
    float* own_lse = part_lse + splits * rows;
    if (a.f16) own_rows_kernel<F16><<<blocks, kWarps * 32, 0, st>>>(a, own_o, own_lse);
    else own_rows_kernel<Bf16><<<blocks, kWarps * 32, 0, st>>>(a, own_o, own_lse);
    VGPU_LAUNCH("own_rows_kernel");
    launch_join(a.f16, splits + 1, rows, a.dim, part_o, part_lse, a.out, a.lse, st);
}

}  // namespace vgpu

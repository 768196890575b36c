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
        if (fa.numRegs * kThreads < 256 * (attn::kSoftmaxRegs + attn::kServiceRegs))
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
// Own pages of each request: bound by reading keys and values once.  A block takes one
// request, one key head, up to 16 of its query heads and a range of keys; each of its
// warps takes 16 keys at a time, with its own running maximum and sum, and the four are
// joined at the end.  The products are m16n8k16 steps of one warp: 16 query heads by 8
// keys, then by 8 values.  Operands go from global memory to registers in 16-byte loads,
// without a stop in shared memory:
//   * keys: the order of the contraction index is free, so lane (g, t) = (lane / 4,
//     lane % 4) holds chunks t, t + 4, ... (eight values each) of key g, and the queries are
//     laid out the same way;
//   * values: the order of the output columns is free, so lane (g, t) holds chunks g and
//     g + 8 of keys 2t, 2t + 1, 2t + 8 and 2t + 9, and column n of step (i, e) is value
//     (8 i + n) 8 + e: one byte permutation makes each operand register.
// The next keys are loaded while the scores become probabilities, the next values while
// the next scores are made.
// ---------------------------------------------------------------------------------
constexpr int kOwnWarps = 4;

template <class H>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (std::is_same<H, Bf16>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t word(const uint4& u, int i) { return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w; }

template <class H, int D>
__global__ void __launch_bounds__(kOwnWarps * 32) own_pages_kernel(const __grid_constant__ SharedArgs a, int splits, int chunk,
                                                                   float* __restrict__ part_o, float* __restrict__ part_lse) {
    using T = typename H::type;
    constexpr int KC = D / 32, VC = D / 64;  // chunks a lane holds of a key row, of a value row
    constexpr int kPad = D + 4;
    __shared__ float s_o[kOwnWarps][16][kPad];
    __shared__ float s_m[kOwnWarps][16], s_l[kOwnWarps][16];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int group = a.heads / a.kv_heads, mt = (group + 15) / 16;
    int x = blockIdx.x;  // key heads fastest: blocks that run together read neighbouring memory
    const int kh = x % a.kv_heads;
    x /= a.kv_heads;
    const int m0 = (x % mt) * 16;
    x /= mt;
    const int split = x % splits, b = x / splits;
    const int rows_here = min(16, group - m0);
    const long long rows = (long long)a.n_requests * a.heads;
    const long long row0 = (long long)b * a.heads + kh * group + m0;

    const int n = min(max(a.lengths[b], 0), a.table_width << a.page_shift);
    const int begin = min((long long)split * chunk, (long long)n), end = min(n, begin + chunk);
    if (begin >= end) {
        if (tid < rows_here) part_lse[split * rows + row0 + tid] = -INFINITY;
        return;
    }
    const int blocks = (end - begin + 15) / 16;
    const int32_t* pages = a.table + (long long)b * a.table_stride;
    const int mask = (1 << a.page_shift) - 1;

    // Queries, laid out as the keys are.
    uint32_t qa[2 * KC][4];
#pragma unroll
    for (int i = 0; i < KC; ++i) {
        const int c = (i * 4 + t) * 8;
        uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
        const T* q = static_cast<const T*>(a.q.p) + b * a.q.tok + (kh * group + m0) * a.q.head;
        if (c < a.dim && g < rows_here) lo = *reinterpret_cast<const uint4*>(q + g * a.q.head + c);
        if (c < a.dim && g + 8 < rows_here) hi = *reinterpret_cast<const uint4*>(q + (g + 8) * a.q.head + c);
        qa[2 * i][0] = lo.x; qa[2 * i][1] = hi.x; qa[2 * i][2] = lo.y; qa[2 * i][3] = hi.y;
        qa[2 * i + 1][0] = lo.z; qa[2 * i + 1][1] = hi.z; qa[2 * i + 1][2] = lo.w; qa[2 * i + 1][3] = hi.w;
    }

    uint4 kf[2][KC], vf[4][VC];
    // 16 keys lie in one page.  Rows past the end are not read: they may hold anything.
    auto load_k = [&](int ib, int pg) {
        const int key = begin + ib * 16;
        const bool ok = ib < blocks && pg >= 0 && pg < a.n_pages;
        const T* p = static_cast<const T*>(a.k_cache.p) + pg * a.k_cache.page + (key & mask) * a.k_cache.tok + kh * a.k_cache.head;
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int i = 0; i < KC; ++i) {
                const int c = (i * 4 + t) * 8;
                kf[r][i] = make_uint4(0, 0, 0, 0);
                if (ok && c < a.dim && key + r * 8 + g < end)
                    kf[r][i] = *reinterpret_cast<const uint4*>(p + (r * 8 + g) * a.k_cache.tok + c);
            }
    };
    auto load_v = [&](int ib, int pg) {
        const int key = begin + ib * 16;
        const bool ok = ib < blocks && pg >= 0 && pg < a.n_pages;
        const T* p = static_cast<const T*>(a.v_cache.p) + pg * a.v_cache.page + (key & mask) * a.v_cache.tok + kh * a.v_cache.head;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < VC; ++i) {
                const int c = (i * 8 + g) * 8, k = 2 * t + (r & 1) + (r >> 1) * 8;
                vf[r][i] = make_uint4(0, 0, 0, 0);
                if (ok && c < a.dim && key + k < end) vf[r][i] = *reinterpret_cast<const uint4*>(p + k * a.v_cache.tok + c);
            }
    };
    auto page_of = [&](int ib) { return ib < blocks ? pages[(begin + ib * 16) >> a.page_shift] : -1; };

    float o[VC][8][4];
#pragma unroll
    for (int i = 0; i < VC; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[i][e][c] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    const float scale = a.scale * kLog2e;
    int ib = warp, pg = page_of(ib), pg_next = page_of(ib + kOwnWarps);
    load_k(ib, pg);
    load_v(ib, pg);
    for (; ib < blocks; ib += kOwnWarps) {
        float s[2][4] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
#pragma unroll
        for (int i = 0; i < KC; ++i)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                mma16816<H>(s[r], qa[2 * i], kf[r][i].x, kf[r][i].y);
                mma16816<H>(s[r], qa[2 * i + 1], kf[r][i].z, kf[r][i].w);
            }
        const int pg_after = page_of(ib + 2 * kOwnWarps);
        load_k(ib + kOwnWarps, pg_next);
        const int key = begin + ib * 16;
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                s[r][c] = key + r * 8 + 2 * t + (c & 1) < end ? s[r][c] * scale : -INFINITY;
                top[c >> 1] = fmaxf(top[c >> 1], s[r][c]);
            }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
            top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
        }
        if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float up = fmaxf(m[h], top[h]), f = up == -INFINITY ? 1.0f : attn::ex2(m[h] - up);
                m[h] = up;
                l[h] *= f;
#pragma unroll
                for (int i = 0; i < VC; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        o[i][e][2 * h] *= f;
                        o[i][e][2 * h + 1] *= f;
                    }
            }
        }
        const float ref0 = m[0] == -INFINITY ? 0.0f : m[0], ref1 = m[1] == -INFINITY ? 0.0f : m[1];
        uint32_t pa[4];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const float p0 = attn::ex2(s[r][0] - ref0), p1 = attn::ex2(s[r][1] - ref0);
            const float p2 = attn::ex2(s[r][2] - ref1), p3 = attn::ex2(s[r][3] - ref1);
            l[0] += p0 + p1;
            l[1] += p2 + p3;
            pa[2 * r] = H::pack(p0, p1);
            pa[2 * r + 1] = H::pack(p2, p3);
        }
#pragma unroll
        for (int i = 0; i < VC; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t sel = (e & 1) ? 0x7632u : 0x5410u;
                const uint32_t b0 = __byte_perm(word(vf[0][i], e / 2), word(vf[1][i], e / 2), sel);
                const uint32_t b1 = __byte_perm(word(vf[2][i], e / 2), word(vf[3][i], e / 2), sel);
                mma16816<H>(o[i][e], pa, b0, b1);
            }
        load_v(ib + kOwnWarps, pg_next);
        pg_next = pg_after;
    }

    // Join of the four warps.
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        const int r = g + 8 * h;
        if (t == 0) {
            s_m[warp][r] = m[h];
            s_l[warp][r] = l[h];
        }
#pragma unroll
        for (int i = 0; i < VC; ++i)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float4* dst = reinterpret_cast<float4*>(&s_o[warp][r][(i * 8 + 2 * t + c) * 8]);
                dst[0] = make_float4(o[i][0][2 * h + c], o[i][1][2 * h + c], o[i][2][2 * h + c], o[i][3][2 * h + c]);
                dst[1] = make_float4(o[i][4][2 * h + c], o[i][5][2 * h + c], o[i][6][2 * h + c], o[i][7][2 * h + c]);
            }
    }
    __syncthreads();
    const int r = tid >> 3;
    if (r >= rows_here) return;
    float top = -INFINITY, total = 0.0f, w[kOwnWarps];
#pragma unroll
    for (int i = 0; i < kOwnWarps; ++i) top = fmaxf(top, s_m[i][r]);
#pragma unroll
    for (int i = 0; i < kOwnWarps; ++i) {
        w[i] = s_m[i][r] == -INFINITY ? 0.0f : attn::ex2(s_m[i][r] - top);
        if (i >= blocks) w[i] = 0.0f;  // a warp without keys
        total += s_l[i][r] * w[i];
    }
    const float inv = total > 0.0f ? 1.0f / total : (total == 0.0f ? 0.0f : total);
    for (int d = (tid & 7) * 4; d < a.dim; d += 32) {
        float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < kOwnWarps; ++i) {
            const float4 v = *reinterpret_cast<const float4*>(&s_o[i][r][d]);
            acc = make_float4(acc.x + w[i] * v.x, acc.y + w[i] * v.y, acc.z + w[i] * v.z, acc.w + w[i] * v.w);
        }
        *reinterpret_cast<float4*>(part_o + (split * rows + row0 + r) * a.dim + d) =
            make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    }
    if ((tid & 7) == 0) part_lse[split * rows + row0 + r] = top + log2f(total);
}

struct OwnPlan {
    int splits, chunk;  // ranges of `chunk` keys
};
// The lengths are on the device: ranges are cut for what the table can hold.  Six blocks an
// SM fill the GPU; no range is below 128 keys, none above 1,024, so that the longest request
// does not run on alone.  A range past a request's length costs one write a row.
OwnPlan own_plan(const SharedArgs& a) {
    const long long cap = (long long)a.table_width << a.page_shift;
    const long long base = (long long)a.n_requests * a.kv_heads * ((a.heads / a.kv_heads + 15) / 16);
    long long s = std::max<long long>(ceil_div(6 * kSms, base), ceil_div(cap, 1024));
    s = std::max<long long>(1, std::min<long long>({s, (cap + 127) / 128, 256}));
    OwnPlan p;
    p.chunk = (int)((ceil_div(cap, s) + 63) / 64 * 64);
    p.splits = p.chunk ? (int)((cap + p.chunk - 1) / p.chunk) : 0;
    return p;
}

template <class H>
void launch_own(const SharedArgs& a, const OwnPlan& pl, float* part_o, float* part_lse, cudaStream_t st) {
    const long long blocks = (long long)a.n_requests * a.kv_heads * ((a.heads / a.kv_heads + 15) / 16) * pl.splits;
    if (blocks > 0x7fffffffLL) throw CudaError("attention: too many requests for one launch");
    if (a.dim <= 64)
        own_pages_kernel<H, 64><<<(unsigned)blocks, kOwnWarps * 32, 0, st>>>(a, pl.splits, pl.chunk, part_o, part_lse);
    else
        own_pages_kernel<H, 128><<<(unsigned)blocks, kOwnWarps * 32, 0, st>>>(a, pl.splits, pl.chunk, part_o, part_lse);
    VGPU_LAUNCH("own_pages_kernel");
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
    return part_bytes(own_plan(a).splits + (a.prefix_len ? shared_splits(a) : 0), (long long)a.n_requests * a.heads, a.dim);
}

void launch_shared_attention(const SharedArgs& a, cudaStream_t st) {
    const long long rows = (long long)a.n_requests * a.heads;
    const int splits = a.prefix_len ? shared_splits(a) : 0;
    const OwnPlan own = own_plan(a);
    float* part_o = static_cast<float*>(a.workspace);
    float* part_lse = part_o + (splits + own.splits) * rows * a.dim;
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
    if (own.splits) {
        float* own_o = part_o + splits * rows * a.dim;
        float* own_lse = part_lse + splits * rows;
        if (a.f16) launch_own<F16>(a, own, own_o, own_lse, st);
        else launch_own<Bf16>(a, own, own_o, own_lse, st);
    }
    launch_join(a.f16, splits + own.splits, rows, a.dim, part_o, part_lse, a.out, a.lse, st);
}

}  // namespace vgpu

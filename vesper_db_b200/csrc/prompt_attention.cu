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
// Prefix rows in tiles of 8 or 16: up to this many of them, re-reading the prefix for each
// from L2 is quicker than a tensor-core tile.
constexpr int kFewRowTiles = 4;
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
// Pages of a cache with few query rows: each request's own pages, and the prefix when the
// whole batch has few rows.  Bound by reading keys and values once.  A block takes one key
// head, up to 8 * NT query rows and a range of keys; each of its warps takes 16 keys at a
// time, with its own running maximum and sum, and the four are joined at the end.  The
// products are m16n8k16 steps of one warp, S^T = K Q^T (16 keys by 8 rows) and O^T = V^T P^T
// (16 values by 8 rows): with the rows on the short side few of them waste little.  Operands
// go from global memory to registers in 16-byte loads, without a stop in shared memory:
//   * keys: the order of the contraction index is free, so lane (g, t) = (lane / 4,
//     lane % 4) holds chunks t, t + 4, ... (eight values each) of keys g and g + 8, and the
//     queries are laid out the same way;
//   * values: the order of the output rows is free, so lane (g, t) holds chunks g and g + 8
//     of keys 2t, 2t + 1, 2t + 8 and 2t + 9, and rows g and g + 8 of step (i, e) are values e
//     and e + 4 of chunk 8 i + g: one byte permutation makes each operand register;
//   * probabilities: one 8 x 8 transposition between registers turns S^T into P^T.
// The next keys are loaded while the scores become probabilities, the next values while
// the next scores are made.
// ---------------------------------------------------------------------------------
constexpr int kOwnWarps = 4;

template <class H>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    if (std::is_same<H, Bf16>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transposed8x8(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

__device__ __forceinline__ uint32_t word(const uint4& u, int i) { return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w; }

// Blocks below `prefix_blocks` take the prefix, the others the requests' own pages; a range
// is `chunk` keys.  Results of range i go to part i of the prefix's or of the own parts.
struct PagesPlan {
    int prefix_blocks, prefix_splits, prefix_chunk;
    int own_splits, own_chunk;
    float* prefix_o;
    float* prefix_lse;
    float* own_o;
    float* own_lse;
};

template <class H, int D, int NT>
__global__ void __launch_bounds__(kOwnWarps * 32, NT == 1 ? 4 : 2)
    pages_kernel(const __grid_constant__ SharedArgs a, const __grid_constant__ PagesPlan pl) {
    using T = typename H::type;
    constexpr int KC = D / 32, VC = D / 64;  // chunks a lane holds of a key, of a value row
    constexpr int kRowsHere = 8 * NT;
    __shared__ float s_o[kOwnWarps][kRowsHere][D + 4];
    __shared__ float s_m[kOwnWarps][kRowsHere], s_l[kOwnWarps][kRowsHere];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int group = a.heads / a.kv_heads;
    const bool prefix = (int)blockIdx.x < pl.prefix_blocks;
    int x = prefix ? blockIdx.x : blockIdx.x - pl.prefix_blocks;
    const int kh = x % a.kv_heads;  // key heads fastest: blocks that run together read neighbouring memory
    x /= a.kv_heads;
    // Rows of this block: row r is query head kh * group + (m0 + r) % group of request
    // b + (m0 + r) / group.
    int b, split, m0, n_rows, n, chunk;
    const int32_t* pages;
    if (prefix) {
        split = x % pl.prefix_splits;
        m0 = x / pl.prefix_splits * kRowsHere;
        b = 0;
        n_rows = min(kRowsHere, a.n_requests * group - m0);
        n = (int)a.prefix_len;
        chunk = pl.prefix_chunk;
        pages = a.prefix_pages;
    } else {
        const int mt = (group + kRowsHere - 1) / kRowsHere;
        m0 = x % mt * kRowsHere;
        x /= mt;
        split = x % pl.own_splits;
        b = x / pl.own_splits;
        n_rows = min(kRowsHere, group - m0);
        n = min(max(a.lengths[b], 0), a.table_width << a.page_shift);
        chunk = pl.own_chunk;
        pages = a.table + (long long)b * a.table_stride;
    }
    const long long rows = (long long)a.n_requests * a.heads;
    auto row_of = [&](int r) { return (long long)(b + (m0 + r) / group) * a.heads + kh * group + (m0 + r) % group; };
    float* const out_o = (prefix ? pl.prefix_o : pl.own_o) + split * rows * a.dim;
    float* const out_lse = (prefix ? pl.prefix_lse : pl.own_lse) + split * rows;

    const int begin = (int)min((long long)split * chunk, (long long)n), end = min(n, begin + chunk);
    if (begin >= end) {
        if (tid < n_rows) out_lse[row_of(tid)] = -INFINITY;
        return;
    }
    const int blocks = (end - begin + 15) / 16;
    const int mask = (1 << a.page_shift) - 1;

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

    int ib = warp, pg = page_of(ib), pg_next = page_of(ib + kOwnWarps);
    load_k(ib, pg);
    load_v(ib, pg);
    // Queries, laid out as the keys are.
    uint32_t qb[NT][2 * KC][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
        const int r = nt * 8 + g;
        const T* q = static_cast<const T*>(a.q.p);
        if (r < n_rows) q += (long long)(b + (m0 + r) / group) * a.q.tok + (kh * group + (m0 + r) % group) * a.q.head;
#pragma unroll
        for (int i = 0; i < KC; ++i) {
            const int c = (i * 4 + t) * 8;
            uint4 u = make_uint4(0, 0, 0, 0);
            if (c < a.dim && r < n_rows) u = *reinterpret_cast<const uint4*>(q + c);
            qb[nt][2 * i][0] = u.x; qb[nt][2 * i][1] = u.y;
            qb[nt][2 * i + 1][0] = u.z; qb[nt][2 * i + 1][1] = u.w;
        }
    }

    float o[NT][VC][4][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < VC; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[nt][i][e][c] = 0.0f;
    float m[NT][2], l[NT][2];  // of rows 2t and 2t + 1; l over this lane's keys only
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) m[nt][0] = m[nt][1] = -INFINITY, l[nt][0] = l[nt][1] = 0.0f;
    const float scale = a.scale * kLog2e;
    for (; ib < blocks; ib += kOwnWarps) {
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
#pragma unroll
            for (int i = 0; i < KC; ++i) {
                mma16816<H>(s[nt], kf[0][i].x, kf[1][i].x, kf[0][i].y, kf[1][i].y, qb[nt][2 * i][0], qb[nt][2 * i][1]);
                mma16816<H>(s[nt], kf[0][i].z, kf[1][i].z, kf[0][i].w, kf[1][i].w, qb[nt][2 * i + 1][0], qb[nt][2 * i + 1][1]);
            }
        }
        const int pg_after = page_of(ib + 2 * kOwnWarps);
        load_k(ib + kOwnWarps, pg_next);
        const int key = begin + ib * 16 + g;
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float top[2];
#pragma unroll
            for (int c = 0; c < 4; ++c) s[nt][c] = key + (c >> 1) * 8 < end ? s[nt][c] * scale : -INFINITY;
            top[0] = fmaxf(s[nt][0], s[nt][2]);
            top[1] = fmaxf(s[nt][1], s[nt][3]);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 4; e < 32; e *= 2) top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], e));
            if (__any_sync(0xffffffffu, top[0] > m[nt][0] || top[1] > m[nt][1])) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float up = fmaxf(m[nt][h], top[h]), f = up == -INFINITY ? 1.0f : attn::ex2(m[nt][h] - up);
                    m[nt][h] = up;
                    l[nt][h] *= f;
#pragma unroll
                    for (int i = 0; i < VC; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            o[nt][i][e][h] *= f;
                            o[nt][i][e][2 + h] *= f;
                        }
                }
            }
            const float ref0 = m[nt][0] == -INFINITY ? 0.0f : m[nt][0], ref1 = m[nt][1] == -INFINITY ? 0.0f : m[nt][1];
#pragma unroll
            for (int h = 0; h < 2; ++h) {  // keys g and g + 8
                const float p0 = attn::ex2(s[nt][2 * h] - ref0), p1 = attn::ex2(s[nt][2 * h + 1] - ref1);
                l[nt][0] += p0;
                l[nt][1] += p1;
                pb[nt][h] = transposed8x8(H::pack(p0, p1));
            }
        }
#pragma unroll
        for (int i = 0; i < VC; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t sel = (e & 1) ? 0x7632u : 0x5410u;
                const uint32_t a0 = __byte_perm(word(vf[0][i], e / 2), word(vf[1][i], e / 2), sel);
                const uint32_t a1 = __byte_perm(word(vf[0][i], e / 2 + 2), word(vf[1][i], e / 2 + 2), sel);
                const uint32_t a2 = __byte_perm(word(vf[2][i], e / 2), word(vf[3][i], e / 2), sel);
                const uint32_t a3 = __byte_perm(word(vf[2][i], e / 2 + 2), word(vf[3][i], e / 2 + 2), sel);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma16816<H>(o[nt][i][e], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
            }
        load_v(ib + kOwnWarps, pg_next);
        pg_next = pg_after;
    }

    // Join of the four warps.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = nt * 8 + 2 * t + h;
#pragma unroll
            for (int e = 4; e < 32; e *= 2) l[nt][h] += __shfl_xor_sync(0xffffffffu, l[nt][h], e);
            if (g == 0) {
                s_m[warp][r] = m[nt][h];
                s_l[warp][r] = l[nt][h];
            }
#pragma unroll
            for (int i = 0; i < VC; ++i) {
                float4* dst = reinterpret_cast<float4*>(&s_o[warp][r][(i * 8 + g) * 8]);
                dst[0] = make_float4(o[nt][i][0][h], o[nt][i][1][h], o[nt][i][2][h], o[nt][i][3][h]);
                dst[1] = make_float4(o[nt][i][0][2 + h], o[nt][i][1][2 + h], o[nt][i][2][2 + h], o[nt][i][3][2 + h]);
            }
        }
    __syncthreads();
    constexpr int kPerRow = kOwnWarps * 32 / kRowsHere;
    const int r = tid / kPerRow;
    if (r >= n_rows) return;
    float top = -INFINITY, total = 0.0f, w[kOwnWarps];
#pragma unroll
    for (int i = 0; i < kOwnWarps; ++i) top = fmaxf(top, s_m[i][r]);
#pragma unroll
    for (int i = 0; i < kOwnWarps; ++i) {
        // a warp without keys has m = -inf, and zeros
        w[i] = s_m[i][r] == -INFINITY ? 0.0f : attn::ex2(s_m[i][r] - top);
        total += s_l[i][r] * (i < blocks && s_m[i][r] == -INFINITY ? 1.0f : w[i]);
    }
    const float inv = total > 0.0f ? 1.0f / total : (total == 0.0f ? 0.0f : total);
    const long long row = row_of(r);
    for (int d = tid % kPerRow * 4; d < a.dim; d += kPerRow * 4) {
        float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < kOwnWarps; ++i) {
            const float4 v = *reinterpret_cast<const float4*>(&s_o[i][r][d]);
            acc = make_float4(acc.x + w[i] * v.x, acc.y + w[i] * v.y, acc.z + w[i] * v.z, acc.w + w[i] * v.w);
        }
        *reinterpret_cast<float4*>(out_o + row * a.dim + d) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    }
    if (tid % kPerRow == 0) out_lse[row] = top + log2f(total);
}

// The lengths are on the device: ranges are cut for what the table can hold.  A range past a
// request's length costs one write a row.
int keys_a_range(long long cap, long long blocks_a_range) {
    // four blocks an SM fill the GPU; 128 keys at least a range, 512 at most, so that the
    // longest request does not run on alone
    long long s = std::max<long long>(ceil_div(4 * kSms, std::max<long long>(blocks_a_range, 1)), ceil_div(cap, 512));
    s = std::max<long long>(1, std::min<long long>(s, (cap + 127) / 128));
    return (int)((ceil_div(cap, s) + 63) / 64 * 64);
}

template <class H>
void launch_pages(const SharedArgs& a, const PagesPlan& pl, int nt, cudaStream_t st) {
    const int group = a.heads / a.kv_heads;
    const long long blocks =
        pl.prefix_blocks + (long long)a.n_requests * a.kv_heads * ((group + 8 * nt - 1) / (8 * nt)) * pl.own_splits;
    if (blocks > 0x7fffffffLL) throw CudaError("attention: too many requests for one launch");
    if (blocks == 0) return;
    auto launch = [&](auto* kernel) { kernel<<<(unsigned)blocks, kOwnWarps * 32, 0, st>>>(a, pl); };
    if (a.dim <= 64) launch(nt == 1 ? pages_kernel<H, 64, 1> : pages_kernel<H, 64, 2>);
    else launch(nt == 1 ? pages_kernel<H, 128, 1> : pages_kernel<H, 128, 2>);
    VGPU_LAUNCH("pages_kernel");
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
    const bool live = lane * 4 < dim;
    float m = -INFINITY, total = 0.0f;
    bool nan = false;
    float4 o = make_float4(0, 0, 0, 0);
    for (int p0 = 0; p0 < parts; p0 += 32) {  // the weights of 32 parts, one a lane
        const float x = p0 + lane < parts ? part_lse[(p0 + lane) * rows + row] : -INFINITY;
        float up = m;
        nan |= __any_sync(0xffffffffu, isnan(x)) != 0;
        up = fmaxf(up, x);
#pragma unroll
        for (int e = 16; e > 0; e >>= 1) up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, e));
        const float ref = up == -INFINITY ? 0.0f : up, f = exp2f(m - ref), w = exp2f(x - ref);
        m = up;
        total = total * f + w;  // this lane's share
        o = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
        unsigned some = __ballot_sync(0xffffffffu, w > 0.0f);  // parts without keys hold no rows
        while (some) {
            float4 v[4];
            float wi[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = some ? __ffs(some) - 1 : -1;
                wi[e] = __shfl_sync(0xffffffffu, w, i < 0 ? 0 : i);
                v[e] = make_float4(0, 0, 0, 0);
                if (i < 0) wi[e] = 0.0f;
                else if (live) v[e] = *reinterpret_cast<const float4*>(part_o + ((p0 + i) * rows + row) * dim + lane * 4);
                some &= some - 1;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                o = make_float4(o.x + wi[e] * v[e].x, o.y + wi[e] * v[e].y, o.z + wi[e] * v[e].z, o.w + wi[e] * v[e].w);
        }
    }
#pragma unroll
    for (int e = 16; e > 0; e >>= 1) total += __shfl_xor_sync(0xffffffffu, total, e);
    const float inv = nan ? __int_as_float(0x7fc00000) : (total > 0.0f ? 1.0f / total : 0.0f);
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

// Parts of the prefix, then of the own pages.
struct SharedPlan {
    bool tiles;  // the prefix goes to the tensor cores' tiles
    int prefix_splits, prefix_chunk, own_splits, own_chunk, nt;
};
SharedPlan shared_plan(const SharedArgs& a) {
    SharedPlan p{};
    const int group = a.heads / a.kv_heads;
    const long long rows = (long long)a.n_requests * group;  // of one key head
    p.nt = group > 8 ? 2 : 1;
    const long long cap = (long long)a.table_width << a.page_shift;
    const long long own_blocks = (long long)a.n_requests * a.kv_heads * ((group + 8 * p.nt - 1) / (8 * p.nt));
    p.own_chunk = cap ? keys_a_range(cap, own_blocks) : 0;
    p.own_splits = cap ? (int)((cap + p.own_chunk - 1) / p.own_chunk) : 0;
    if (a.prefix_len == 0) return p;
    const long long row_tiles = (rows + 8 * p.nt - 1) / (8 * p.nt);
    p.tiles = row_tiles > kFewRowTiles;
    if (p.tiles) {
        const int span = 2 * (kRows / group);
        p.prefix_splits = splits_for((long long)ceil_div(a.n_requests, span) * a.kv_heads, a.prefix_len / kKeys);
    } else {
        p.prefix_chunk = keys_a_range(a.prefix_len, row_tiles * a.kv_heads);
        p.prefix_splits = (int)((a.prefix_len + p.prefix_chunk - 1) / p.prefix_chunk);
    }
    return p;
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
    const SharedPlan sp = shared_plan(a);
    return part_bytes(sp.prefix_splits + sp.own_splits, (long long)a.n_requests * a.heads, a.dim);
}

void launch_shared_attention(const SharedArgs& a, cudaStream_t st) {
    const long long rows = (long long)a.n_requests * a.heads;
    const SharedPlan sp = shared_plan(a);
    const int parts = sp.prefix_splits + sp.own_splits;
    float* part_o = static_cast<float*>(a.workspace);
    float* part_lse = part_o + parts * rows * a.dim;
    PagesPlan pl{};
    pl.own_splits = sp.own_splits;
    pl.own_chunk = sp.own_chunk;
    pl.own_o = part_o + sp.prefix_splits * rows * a.dim;
    pl.own_lse = part_lse + sp.prefix_splits * rows;
    if (sp.tiles) {
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
        p.splits = sp.prefix_splits;
        p.part = true;
        p.part_o = part_o;
        p.part_lse = part_lse;
        launch_tiles<true>(p, a.f16, (long long)ceil_div(a.n_requests, 2 * p.tile_tokens) * a.kv_heads * p.splits, st);
    } else if (sp.prefix_splits) {
        const long long row_tiles = ((long long)a.n_requests * (a.heads / a.kv_heads) + 8 * sp.nt - 1) / (8 * sp.nt);
        pl.prefix_blocks = (int)(row_tiles * a.kv_heads * sp.prefix_splits);
        pl.prefix_splits = sp.prefix_splits;
        pl.prefix_chunk = sp.prefix_chunk;
        pl.prefix_o = part_o;
        pl.prefix_lse = part_lse;
    }
    if (a.f16) launch_pages<F16>(a, pl, sp.nt, st);
    else launch_pages<Bf16>(a, pl, sp.nt, st);
    launch_join(a.f16, parts, rows, a.dim, part_o, part_lse, a.out, a.lse, st);
}

}  // namespace vgpu

// Page tables of a paged key/value cache, and the norm + rotation that fills it.
#include <algorithm>

#include "attention.cuh"
#include "common.cuh"
#include "half_types.cuh"

namespace vgpu {

namespace {

// ---------------------------------------------------------------------------------
// Page tables.  Request b holds cached_b tokens and gets fresh_b more:
//   had_b = ceil(cached_b / P), need_b = ceil((cached_b + fresh_b) / P),
//   first_b = sum_{a < b} (need_a - had_a),
//   table[b, had_b + i] = free[first_b + i],
//   starts_b = sum_{a < b} fresh_a; token t of request b has n = cached_b + t - starts_b,
//   slot table[b, n / P] * P + n % P, position base + n.
// One launch: every block scans all requests itself (two int32 loads each, from L2), so
// no block waits for another; then each block fills its share of tokens and table rows.
// A token's new page is taken from the free list directly, never from a table entry that
// another block may still be writing.
// ---------------------------------------------------------------------------------
constexpr int kScanThreads = 512;

__device__ __forceinline__ int clamp_int(long long v) {
    return (int)(v < 0 ? 0 : (v > 0x7fffffffLL ? 0x7fffffffLL : v));
}

__global__ void __launch_bounds__(kScanThreads) page_tables_kernel(const __grid_constant__ PageTablesArgs a) {
    extern __shared__ int smem[];
    int* s_start = smem;                        // [n + 1] first token of each request
    int* s_first = smem + a.n_requests + 1;     // [n + 1] first free-list entry of each request
    __shared__ long long s_warp[2][kScanThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.n_requests;
    const int page = 1 << a.page_shift;

    // Exclusive scans, kScanThreads requests at a time; sums in 64 bits.
    long long run_t = 0, run_p = 0;
    for (int r0 = 0; r0 < n; r0 += kScanThreads) {
        const int r = r0 + tid;
        long long fresh = 0, pages = 0;
        if (r < n) {
            const long long old = max(a.cached[r], 0);
            fresh = max(a.fresh[r], 0);
            pages = ((old + fresh + page - 1) >> a.page_shift) - ((old + page - 1) >> a.page_shift);
            if (blockIdx.x == 0) a.lengths[r] = clamp_int(old + fresh);
        }
        long long it = fresh, ip = pages;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long ut = __shfl_up_sync(0xffffffffu, it, o), up = __shfl_up_sync(0xffffffffu, ip, o);
            if (lane >= o) { it += ut; ip += up; }
        }
        if (lane == 31) { s_warp[0][warp] = it; s_warp[1][warp] = ip; }
        __syncthreads();
        long long bt = run_t, bp = run_p;
        for (int w = 0; w < kScanThreads / 32; ++w) {
            if (w < warp) { bt += s_warp[0][w]; bp += s_warp[1][w]; }
            run_t += s_warp[0][w];
            run_p += s_warp[1][w];
        }
        if (r < n) {
            s_start[r] = clamp_int(bt + it - fresh);
            s_first[r] = clamp_int(bp + ip - pages);
        }
        __syncthreads();
    }
    if (tid == 0) {
        s_start[n] = clamp_int(run_t);
        s_first[n] = clamp_int(run_p);
        if (blockIdx.x == 0) a.used[0] = clamp_int(run_p);
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int r = tid; r <= n; r += kScanThreads) a.starts[r] = s_start[r];

    // New table entries: one warp a request.
    for (int r = blockIdx.x * (kScanThreads / 32) + warp; r < n; r += gridDim.x * (kScanThreads / 32)) {
        const long long had = ((long long)max(a.cached[r], 0) + page - 1) >> a.page_shift;
        const int first = s_first[r], more = s_first[r + 1] - first;
        for (int i = lane; i < more; i += 32) {
            if (had + i >= a.table_width) break;
            const long long f = (long long)first + i;
            a.table[(long long)r * a.table_stride + had + i] = f < a.n_free ? a.free_pages[f] : -1;
        }
    }

    // Tokens: a run of kRun consecutive ones a thread, one search for the first of them.
    constexpr int kRun = 4;
    for (long long t0 = ((long long)blockIdx.x * kScanThreads + tid) * kRun; t0 < a.n_tokens;
         t0 += (long long)gridDim.x * kScanThreads * kRun) {
        int lo = 0, hi = n;  // the last request whose start is <= t0
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s_start[mid] <= t0) lo = mid; else hi = mid;
        }
        int r = lo;
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
            const long long t = t0 + i;
            if (t >= a.n_tokens) break;
            while (r < n && s_start[r + 1] <= t) ++r;
            int pos = 0;
            int64_t slot = -1;
            if (r < n) {
                const long long old = max(a.cached[r], 0), at = old + t - s_start[r];
                const long long col = at >> a.page_shift, had = (old + page - 1) >> a.page_shift;
                int32_t pg = -1;
                if (col < a.table_width) {
                    if (col < had) {
                        pg = a.table[(long long)r * a.table_stride + col];
                    } else {
                        const long long f = s_first[r] + col - had;
                        if (f < a.n_free) pg = a.free_pages[f];
                    }
                }
                if (pg >= 0) slot = ((int64_t)pg << a.page_shift) + (at & (page - 1));
                pos = clamp_int(at + a.base);
            }
            a.positions[t] = pos;
            a.slots[t] = slot;
        }
    }
}

// ---------------------------------------------------------------------------------
// Norm of each head, rotation, cache write.  x of one head (dim values):
//   y = x * rsqrt(mean(x^2) + eps) * w, then for each pair (a, b) of the first `turned`
//   values, a' = a cos - b sin, b' = b cos + a sin.
// All of it in 32 bits, one rounding at the store.  Bound by reading and writing each row
// once.  A group of W lanes holds one head, eight values (16 bytes) a lane; the partner of
// a half-split pair is in another lane of the group.  A block takes whole tokens, so that a
// lane's cosines and sines serve all heads and its weights all tokens; the rows of kBatch
// heads are requested before the first of them is used.
// ---------------------------------------------------------------------------------
constexpr int kRotThreads = 256;
constexpr int kBatch = 4;

template <class H, int W, bool PAIRS>
__global__ void __launch_bounds__(kRotThreads, 3) norm_rotate_kernel(const __grid_constant__ NormRotateArgs a) {
    using T = typename H::type;
    const int c = threadIdx.x % W;  // this lane's chunk of eight values
    const int group = threadIdx.x / W;
    constexpr int kGroups = kRotThreads / W;
    const int half = a.turned / 2, total = a.heads + 2 * a.kv_heads;
    const bool live = c * 8 < a.dim, turns_here = c * 8 < a.turned;
    // Angles of the chunk: half-split pairs use angle i % (turned / 2), neighbouring pairs
    // angle i / 2.
    const int angle = PAIRS ? c * 4 : (c * 8 < half ? c * 8 : c * 8 - half);
    const int mate = !turns_here || PAIRS ? c : (c * 8 < half ? c + half / 8 : c - half / 8);
    const float sign = c * 8 < half ? -1.0f : 1.0f;
    uint4 wq = make_uint4(0, 0, 0, 0), wk = wq;
    if (live && a.q_weight) wq = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q_weight) + c * 8);
    if (live && a.k_weight) wk = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.k_weight) + c * 8);

    for (int t = blockIdx.x; t < a.n_tokens; t += gridDim.x) {
        const int pos = a.positions[t];
        int64_t slot = a.slots ? a.slots[t] : -1;
        const bool known = pos >= 0 && pos < a.n_positions;
        if (slot >= (a.n_pages << a.page_shift)) slot = -1;
        const int64_t page = slot >> a.page_shift, off = slot & ((1 << a.page_shift) - 1);
        constexpr int kAngles = PAIRS ? 4 : 8;
        float cs[kAngles], sn[kAngles];
#pragma unroll
        for (int i = 0; i < kAngles; i += 4) {
            float4 x = make_float4(1, 1, 1, 1), y = make_float4(0, 0, 0, 0);
            if (turns_here) {
                const float nan = __int_as_float(0x7fc00000);
                x = y = make_float4(nan, nan, nan, nan);
                if (known) {
                    const float* row = a.turns + (long long)pos * a.turned + angle + i;
                    x = __ldg(reinterpret_cast<const float4*>(row));
                    y = __ldg(reinterpret_cast<const float4*>(row + half));
                }
            }
            cs[i] = x.x; cs[i + 1] = x.y; cs[i + 2] = x.z; cs[i + 3] = x.w;
            sn[i] = y.x; sn[i + 1] = y.y; sn[i + 2] = y.z; sn[i + 3] = y.w;
        }
        for (int u0 = group; u0 - group < total; u0 += kGroups * kBatch) {  // uniform trip count: shuffles below
            uint4 raw[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int u = u0 + b * kGroups;
                raw[b] = make_uint4(0, 0, 0, 0);
                if (!live || u >= total) continue;
                const T* src;
                if (u < a.heads) src = static_cast<const T*>(a.q.p) + t * a.q.tok + u * a.q.head;
                else if (u < a.heads + a.kv_heads) src = static_cast<const T*>(a.k.p) + t * a.k.tok + (u - a.heads) * a.k.head;
                else if (slot < 0) continue;
                else src = static_cast<const T*>(a.v.p) + t * a.v.tok + (u - a.heads - a.kv_heads) * a.v.head;
                raw[b] = *reinterpret_cast<const uint4*>(src + c * 8);
            }
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int u = u0 + b * kGroups;
                if (u0 - group + b * kGroups >= total) break;  // the same for the whole block
                const bool is_q = u < a.heads, is_k = !is_q && u < a.heads + a.kv_heads;
                float x[8], w[8];
                unpack8<H>(raw[b], x);
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
                for (int o = W / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o, W);
                if (is_q ? a.q_weight != nullptr : a.k_weight != nullptr) {
                    const float inv = rsqrtf(ss / a.dim + a.eps);
                    unpack8<H>(is_q ? wq : wk, w);
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * w[i];
                }
                float y[8];
                if (PAIRS) {
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        y[i] = turns_here ? x[i] * cs[i / 2] - x[i + 1] * sn[i / 2] : x[i];
                        y[i + 1] = turns_here ? x[i + 1] * cs[i / 2] + x[i] * sn[i / 2] : x[i + 1];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float o = __shfl_sync(0xffffffffu, x[i], mate, W);
                        y[i] = turns_here ? x[i] * cs[i % kAngles] + sign * o * sn[i % kAngles] : x[i];
                    }
                }
                if (!live || u >= total) continue;
                if (!is_q && !is_k) {  // values are copied as they are
                    if (slot >= 0)
                        *reinterpret_cast<uint4*>(static_cast<T*>(a.v_cache.p) + page * a.v_cache.page + off * a.v_cache.tok +
                                                  (u - a.heads - a.kv_heads) * a.v_cache.head + c * 8) = raw[b];
                    continue;
                }
                const uint4 r = pack8<H>(y);
                if (is_q) {
                    *reinterpret_cast<uint4*>(static_cast<T*>(a.out_q) + ((long long)t * a.heads + u) * a.dim + c * 8) = r;
                    continue;
                }
                const int h = u - a.heads;
                if (a.out_k)
                    *reinterpret_cast<uint4*>(static_cast<T*>(a.out_k) + ((long long)t * a.kv_heads + h) * a.dim + c * 8) = r;
                if (slot >= 0)
                    *reinterpret_cast<uint4*>(static_cast<T*>(a.k_cache.p) + page * a.k_cache.page + off * a.k_cache.tok +
                                              h * a.k_cache.head + c * 8) = r;
            }
            __syncwarp();
        }
    }
}

template <class H, bool PAIRS>
void norm_rotate_width(const NormRotateArgs& a, cudaStream_t st) {
    const int chunks = a.dim / 8;
    const unsigned grid = (unsigned)std::min(a.n_tokens, 148 * 3 * 8);  // a few tokens a block where there are many
    if (chunks <= 8) norm_rotate_kernel<H, 8, PAIRS><<<grid, kRotThreads, 0, st>>>(a);
    else if (chunks <= 16) norm_rotate_kernel<H, 16, PAIRS><<<grid, kRotThreads, 0, st>>>(a);
    else norm_rotate_kernel<H, 32, PAIRS><<<grid, kRotThreads, 0, st>>>(a);
    VGPU_LAUNCH("norm_rotate_kernel");
}

}  // namespace

void launch_page_tables(const PageTablesArgs& a, cudaStream_t st) {
    const size_t smem = 2 * ((size_t)a.n_requests + 1) * sizeof(int);
    if (smem > 48 * 1024)
        VGPU_CHECK(cudaFuncSetAttribute(page_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    const long long per_block = kScanThreads * 4;
    const long long want = std::max<long long>((a.n_tokens + per_block - 1) / per_block, (a.n_requests + 63) / 64);
    const int blocks = (int)std::min<long long>(std::max<long long>(want, 1), 148 * 2);
    page_tables_kernel<<<blocks, kScanThreads, smem, st>>>(a);
    VGPU_LAUNCH("page_tables_kernel");
}

void launch_norm_rotate(const NormRotateArgs& a, cudaStream_t st) {
    if (a.f16) {
        if (a.pairs) norm_rotate_width<F16, true>(a, st);
        else norm_rotate_width<F16, false>(a, st);
    } else {
        if (a.pairs) norm_rotate_width<Bf16, true>(a, st);
        else norm_rotate_width<Bf16, false>(a, st);
    }
}

}  // namespace vgpu

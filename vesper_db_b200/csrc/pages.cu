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
// All of it in 32 bits, two values an instruction, one rounding at the store.  The bound is
// reading and writing each row once; getting near it took fewer instructions rather than
// more loads in flight.  A group of W lanes holds one head; a lane holds two chunks of eight
// values that rotate into each other (half-split pairs: chunks l and l + turned / 16, which
// share their eight angles; neighbouring pairs: chunks 2 l and 2 l + 1), so that the partners
// need no exchange.  A block takes whole tokens: a lane's cosines and sines serve all its
// heads and its weights all tokens, and the next rows are requested before the current ones
// are used.
// ---------------------------------------------------------------------------------
constexpr int kRotThreads = 256;

using Pairs = uint64_t[4];  // eight 32-bit values

template <class H>
__device__ __forceinline__ void unpack_pairs(const uint4& u, Pairs& x) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = H::unpack(w[i]);
        x[i] = pair(f.x, f.y);
    }
}

template <class H>
__device__ __forceinline__ uint4 pack_pairs(const Pairs& x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = halves(x[i]);
        w[i] = H::pack(f.x, f.y);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

struct TwoChunks {
    uint4 a, b;
};

template <class H, int W, bool PAIRS>
__global__ void __launch_bounds__(kRotThreads, 2) norm_rotate_kernel(const __grid_constant__ NormRotateArgs a) {
    using T = typename H::type;
    constexpr int kGroups = kRotThreads / W;
    const int l = threadIdx.x % W, group = threadIdx.x / W;
    const unsigned mask = W == 32 ? 0xffffffffu : ((1u << (W & 31)) - 1u) << (threadIdx.x & 31 & ~(W - 1));
    const int half = a.turned / 2, turning = a.turned / 16;  // lanes whose chunks rotate
    const bool turns_here = l < turning;
    // Values at which the lane's chunks start; the second may lie past the head.
    const int c0 = !PAIRS && turns_here ? l * 8 : (PAIRS ? l * 16 : a.turned + (l - turning) * 16);
    const int c1 = !PAIRS && turns_here ? c0 + half : c0 + 8;
    const bool live0 = c0 < a.dim, live1 = c1 < a.dim;
    const float inv_dim = 1.0f / a.dim;

    auto load2 = [&](const T* row) {
        TwoChunks x;
        x.a = x.b = make_uint4(0, 0, 0, 0);
        if (live0) x.a = __ldcs(reinterpret_cast<const uint4*>(row + c0));
        if (live1) x.b = __ldcs(reinterpret_cast<const uint4*>(row + c1));
        return x;
    };
    auto store2 = [&](T* row, const TwoChunks& x) {
        if (live0) __stcs(reinterpret_cast<uint4*>(row + c0), x.a);
        if (live1) __stcs(reinterpret_cast<uint4*>(row + c1), x.b);
    };
    TwoChunks wq = {}, wk = {};
    if (a.q_weight) wq = load2(static_cast<const T*>(a.q_weight));
    if (a.k_weight) wk = load2(static_cast<const T*>(a.k_weight));

    // Round r of a token: one query head, one key head and one value head for each group.
    // Keys and values start at the groups that the queries leave free.
    const int hk0 = (group + kGroups - a.heads % kGroups) % kGroups;
    const int hv0 = (group + kGroups - (a.heads + a.kv_heads) % kGroups) % kGroups;
    const int rounds = max((a.heads + kGroups - 1) / kGroups, (a.kv_heads + kGroups - 1) / kGroups);
    TwoChunks q = {}, k = {}, v = {};
    // Values are read even where the slot says to skip them: the read does not wait for it.
    auto request = [&](int t, int r) {
        const int hq = group + r * kGroups, hk = hk0 + r * kGroups, hv = hv0 + r * kGroups;
        if (hq < a.heads) q = load2(static_cast<const T*>(a.q.p) + t * a.q.tok + hq * a.q.head);
        if (hk < a.kv_heads) k = load2(static_cast<const T*>(a.k.p) + t * a.k.tok + hk * a.k.head);
        if (hv < a.kv_heads && a.slots) v = load2(static_cast<const T*>(a.v.p) + t * a.v.tok + hv * a.v.head);
    };
    const int step = gridDim.x;
    int pos = a.positions[blockIdx.x];
    int64_t slot = a.slots ? a.slots[blockIdx.x] : -1;
    request(blockIdx.x, 0);
    for (int t = blockIdx.x; t < a.n_tokens; t += step) {
        Pairs cs, sn;  // of angles l * 8 .. l * 8 + 7
        if (turns_here) {
            const bool known = pos >= 0 && pos < a.n_positions;
            const float nan = __int_as_float(0x7fc00000);
            float4 x[2], y[2];
            x[0] = x[1] = y[0] = y[1] = make_float4(nan, nan, nan, nan);
            if (known) {
                const float* row = a.turns + (long long)pos * a.turned + l * 8;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    x[i] = __ldg(reinterpret_cast<const float4*>(row) + i);
                    y[i] = __ldg(reinterpret_cast<const float4*>(row + half) + i);
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                cs[2 * i] = pair(x[i].x, x[i].y); cs[2 * i + 1] = pair(x[i].z, x[i].w);
                sn[2 * i] = pair(y[i].x, y[i].y); sn[2 * i + 1] = pair(y[i].z, y[i].w);
            }
        }
        auto rotated = [&](const TwoChunks& in, const TwoChunks& weight, bool norm) {
            Pairs x, y;
            unpack_pairs<H>(in.a, x);
            unpack_pairs<H>(in.b, y);
            if (norm) {
                uint64_t s2 = 0, s3 = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s2 = fma2(x[i], x[i], s2);
                    s3 = fma2(y[i], y[i], s3);
                }
                const float2 s = halves(add2(s2, s3));
                float ss = s.x + s.y;
#pragma unroll
                for (int o = W / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o, W);
                const float inv = rsqrtf(fmaf(ss, inv_dim, a.eps));
                const uint64_t inv2 = pair(inv, inv);
                Pairs w;
                unpack_pairs<H>(weight.a, w);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = mul2(mul2(x[i], inv2), w[i]);
                unpack_pairs<H>(weight.b, w);
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = mul2(mul2(y[i], inv2), w[i]);
            }
            if (turns_here) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (PAIRS) {  // chunk a has angles 0 to 3, chunk b angles 4 to 7
                        const float2 u = halves(x[i]), w = halves(y[i]);
                        const float2 c_lo = halves(cs[i / 2]), s_lo = halves(sn[i / 2]);
                        const float2 c_hi = halves(cs[2 + i / 2]), s_hi = halves(sn[2 + i / 2]);
                        const float c = i & 1 ? c_lo.y : c_lo.x, s = i & 1 ? s_lo.y : s_lo.x;
                        const float e = i & 1 ? c_hi.y : c_hi.x, f = i & 1 ? s_hi.y : s_hi.x;
                        x[i] = pair(u.x * c - u.y * s, u.y * c + u.x * s);
                        y[i] = pair(w.x * e - w.y * f, w.y * e + w.x * f);
                    } else {
                        const uint64_t u = x[i], w = y[i];
                        y[i] = fma2(u, sn[i], mul2(w, cs[i]));
                        x[i] = fma2(w, mul2(sn[i], pair(-1.0f, -1.0f)), mul2(u, cs[i]));
                    }
                }
            }
            return TwoChunks{pack_pairs<H>(x), pack_pairs<H>(y)};
        };
        int64_t at = slot;
        if (at >= (a.n_pages << a.page_shift)) at = -1;
        const int64_t page = at >> a.page_shift, off = at & ((1 << a.page_shift) - 1);
        const int next = t + step;
        if (next < a.n_tokens) {
            pos = a.positions[next];
            if (a.slots) slot = a.slots[next];
        }
        for (int r = 0; r < rounds; ++r) {
            const TwoChunks q_now = q, k_now = k, v_now = v;
            if (r + 1 < rounds) request(t, r + 1);
            else if (next < a.n_tokens) request(next, 0);
            const int hq = group + r * kGroups, hk = hk0 + r * kGroups, hv = hv0 + r * kGroups;
            if (hv < a.kv_heads && at >= 0)  // values are copied as they are
                store2(static_cast<T*>(a.v_cache.p) + page * a.v_cache.page + off * a.v_cache.tok + hv * a.v_cache.head, v_now);
            if (hq < a.heads)  // the same for a whole group
                store2(static_cast<T*>(a.out_q) + ((long long)t * a.heads + hq) * a.dim,
                       rotated(q_now, wq, a.q_weight != nullptr));
            if (hk < a.kv_heads) {
                const TwoChunks y = rotated(k_now, wk, a.k_weight != nullptr);
                if (a.out_k) store2(static_cast<T*>(a.out_k) + ((long long)t * a.kv_heads + hk) * a.dim, y);
                if (at >= 0)
                    store2(static_cast<T*>(a.k_cache.p) + page * a.k_cache.page + off * a.k_cache.tok + hk * a.k_cache.head, y);
            }
        }
    }
}

template <class H, bool PAIRS>
void norm_rotate_width(const NormRotateArgs& a, cudaStream_t st) {
    const unsigned grid = (unsigned)std::min(a.n_tokens, 148 * 2 * 8);  // a few tokens a block where there are many
    if (a.dim <= 64) norm_rotate_kernel<H, 4, PAIRS><<<grid, kRotThreads, 0, st>>>(a);
    else if (a.dim <= 128) norm_rotate_kernel<H, 8, PAIRS><<<grid, kRotThreads, 0, st>>>(a);
    else norm_rotate_kernel<H, 16, PAIRS><<<grid, kRotThreads, 0, st>>>(a);
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

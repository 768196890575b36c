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
// One launch: every block scans all requests itself (two int32 loads each, from L2; a
// thread takes a run of neighbouring ones), so no block waits for another; then each block
// fills its share of tokens and table rows.  What the tokens need of a request is in shared
// memory by then, and a token's new page is taken from the free list directly, never from a
// table entry that another block may still be writing.  Bound by the latency of its chain of
// loads: lengths, then pages, then the stores.  Measured: 64 requests of one token 4.7 us,
// 1,500 prompts with 778,000 tokens (9.6 MB read and written) 10.4 us.
// ---------------------------------------------------------------------------------
constexpr int kScanThreads = 512, kRun = 4;  // tokens a thread takes at once

__device__ __forceinline__ int clamp_int(long long v) {
    return (int)(v < 0 ? 0 : (v > 0x7fffffffLL ? 0x7fffffffLL : v));
}

__global__ void __launch_bounds__(kScanThreads) page_tables_kernel(const __grid_constant__ PageTablesArgs a) {
    extern __shared__ int smem[];
    const int n = a.n_requests;
    int* s_start = smem;              // [n + 1] first token of each request
    int* s_first = smem + n + 1;      // [n + 1] first free-list entry of each request
    int* s_old = smem + 2 * (n + 1);  // [n] tokens held
    __shared__ long long s_warp[2][kScanThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int page = 1 << a.page_shift;

    // Exclusive scans of the new tokens and new pages; sums in 64 bits.
    const int per = (n + kScanThreads - 1) / kScanThreads, r0 = min(tid * per, n), r1 = min(r0 + per, n);
    long long sum_t = 0, sum_p = 0;
#pragma unroll 4
    for (int r = r0; r < r1; ++r) {
        const long long old = max(__ldg(a.cached + r), 0), fresh = max(__ldg(a.fresh + r), 0);
        s_old[r] = (int)old;
        s_start[r] = clamp_int(sum_t);  // within the run, for now
        s_first[r] = clamp_int(sum_p);
        sum_t += fresh;
        sum_p += ((old + fresh + page - 1) >> a.page_shift) - ((old + page - 1) >> a.page_shift);
        if (blockIdx.x == 0) a.lengths[r] = clamp_int(old + fresh);
    }
    long long it = sum_t, ip = sum_p;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long ut = __shfl_up_sync(0xffffffffu, it, o), up = __shfl_up_sync(0xffffffffu, ip, o);
        if (lane >= o) { it += ut; ip += up; }
    }
    if (lane == 31) { s_warp[0][warp] = it; s_warp[1][warp] = ip; }
    __syncthreads();
    long long bt = it - sum_t, bp = ip - sum_p, all_t = 0, all_p = 0;
#pragma unroll
    for (int w = 0; w < kScanThreads / 32; ++w) {
        if (w < warp) { bt += s_warp[0][w]; bp += s_warp[1][w]; }
        all_t += s_warp[0][w];
        all_p += s_warp[1][w];
    }
    for (int r = r0; r < r1; ++r) {
        s_start[r] = clamp_int(bt + s_start[r]);
        s_first[r] = clamp_int(bp + s_first[r]);
        if (blockIdx.x == 0) a.starts[r] = s_start[r];
    }
    if (tid == 0) {
        s_start[n] = clamp_int(all_t);
        s_first[n] = clamp_int(all_p);
        if (blockIdx.x == 0) {
            a.starts[n] = s_start[n];
            a.used[0] = s_first[n];
        }
    }
    __syncthreads();

    // New table entries: one warp a request.
    for (int r = blockIdx.x * (kScanThreads / 32) + warp; r < n; r += gridDim.x * (kScanThreads / 32)) {
        const long long had = ((long long)s_old[r] + page - 1) >> a.page_shift;
        const int first = s_first[r], more = s_first[r + 1] - first;
        for (int i = lane; i < more; i += 32) {
            if (had + i >= a.table_width) break;
            const long long f = (long long)first + i;
            a.table[(long long)r * a.table_stride + had + i] = f < a.n_free ? a.free_pages[f] : -1;
        }
    }

    // Tokens: a run of kRun consecutive ones a thread, one search for the first of them.
    for (long long t0 = ((long long)blockIdx.x * kScanThreads + tid) * kRun; t0 < a.n_tokens;
         t0 += (long long)gridDim.x * kScanThreads * kRun) {
        int lo = 0, hi = n;  // the last request whose start is <= t0
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s_start[mid] <= t0) lo = mid; else hi = mid;
        }
        int r = lo, pos[kRun];
        long long from[kRun];  // where the page's number stands: an index of the table, or -2 - one of the free list
        int off[kRun];
#pragma unroll
        for (int i = 0; i < kRun; ++i) {
            const long long t = t0 + i;
            while (r < n && s_start[r + 1] <= t) ++r;
            pos[i] = 0;
            from[i] = -1;
            off[i] = 0;
            if (r < n) {
                const long long old = s_old[r], at = old + t - s_start[r];
                const long long col = at >> a.page_shift, had = (old + page - 1) >> a.page_shift;
                const long long f = s_first[r] + col - had;
                if (col < a.table_width) {
                    if (col < had) from[i] = (long long)r * a.table_stride + col;
                    else if (f < a.n_free) from[i] = -2 - f;
                }
                off[i] = (int)(at & (page - 1));
                pos[i] = clamp_int(at + a.base);
            }
        }
        int32_t pg[kRun];
#pragma unroll
        for (int i = 0; i < kRun; ++i)
            pg[i] = from[i] >= 0 ? a.table[from[i]] : (from[i] < -1 ? __ldg(a.free_pages - 2 - from[i]) : -1);
        int64_t slot[kRun];
#pragma unroll
        for (int i = 0; i < kRun; ++i) slot[i] = pg[i] >= 0 ? ((int64_t)pg[i] << a.page_shift) + off[i] : -1;
        if (t0 + kRun <= a.n_tokens && a.wide) {
#pragma unroll
            for (int i = 0; i < kRun; i += 4)
                *reinterpret_cast<int4*>(a.positions + t0 + i) = make_int4(pos[i], pos[i + 1], pos[i + 2], pos[i + 3]);
#pragma unroll
            for (int i = 0; i < kRun; i += 2)
                *reinterpret_cast<longlong2*>(a.slots + t0 + i) = make_longlong2(slot[i], slot[i + 1]);
        } else {
            for (int i = 0; i < kRun && t0 + i < a.n_tokens; ++i) {
                a.positions[t0 + i] = pos[i];
                a.slots[t0 + i] = slot[i];
            }
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
// need no exchange.  Groups step over the (token, head) rows of the batch, neighbouring
// groups on neighbouring heads, and request the next row before the current one is used.
// Measured (bf16, 32 + 8 heads of 128, 50,000 tokens, 1.36 GB with the cache): 249 us, 5.5 TB/s
// (264 among calls whose inputs change); 33 tokens: 2.4 us.
// ---------------------------------------------------------------------------------
constexpr int kRotThreads = 256, kRotBlocks = 3;  // threads a block, blocks an SM

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
__global__ void __launch_bounds__(kRotThreads, kRotBlocks) norm_rotate_kernel(const __grid_constant__ NormRotateArgs a) {
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
    // Rows of a token: query heads, key heads, value heads.
    const int qk = a.heads + a.kv_heads, units = a.slots ? qk + a.kv_heads : qk;
    const long long first = (long long)blockIdx.x * kGroups + group, stride = (long long)gridDim.x * kGroups;
    unsigned t = (unsigned)(first / units);  // may pass 2^31 by a stride
    int u = (int)(first % units);
    const int dt = (int)(stride / units), du = (int)(stride % units);
    TwoChunks next = {};
    int next_pos = 0;
    int64_t next_slot = -1;
    const unsigned n_tokens = (unsigned)a.n_tokens;
    auto request = [&](unsigned t, int u) {
        if (t >= n_tokens) return;
        next_pos = a.positions[t];
        if (a.slots && u >= a.heads) next_slot = a.slots[t];
        const HeadsView& x = u < a.heads ? a.q : (u < qk ? a.k : a.v);
        const int h = u < a.heads ? u : (u < qk ? u - a.heads : u - qk);
        next = load2(static_cast<const T*>(x.p) + t * x.tok + h * x.head);
    };
    request(t, u);
    while (t < n_tokens) {
        const TwoChunks in = next;
        const unsigned here_t = t;
        const int pos = next_pos, here_u = u;
        int64_t at = next_slot;
        // Cosines and sines of angles l * 8 .. l * 8 + 7
        float4 cs[2], sn[2];
        const float nan = __int_as_float(0x7fc00000);
        cs[0] = cs[1] = sn[0] = sn[1] = make_float4(nan, nan, nan, nan);
        if (turns_here && here_u < qk && pos >= 0 && pos < a.n_positions) {
            const float4* row = reinterpret_cast<const float4*>(a.turns + (long long)pos * a.turned + l * 8);
            cs[0] = __ldg(row);
            cs[1] = __ldg(row + 1);
            sn[0] = __ldg(row + half / 4);
            sn[1] = __ldg(row + half / 4 + 1);
        }
        t += dt;
        u += du;
        if (u >= units) {
            u -= units;
            ++t;
        }
        request(t, u);
        if (at >= (a.n_pages << a.page_shift)) at = -1;
        const int64_t page = at >> a.page_shift, off = at & ((1 << a.page_shift) - 1);
        if (here_u >= qk) {  // values are copied as they are
            if (at >= 0)
                store2(static_cast<T*>(a.v_cache.p) + page * a.v_cache.page + off * a.v_cache.tok + (here_u - qk) * a.v_cache.head, in);
            continue;
        }
        const bool is_q = here_u < a.heads;
        const T* weight = static_cast<const T*>(is_q ? a.q_weight : a.k_weight);
        Pairs x, y;
        unpack_pairs<H>(in.a, x);
        unpack_pairs<H>(in.b, y);
        if (weight) {
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
            uint4 wa = make_uint4(0, 0, 0, 0), wb = wa;
            if (live0) wa = __ldg(reinterpret_cast<const uint4*>(weight + c0));
            if (live1) wb = __ldg(reinterpret_cast<const uint4*>(weight + c1));
            Pairs w;
            unpack_pairs<H>(wa, w);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = mul2(mul2(x[i], inv2), w[i]);
            unpack_pairs<H>(wb, w);
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i] = mul2(mul2(y[i], inv2), w[i]);
        }
        if (turns_here) {
            const float c[8] = {cs[0].x, cs[0].y, cs[0].z, cs[0].w, cs[1].x, cs[1].y, cs[1].z, cs[1].w};
            const float s[8] = {sn[0].x, sn[0].y, sn[0].z, sn[0].w, sn[1].x, sn[1].y, sn[1].z, sn[1].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (PAIRS) {  // chunk a has angles 0 to 3, chunk b angles 4 to 7
                    const float2 f = halves(x[i]), g = halves(y[i]);
                    x[i] = pair(f.x * c[i] - f.y * s[i], f.y * c[i] + f.x * s[i]);
                    y[i] = pair(g.x * c[4 + i] - g.y * s[4 + i], g.y * c[4 + i] + g.x * s[4 + i]);
                } else {
                    const uint64_t f = x[i], g = y[i], c2 = pair(c[2 * i], c[2 * i + 1]), s2 = pair(s[2 * i], s[2 * i + 1]);
                    y[i] = fma2(f, s2, mul2(g, c2));
                    x[i] = fma2(g, pair(-s[2 * i], -s[2 * i + 1]), mul2(f, c2));
                }
            }
        }
        const TwoChunks out{pack_pairs<H>(x), pack_pairs<H>(y)};
        if (is_q) {
            store2(static_cast<T*>(a.out_q) + ((long long)here_t * a.heads + here_u) * a.dim, out);
            continue;
        }
        const int h = here_u - a.heads;
        if (a.out_k) store2(static_cast<T*>(a.out_k) + ((long long)here_t * a.kv_heads + h) * a.dim, out);
        if (at >= 0)
            store2(static_cast<T*>(a.k_cache.p) + page * a.k_cache.page + off * a.k_cache.tok + h * a.k_cache.head, out);
    }
}

template <class H, bool PAIRS>
void norm_rotate_width(const NormRotateArgs& a, cudaStream_t st) {
    const long long rows = (long long)a.n_tokens * (a.heads + (a.slots ? 2 : 1) * a.kv_heads);
    auto launch = [&](auto* kernel, int width) {
        const long long blocks = (rows * width + kRotThreads - 1) / kRotThreads;
        kernel<<<(unsigned)std::min<long long>(blocks, 148 * kRotBlocks * 4), kRotThreads, 0, st>>>(a);
    };
    if (a.dim <= 64) launch(norm_rotate_kernel<H, 4, PAIRS>, 4);
    else if (a.dim <= 128) launch(norm_rotate_kernel<H, 8, PAIRS>, 8);
    else launch(norm_rotate_kernel<H, 16, PAIRS>, 16);
    VGPU_LAUNCH("norm_rotate_kernel");
}

}  // namespace

void launch_page_tables(const PageTablesArgs& a, cudaStream_t st) {
    const size_t smem = 3 * ((size_t)a.n_requests + 1) * sizeof(int);
    // To the most that any call needs, whatever this one does: calls of other threads, and what the
    // kernel has of shared memory besides, then do not matter.
    static std::atomic<uint64_t> devices{0};
    opt_in(devices, page_tables_kernel, (int)(3 * (kMaxTableRequests + 1) * sizeof(int)), [] {});
    const long long per_block = kScanThreads * kRun;
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

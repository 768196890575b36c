// Attention of short prompts: the same rows and masks as attn_tile.cuh, in small blocks.
//
// A prompt of a few hundred tokens gives a tensor-memory tile little to overlap: setting it
// up and draining it costs an SM that holds one block more than the products do.  Here a block is four warps of
// 16 rows (64 / group tokens with the query heads of one key head), takes the keys 64 at a
// time through two shared-memory stages filled by asynchronous copies, multiplies with
// m16n8k16 steps of each warp, and an SM holds three or more such blocks.
//
// Rows of the stages are 16-byte chunks XORed with the row, so that the eight rows of a
// matrix load lie in different banks.  Softmax as in attn_tile.cuh: one pass, running maximum
// and sum in 32 bits, P rounded to the data's type for the second product, which takes both
// operands in that type.  Value rows past
// the last key are filled with zeros by the copy, and non-finite values of tokens that not every
// row of the block sees (the diagonal tiles') are taken out in shared memory and added back by
// the rows that do see them.
//
// Bound by the latency of one block: loads, two products and the softmax of a few key tiles.
// Measured: three prompts of 92 tokens in all (32 + 8 heads of 128, causal): 6.3 us; both
// kernels side by side at other sizes stand where one of them is chosen.
#pragma once

#include "attn_tile.cuh"

namespace vgpu {
namespace attn {

constexpr int kShortRows = 64, kShortKeys = 64, kShortThreads = 128;

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

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
// 16 bytes to shared memory, zeros where `some` is false.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool some) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(some ? 16 : 0) : "memory");
}

template <class H, int D>
__global__ void __launch_bounds__(kShortThreads, D == 64 ? 4 : 3) attn_short_kernel(const __grid_constant__ TileParams p) {
    using T = typename H::type;
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int kChunks = D / 8, kRowBytes = D * 2, kTileBytes = kShortKeys * kRowBytes;
    __shared__ Work s_work;
    __shared__ int s_leak;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int kh = blockIdx.x % p.kv_heads;
    if (warp == 0) {
        int near = -1;
        const Work w = find_work(p, blockIdx.x / p.kv_heads, lane, p.tile_tokens, near);
        if (lane == 0) {
            s_work = w;
            s_leak = 0;
        }
    }
    __syncthreads();
    const Work w = s_work;
    const int tokens = min(w.tokens, p.tile_tokens);
    if (tokens <= 0) return;
    const int last = min(w.len_k, w.first_lim + w.step * (tokens - 1));  // keys the last row sees
    const int n = (max(last, 0) + kShortKeys - 1) / kShortKeys;
    const int min_lim = min(max(w.first_lim, 0), w.len_k);  // keys that every row sees

    // A thread copies the same 16-byte chunk of every kRowStep-th row; rows past the last key
    // are filled with zeros (nothing is read for them).
    const uint32_t s_kv = tc::smem_u32(smem);
    constexpr int kRowStep = kShortThreads / kChunks;
    const int row0 = tid / kChunks, chunk = tid % kChunks;
    const uint32_t at0 = row0 * kRowBytes + ((chunk ^ (row0 & 7)) << 4);  // kRowStep is a multiple of 8
    const bool here = chunk * 8 < p.dim;
    const T* k_at = static_cast<const T*>(p.k.p) + (w.k0 + row0) * p.k.tok + kh * p.k.head + (here ? chunk * 8 : 0);
    const T* v_at = static_cast<const T*>(p.v.p) + (w.k0 + row0) * p.v.tok + kh * p.v.head + (here ? chunk * 8 : 0);
    const long long k_step = kRowStep * p.k.tok, v_step = kRowStep * p.v.tok;
    auto request = [&](int j) {
        const uint32_t dst = s_kv + (j & 1) * 2 * kTileBytes + at0;
        const int left = here ? w.len_k - j * kShortKeys - row0 : 0;
#pragma unroll
        for (int i = 0; i < kShortKeys / kRowStep; ++i) {
            const bool some = i * kRowStep < left;
            copy16(dst + i * kRowStep * kRowBytes, some ? k_at : p.k.p, some);
            copy16(dst + kTileBytes + i * kRowStep * kRowBytes, some ? v_at : p.v.p, some);
            k_at += k_step;
            v_at += v_step;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if (n > 0) request(0);

    // Rows g and g + 8 of the warp's 16.
    int lim[2];
    long long out_row[2];
    bool valid[2];
    const T* q_row[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int row = warp * 16 + g + 8 * h, tok = row / p.group, head = kh * p.group + row - tok * p.group;
        valid[h] = tok < tokens;
        lim[h] = valid[h] ? min(max(w.first_lim + w.step * tok, 0), w.len_k) : 0;
        out_row[h] = (long long)(w.q0 + tok) * p.heads + head;
        q_row[h] = static_cast<const T*>(p.q.p) + (w.q0 + (valid[h] ? tok : 0)) * p.q.tok + (valid[h] ? head : kh * p.group) * p.q.head;
    }
    uint32_t qa[D / 16][4];
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int d = k * 16 + 2 * t + (i >> 1) * 8;
            qa[k][i] = d < p.dim ? *reinterpret_cast<const uint32_t*>(q_row[i & 1] + d) : 0u;
        }

    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    // Matrix loads: lane's row and chunk within a 16 x 16 piece.
    const int r16 = (lane & 7) + ((lane >> 4) << 3), c16 = (lane >> 3) & 1;    // keys: rows 0-7, 8-15 by lane / 16
    const int rv = (lane & 7) + (((lane >> 3) & 1) << 3), cv = lane >> 4;      // values: rows by lane / 8, columns by lane / 16
    for (int j = 0; j < n; ++j) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();
        if (j + 1 < n) request(j + 1);
        const uint32_t sk = s_kv + (j & 1) * 2 * kTileBytes, sv = sk + kTileBytes;
        const int key = j * kShortKeys;
        const bool guarded = w.step && key + kShortKeys > min_lim;  // value rows that some row must not see
        if (guarded) {
            const int from = max(min_lim - key, 0), end = min(w.len_k - key, kShortKeys);
            for (int i = from * kChunks + tid; i < end * kChunks; i += kShortThreads) {
                uint4* const at = reinterpret_cast<uint4*>(smem + (j & 1) * 2 * kTileBytes + kTileBytes + i * 16);
                if (not_finite<H>(*at)) {
                    *at = finite_part<H>(*at);
                    s_leak = 1;
                }
            }
        }
        float s[kShortKeys / 8][4];
#pragma unroll
        for (int i = 0; i < kShortKeys / 8; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
            for (int i = 0; i < kShortKeys / 16; ++i) {
                uint32_t b[4];
                const int row = i * 16 + r16;
                ldsm4(b, sk + row * kRowBytes + (((2 * k + c16) ^ (row & 7)) << 4));
                mma16816<H>(s[2 * i], qa[k][0], qa[k][1], qa[k][2], qa[k][3], b[0], b[1]);
                mma16816<H>(s[2 * i + 1], qa[k][0], qa[k][1], qa[k][2], qa[k][3], b[2], b[3]);
            }
        if (key + kShortKeys > min_lim) {
#pragma unroll
            for (int i = 0; i < kShortKeys / 8; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (key + i * 8 + 2 * t + (c & 1) >= lim[c >> 1]) s[i][c] = -INFINITY;
        }
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < kShortKeys / 8; ++i) {
            top[0] = max3(top[0], s[i][0], s[i][1]);
            top[1] = max3(top[1], s[i][2], s[i][3]);
        }
        float f[2], ref[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float a = __shfl_xor_sync(0xffffffffu, top[h], 1);
            const float b = max3(top[h], a, a), c = __shfl_xor_sync(0xffffffffu, b, 2);
            float up = max3(m[h], b * p.scale_log2, c * p.scale_log2);
            if (up == INFINITY) up = __int_as_float(0x7fc00000);
            f[h] = up == m[h] ? 1.0f : ex2(m[h] - up);
            m[h] = up;
            ref[h] = up == -INFINITY ? 0.0f : up;
            l[h] *= f[h];
        }
        if (__any_sync(0xffffffffu, f[0] != 1.0f || f[1] != 1.0f)) {
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
                o[i][0] *= f[0];
                o[i][1] *= f[0];
                o[i][2] *= f[1];
                o[i][3] *= f[1];
            }
        }
        if (guarded) __syncthreads();  // the values are as they are multiplied
#pragma unroll
        for (int k = 0; k < kShortKeys / 16; ++k) {
            uint32_t pa[4];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float* x = s[2 * k + e];
                const float p0 = ex2(fmaf(x[0], p.scale_log2, -ref[0])), p1 = ex2(fmaf(x[1], p.scale_log2, -ref[0]));
                const float p2 = ex2(fmaf(x[2], p.scale_log2, -ref[1])), p3 = ex2(fmaf(x[3], p.scale_log2, -ref[1]));
                l[0] += p0 + p1;
                l[1] += p2 + p3;
                pa[2 * e] = H::pack(p0, p1);
                pa[2 * e + 1] = H::pack(p2, p3);
            }
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                uint32_t b[4];
                const int row = k * 16 + rv;
                ldsm4_t(b, sv + row * kRowBytes + (((2 * i + cv) ^ (row & 7)) << 4));
                mma16816<H>(o[2 * i], pa[0], pa[1], pa[2], pa[3], b[0], b[1]);
                mma16816<H>(o[2 * i + 1], pa[0], pa[1], pa[2], pa[3], b[2], b[3]);
            }
        }
    }
    __syncthreads();
    if (*static_cast<volatile int*>(&s_leak) != 0) {
        // The rows see at most 64 keys that not all of them see; a lane looks through one.
        const T* const v = static_cast<const T*>(p.v.p) + w.k0 * p.v.tok + kh * p.v.head;
        const int until = __reduce_max_sync(0xffffffffu, max(lim[0], lim[1]));
#pragma unroll 1
        for (int first = min_lim; first < until; first += 32) {
            bool odd = false;
            if (first + lane < until)
#pragma unroll 4
                for (int c = 0; c < p.dim; c += 8)
                    odd |= not_finite<H>(__ldg(reinterpret_cast<const uint4*>(v + (first + lane) * p.v.tok + c)));
#pragma unroll 1
            for (unsigned some = __ballot_sync(0xffffffffu, odd); some; some &= some - 1) {
                const int key = first + __ffs(some) - 1;
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    if (i * 8 >= p.dim) break;
                    const float2 x = H::unpack(finite_part<H>(
                        __ldg(reinterpret_cast<const uint32_t*>(v + key * p.v.tok + i * 8 + 2 * t)), true));
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (key >= lim[h]) continue;
                        o[i][2 * h] += x.x;
                        o[i][2 * h + 1] += x.y;
                    }
                }
            }
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        if (!valid[h]) continue;
        const float inv = l[h] > 0.0f ? 1.0f / l[h] : (l[h] == 0.0f ? 0.0f : l[h]);
        // through the warp's own part of the stages: whole rows are stored below
        const int r = warp * 16 + g + 8 * h;
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
            const float x = l[h] == 0.0f ? 0.0f : o[i][2 * h] * inv, y = l[h] == 0.0f ? 0.0f : o[i][2 * h + 1] * inv;
            *reinterpret_cast<uint32_t*>(smem + r * kRowBytes + ((i ^ (r & 7)) << 4) + t * 4) = H::pack(x, y);
        }
        if (p.lse && t == 0) p.lse[out_row[h]] = (m[h] + log2f(l[h])) * 0.6931471805599453f;
    }
    __syncwarp();
#pragma unroll
    for (int e = lane; e < 16 * kChunks; e += 32) {
        const int r = warp * 16 + e / kChunks, c = e % kChunks, tok = r / p.group, head = kh * p.group + r - tok * p.group;
        if (tok < tokens && c * 8 < p.dim)
            *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + ((long long)(w.q0 + tok) * p.heads + head) * p.dim + c * 8) =
                *reinterpret_cast<const uint4*>(smem + r * kRowBytes + ((c ^ (r & 7)) << 4));
    }
}

template <int D>
constexpr int short_smem_bytes() {
    return 4 * kShortKeys * D * 2;
}

}  // namespace attn
}  // namespace vgpu

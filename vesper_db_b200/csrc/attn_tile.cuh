// Attention of query tiles on the tensor cores (tcgen05): the kernel that prompts and the
// shared prefix both run.
//
//   S = Q K^T, P = exp2(scale' S - m) with scale' = scale log2(e), O = sum P V / sum P,
// one pass over the keys with a running maximum m and sum l of each row in 32 bits.
//
// A tile is 128 rows: floor(128 / group) tokens with the `group` query heads of one key
// head each, so that one key tile serves the whole group.  A block holds two query tiles
// and takes the keys 128 at a time:
//   * warp 8 copies Q, then K and V tiles by TMA into a ring of shared-memory slots;
//   * warps 9 and 10 issue the products of tile 0 and tile 1: S_t = Q_t K^T (both operands
//     from shared memory) and O_t += P_t V (P from tensor memory);
//   * warps 0-3 and 4-7 hold one row a thread of tile 0 and tile 1: they read S, keep m and
//     l, and write P over S as 16-bit values, in two halves, so that the first half's
//     product runs while the second half is made;
//   * warps 12 to 15 clean the value tiles that hold keys some row must not see.
// The two query tiles are independent of each other: while one is in the tensor cores the
// other is in the exponentials.  Tensor memory: S0, S1 (128 columns each), O0, O1.
//
// What bounds it: a pair of tiles takes 2,048 cycles in the tensor cores (heads of 128), as
// many in the special-function units (32,768 exponentials, 16 a cycle) and as many in
// shared memory (256 KB read and written, 128 bytes a cycle).  Making a quarter or three
// eighths of the exponentials by a polynomial on the FMA units instead cost 1 to 7 %: the
// issue slots it takes are worth more than the special-function cycles it frees.
//
// m only moves when a row's maximum has grown by more than 2^8: until then P may reach 2^8,
// which both types hold at full relative precision, and O need not be rescaled.
//
// Masked scores become -inf by selection, so what unseen keys hold does not matter; unseen
// values meet P = 0, and 0 * NaN is NaN: value rows past the last key are zeroed in shared
// memory, and where a later token of the same prompt holds a non-finite value (checked on
// the diagonal tiles) the block recomputes its rows one key at a time.
//
// Every wait is bounded; a block whose wait ran out issues no further work, gives NaN rows
// and frees its tensor memory.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "attention.cuh"
#include "common.cuh"
#include "half_types.cuh"
#include "tc_common.cuh"

namespace vgpu {
namespace attn {

constexpr int kRows = 128;     // query rows of a tile
constexpr int kKeys = 128;     // keys of a tile
constexpr int kThreads = 512;  // two softmax warpgroups, two of service warps
constexpr int kSlots = 4;      // K and V tiles in flight
constexpr float kGrow = 8.0f;  // log2 of how far P may pass 1 before O is rescaled
constexpr int kSoftmaxRegs = 208, kServiceRegs = 40;  // 256 * 208 + 256 * 40 <= 512 * 128

struct TileParams {
    CUtensorMap mq, mk, mv;
    int heads, kv_heads, group, dim;
    int tile_tokens;  // tokens of one query tile
    int n_q, n_k;     // rows of q; rows of k and v, or keys of the prefix
    // Packed prompts: requests' first rows.  Shared prefix: one request of all rows.
    const int32_t* starts;
    const int32_t* starts_k;
    int n_requests;
    bool causal;
    // Paged keys: pages of the prefix.
    const int32_t* pages;
    int page_shift;
    // Packed keys again, for the rows recomputed one key at a time.
    HeadsView q, k, v;
    float scale_log2;
    int splits;
    bool part;       // results of each split for a later join, in 32 bits
    void* out;       // otherwise: [n_q, heads, dim]
    float* lse;
    float* part_o;   // [splits, n_q * heads, dim], and their log2-sum-exp
    float* part_lse;
};

template <int D>
constexpr int smem_bytes() {
    return 2 * kRows * D * 2 + kSlots * kKeys * D * 2 + 1024 + 512;
}

// Bounded wait for the barrier's phase; false when it ran out (a tile takes microseconds).
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity) {
    const uint32_t a = tc::smem_u32(bar);
    for (uint32_t i = 0; i < (1u << 20); ++i) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(a), "r"(parity)
            : "memory");
        if (done) return true;
    }
    return false;
}

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Maximum of three; NaN if one of them is.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

__device__ __forceinline__ void tma4(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(dst), "l"(map), "r"(tc::smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
        : "memory");
}

// Operand whose 64-value blocks run along the output dimension (values: rows are keys),
// 128-byte swizzle: 8-key groups 1024 bytes apart, 64-value blocks `block_bytes` apart.
__device__ __forceinline__ uint64_t values_desc(uint32_t saddr, uint32_t block_bytes) {
    uint64_t d = (uint64_t)((saddr >> 4) & 0x3FFFu);
    d |= (uint64_t)(block_bytes >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

// Issued by one elected lane of a converged warp: the election inside the statement keeps
// the operands in uniform registers.  (Under `if (lane == 0)` each product took 120 cycles
// to issue, twice what it takes to run.)
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred e, p;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred e, p;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(tc::smem_u32(bar))
        : "memory");
}

// What a block works on.
struct Work {
    int q0;        // first row of q of the block's first tile
    int tokens;    // rows of the request from there on (those past the block's tiles do not count)
    int k0, len_k; // first key row, keys of the request
    int first_lim; // keys that the first of these rows sees; each later one sees `step` more
    int step;
    int split;
};

// Piece `idx` of the packed requests, each cut into `span` tokens.  Run by one whole warp;
// tokens <= 0: no such piece.  Request b's pieces have the numbers from starts[b] / span + b
// on, which leaves room for each (some numbers stay unused) and can be searched without
// adding up lengths: 32 candidates a step.  Rows before the first and after the last request
// are requests without keys.  Last pieces come first: the rows of a causal prompt's end see
// the most keys.
__device__ __forceinline__ Work find_work(const TileParams& p, int idx, int lane, int span) {
    const int n = p.n_requests + 2;
    auto bound = [&](int b) {  // first row of request b
        if (b == 0) return 0;
        if (b >= n) return p.n_q;
        return min(max(p.starts[b - 1], 0), p.n_q);
    };
    const int want = p.n_q / span + n - 1 - idx;
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, c = lo + (lane + 1) * step;
        const bool before = c < hi && bound(c) / span + c <= want;
        lo += __popc(__ballot_sync(0xffffffffu, before)) * step;
        hi = min(hi, lo + step);
    }
    Work w{};
    const int q0 = bound(lo), len_q = bound(lo + 1) - q0, tok = (want - q0 / span - lo) * span;
    w.q0 = q0 + tok;
    w.tokens = tok >= 0 ? len_q - tok : 0;
    int k0 = 0, k1 = 0;
    if (lo > 0 && lo <= p.n_requests) {
        k0 = min(max(p.starts_k[lo - 1], 0), p.n_k);
        k1 = min(max(p.starts_k[lo], k0), p.n_k);
    }
    w.k0 = k0;
    w.len_k = k1 - k0;
    w.step = p.causal ? 1 : 0;
    w.first_lim = p.causal ? tok + 1 + w.len_k - len_q : w.len_k;
    return w;
}

template <class H>
__device__ __forceinline__ bool not_finite(uint4 u) {
    constexpr uint32_t lo = sizeof(H) && std::is_same<H, Bf16>::value ? 0x7f80u : 0x7c00u, hi = lo << 16;
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) bad |= (w[i] & lo) == lo || (w[i] & hi) == hi;
    return bad;
}

template <class H, int D, bool PAGED>
__global__ void __launch_bounds__(kThreads, 1) attn_tile_kernel(const __grid_constant__ TileParams p) {
    extern __shared__ uint8_t smem_raw[];
    constexpr int kHalves = D / 64, kHalfBytes = kKeys * 128, kTileBytes = kHalves * kHalfBytes;
    const uint32_t raw = tc::smem_u32(smem_raw), base = (raw + 1023) & ~1023u;
    uint8_t* const smem = smem_raw + (base - raw);
    const uint32_t s_q = base, s_kv = base + 2 * kTileBytes;
    uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + (2 + kSlots) * kTileBytes);
    uint64_t* const q_full = bars;                // [2]
    uint64_t* const kv_full = bars + 2;           // [kSlots]
    uint64_t* const kv_empty = kv_full + kSlots;  // [kSlots]
    uint64_t* const s_full = kv_empty + kSlots;   // [2]
    uint64_t* const p_full = s_full + 2;          // [2][2]: tile, half of the keys
    uint64_t* const turn = p_full + 4;            // [2]
    uint64_t* const o_full = turn + 2;            // [2]
    uint64_t* const drained = o_full + 2;         // [2]
    uint64_t* const clean = drained + 2;
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(clean + 1);
    int* const s_leak = reinterpret_cast<int*>(tmem_slot + 1);
    Work* const s_work = reinterpret_cast<Work*>(tmem_slot + 2);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // The own pages' kernel may be queued behind this one and does not depend on it.
    if (PAGED) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    int block = blockIdx.x;
    const int kh = block % p.kv_heads;
    block /= p.kv_heads;
    const int split = block % p.splits;
    block /= p.splits;

    if (warp == 0) {
        Work w{};
        if (PAGED) {  // every row sees the whole prefix
            w.q0 = block * 2 * p.tile_tokens;
            w.tokens = p.n_q - w.q0;
            w.len_k = w.first_lim = p.n_k;
        } else {
            w = find_work(p, block, lane, 2 * p.tile_tokens);
        }
        w.split = split;
        if (lane == 0) *s_work = w;
    } else if (warp == 9) {
        if (lane == 0) {
            for (int i = 0; i < 2; ++i) {
                tc::mbar_init(&q_full[i], 1);
                tc::mbar_init(&s_full[i], 1);
                tc::mbar_init(&p_full[2 * i], 128);
                tc::mbar_init(&p_full[2 * i + 1], 128);
                tc::mbar_init(&turn[i], 1);
                tc::mbar_init(&o_full[i], 1);
                tc::mbar_init(&drained[i], 1);
            }
            for (int i = 0; i < kSlots; ++i) {
                tc::mbar_init(&kv_full[i], 1);
                tc::mbar_init(&kv_empty[i], 2);  // both warps of products
            }
            tc::mbar_init(clean, 4);
            *s_leak = 0;
            tc::mbar_init_fence();
        }
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(tmem_slot)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    const Work w = *s_work;

    // Key tiles of each query tile in this split: [j0, j0 + n_t).
    const int tt = p.tile_tokens;
    int tok[2], nt[2];  // indexed by constants only: they stay in registers
    const int all = (w.len_k + kKeys - 1) / kKeys, per = (all + p.splits - 1) / p.splits, j0 = w.split * per;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        tok[t] = min(max(w.tokens - t * tt, 0), tt);
        const int last = min(w.len_k, w.first_lim + w.step * (t * tt + tok[t] - 1));  // keys its last row sees
        const int tiles = tok[t] > 0 ? (max(last, 0) + kKeys - 1) / kKeys : 0;
        nt[t] = min(max(tiles - j0, 0), per);
    }
    const int n = max(nt[0], nt[1]);
    // From this key on some valid row of the block does not see the keys.
    const int min_lim = min(max(w.first_lim, 0), w.len_k);
    auto guarded_tile = [&](int j) { return (j0 + j + 1) * kKeys > min_lim; };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kServiceRegs));
        if (warp == 8) {
            // ---------------------------------------------------------------- copies
            if (n > 0) {
                if (lane == 0) {
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (nt[t] == 0) continue;
                        const uint32_t rows = (uint32_t)(tt * p.group);
                        tc::mbar_expect_tx(&q_full[t], rows * 128 * kHalves);
                        for (int h = 0; h < kHalves; ++h)
                            tma4(s_q + t * kTileBytes + h * kHalfBytes, &p.mq, h * 64, 0, kh, w.q0 + t * tt, &q_full[t]);
                    }
                }
                bool ok = true;
                int i = 0;
                for (; i < 2 * n; ++i) {  // K, V, K, V, ...
                    const int slot = i % kSlots, round = i / kSlots, key = (j0 + (i >> 1)) * kKeys;
                    if (round > 0) ok = mbar_wait(&kv_empty[slot], (round - 1) & 1);
                    if (!ok) break;
                    const CUtensorMap* map = (i & 1) ? &p.mv : &p.mk;
                    const uint32_t dst = s_kv + slot * kTileBytes;
                    if (!PAGED) {
                        if (lane == 0) {
                            tc::mbar_expect_tx(&kv_full[slot], kTileBytes);
                            for (int h = 0; h < kHalves; ++h)
                                tma4(dst + h * kHalfBytes, map, h * 64, kh, w.k0 + key, 0, &kv_full[slot]);
                        }
                    } else {
                        const int page = 1 << p.page_shift, box = min(page, kKeys);
                        const int boxes = (min(w.len_k - key, kKeys) + box - 1) / box;  // those that hold keys
                        if (lane == 0) tc::mbar_expect_tx(&kv_full[slot], (uint32_t)(boxes * box) * 128 * kHalves);
                        __syncwarp();
                        if (lane < boxes) {
                            const int at = key + lane * box, pg = p.pages[at >> p.page_shift];
                            for (int h = 0; h < kHalves; ++h)
                                tma4(dst + h * kHalfBytes + lane * box * 128, map, h * 64, kh, at & (page - 1), pg,
                                     &kv_full[slot]);
                        }
                        __syncwarp();
                    }
                }
                if (!ok)  // nothing may land after the block has gone
                    for (int e = max(i - kSlots, 0); e < i; ++e) mbar_wait(&kv_full[e % kSlots], (e / kSlots) & 1);
            }
        } else if (warp == 9 || warp == 10) {
            // ---------------------------------------------------------------- products of tile t
            constexpr uint32_t fmt = std::is_same<H, Bf16>::value ? 1u : 0u;
            constexpr uint32_t common = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(kRows >> 4) << 24);
            constexpr uint32_t id_s = common | ((uint32_t)(kKeys >> 3) << 17);
            constexpr uint32_t id_o = common | (1u << 16) | ((uint32_t)(D >> 3) << 17);
            const int t = warp - 9, mine = t ? nt[1] : nt[0];
            const uint32_t t_s = tmem + t * 128, t_o = tmem + 256 + t * 128;
            const uint64_t q_desc = tc::sw128_kmajor_desc(s_q + t * kTileBytes);
            bool ok = true;
            auto wait = [&](uint64_t* b, uint32_t parity) {
                if (ok) ok = mbar_wait(b, parity);
                return ok;
            };
            auto scores = [&](int slot) {
                const uint64_t b = tc::sw128_kmajor_desc(s_kv + slot * kTileBytes);
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {  // columns past dim are zero
                    const uint32_t off = ((k >> 2) * kHalfBytes + (k & 3) * 32) >> 4;
                    mma_ss(t_s, q_desc + off, b + off, id_s, k > 0);
                }
                commit(&s_full[t]);
            };
            // Hands the slot of item i back to the copies, unless they are done with it: an
            // arrival that nobody waits for could come after the block has gone.
            auto release = [&](int i) {
                if (ok && i + kSlots < 2 * n) commit(&kv_empty[i % kSlots]);
            };
            // A warp without rows of its own follows the same waits: it hands a slot back only
            // after what the slot holds has landed.
            if (mine > 0) wait(&q_full[t], 0);
            if (n > 0 && wait(&kv_full[0], 0) && mine > 0) {
                tc::fence_after_sync();
                scores(0);
            }
            release(0);
            // The two warps take turns, one product of values and the next of scores each: left
            // to themselves the tiles fall into step, both in the exponentials and then both in
            // the tensor cores, and half the time of each is lost.
            int cleaned = 0;
            for (int j = 0; j < n; ++j) {
                const int iv = 2 * j + 1, ik = 2 * j + 2, sv = iv % kSlots, sk = ik % kSlots;
                wait(&kv_full[sv], (iv / kSlots) & 1);
                if (guarded_tile(j)) {
                    asm volatile("bar.arrive 1, 192;" ::: "memory");
                    wait(clean, cleaned++ & 1);
                }
                if (t == 1 || j > 0) wait(&turn[t], t == 1 ? j & 1 : (j - 1) & 1);
                if (j < mine) {
                    const uint64_t b = values_desc(s_kv + sv * kTileBytes, kHalfBytes);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {  // halves of P
                        if (!wait(&p_full[2 * t + h], j & 1)) break;
                        tc::fence_after_sync();
#pragma unroll
                        for (int k = h * 4; k < h * 4 + 4; ++k)
                            mma_ts(t_o, t_s + k * 8, b + k * (2048 >> 4), id_o, (j > 0 || k > 0) ? 1u : 0u);
                    }
                    if (ok && j + 1 == mine) commit(&o_full[t]);
                }
                if (j + 1 < n && wait(&kv_full[sk], (ik / kSlots) & 1) && j + 1 < mine) scores(sk);
                if (lane == 0) tc::mbar_arrive(&turn[t ^ 1]);
                release(iv);
                if (j + 1 < n) release(ik);
            }
            if (!ok) {
                commit(&drained[t]);
                mbar_wait(&drained[t], 0);
            }
        } else if (warp >= 12) {
            // ---------------------------------------------------------------- value rows that not every row sees
            const int g = tid - 384;
            for (int j = 0; j < n; ++j) {
                if (!guarded_tile(j)) continue;
                asm volatile("bar.sync 1, 192;" ::: "memory");  // both warps of products have seen the tile land
                uint8_t* const v = smem + (2 + (2 * j + 1) % kSlots) * kTileBytes;
                const int key = (j0 + j) * kKeys;
                const int end = min(max(w.len_k - key, 0), kKeys), from = max(min_lim - key, 0);
                bool bad = false;
                if (!PAGED)
                    for (int i = g; i < (end - from) * 8; i += 128)
                        for (int h = 0; h < kHalves; ++h)
                            bad |= not_finite<H>(*reinterpret_cast<const uint4*>(v + h * kHalfBytes + from * 128 + i * 16));
                for (int i = g; i < (kKeys - end) * 8; i += 128)
                    for (int h = 0; h < kHalves; ++h)
                        *reinterpret_cast<uint4*>(v + h * kHalfBytes + end * 128 + i * 16) = make_uint4(0, 0, 0, 0);
                if (bad) *s_leak = 1;
                tc::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(clean);
            }
        }
    } else {
        // -------------------------------------------------------------------- softmax: one row a thread
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        const int t = warp >> 2, row = tid & 127;
        const int row_tok = row / p.group, row_head = row - row_tok * p.group;
        const int my_tiles = t ? nt[1] : nt[0];
        const bool valid = row_tok < (t ? tok[1] : tok[0]);
        const int lim = valid ? min(max(w.first_lim + w.step * (t * tt + row_tok), 0), w.len_k) : w.len_k;
        const int tile_lim = min(max(w.first_lim + w.step * t * tt, 0), w.len_k);  // the tile's first row's
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + t * 128 + lane_base, to = tmem + 256 + t * 128 + lane_base;
        float m = -INFINITY, l = 0.0f;
        bool ok = true;
        for (int j = 0; j < my_tiles && ok; ++j) {
            ok = mbar_wait(&s_full[t], j & 1);
            if (!ok) break;
            tc::fence_after_sync();
            uint32_t s[4][32];
#pragma unroll
            for (int c = 0; c < 4; ++c) tc::tmem_ld32(ts + c * 32, s[c]);
            tc::tmem_ld_wait();
            const int key = (j0 + j) * kKeys;
            if (key + kKeys > tile_lim) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (key + c * 32 + i >= lim) s[c][i] = 0xff800000u;  // -inf
            }
            float mx[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                auto f = [&](int i) { return __uint_as_float(s[c][i]); };
                mx[c] = max3(f(0), f(1), f(2));
#pragma unroll
                for (int i = 3; i < 31; i += 2) mx[c] = max3(mx[c], f(i), f(i + 1));
                mx[c] = max3(mx[c], mx[c], f(31));
            }
            const float top = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]) * p.scale_log2;
            if (j == 0) {
                m = top == INFINITY ? __int_as_float(0x7fc00000) : top;
            } else if (__any_sync(0xffffffffu, !(top - m <= kGrow))) {
                // Grown too far, or NaN (a score is NaN or infinite, or the row has seen no key)
                float up = !(top - m <= kGrow) ? top : m;
                if (up == INFINITY) up = __int_as_float(0x7fc00000);
                const float f = m == up ? 1.0f : ex2(m - up);
                m = up;
                l *= f;
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t o[32];
                    tc::tmem_ld32(to + c * 32, o);
                    tc::tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                    tc::tmem_st32(to + c * 32, o);
                }
            }
            const float ref = m == -INFINITY ? 0.0f : m;
            const uint64_t scale2 = pair(p.scale_log2, p.scale_log2);
            uint64_t ref2 = pair(-ref, -ref);
            uint64_t sum[4] = {0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < 4; c += 2) {  // halves of 64 keys
                uint32_t pk[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const uint32_t* e = &s[c + i / 16][(2 * i) & 31];
                    const float2 x = halves(fma2(pair(__uint_as_float(e[0]), __uint_as_float(e[1])), scale2, ref2));
                    const float a = ex2(x.x), b = ex2(x.y);
                    sum[i & 3] = add2(sum[i & 3], pair(a, b));
                    pk[i] = H::pack(a, b);
                }
                tc::tmem_st32(ts + c * 16, pk);
                tc::tmem_st_wait();
                tc::fence_before_sync();
                tc::mbar_arrive(&p_full[2 * t + c / 2]);
                // the second half's exponentials stay behind this arrival
                asm volatile("" : "+l"(ref2));
            }
            const float2 s01 = halves(add2(sum[0], sum[1])), s23 = halves(add2(sum[2], sum[3]));
            l += (s01.x + s01.y) + (s23.x + s23.y);
        }
        if (ok && my_tiles > 0) ok = mbar_wait(&o_full[t], 0);
        tc::fence_after_sync();
        // ---- results
        const long long at = ((long long)(w.q0 + t * tt + row_tok) * p.heads + kh * p.group + row_head);
        const bool leak = !PAGED && my_tiles > 0 && *reinterpret_cast<volatile int*>(s_leak) != 0;
        const bool part = p.part;
        const long long rows = (long long)p.n_q * p.heads;
        float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
        if (!ok) inv = __int_as_float(0x7fc00000);
        using T = typename H::type;
        if (!leak) {
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                if (my_tiles > 0) {
                    tc::tmem_ld32(to + c * 32, o);
                    tc::tmem_ld_wait();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = 0;
                }
#pragma unroll
                for (int i = 0; i < 32; i += 8) {
                    if (!valid || c * 32 + i >= p.dim) continue;
                    float x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = l == 0.0f && ok ? 0.0f : __uint_as_float(o[i + e]) * inv;
                    if (part) {
                        float4* dst = reinterpret_cast<float4*>(p.part_o + (split * rows + at) * p.dim + c * 32 + i);
                        dst[0] = make_float4(x[0], x[1], x[2], x[3]);
                        dst[1] = make_float4(x[4], x[5], x[6], x[7]);
                    } else {
                        *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + at * p.dim + c * 32 + i) = pack8<H>(x);
                    }
                }
                __syncwarp();
            }
        } else if (valid) {
            // One key at a time, eight output values a pass, with the maximum and sum that the
            // scores gave: only where an unseen value row is not finite.
            const T* q = static_cast<const T*>(p.q.p) + (w.q0 + t * tt + row_tok) * p.q.tok + (kh * p.group + row_head) * p.q.head;
            const T* k = static_cast<const T*>(p.k.p) + w.k0 * p.k.tok + kh * p.k.head;
            const T* v = static_cast<const T*>(p.v.p) + w.k0 * p.v.tok + kh * p.v.head;
            const int from = j0 * kKeys, to_key = min(lim, (j0 + per) * kKeys);
            const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll 1
            for (int c = 0; c < p.dim; c += 8) {
                float o[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 1
                for (int key = from; key < to_key; ++key) {
                    float s = 0.0f;
#pragma unroll 1
                    for (int e = 0; e < p.dim; e += 8) {
                        float a[8], b[8];
                        unpack8<H>(*reinterpret_cast<const uint4*>(q + e), a);
                        unpack8<H>(*reinterpret_cast<const uint4*>(k + key * p.k.tok + e), b);
#pragma unroll
                        for (int i = 0; i < 8; ++i) s = fmaf(a[i], b[i], s);
                    }
                    const float x = ex2(fmaf(s, p.scale_log2, -ref));
                    float val[8];
                    unpack8<H>(*reinterpret_cast<const uint4*>(v + key * p.v.tok + c), val);
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[i] += x * val[i];
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] *= inv;
                if (part) {
                    float4* dst = reinterpret_cast<float4*>(p.part_o + (split * rows + at) * p.dim + c);
                    dst[0] = make_float4(o[0], o[1], o[2], o[3]);
                    dst[1] = make_float4(o[4], o[5], o[6], o[7]);
                } else {
                    *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + at * p.dim + c) = pack8<H>(o);
                }
            }
        }
        if (valid) {
            const float lse2 = ok ? m + log2f(l) : __int_as_float(0x7fc00000);
            if (part) p.part_lse[split * rows + at] = lse2;
            else if (p.lse) p.lse[at] = lse2 * 0.6931471805599453f;
        }
        tc::fence_before_sync();
    }
    __syncthreads();
    if (warp == 9) {
        tc::fence_after_sync();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

}  // namespace attn
}  // namespace vgpu

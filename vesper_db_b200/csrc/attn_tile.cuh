// Attention of query tiles on the tensor cores (tcgen05): the kernel that prompts and the
// shared prefix both run.
//
//   S = Q K^T, P = exp2(scale' S - m) with scale' = scale log2(e), O = sum P V / sum P,
// one pass over the keys with a running maximum m and sum l of each row in 32 bits.
//
// A tile is 128 rows: floor(128 / group) tokens with the `group` query heads of one key
// head each, so that one key tile serves the whole group.  A block holds two query tiles
// and takes the keys 128 at a time:
//   * warps 0-7 and 8-15 make the probabilities of tile 0 and tile 1, one row of 64 keys a
//     thread: they read S, exchange the two halves' maxima of a row, keep m and l, and write P
//     over S as 16-bit values, 32 keys at a time, so that the first products with the values
//     run while the rest is made.  (With whole rows of 128 keys in four warps a tile, each
//     scheduler had one warp to hide every latency with: 1,900 cycles from S to P, before the
//     other steps named here.)
//   * warp 16 picks what the block works on next, and copies Q, K and V tiles by TMA, K and V
//     into a ring of shared-memory slots;
//   * warps 17 and 18 issue the products of tile 0 and tile 1: S_t = Q_t K^T (both operands
//     from shared memory) and O_t += P_t V (P from tensor memory);
//   * warp 19 cleans the value tiles that hold keys some row must not see.
// The two query tiles are independent of each other: while one is in the tensor cores the
// other is in the exponentials.  Tensor memory: S0, S1 (128 columns each), O0, O1.
//
// What bounds it: a pair of tiles takes 2,048 cycles in the tensor cores (heads of 128), as
// many in the special-function units (32,768 exponentials, 16 a cycle) and as many in
// shared memory (256 KB read and written, 128 bytes a cycle).  Making a quarter or three
// eighths of the exponentials by a polynomial on the FMA units instead cost 1 to 7 %: the
// issue slots it takes are worth more than the special-function cycles it frees.
// Measured (bf16, heads of 128, 32 over 8): 16,384 tokens, causal: 2,030 to 2,060 us in long
// runs, 1,070 to 1,080 TFLOP/s of 1,404 for a library product that runs as long, at 990 W and
// 1.6 GHz: the power limit; 1,750 us in the first milliseconds.  Tensor cores and
// special-function units are 56 % busy each, as cycles go.  24 prompts of 1 to 4,000 tokens:
// 720 us in long runs, 620 in the first milliseconds (1.17 M cycles), 47 % busy.  256 tokens
// over a prefix of 20,000: 93 us with the join, 42 %, on 128 SMs.
//
// P is rounded to the data's type, as a product takes both operands in one 16-bit type; its sum l
// is of the unrounded values.  Against 64 bits the long cases' outputs are off by 0.0021 to 0.0023 of
// their size then, where rounding them once costs 0.0016 (bf16; f16: 0.00025 to 0.00028, 0.00021).
//
// m only moves when a row's maximum has grown by more than 2^8: until then P may reach 2^8,
// which both types hold at full relative precision, and O need not be rescaled.
//
// Masked scores become -inf by selection, so what unseen keys hold does not matter; unseen
// values meet P = 0, and 0 * NaN is NaN: value rows past the last key are zeroed in shared
// memory, and so are the non-finite values among rows that not every query row sees (the
// diagonal tiles').  A row's results then get back those of the keys that it sees, as a sum:
// any positive weight leaves an infinity or NaN what it is.
//
// A block runs from one piece of work to the next (there is one an SM): the copies of the
// next one, and its first scores, go on while the results of the last one are written.
//
// Every wait is bounded; a block whose wait ran out issues no further work, gives NaN to the
// rows of all pieces that it may not have finished and frees its tensor memory.
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
constexpr int kSoftmaxWarps = 16, kThreads = kSoftmaxWarps * 32 + 128;  // and four service warps
constexpr int kSlots = 4;      // K and V tiles in flight
constexpr int kAhead = 4;      // pieces of work known ahead
constexpr float kGrow = 8.0f;  // log2 of how far P may pass 1 before O is rescaled
constexpr int kSoftmaxRegs = 104, kServiceRegs = 56;  // 512 * 104 + 128 * 56 <= 640 * 96

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
    // Packed rows again, as addresses: the small blocks' (attn_short.cuh), and the values of
    // keys that not every row of a piece sees.
    HeadsView q, k, v;
    float scale_log2;
    int items;     // pieces of work at most (two query tiles, key head, split)
    int* counter;  // zero at launch: pieces are taken as blocks come free; null: in turn
    int splits;
    bool part;       // results of each split for a later join, in 32 bits
    void* out;       // otherwise: [n_q, heads, dim]
    float* lse;
    float* part_o;   // [splits, n_q * heads, dim], and their log2-sum-exp
    float* part_lse;
};

template <int D>
constexpr int smem_bytes() {
    return 2 * kRows * D * 2 + kSlots * kKeys * D * 2 + 1024 + 512 + 2 * 2 * 2 * kRows * 4 + kSoftmaxWarps * 1024;
}

// Bounded wait for the barrier's phase; false when it ran out.  A poll suspends for 3.95 us
// (measured), so 2^18 of them are a second.  The longest stretch between two arrivals is the
// results of a piece, with at most 2 * 128 rows of values looked through once more: 0.12 ms where
// all of them hold a non-finite value (eight prompts of 2,000 tokens, 8 heads of 128: 119 us clean,
// 220 with one in thirty tokens, 537 with all).
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity) {
    const uint32_t a = tc::smem_u32(bar);
#pragma unroll 1
    for (uint32_t i = 0; i < (1u << 18); ++i) {
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

// Maximum of three; NaN is passed over.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// 16 columns of tensor memory, one lane's row a thread.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
          "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
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

// Lane 0's value, known to the compiler as one for the warp: descriptors made from it stay in
// uniform registers, which a product's issue needs them in.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

// What a block works on.
struct Work {
    int q0;        // first row of q of the block's first tile
    int tokens;    // rows of the request from there on (those past the block's tiles do not count)
    int k0, len_k; // first key row, keys of the request
    int first_lim; // keys that the first of these rows sees; each later one sees `step` more
    int step;
    int kh, split;
    int stop;      // no more work
};

// What follows from it: tokens and key tiles of each query tile, [j0, j0 + nt) of the keys'.
struct Tiles {
    int tok0, tok1, nt0, nt1, n, j0, per, min_lim;
    // Tiles that hold keys which some valid row does not see.
    __device__ __forceinline__ bool guarded(int j) const { return (j0 + j + 1) * kKeys > min_lim; }
};
__device__ __forceinline__ Tiles tiles_of(const Work& w, int tt, int splits) {
    Tiles x;
    const int all = (w.len_k + kKeys - 1) / kKeys;
    x.per = (all + splits - 1) / splits;
    x.j0 = w.split * x.per;
    auto count = [&](int first, int tok) {
        const int last = min(w.len_k, w.first_lim + w.step * (first + tok - 1));  // keys its last row sees
        const int tiles = tok > 0 ? (max(last, 0) + kKeys - 1) / kKeys : 0;
        return min(max(tiles - x.j0, 0), x.per);
    };
    x.tok0 = min(max(w.tokens, 0), tt);
    x.tok1 = min(max(w.tokens - tt, 0), tt);
    x.nt0 = count(0, x.tok0);
    x.nt1 = count(tt, x.tok1);
    x.n = max(x.nt0, x.nt1);
    x.min_lim = min(max(w.first_lim, 0), w.len_k);
    return x;
}

// Piece `idx` of the packed requests, each cut into `span` tokens.  Run by one whole warp;
// tokens <= 0: no such piece.  Request b's pieces have the numbers from starts[b] / span + b
// on, which leaves room for each (some numbers stay unused) and can be searched without
// adding up lengths: 32 candidates a step.  Rows before the first and after the last request
// are requests without keys.  Last pieces come first: the rows of a causal prompt's end see
// the most keys.
//
// `near` is the request of the last piece that the warp looked for, or -1: the pieces that a
// block takes come in order, so the next one's request is mostly among the 32 up to there,
// and one step of loads finds it with its keys (the search from scratch takes three or four,
// one after the other, 1.5 us).
__device__ __forceinline__ Work find_work(const TileParams& p, int idx, int lane, int span, int& near) {
    const int n = p.n_requests + 2;
    auto bound = [&](int b) {  // first row of request b
        if (b <= 0) return 0;
        if (b >= n) return p.n_q;
        return min(max(__ldg(p.starts + b - 1), 0), p.n_q);
    };
    auto key_bound = [&](int b) {  // first key row of request b, 1 .. n_requests + 1
        return min(max(__ldg(p.starts_k + b - 1), 0), p.n_k);
    };
    const int want = p.n_q / span + n - 1 - idx;
    int lo = 0, q0 = 0, q1 = 0, k0 = 0, k1 = 0;
    bool found = false;
    if (near >= 0) {
        const int b = near - lane;
        int kb = 0, ke = 0;
        const int qb = bound(b), qe = bound(b + 1);
        if (b > 0 && b <= p.n_requests) {
            kb = key_bound(b);
            ke = max(key_bound(b + 1), kb);
        }
        const unsigned at = __ballot_sync(0xffffffffu, b >= 0 && qb / span + b <= want);
        found = at != 0;
        const int src = found ? __ffs(at) - 1 : 0;
        lo = near - src;
        q0 = __shfl_sync(0xffffffffu, qb, src);
        q1 = __shfl_sync(0xffffffffu, qe, src);
        k0 = __shfl_sync(0xffffffffu, kb, src);
        k1 = __shfl_sync(0xffffffffu, ke, src);
    }
    if (!found) {
        int hi = n;
        lo = 0;
        while (hi - lo > 1) {
            const int step = (hi - lo + 31) / 32, c = lo + (lane + 1) * step;
            const bool before = c < hi && bound(c) / span + c <= want;
            lo += __popc(__ballot_sync(0xffffffffu, before)) * step;
            hi = min(hi, lo + step);
        }
        q0 = bound(lo);
        q1 = bound(lo + 1);
        if (lo > 0 && lo <= p.n_requests) {
            k0 = key_bound(lo);
            k1 = max(key_bound(lo + 1), k0);
        }
    }
    near = lo;
    Work w{};
    const int len_q = q1 - q0, tok = (want - q0 / span - lo) * span;
    w.q0 = q0 + tok;
    w.tokens = tok >= 0 ? len_q - tok : 0;
    w.k0 = k0;
    w.len_k = k1 - k0;
    w.step = p.causal ? 1 : 0;
    w.first_lim = p.causal ? w.len_k - (len_q - tok - 1) : w.len_k;
    return w;
}

template <class H>
__device__ __forceinline__ bool not_finite(uint4 u) {
    constexpr uint32_t lo = std::is_same<H, Bf16>::value ? 0x7f80u : 0x7c00u, hi = lo << 16;
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) bad |= (w[i] & lo) == lo || (w[i] & hi) == hi;
    return bad;
}

// Of two values, or eight: the finite ones, zero in the others' places; with `others` those,
// zero in the finite ones' places.
template <class H>
__device__ __forceinline__ uint32_t finite_part(uint32_t u, bool others = false) {
    constexpr uint32_t lo = std::is_same<H, Bf16>::value ? 0x7f80u : 0x7c00u, hi = lo << 16;
    const uint32_t odd = ((u & lo) == lo ? 0xffffu : 0u) | ((u & hi) == hi ? 0xffff0000u : 0u);
    return u & (others ? odd : ~odd);
}
template <class H>
__device__ __forceinline__ uint4 finite_part(uint4 u, bool others = false) {
    return make_uint4(finite_part<H>(u.x, others), finite_part<H>(u.y, others), finite_part<H>(u.z, others),
                      finite_part<H>(u.w, others));
}

// Piece of work number `item`: key heads fastest, then splits.  Run by one whole warp.
template <bool PAGED>
__device__ __forceinline__ Work item_work(const TileParams& p, int item, int lane, int& near) {
    Work w{};
    const int kh = item % p.kv_heads, rest = item / p.kv_heads, split = rest % p.splits, block = rest / p.splits;
    if (PAGED) {  // every row sees the whole prefix
        w.q0 = block * 2 * p.tile_tokens;
        w.tokens = p.n_q - w.q0;
        w.len_k = w.first_lim = p.n_k;
    } else {
        w = find_work(p, block, lane, 2 * p.tile_tokens, near);
    }
    w.kh = kh;
    w.split = split;
    w.stop = 0;
    return w;
}

template <class H, int D, bool PAGED>
__global__ void __launch_bounds__(kThreads, 1) attn_tile_kernel(const __grid_constant__ TileParams p) {
    extern __shared__ uint8_t smem_raw[];
    constexpr int kHalves = D / 64, kHalfBytes = kKeys * 128, kTileBytes = kHalves * kHalfBytes;
    const uint32_t raw = tc::smem_u32(smem_raw), base = (raw + 1023) & ~1023u;
    uint8_t* const smem = smem_raw + (base - raw);
    const uint32_t s_q = base, s_kv = base + 2 * kTileBytes;
    uint64_t* const bars = reinterpret_cast<uint64_t*>(smem + (2 + kSlots) * kTileBytes);
    uint64_t* const q_full = bars;                   // [2]
    uint64_t* const q_empty = q_full + 2;            // [2]
    uint64_t* const kv_full = q_empty + 2;           // [kSlots]
    uint64_t* const kv_empty = kv_full + kSlots;     // [kSlots]
    uint64_t* const s_full = kv_empty + kSlots;      // [2]
    uint64_t* const p_full = s_full + 2;             // [2][2]: tile, part of the keys
    uint64_t* const o_full = p_full + 4;             // [2]
    uint64_t* const turn = o_full + 2;               // [2]
    uint64_t* const drained = turn + 2;              // [2]
    uint64_t* const landed = drained + 2;
    uint64_t* const clean = landed + 1;
    uint64_t* const work_full = clean + 1;           // [kAhead]
    uint64_t* const work_empty = work_full + kAhead; // [kAhead]
    // [kAhead], and the piece that was taken but not begun when a wait ran out
    Work* const s_work = reinterpret_cast<Work*>(work_empty + kAhead);
    int* const s_leak = reinterpret_cast<int*>(s_work + kAhead + 1);  // [kAhead][2]: piece, query tile
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(s_leak + 2 * kAhead);
    volatile int* const s_lost = reinterpret_cast<int*>(tmem_slot + 1);  // a wait ran out
    volatile uint32_t* const s_copies = tmem_slot + 2;                   // key and value tiles asked for
    // Rows' maxima (and sums) of each half of the keys: [turn][tile][half][row]
    float* const s_half = reinterpret_cast<float*>(bars + 64);
    const uint32_t s_stage = tc::smem_u32(s_half + 2 * 2 * 2 * kRows);  // 1 KB a softmax warp, for the results
    static_assert((2 + 2 + 2 * kSlots + 2 + 4 + 2 + 2 + 2 + 2 + 2 * kAhead) * 8 + (kAhead + 1) * sizeof(Work) + 2 * kAhead * 4 + 12 <= 512, "");

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // The own pages' kernel may be queued behind this one and does not depend on it.
    if (PAGED) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (warp == 16 && lane < 3 && p.n_k > 0) {
        const CUtensorMap* map = lane == 0 ? &p.mq : (lane == 1 ? &p.mk : &p.mv);
        asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
    }
    if (warp == 17) {
        if (lane == 0) {
            for (int i = 0; i < 2; ++i) {
                tc::mbar_init(&q_full[i], 1);
                tc::mbar_init(&q_empty[i], 1);
                tc::mbar_init(&s_full[i], 1);
                tc::mbar_init(&p_full[2 * i], 256);
                tc::mbar_init(&p_full[2 * i + 1], 256);
                tc::mbar_init(&turn[i], 1);
                tc::mbar_init(&o_full[i], 1);
                tc::mbar_init(&drained[i], 1);
            }
            for (int i = 0; i < kSlots; ++i) {
                tc::mbar_init(&kv_full[i], 1);
                tc::mbar_init(&kv_empty[i], 2);  // both warps of products
            }
            for (int i = 0; i < kAhead; ++i) {
                tc::mbar_init(&work_full[i], 1);
                tc::mbar_init(&work_empty[i], kSoftmaxWarps + 3);  // all warps but the one that fills it
            }
            for (int i = 0; i <= kAhead; ++i) s_work[i].tokens = 0;
            *s_lost = 0;
            *s_copies = 0;
            tc::mbar_init(landed, 2);
            tc::mbar_init(clean, 1);
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
    const uint32_t tmem = (uint32_t)uniform((int)*tmem_slot);
    const int tt = p.tile_tokens;

    bool ok = true;  // sticky: after a wait that ran out a warp waits no more
    auto wait = [&](uint64_t* b, uint32_t parity) {
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(b, parity)) != 0;
        return ok;
    };
    // A wait that may last for all key tiles of a piece (2.3 us each), however many they are: it runs
    // out when the block has asked for none in a second.  Only where that can be, as the second loop
    // costs: 200 short passages took 158 us instead of 125 with it in every wait.
    auto wait_on = [&](uint64_t* b, uint32_t parity) {
        uint32_t before = ~0u;
#pragma unroll 1
        while (ok && !__all_sync(0xffffffffu, mbar_wait(b, parity))) {
            const uint32_t now = (uint32_t)uniform((int)*s_copies);
            ok = now != before;
            before = now;
        }
        return ok;
    };
    // The piece of work number `it` of the block; false when a wait ran out.  `done` hands its
    // place back; whoever reads the leak flag does that at the end.
    auto work_done = [&](uint32_t it) {
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&work_empty[it % kAhead]);
    };
    auto next_work = [&](Work& w, uint32_t it) {
        if (!wait_on(&work_full[it % kAhead], (it / kAhead) & 1)) return false;
        w = s_work[it % kAhead];
        return true;
    };

    if (warp >= kSoftmaxWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kServiceRegs));
        if (warp == 16) {
            // ---------------------------------------------------------------- work and copies
            uint32_t it = 0, kv = 0, qn0 = 0, qn1 = 0;
            auto load_q = [&](const Work& w, int t, uint32_t& qn) {
                if (qn > 0 && !wait(&q_empty[t], (qn - 1) & 1)) return;
                ++qn;
                if (lane == 0) {
                    tc::mbar_expect_tx(&q_full[t], (uint32_t)(tt * p.group) * 128 * kHalves);
                    for (int h = 0; h < kHalves; ++h)
                        tma4(s_q + t * kTileBytes + h * kHalfBytes, &p.mq, h * 64, 0, w.kh, w.q0 + t * tt, &q_full[t]);
                }
            };
            int item = blockIdx.x, near = -1;
            while (true) {
                Work w{};
                w.stop = 1;
                // pieces that turn out to be empty are passed over
                while (item < p.items) {
                    w = item_work<PAGED>(p, item, lane, near);
                    if (w.tokens > 0) break;
                    w.stop = 1;
                    if (p.counter) {
                        if (lane == 0) item = gridDim.x + atomicAdd(p.counter, 1);
                        item = __shfl_sync(0xffffffffu, item, 0);
                    } else {
                        item += gridDim.x;
                    }
                }
                const int r = it % kAhead;
                if (it >= kAhead) wait(&work_empty[r], (it / kAhead - 1) & 1);
                if (!ok) {
                    if (lane == 0) s_work[kAhead] = w;
                    break;
                }
                if (lane == 0) {
                    s_work[r] = w;
                    s_leak[2 * r] = s_leak[2 * r + 1] = 0;
                    tc::mbar_arrive(&work_full[r]);
                }
                __syncwarp();
                ++it;
                if (w.stop) break;
                int after = item + gridDim.x;
                if (p.counter && lane == 0) after = gridDim.x + atomicAdd(p.counter, 1);
                const Tiles x = tiles_of(w, tt, p.splits);
                for (int i = 0; i < 2 * x.n; ++i, ++kv) {  // K, V, K, V, ...
                    const int slot = kv % kSlots, round = kv / kSlots, key = (x.j0 + (i >> 1)) * kKeys;
                    if (round > 0 && !wait(&kv_empty[slot], (round - 1) & 1)) break;
                    if (lane == 0) *s_copies = kv;
                    const CUtensorMap* map = (i & 1) ? &p.mv : &p.mk;
                    const uint32_t dst = s_kv + slot * kTileBytes;
                    if (!PAGED) {
                        if (lane == 0) {
                            tc::mbar_expect_tx(&kv_full[slot], kTileBytes);
                            for (int h = 0; h < kHalves; ++h)
                                tma4(dst + h * kHalfBytes, map, h * 64, w.kh, w.k0 + key, 0, &kv_full[slot]);
                        }
                    } else {
                        const int page = 1 << p.page_shift, box = min(page, kKeys);
                        const int boxes = (min(w.len_k - key, kKeys) + box - 1) / box;  // those that hold keys
                        if (lane == 0) tc::mbar_expect_tx(&kv_full[slot], (uint32_t)(boxes * box) * 128 * kHalves);
                        __syncwarp();
                        if (lane < boxes) {
                            const int at = key + lane * box, pg = p.pages[at >> p.page_shift];
                            for (int h = 0; h < kHalves; ++h)
                                tma4(dst + h * kHalfBytes + lane * box * 128, map, h * 64, w.kh, at & (page - 1), pg,
                                     &kv_full[slot]);
                        }
                        __syncwarp();
                    }
                    if (i == 0) {
                        if (x.nt0 > 0) load_q(w, 0, qn0);
                        if (x.nt1 > 0) load_q(w, 1, qn1);
                    }
                }
                item = __shfl_sync(0xffffffffu, after, 0);
            }
            // Nothing may land, or arrive, after the block has gone.
            const bool sound = ok;
            ok = true;
            for (uint32_t e = kv > kSlots ? kv - kSlots : 0; e < kv; ++e) {
                wait(&kv_full[e % kSlots], (e / kSlots) & 1);
                if (sound) wait(&kv_empty[e % kSlots], (e / kSlots) & 1);
            }
            if (sound && qn0 > 0) wait(&q_empty[0], (qn0 - 1) & 1);
            if (sound && qn1 > 0) wait(&q_empty[1], (qn1 - 1) & 1);
        } else if (warp == 17 || warp == 18) {
            // ---------------------------------------------------------------- products of tile t
            constexpr uint32_t fmt = std::is_same<H, Bf16>::value ? 1u : 0u;
            constexpr uint32_t common = (1u << 4) | (fmt << 7) | (fmt << 10) | ((uint32_t)(kRows >> 4) << 24);
            constexpr uint32_t id_s = common | ((uint32_t)(kKeys >> 3) << 17);
            constexpr uint32_t id_o = common | (1u << 16) | ((uint32_t)(D >> 3) << 17);
            const int t = uniform(warp - 17);
            const uint32_t t_s = tmem + t * 128, t_o = tmem + 256 + t * 128;
            const uint64_t q_desc = tc::sw128_kmajor_desc(s_q + t * kTileBytes);
            auto scores = [&](int slot) {
                const uint64_t b = tc::sw128_kmajor_desc(s_kv + slot * kTileBytes);
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {  // columns past dim are zero
                    const uint32_t off = ((k >> 2) * kHalfBytes + (k & 3) * 32) >> 4;
                    mma_ss(t_s, q_desc + off, b + off, id_s, k > 0);
                }
                commit(&s_full[t]);
            };
            // Counts over all pieces of work: items of the ring, turns, tiles, Q tiles, cleanings.
            uint32_t kv = 0, turns = 0, tiles = 0, qn = 0, cleaned = 0;
            Work w;
            for (uint32_t it = 0; next_work(w, it); ++it) {
                work_done(it);
                if (w.stop) break;
                const Tiles x = tiles_of(w, tt, p.splits);
                const int n = uniform(x.n), mine = uniform(t ? x.nt1 : x.nt0);
                if (n == 0) continue;
                auto slot_of = [&](int i) { return (int)((kv + i) % kSlots); };
                auto arrived = [&](int i) { return wait(&kv_full[slot_of(i)], ((kv + i) / kSlots) & 1); };
                auto release = [&](int i) {
                    if (ok) commit(&kv_empty[slot_of(i)]);
                };
                // A warp without rows of its own follows the same waits: it hands a slot back only
                // after what the slot holds has landed.
                if (mine > 0) wait(&q_full[t], qn++ & 1);
                if (arrived(0) && mine > 0) {
                    tc::fence_after_sync();
                    scores(slot_of(0));
                    if (mine == 1) commit(&q_empty[t]);
                }
                release(0);
                // The two warps take turns, one product of values and the next of scores each:
                // left to themselves the tiles fall into step, both in the exponentials and then
                // both in the tensor cores, and half the time of each is lost.
                for (int j = 0; j < n && ok; ++j, ++turns) {
                    const int iv = 2 * j + 1, ik = 2 * j + 2;
                    arrived(iv);
                    if (x.guarded(j)) {
                        if (lane == 0) tc::mbar_arrive(landed);
                        wait(clean, cleaned++ & 1);
                    }
                    if (j + 1 < n) arrived(ik);
                    if (t == 1 || turns > 0) wait(&turn[t], t == 1 ? turns & 1 : (turns - 1) & 1);
                    if (j < mine) {
                        const uint64_t b = values_desc(s_kv + slot_of(iv) * kTileBytes, kHalfBytes);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {  // keys 0-31 and 64-95, then the others
                            if (!wait(&p_full[2 * t + h], tiles & 1)) break;
                            tc::fence_after_sync();
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int k = 2 * h + (e & 1) + (e >> 1) * 4;
                                mma_ts(t_o, t_s + k * 8, b + k * (2048 >> 4), id_o, (j > 0 || h > 0 || e > 0) ? 1u : 0u);
                            }
                        }
                        ++tiles;
                        if (ok && j + 1 == mine) commit(&o_full[t]);
                    }
                    if (ok && j + 1 < mine) {
                        scores(slot_of(ik));
                        if (j + 2 == mine) commit(&q_empty[t]);
                    }
                    if (lane == 0) tc::mbar_arrive(&turn[t ^ 1]);
                    release(iv);
                    if (j + 1 < n) release(ik);
                }
                kv += 2 * n;
            }
            if (!ok) {
                commit(&drained[t]);
                mbar_wait(&drained[t], 0);
            }
        } else {
            // ---------------------------------------------------------------- value rows that not every row sees
            uint32_t kv = 0, seen = 0;
            Work w;
            for (uint32_t it = 0; next_work(w, it); ++it) {
                work_done(it);
                if (w.stop) break;
                const Tiles x = tiles_of(w, tt, p.splits);
                for (int j = 0; j < x.n; ++j) {
                    if (!x.guarded(j)) continue;
                    if (!wait_on(landed, seen++ & 1)) break;  // both warps of products have seen the tile land
                    uint8_t* const v = smem + (2 + (kv + 2 * j + 1) % kSlots) * kTileBytes;
                    const int key = (x.j0 + j) * kKeys;
                    const int end = min(max(w.len_k - key, 0), kKeys), from = max(x.min_lim - key, 0);
                    bool bad = false;
                    if (!PAGED)
                        for (int i = lane; i < (end - from) * 8; i += 32)
                            for (int h = 0; h < kHalves; ++h) {
                                uint4* const at = reinterpret_cast<uint4*>(v + h * kHalfBytes + from * 128 + i * 16);
                                if (not_finite<H>(*at)) {
                                    *at = finite_part<H>(*at);
                                    bad = true;
                                }
                            }
                    for (int i = lane; i < (kKeys - end) * 8; i += 32)
                        for (int h = 0; h < kHalves; ++h)
                            *reinterpret_cast<uint4*>(v + h * kHalfBytes + end * 128 + i * 16) = make_uint4(0, 0, 0, 0);
                    // Of each query tile that has this key tile to come: its results, which read the
                    // flag, then wait for a product that waits for this.  A tile that is done with
                    // its keys may be reading by now, and sees none of these rows.
                    if (bad && j < x.nt0) s_leak[it % kAhead * 2] = 1;
                    if (bad && j < x.nt1) s_leak[it % kAhead * 2 + 1] = 1;
                    tc::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(clean);
                }
                kv += 2 * x.n;
            }
        }
    } else {
        // -------------------------------------------------------------------- softmax: 64 keys of a row a thread
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        const int t = warp >> 3, half = (warp >> 2) & 1, row = tid & 127;
        const int row_tok = row / p.group, row_head = row - row_tok * p.group;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t ts = tmem + t * 128 + lane_base, to = tmem + 256 + t * 128 + half * (D / 2) + lane_base;
        // The two warps of a row meet: each gives a value and gets the other's.
        uint32_t meetings = 0;
        auto exchange = [&](float x) {
            float* const ex = s_half + (meetings++ & 1) * 512 + t * 256;
            ex[half * 128 + row] = x;
            asm volatile("bar.sync %0, 64;" ::"r"(2 + t * 4 + (warp & 3)) : "memory");
            return ex[(half ^ 1) * 128 + row];
        };
        uint32_t tiles = 0, outs = 0;  // over all pieces of work
        Work w;
        uint32_t it = 0;
        while (true) {
            // Both warps of a row stop together, or one would wait for the other for good.
            next_work(w, it);
            if (exchange(ok ? 0.0f : 1.0f) != 0.0f) ok = false;
            if (!ok || w.stop) break;
            const Tiles x = tiles_of(w, tt, p.splits);
            const int my_tiles = t ? x.nt1 : x.nt0, j0 = x.j0, per = x.per;
            const bool valid = row_tok < (t ? x.tok1 : x.tok0);
            const int lim = valid ? min(max(w.first_lim + w.step * (t * tt + row_tok), 0), w.len_k) : w.len_k;
            const int tile_lim = min(max(w.first_lim + w.step * t * tt, 0), w.len_k);  // the tile's first row's
            // Keys that some row of the warp sees, at most; a warp without rows makes no
            // probabilities (what stands in its lanes only reaches results that are not stored).
            const bool idle = !__any_sync(0xffffffffu, valid);
            const int warp_lim = __reduce_max_sync(0xffffffffu, valid ? lim : 0);
            float m = -INFINITY, l = 0.0f;
            // Moves the reference m to a row's new maximum where it has grown too far.  Each of the
            // two warps of a row sees the same values, and rescales half of O.
            auto settle = [&](float top, bool first) {
                if (first) {
                    m = top == INFINITY ? __int_as_float(0x7fc00000) : top;
                } else if (__any_sync(0xffffffffu, !(top - m <= kGrow))) {
                    // grown, or NaN (a score is NaN or infinite, or the row has seen no key)
                    float up = !(top - m <= kGrow) ? top : m;
                    if (up == INFINITY) up = __int_as_float(0x7fc00000);
                    const float f = m == up ? 1.0f : ex2(m - up);
                    m = up;
                    l *= f;
#pragma unroll 1
                    for (int c = 0; c < D / 32; ++c) {
                        uint32_t o[16];
                        tmem_ld16(to + c * 16, o);
                        tc::tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        tmem_st16(to + c * 16, o);
                    }
                }
            };
            for (int j = 0; j < my_tiles; ++j) {
                // after a wait that ran out the row's warps only keep meeting
                // (the first scores may come after the other tile's keys of the piece before)
                if (j == 0) wait_on(&s_full[t], tiles++ & 1);
                else wait(&s_full[t], tiles++ & 1);
                tc::fence_after_sync();
                const int key = (j0 + j) * kKeys + half * 64;
                if (key >= warp_lim) {  // no row of the warp sees these keys: P is zero
                    const float top = exchange(-INFINITY) * p.scale_log2;
                    if (!idle) {
                        settle(top, j == 0);
                        uint32_t zero[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) zero[i] = 0;
                        tmem_st16(ts + half * 32, zero);
                        tmem_st16(ts + half * 32 + 16, zero);
                        tc::tmem_st_wait();
                        tc::fence_before_sync();
                    }
                    tc::mbar_arrive(&p_full[2 * t]);
                    tc::mbar_arrive(&p_full[2 * t + 1]);
                    continue;
                }
                uint32_t s[2][32];
                tc::tmem_ld32(ts + half * 64, s[0]);
                tc::tmem_ld32(ts + half * 64 + 32, s[1]);
                tc::tmem_ld_wait();
                if (key + 64 > tile_lim) {
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if (key + c * 32 + i >= lim) s[c][i] = 0xff800000u;  // -inf
                }
                float mx[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    auto f = [&](int i) { return __uint_as_float(s[c >> 1][(c & 1) * 16 + i]); };
                    mx[c] = max3(f(0), f(1), f(2));
#pragma unroll
                    for (int i = 3; i < 15; i += 2) mx[c] = max3(mx[c], f(i), f(i + 1));
                    mx[c] = max3(mx[c], f(15), f(15));
                }
                float top = max3(max3(mx[0], mx[1], mx[2]), mx[3], mx[3]);
                // also: both halves of S are in registers after this, and P may take their place
                top = fmaxf(top, exchange(top)) * p.scale_log2;
                settle(top, j == 0);
                const float ref = m == -INFINITY ? 0.0f : m;
                const uint64_t scale2 = pair(p.scale_log2, p.scale_log2);
                uint64_t ref2 = pair(-ref, -ref);
                uint64_t sum[2] = {0, 0};
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t pk[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float2 x =
                            halves(fma2(pair(__uint_as_float(s[c][2 * i]), __uint_as_float(s[c][2 * i + 1])), scale2,
                                        ref2));
                        const float a = ex2(x.x), b = ex2(x.y);
                        sum[i & 1] = add2(sum[i & 1], pair(a, b));
                        pk[i] = H::pack(a, b);
                    }
                    tmem_st16(ts + half * 32 + c * 16, pk);
                    tc::tmem_st_wait();
                    tc::fence_before_sync();
                    tc::mbar_arrive(&p_full[2 * t + c]);
                    // the second part's exponentials stay behind this arrival
                    asm volatile("" : "+l"(ref2));
                }
                const float2 both = halves(add2(sum[0], sum[1]));
                l += both.x + both.y;
            }
            if (my_tiles > 0) {
                wait(&o_full[t], outs++ & 1);
                const float other = exchange(ok ? l : __int_as_float(0x7fc00000));
                // one order of the two, so that both warps hold the same sum
                l = half ? other + l : l + other;
                if (!ok) l = __int_as_float(0x7fc00000);
            }
            tc::fence_after_sync();
            // ---- results
            using T = typename H::type;
            const long long at = ((long long)(w.q0 + t * tt + row_tok) * p.heads + w.kh * p.group + row_head);
            const bool leak = !PAGED && my_tiles > 0 && ok && *reinterpret_cast<volatile int*>(&s_leak[it % kAhead * 2 + t]) != 0;
            // The piece's place is handed back before the stores: the arrival would wait for them.
            work_done(it++);
            if (leak) {
                // Non-finite values were taken out of the tiles that not every row of the piece sees:
                // each row adds those of the keys that it does see.  At most 2 * 128 keys, as a row
                // sees one more than the row before it.
                const T* const v = static_cast<const T*>(p.v.p) + w.k0 * p.v.tok + w.kh * p.v.head;
                const int begin = j0 * kKeys, from = max(x.min_lim, begin);
                const int mine = valid ? begin + min(max(lim - begin, 0), per * kKeys) : 0;
                const int until = __reduce_max_sync(0xffffffffu, mine);
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    const int d = half * (D / 2) + c * 16;
                    if (d >= p.dim) break;
                    uint32_t o[16];
                    tmem_ld16(to + c * 16, o);
                    tc::tmem_ld_wait();
#pragma unroll 1
                    for (int first = from; first < until; first += 32) {  // a lane looks through one key
                        auto values = [&](int key, int h) {
                            if (key >= until || d + h * 8 >= p.dim) return make_uint4(0, 0, 0, 0);
                            return __ldg(reinterpret_cast<const uint4*>(v + key * p.v.tok + d) + h);
                        };
                        unsigned some = __ballot_sync(
                            0xffffffffu, not_finite<H>(values(first + lane, 0)) || not_finite<H>(values(first + lane, 1)));
#pragma unroll 1
                        for (; some; some &= some - 1) {
                            const int key = first + __ffs(some) - 1;
                            if (key >= mine) continue;
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                float val[8];
                                unpack8<H>(finite_part<H>(values(key, h), true), val);
#pragma unroll
                                for (int i = 0; i < 8; ++i)
                                    o[h * 8 + i] = __float_as_uint(__uint_as_float(o[h * 8 + i]) + val[i]);
                            }
                        }
                    }
                    __syncwarp();
                    tmem_st16(to + c * 16, o);
                    tc::tmem_st_wait();
                }
            }
            const bool part = p.part;
            const long long rows = (long long)p.n_q * p.heads;
            const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
            // A thread has part of one row, rows lie heads * dim apart: stored from here, each
            // 16 bytes are a line of their own (3,000 cycles a piece with heads of 64, 6,000 with
            // 128).  So a warp passes its rows through 1 KB of shared memory, a few at a time, and
            // stores each row's part in one go.
            const uint32_t stage = s_stage + warp * 1024;
            auto scaled = [&](uint32_t o) { return l == 0.0f ? 0.0f : __uint_as_float(o) * inv; };
            // kRowsAt rows of kPieces 16-byte pieces; `piece` gives this lane's, `put` stores one
            // of the row of another lane.
            auto through = [&](auto pieces, auto&& piece, auto&& put) {
                constexpr int kPieces = decltype(pieces)::value, kRowsAt = 64 / kPieces;
                const int mine = lane % kRowsAt;
#pragma unroll
                for (int r0 = 0; r0 < 32; r0 += kRowsAt) {
                    __syncwarp();
                    if (lane / kRowsAt == r0 / kRowsAt)
#pragma unroll
                        for (int i = 0; i < kPieces; ++i) {
                            const uint4 u = piece(i);
                            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(
                                             stage + (mine * kPieces + (i ^ (mine & 7 & (kPieces - 1)))) * 16),
                                         "r"(u.x), "r"(u.y), "r"(u.z), "r"(u.w)
                                         : "memory");
                        }
                    __syncwarp();
#pragma unroll
                    for (int e = lane; e < 64; e += 32) {
                        const int r = e / kPieces, i = e % kPieces;
                        uint4 u;
                        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                                     : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                                     : "r"(stage + (r * kPieces + (i ^ (r & 7 & (kPieces - 1)))) * 16)
                                     : "memory");
                        const long long row_at = __shfl_sync(0xffffffffu, at, r0 + r);
                        if (__shfl_sync(0xffffffffu, (int)valid, r0 + r)) put(row_at, i, u);
                    }
                }
            };
            if (!part) {
                uint32_t pk[D / 4];
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t o[16];
                    if (my_tiles > 0) {
                        tmem_ld16(to + c * 16, o);
                        tc::tmem_ld_wait();
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = 0;
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) pk[c * 8 + i] = H::pack(scaled(o[2 * i]), scaled(o[2 * i + 1]));
                }
                through(std::integral_constant<int, D / 16>{},
                        [&](int i) { return make_uint4(pk[4 * i], pk[4 * i + 1], pk[4 * i + 2], pk[4 * i + 3]); },
                        [&](long long row_at, int i, const uint4& u) {
                            const int d = half * (D / 2) + i * 8;
                            if (d < p.dim) *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + row_at * p.dim + d) = u;
                        });
            } else {
#pragma unroll 1
                for (int c = 0; c < D / 64; ++c) {  // 32 values at a time
                    uint32_t o[2][16];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (my_tiles > 0) {
                            tmem_ld16(to + c * 32 + h * 16, o[h]);
                            tc::tmem_ld_wait();
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[h][i] = 0;
                        }
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[h][i] = __float_as_uint(scaled(o[h][i]));
                    }
                    through(std::integral_constant<int, 8>{},
                            [&](int i) {
                                const uint32_t* e = &o[i >> 2][(i & 3) * 4];
                                return make_uint4(e[0], e[1], e[2], e[3]);
                            },
                            [&](long long row_at, int i, const uint4& u) {
                                const int d = half * (D / 2) + c * 32 + i * 4;
                                if (d < p.dim)
                                    *reinterpret_cast<uint4*>(p.part_o + (w.split * rows + row_at) * p.dim + d) = u;
                            });
                }
            }
            if (valid && half == 0) {
                const float lse2 = m + log2f(l);
                if (part) p.part_lse[w.split * rows + at] = lse2;
                else if (p.lse) p.lse[at] = lse2 * 0.6931471805599453f;
            }
            // the next piece's first P, and with it the first product into O, comes after these reads
            tc::fence_before_sync();
        }
        if (!ok) *s_lost = 1;
    }
    __syncthreads();
    if (warp < kSoftmaxWarps && *s_lost) {
        // A wait ran out: the rows of all pieces that the block may not have finished are NaN.
        // (Without a counter a block has at most two pieces.)
        const int t = warp >> 3, row = tid & 127, row_tok = row / p.group, row_head = row - row_tok * p.group;
        auto lost = [&](const Work& v) {
            if ((warp & 4) || row_tok >= min(max(v.tokens - t * tt, 0), tt)) return;
            const long long at = (long long)(v.q0 + t * tt + row_tok) * p.heads + v.kh * p.group + row_head;
            for (int d = 0; d < p.dim && !p.part; ++d) static_cast<uint16_t*>(p.out)[at * p.dim + d] = 0x7fff;
            if (p.part) p.part_lse[v.split * (long long)p.n_q * p.heads + at] = __int_as_float(0x7fc00000);
            else if (p.lse) p.lse[at] = __int_as_float(0x7fc00000);
        };
        for (int i = 0; i <= kAhead; ++i) lost(s_work[i]);
    }
    if (warp == 17) {
        tc::fence_after_sync();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

}  // namespace attn
}  // namespace vgpu

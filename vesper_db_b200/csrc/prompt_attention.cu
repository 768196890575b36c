// Attention over packed prompts, and over a shared prefix joined with each request's own
// pages: launchers, the kernel of the own pages, and the join of partial results.
#include <algorithm>

#include "attention.cuh"
#include "attn_short.cuh"
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
// Prompts go to the small blocks when their mean is at most this many query rows (tokens
// times group) and keys: twice as many rows, and more, while the tiles would not give every
// SM a block, as it is the latency of one that counts then.  30,000 tokens of one length, us
// in small blocks / tiles: 32 + 8 heads of 128, 16 tokens (64 rows) 334 / 465, 32 tokens
// 302 / 284; 12 heads of 64, 100 tokens 89 / 111, 200 tokens 107 / 113 (causal), 136 / 93
// (full).  1,500 tokens: 32 + 8 heads, 64 tokens 20 / 26, 150 tokens 25 / 25.  The lengths are
// on the device, so the rule goes by means: one prompt of 16,000 tokens beside 1,000 of one token
// takes 5.8 ms in small blocks (1.66 ms alone, in tiles).
constexpr int kShortMeanRows = 128, kShortMeanRowsFew = 384, kShortMeanKeys = 512;
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
void launch_tiles_as(const TileParams& p, unsigned blocks, cudaStream_t st) {
    auto* kernel = attn::attn_tile_kernel<H, D, PAGED>;
    constexpr int smem = attn::smem_bytes<D>();
    static std::atomic<uint64_t> devices{0};
    opt_in(devices, kernel, smem, [&] {
        cudaFuncAttributes fa;
        VGPU_CHECK(cudaFuncGetAttributes(&fa, kernel));
        // the softmax warps' registers come out of what the block is launched with
        if (fa.numRegs * kThreads < attn::kSoftmaxWarps * 32 * attn::kSoftmaxRegs + 128 * attn::kServiceRegs)
            throw CudaError("attn_tile_kernel: launched with too few registers for its split");
    });
    kernel<<<blocks, kThreads, smem, st>>>(p);
    VGPU_LAUNCH("attn_tile_kernel");
}

// Pieces of work are handed out by a counter when every block gets several: their lengths
// differ, and are known on the device only.
bool counted(long long items) { return items > 2 * kSms; }

template <bool PAGED>
void launch_tiles(TileParams p, bool f16, long long items, int* counter, cudaStream_t st) {
    if (items <= 0) return;
    if (items > 0x7fffffffLL - kSms) throw CudaError("attention: too many tiles for one launch");
    p.items = (int)items;
    if (counted(items)) {
        p.counter = counter;
        VGPU_CHECK(cudaMemsetAsync(counter, 0, sizeof(int), st));
    }
    const unsigned blocks = (unsigned)std::min<long long>(items, kSms);
    if (f16) {
        if (p.dim <= 64) launch_tiles_as<F16, 64, PAGED>(p, blocks, st);
        else launch_tiles_as<F16, 128, PAGED>(p, blocks, st);
    } else {
        if (p.dim <= 64) launch_tiles_as<Bf16, 64, PAGED>(p, blocks, st);
        else launch_tiles_as<Bf16, 128, PAGED>(p, blocks, st);
    }
}

template <class H, int D>
void launch_short_as(const TileParams& p, long long blocks, cudaStream_t st) {
    constexpr int smem = attn::short_smem_bytes<D>();
    static std::atomic<uint64_t> devices{0};
    opt_in(devices, attn::attn_short_kernel<H, D>, smem, [] {});
    attn::attn_short_kernel<H, D><<<(unsigned)blocks, attn::kShortThreads, smem, st>>>(p);
    VGPU_LAUNCH("attn_short_kernel");
}

void launch_short(const TileParams& p, bool f16, long long blocks, cudaStream_t st) {
    if (blocks > 0x7fffffffLL) throw CudaError("attention: too many tiles for one launch");
    if (f16) {
        if (p.dim <= 64) launch_short_as<F16, 64>(p, blocks, st);
        else launch_short_as<F16, 128>(p, blocks, st);
    } else {
        if (p.dim <= 64) launch_short_as<Bf16, 64>(p, blocks, st);
        else launch_short_as<Bf16, 128>(p, blocks, st);
    }
}

// A launch that may overlap the end of the stream's last kernel, if that one allows it.
template <class K, class... Args>
void launch_ahead(K* kernel, unsigned blocks, unsigned threads, int smem, bool ahead, cudaStream_t st, const Args&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = ahead ? 1 : 0;
    VGPU_CHECK(cudaLaunchKernelEx(&cfg, kernel, args...));
}

// ---------------------------------------------------------------------------------
// Pages of a cache with few query rows: each request's own pages, and the prefix when the
// whole batch has few rows.  Bound by reading keys and values once.
//
// A job is up to 8 * NT query rows of one key head with the keys they share: a request's
// own pages (jobs 0 ..), then the prefix for each tile of the batch's rows.  Requests differ
// widely in length, so the work is cut by keys, not by requests: the jobs' blocks of 16 keys
// are laid end to end, and each warp takes the next `range` of them, across jobs.  What it
// has of a job when the job or the range ends goes to slot job + warp (which grows from one
// such segment to the next, so it is unique); the join adds up a job's slots.  (A grid of
// requests by fixed ranges took 67 us for 256 requests of 1 to 1,500 tokens, 175 MB: most
// of its blocks were empty or short.)
//
// The products are m16n8k16 steps of one warp, S^T = K Q^T (16 keys by 8 rows) and
// O^T = V^T P^T (16 values by 8 rows): with the rows on the short side few of them waste
// little.  Each warp copies its blocks into shared-memory stages of its own, two blocks ahead
// (asynchronous copies: what is in flight costs no registers; with the next block in registers
// instead, the same took longer), and reads operands from there in 16-byte pieces:
//   * keys: the order of the contraction index is free, so lane (g, t) = (lane / 4,
//     lane % 4) takes chunks t, t + 4, ... (eight values each) of keys g and g + 8, and the
//     queries are laid out the same way;
//   * values: the order of the output rows is free, so lane (g, t) takes chunks g and g + 8
//     of keys 2t, 2t + 1, 2t + 8 and 2t + 9, and rows g and g + 8 of step (i, e) are values e
//     and e + 4 of chunk 8 i + g: one byte permutation makes each operand register;
//   * probabilities: rounded to the data's type, which the product takes them in (their sum is of
//     the unrounded ones); one 8 x 8 transposition between registers turns S^T into P^T.
// Chunk c of row r stands at c ^ (r & 6) ^ 4 (r & 1): both ways of reading then take eight
// different bank groups at a time.
// Measured (32 + 8 heads of 128, bf16): 256 requests of 1 to 1,500 tokens, 175 MB: 50 us
// with the join of the results.
// ---------------------------------------------------------------------------------
constexpr int kOwnWarps = 4;

__device__ __forceinline__ uint32_t transposed8x8(uint32_t x) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}

__device__ __forceinline__ uint32_t word(const uint4& u, int i) { return i == 0 ? u.x : i == 1 ? u.y : i == 2 ? u.z : u.w; }

constexpr int kBlockKeys = 16;
constexpr int kMinRange = 2;  // blocks a warp takes at least
constexpr int kStages = 3;

struct PagesPlan {
    int own_jobs, tiles;  // jobs of own pages: `tiles` of them a request
    int prefix_jobs;      // 0: the prefix is not taken here
    int warps;            // of each key head
    bool alone;           // the only kernel of the call before the join
    // Results: [slots][kv_heads][8 * NT][dim], their log2-sum-exp, and of each job its first
    // warp and how many warps it has.
    float* o;
    float* lse;
    int2* where;
};

// A block of keys: its job, the job's keys, its number in the job and in all.
struct Cursor {
    int job, keys, block, at;
};

__device__ __forceinline__ int job_keys(const SharedArgs& a, const PagesPlan& pl, int job) {
    if (job >= pl.own_jobs) return (int)a.prefix_len;
    return min(max(a.lengths[job / pl.tiles], 0), a.table_width << a.page_shift);
}

template <class H, int D, int NT>
__global__ void __launch_bounds__(kOwnWarps * 32, NT == 1 && D == 64 ? 4 : 2)
    pages_kernel(const __grid_constant__ SharedArgs a, const __grid_constant__ PagesPlan pl) {
    using T = typename H::type;
    constexpr int KC = D / 32, VC = D / 64;  // chunks a lane holds of a key, of a value row
    constexpr int kThreadsHere = kOwnWarps * 32;
    __shared__ int s_sum[kThreadsHere + 1];
    if (pl.alone) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int tid = threadIdx.x, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int group = a.heads / a.kv_heads, jobs = pl.own_jobs + pl.prefix_jobs;
    const int warp_all = blockIdx.x * kOwnWarps + (tid >> 5);
    const int kh = warp_all % a.kv_heads, warp = warp_all / a.kv_heads;  // key heads fastest: neighbours in memory
    auto blocks_of = [&](int job) { return (job_keys(a, pl, job) + kBlockKeys - 1) / kBlockKeys; };

    // Blocks before each thread's share of the jobs.
    const int per = (jobs + kThreadsHere - 1) / kThreadsHere;
    int mine = 0;
    for (int j = tid * per; j < min(jobs, (tid + 1) * per); ++j) {
        const int n = blocks_of(j);
        mine += n;
        if (n == 0 && blockIdx.x == 0) pl.where[j] = make_int2(0, 0);  // the others' is written with their first block
    }
    s_sum[tid + 1] = mine;
    if (tid == 0) s_sum[0] = 0;
    __syncthreads();
    if (tid < 32) {  // four entries a lane
        int v[kThreadsHere / 32], sum = 0;
#pragma unroll
        for (int i = 0; i < kThreadsHere / 32; ++i) sum += v[i] = s_sum[1 + lane * (kThreadsHere / 32) + i];
        int incl = sum;
#pragma unroll
        for (int e = 1; e < 32; e <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, incl, e);
            if (lane >= e) incl += u;
        }
        int run = incl - sum;
#pragma unroll
        for (int i = 0; i < kThreadsHere / 32; ++i) s_sum[1 + lane * (kThreadsHere / 32) + i] = run += v[i];
    }
    __syncthreads();
    const int all = s_sum[kThreadsHere], range = max(kMinRange, (all + pl.warps - 1) / pl.warps);
    const int begin = (int)min((long long)warp * range, (long long)all), end = min(all, begin + range);
    // Behind the prefix's tiles this grid starts before they end, and the join is ordered behind
    // this grid alone: it must not end before the tiles have.  One block that waits at its end
    // is enough for that; the others make room for the next ones.
    auto leave = [&] {
        if (blockIdx.x + 1 == gridDim.x) asm volatile("griddepcontrol.wait;" ::: "memory");
    };
    if (warp >= pl.warps || begin >= end) {
        leave();
        return;
    }

    // The job of the warp's first block: the share that holds it, then the job in the share.
    Cursor cur;
    {
        int lo = 0, hi = kThreadsHere;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s_sum[mid] <= begin) lo = mid; else hi = mid;
        }
        int at = s_sum[lo], job = lo * per, n = blocks_of(job);
        while (at + n <= begin) {
            at += n;
            n = blocks_of(++job);
        }
        cur = {job, job_keys(a, pl, job), begin - at, begin};
    }
    // The block after c; past the warp's range its contents do not matter.
    auto after = [&](Cursor c) {
        ++c.at;
        ++c.block;
        if (c.block * kBlockKeys >= c.keys && c.at < end) {
            c.block = 0;
            do c.keys = job_keys(a, pl, ++c.job);
            while (c.keys == 0);
        }
        return c;
    };
    auto page_of = [&](const Cursor& c) {
        if (c.at >= end) return -1;
        const int i = (c.block * kBlockKeys) >> a.page_shift;
        return c.job >= pl.own_jobs ? a.prefix_pages[i] : a.table[(long long)(c.job / pl.tiles) * a.table_stride + i];
    };
    const int mask = (1 << a.page_shift) - 1;
    // Stages of this warp: 16 rows of keys, 16 of values.  16 keys lie in one page; rows past
    // the job's keys are filled with zeros, nothing is read for them.
    extern __shared__ __align__(128) uint8_t stages[];
    constexpr int kChunks = D / 8, kRowBytes = D * 2, kHalf = kBlockKeys * kRowBytes;
    constexpr int kRowStep = 32 / kChunks;  // rows a pass of the warp copies
    const uint32_t stage0 = tc::smem_u32(stages) + (tid >> 5) * kStages * 2 * kHalf;
    auto place = [](int row, int chunk) { return row * kRowBytes + ((chunk ^ (row & 6) ^ ((row & 1) << 2)) << 4); };
    const int chunk = lane % kChunks, row0 = lane / kChunks;
    const bool here = chunk * 8 < a.dim;
    const T* const k_lane = static_cast<const T*>(a.k_cache.p) + kh * a.k_cache.head + row0 * a.k_cache.tok + (here ? chunk * 8 : 0);
    const T* const v_lane = static_cast<const T*>(a.v_cache.p) + kh * a.v_cache.head + row0 * a.v_cache.tok + (here ? chunk * 8 : 0);
    const long long k_step = kRowStep * a.k_cache.tok, v_step = kRowStep * a.v_cache.tok;
    auto request = [&](const Cursor& c, int pg, int stage) {
        const int first = c.block * kBlockKeys;
        const int left = pg >= 0 && pg < a.n_pages && c.at < end && here ? c.keys - first - row0 : 0;
        const T* kp = k_lane + pg * a.k_cache.page + (first & mask) * a.k_cache.tok;
        const T* vp = v_lane + pg * a.v_cache.page + (first & mask) * a.v_cache.tok;
        const uint32_t dst = stage0 + stage * 2 * kHalf;
#pragma unroll
        for (int i = 0; i < kBlockKeys / kRowStep; ++i) {
            const bool some = i * kRowStep < left;
            const uint32_t at = dst + place(row0 + i * kRowStep, chunk);
            attn::copy16(at, some ? static_cast<const void*>(kp) : a.k_cache.p, some);
            attn::copy16(at + kHalf, some ? static_cast<const void*>(vp) : a.v_cache.p, some);
            kp += k_step;
            vp += v_step;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto piece = [&](uint32_t base, int row, int ch) {
        uint4 u;
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(base + place(row, ch)));
        return u;
    };
    // Rows of a job: row r is query head kh * group + (m0 + r) % group of request
    // b + (m0 + r) / group.
    auto first_row = [&](int job) {
        return job >= pl.own_jobs ? make_int2(0, (job - pl.own_jobs) * 8 * NT) : make_int2(job / pl.tiles, job % pl.tiles * 8 * NT);
    };
    auto rows_of = [&](int job) {
        return min(8 * NT, job >= pl.own_jobs ? a.n_requests * group - (job - pl.own_jobs) * 8 * NT
                                              : group - job % pl.tiles * 8 * NT);
    };
    uint32_t qb[NT][2 * KC][2];
    auto load_q = [&](int job) {  // laid out as the keys are
        const int2 bm = first_row(job);
        const int n_rows = rows_of(job);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = nt * 8 + g;
            const T* q = static_cast<const T*>(a.q.p);
            if (r < n_rows) q += (long long)(bm.x + (bm.y + r) / group) * a.q.tok + (kh * group + (bm.y + r) % group) * a.q.head;
#pragma unroll
            for (int i = 0; i < KC; ++i) {
                const int ch = (i * 4 + t) * 8;
                uint4 u = make_uint4(0, 0, 0, 0);
                if (ch < a.dim && r < n_rows) u = *reinterpret_cast<const uint4*>(q + ch);
                qb[nt][2 * i][0] = u.x; qb[nt][2 * i][1] = u.y;
                qb[nt][2 * i + 1][0] = u.z; qb[nt][2 * i + 1][1] = u.w;
            }
        }
    };

    float o[NT][VC][4][4];
    float m[NT][2], l[NT][2];  // of rows 2t and 2t + 1; l over this lane's keys only
    auto clear = [&] {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
            for (int i = 0; i < VC; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int c = 0; c < 4; ++c) o[nt][i][e][c] = 0.0f;
        }
    };
    auto flush = [&](int job) {
        const long long slot = ((long long)(job + warp) * a.kv_heads + kh) * (8 * NT);
        const int n_rows = rows_of(job);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = nt * 8 + 2 * t + h;
                float sum = l[nt][h];
#pragma unroll
                for (int e = 4; e < 32; e *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, e);
                if (r >= n_rows) continue;
                const float inv = sum > 0.0f ? 1.0f / sum : (sum == 0.0f ? 0.0f : sum);
#pragma unroll
                for (int i = 0; i < VC; ++i) {
                    const int d = (i * 8 + g) * 8;
                    if (d >= a.dim) continue;
                    float4* dst = reinterpret_cast<float4*>(pl.o + (slot + r) * a.dim + d);
                    dst[0] = make_float4(o[nt][i][0][h] * inv, o[nt][i][1][h] * inv, o[nt][i][2][h] * inv, o[nt][i][3][h] * inv);
                    dst[1] = make_float4(o[nt][i][0][2 + h] * inv, o[nt][i][1][2 + h] * inv, o[nt][i][2][2 + h] * inv,
                                         o[nt][i][3][2 + h] * inv);
                }
                if (g == 0) pl.lse[slot + r] = m[nt][h] + log2f(sum);
            }
        __syncwarp();
        clear();
    };

    Cursor next = after(cur), then = after(next);
    {
        const int pg0 = page_of(cur), pg1 = page_of(next);
        request(cur, pg0, 0);
        request(next, pg1, 1);
    }
    int pg = page_of(then), stage = 0;
    load_q(cur.job);
    clear();
    const float scale = a.scale * kLog2e;
    while (true) {
        if (cur.block == 0 && kh == 0 && lane == 0) {
            const int last = cur.at + (cur.keys + kBlockKeys - 1) / kBlockKeys - 1;
            pl.where[cur.job] = make_int2(warp, last / range - warp + 1);
        }
        __syncwarp();  // every lane is done with the stage that is filled next
        request(then, pg, stage == 0 ? 2 : stage - 1);
        const Cursor last = after(then);
        pg = page_of(last);
        asm volatile("cp.async.wait_group 2;" ::: "memory");
        __syncwarp();
        const uint32_t sk = stage0 + stage * 2 * kHalf, sv = sk + kHalf;
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
#pragma unroll
        for (int i = 0; i < KC; ++i) {
            const uint4 lo = piece(sk, g, i * 4 + t), hi = piece(sk, g + 8, i * 4 + t);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                attn::mma16816<H>(s[nt], lo.x, hi.x, lo.y, hi.y, qb[nt][2 * i][0], qb[nt][2 * i][1]);
                attn::mma16816<H>(s[nt], lo.z, hi.z, lo.w, hi.w, qb[nt][2 * i + 1][0], qb[nt][2 * i + 1][1]);
            }
        }
        const bool ends = next.at >= end || next.job != cur.job;
        if (next.at < end && next.job != cur.job) load_q(next.job);
        const int key = cur.block * kBlockKeys + g;
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float top[2];
#pragma unroll
            for (int c = 0; c < 4; ++c) s[nt][c] = key + (c >> 1) * 8 < cur.keys ? s[nt][c] * scale : -INFINITY;
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
        for (int i = 0; i < VC; ++i) {
            uint4 vf[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) vf[r] = piece(sv, 2 * t + (r & 1) + (r >> 1) * 8, i * 8 + g);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t sel = (e & 1) ? 0x7632u : 0x5410u;
                const uint32_t a0 = __byte_perm(word(vf[0], e / 2), word(vf[1], e / 2), sel);
                const uint32_t a1 = __byte_perm(word(vf[0], e / 2 + 2), word(vf[1], e / 2 + 2), sel);
                const uint32_t a2 = __byte_perm(word(vf[2], e / 2), word(vf[3], e / 2), sel);
                const uint32_t a3 = __byte_perm(word(vf[2], e / 2 + 2), word(vf[3], e / 2 + 2), sel);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) attn::mma16816<H>(o[nt][i][e], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
            }
        }
        if (ends) flush(cur.job);
        if (next.at >= end) break;
        cur = next;
        next = then;
        then = last;
        stage = stage == kStages - 1 ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    leave();
}

template <class H, int D, int NT>
void launch_pages_as(const SharedArgs& a, const PagesPlan& pl, unsigned blocks, bool after_tiles, cudaStream_t st) {
    constexpr int smem = kOwnWarps * kStages * 2 * kBlockKeys * D * 2;
    static std::atomic<uint64_t> devices{0};
    opt_in(devices, pages_kernel<H, D, NT>, smem, [] {});
    launch_ahead(pages_kernel<H, D, NT>, blocks, kOwnWarps * 32, smem, after_tiles, st, a, pl);
    VGPU_LAUNCH("pages_kernel");
}

template <class H>
void launch_pages(const SharedArgs& a, const PagesPlan& pl, int nt, bool after_tiles, cudaStream_t st) {
    if (pl.own_jobs + pl.prefix_jobs == 0) return;
    const unsigned blocks = (unsigned)ceil_div((long long)pl.warps * a.kv_heads, kOwnWarps);
    // After the prefix's tiles: nothing here depends on them, and they leave SMs idle, so
    // the blocks may start as soon as all of the tiles' blocks have; the last one ends after them.
    if (a.dim <= 64) {
        if (nt == 1) launch_pages_as<H, 64, 1>(a, pl, blocks, after_tiles, st);
        else launch_pages_as<H, 64, 2>(a, pl, blocks, after_tiles, st);
    } else {
        if (nt == 1) launch_pages_as<H, 128, 1>(a, pl, blocks, after_tiles, st);
        else launch_pages_as<H, 128, 2>(a, pl, blocks, after_tiles, st);
    }
}

// ---------------------------------------------------------------------------------
// Join of partial results: with L_i their log2-sum-exp and M = max L_i, the weights are
// 2^(L_i - M) and out = sum w_i O_i / sum w_i.  One warp a row, one part a lane.  A row's
// parts are `splits` of the tile kernel ([splits][rows][dim]) and the slots of its jobs in
// the pages kernel.
// ---------------------------------------------------------------------------------
struct JoinArgs {
    long long rows;  // n * heads
    int heads, kv_heads, dim;
    int splits;
    const float* tile_o;
    const float* tile_lse;
    bool paged;
    int nt;
    PagesPlan pages;
    bool own;  // there are own pages
    void* out;
    float* lse;
};

template <class H>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ JoinArgs a) {
    const int lane = threadIdx.x & 31;
    const long long row = blockIdx.x * 4LL + (threadIdx.x >> 5);
    asm volatile("griddepcontrol.wait;" ::: "memory");  // no wait unless launched ahead
    if (row >= a.rows) return;
    const bool live = lane * 4 < a.dim;
    // Slots of the row's own job, then of its prefix job.
    const int head = (int)(row % a.heads), group = a.heads / a.kv_heads, kh = head / group, g = head - kh * group;
    const int b = (int)(row / a.heads);
    int own = 0, shared = 0;
    long long own_at = 0, shared_at = 0;  // rows of slots
    if (a.paged) {
        const int tall = 8 * a.nt;
        if (a.own) {
            const int job = b * a.pages.tiles + g / tall;
            const int2 w = a.pages.where[job];
            own = w.y;
            own_at = ((long long)(job + w.x) * a.kv_heads + kh) * tall + g % tall;
        }
        if (a.pages.prefix_jobs) {
            const long long r = (long long)b * group + g;
            const int job = a.pages.own_jobs + (int)(r / tall);
            const int2 w = a.pages.where[job];
            shared = w.y;
            shared_at = ((long long)(job + w.x) * a.kv_heads + kh) * tall + (int)(r % tall);
        }
    }
    const long long slot_rows = (long long)a.kv_heads * 8 * a.nt;
    const int parts = a.splits + own + shared;
    float m = -INFINITY, total = 0.0f;
    bool nan = false;
    float4 o = make_float4(0, 0, 0, 0);
    for (int p0 = 0; p0 < parts; p0 += 32) {
        const int p = p0 + lane;
        const float* src = a.pages.o;  // the lane's part
        float x = -INFINITY;
        if (p < a.splits) {
            x = a.tile_lse[p * a.rows + row];
            src = a.tile_o + (p * a.rows + row) * a.dim;
        } else if (p < parts) {
            const int i = p - a.splits;
            const long long at = i < own ? own_at + i * slot_rows : shared_at + (i - own) * slot_rows;
            x = a.pages.lse[at];
            src = a.pages.o + at * a.dim;
        }
        float up = fmaxf(m, x);
        nan |= __any_sync(0xffffffffu, isnan(x)) != 0;
#pragma unroll
        for (int e = 16; e > 0; e >>= 1) up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, e));
        const float ref = up == -INFINITY ? 0.0f : up, f = exp2f(m - ref), w = exp2f(x - ref);
        m = up;
        total = total * f + w;  // this lane's share
        o = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
        // Parts without keys may hold anything.  One whose weight is zero in 32 bits takes part: a
        // value in it that is not finite is seen by the row.
        unsigned some = __ballot_sync(0xffffffffu, x != -INFINITY);
        while (some) {
            float4 v[4];
            float wi[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = some ? __ffs(some) - 1 : -1, from = i < 0 ? 0 : i;
                wi[e] = __shfl_sync(0xffffffffu, w, from);
                const float* s = reinterpret_cast<const float*>(
                    __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), from));
                v[e] = make_float4(0, 0, 0, 0);
                if (i < 0) wi[e] = 0.0f;
                else if (live) v[e] = *reinterpret_cast<const float4*>(s + lane * 4);
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
        *reinterpret_cast<uint2*>(static_cast<typename H::type*>(a.out) + row * a.dim + lane * 4) =
            make_uint2(H::pack(o.x * inv, o.y * inv), H::pack(o.z * inv, o.w * inv));
    if (a.lse && lane == 0) a.lse[row] = nan ? __int_as_float(0x7fc00000) : (m + log2f(total)) / kLog2e;
}

// `ahead`: the one kernel whose results are joined is the last one queued, and lets this one
// be set up while it runs.
void launch_join(bool f16, const JoinArgs& a, bool ahead, cudaStream_t st) {
    launch_ahead(f16 ? join_kernel<F16> : join_kernel<Bf16>, (unsigned)ceil_div(a.rows, 4), 128, 0, ahead, st, a);
    VGPU_LAUNCH("join_kernel");
}

size_t part_bytes(long long parts, long long rows, int dim) { return (size_t)(parts * rows * (dim + 1)) * sizeof(float); }

// How many ways to split the keys: as many as give each SM a block, but at least four key
// tiles a split.
int splits_for(long long blocks, long long key_tiles) {
    const long long by_sms = kSms / std::max<long long>(blocks, 1), by_keys = key_tiles / 4;
    return (int)std::max<long long>(1, std::min<long long>({by_sms, by_keys, 64}));
}

constexpr size_t kCounterBytes = 16;

struct PromptPlan {
    bool small;       // small blocks, see attn_short.cuh
    long long tiles;  // upper bound of block tiles: the requests' lengths are on the device
    int splits;
};
PromptPlan prompt_plan(const PromptArgs& a) {
    const int group = a.heads / a.kv_heads;
    PromptPlan pl;
    const long long blocks = ((a.n_q + 2 * (kRows / group) - 1) / (2 * (kRows / group)) + a.n_requests) * a.kv_heads;
    const int rows = blocks <= kSms ? kShortMeanRowsFew : kShortMeanRows;
    pl.small = group <= attn::kShortRows && a.n_q * group <= (long long)rows * a.n_requests &&
               a.n_k <= (long long)kShortMeanKeys * a.n_requests;
    if (pl.small) {
        pl.tiles = a.n_q / (attn::kShortRows / group) + a.n_requests + 2;
        pl.splits = 1;
        return pl;
    }
    const int span = 2 * (kRows / group);
    pl.tiles = a.n_q / span + a.n_requests + 2;
    const long long likely = (a.n_q + span - 1) / span + std::max(a.n_requests - 1, 0);
    pl.splits = splits_for(likely * a.kv_heads, a.n_k / kKeys / std::max(a.n_requests, 1));
    return pl;
}

// Workspace of a shared-prefix call: the tile kernel's parts, the pages kernel's slots.
struct SharedPlan {
    int splits;  // of the prefix on the tensor cores' tiles; 0: the pages kernel takes it
    int nt;
    PagesPlan pages;
    // In floats: the tiles' rows come first, then the slots' rows (both 16-byte aligned, as
    // dim is a multiple of 8), then both log2-sum-exps and the jobs' slots.
    size_t slots_at, tile_lse_at, slot_lse_at, where_at;
    size_t bytes;
};
SharedPlan shared_plan(const SharedArgs& a) {
    SharedPlan p{};
    const int group = a.heads / a.kv_heads;
    p.nt = group > 8 ? 2 : 1;
    const int tall = 8 * p.nt;
    const long long rows = (long long)a.n_requests * a.heads;
    const long long row_tiles = ((long long)a.n_requests * group + tall - 1) / tall;
    p.pages.tiles = (group + tall - 1) / tall;
    p.pages.own_jobs = a.table_width ? a.n_requests * p.pages.tiles : 0;
    if (a.prefix_len) {
        if (row_tiles <= kFewRowTiles) p.pages.prefix_jobs = (int)row_tiles;
        else p.splits = splits_for((long long)ceil_div(a.n_requests, 2 * (kRows / group)) * a.kv_heads, a.prefix_len / kKeys);
    }
    const long long jobs = (long long)p.pages.own_jobs + p.pages.prefix_jobs;
    // as many warps as are resident at once, and no more than the keys can use
    const long long cap = (((long long)a.table_width << a.page_shift) + kBlockKeys - 1) / kBlockKeys;
    const long long most = p.pages.own_jobs * cap + p.pages.prefix_jobs * ((a.prefix_len + kBlockKeys - 1) / kBlockKeys);
    // (twice that after the tiles: their SMs come free one by one)
    const long long resident = (long long)kSms * (p.nt == 1 && a.dim <= 64 ? 4 : 2) * kOwnWarps * (p.splits ? 2 : 1) / a.kv_heads;
    p.pages.warps = (int)std::max<long long>(1, std::min<long long>(resident, (most + kMinRange - 1) / kMinRange));
    const size_t slot_rows = jobs ? (size_t)(jobs + p.pages.warps) * a.kv_heads * tall : 0;
    p.slots_at = (size_t)p.splits * rows * a.dim;
    p.tile_lse_at = p.slots_at + slot_rows * a.dim;
    p.slot_lse_at = p.tile_lse_at + (size_t)p.splits * rows;
    p.where_at = (p.slot_lse_at + slot_rows + 1) / 2 * 2;
    p.bytes = kCounterBytes + (p.where_at + 2 * (size_t)jobs) * sizeof(float);
    return p;
}

}  // namespace

size_t prompt_attention_workspace(const PromptArgs& a) {
    if (a.n_q == 0) return 0;
    const PromptPlan pl = prompt_plan(a);
    // the counter of pieces comes first
    return pl.splits > 1 ? kCounterBytes + part_bytes(pl.splits, a.n_q * a.heads, a.dim)
                         : (!pl.small && counted(pl.tiles * a.kv_heads) ? kCounterBytes : 0);
}

void launch_prompt_attention(const PromptArgs& a, cudaStream_t st) {
    const PromptPlan pl = prompt_plan(a);
    const long long rows = a.n_q * a.heads;
    TileParams p{};
    if (pl.small) {
        p.heads = a.heads;
        p.kv_heads = a.kv_heads;
        p.group = a.heads / a.kv_heads;
        p.dim = a.dim;
        p.tile_tokens = attn::kShortRows / p.group;
        p.n_q = (int)a.n_q;
        p.q = a.q;
    } else {
        fill_queries(p, a.f16, a.q, a.heads, a.kv_heads, a.dim, a.n_q);
    }
    p.n_k = (int)a.n_k;
    if (a.n_k && !pl.small) {
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
    p.part_o = static_cast<float*>(a.workspace) + kCounterBytes / sizeof(float);
    p.part_lse = p.part_o + pl.splits * rows * a.dim;
    if (pl.small) {
        launch_short(p, a.f16, pl.tiles * a.kv_heads, st);
        return;
    }
    launch_tiles<false>(p, a.f16, pl.tiles * a.kv_heads * pl.splits, static_cast<int*>(a.workspace), st);
    if (!p.part) return;
    JoinArgs j{};
    j.rows = rows;
    j.heads = a.heads;
    j.kv_heads = a.kv_heads;
    j.dim = a.dim;
    j.splits = pl.splits;
    j.tile_o = p.part_o;
    j.tile_lse = p.part_lse;
    j.out = a.out;
    j.lse = a.lse;
    launch_join(a.f16, j, false, st);
}

size_t shared_attention_workspace(const SharedArgs& a) { return a.n_requests == 0 ? 0 : shared_plan(a).bytes; }

void launch_shared_attention(const SharedArgs& a, cudaStream_t st) {
    SharedPlan sp = shared_plan(a);
    const long long rows = (long long)a.n_requests * a.heads;
    float* const base = static_cast<float*>(a.workspace) + kCounterBytes / sizeof(float);
    JoinArgs j{};
    j.rows = rows;
    j.heads = a.heads;
    j.kv_heads = a.kv_heads;
    j.dim = a.dim;
    j.splits = sp.splits;
    j.tile_o = base;
    j.tile_lse = base + sp.tile_lse_at;
    if (sp.splits) {
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
        p.splits = sp.splits;
        p.part = true;
        p.part_o = base;
        p.part_lse = base + sp.tile_lse_at;
        launch_tiles<true>(p, a.f16, (long long)ceil_div(a.n_requests, 2 * p.tile_tokens) * a.kv_heads * p.splits,
                           static_cast<int*>(a.workspace), st);
    }
    sp.pages.alone = sp.splits == 0 && sp.pages.own_jobs + sp.pages.prefix_jobs > 0;
    sp.pages.o = base + sp.slots_at;
    sp.pages.lse = base + sp.slot_lse_at;
    sp.pages.where = reinterpret_cast<int2*>(base + sp.where_at);
    if (a.f16) launch_pages<F16>(a, sp.pages, sp.nt, sp.splits > 0, st);
    else launch_pages<Bf16>(a, sp.pages, sp.nt, sp.splits > 0, st);
    j.paged = true;
    j.nt = sp.nt;
    j.pages = sp.pages;
    j.own = sp.pages.own_jobs > 0;
    j.out = a.out;
    j.lse = a.lse;
    launch_join(a.f16, j, sp.pages.alone, st);
}

}  // namespace vgpu

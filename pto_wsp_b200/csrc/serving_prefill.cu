// Attention over a paged KV cache held in 8 bits, for many query rows per request (prefill chunks), on tcgen05.
//
// The mathematics is that of the kernel for few rows: with code c and page scale s, the logit takes s_k, and the weight
// w = 2^(a s_k q.c_k + log2 s_v - M) takes s_v, so both products run on codes, which f16 holds exactly, and the
// denominator sums w / s_v.  w is kept between 2^7 and 2^15 of its row's largest, as f16 for the second product; sums are
// f32.  A group of 16 tokens is in one page, so a row pays one product per group for the scales, not one per key.
//
// A CTA works on up to 256 rows (tokens x heads of one group) of one request and KV head, as two tiles A and B of 128 rows
// that share every converted K and V tile of 128 tokens:
//   warps 0-15      softmax, eight warps per tile: a row's two threads take 64 keys each and agree on the maximum through
//                   shared memory.  The row's q as f16 into shared memory, then per step the maximum, the weights as
//                   f16 over the scores they came from in TMEM, the rescaling of O; at the end O / sum to the row, or
//                   to the workspace.  One thread per row took 3500 cycles a step, longer than both tiles' MMAs, and
//                   nothing of the row's chain -- scores, softmax, product, scores -- overlaps within a tile
//   warps 16-19     codes from the landing place in shared memory, converted into the 128-byte-swizzled layouts of the
//                   MMAs: K as rows of dims (K-major), V as rows of tokens (MN-major)
//   warp 20         issues the MMAs from one thread: S_A S_B | PV_A S_A' | PV_B S_B' | ...: while the tensor cores work
//                   on one tile's products the other tile's softmax runs
//   warp 21         asks for the codes by TMA, a box per 16 tokens, and gives the groups' scales
// TMEM: S_A, S_B (128 columns each; P over the first 32 of either half), O_A, O_B.  The tensor pipe runs one thread's MMAs
// in order, so S' may follow PV into the columns that P is read from, and S' being done means that PV is.
//
// Bound by the chain score - softmax - product of a tile, beside which the tensor pipe stands idle for two thirds of the
// time.  Chunks of 1142-1516 rows over 2791-6204 keys (8 KV heads, groups of four, D = 128: 355 GFLOP) take 541 us, 656
// TFLOP/s, as a whole call.  Of the main kernel's 906 thousand cycles (148 steps a CTA, 6100 a step) the tensor pipe works
// 34 %, the 2048 that both products of a step take at the full rate; instructions issue in 56 % of the cycles.  The
// list takes 7 us, the join 25 and the few-rows kernel and its join 23, one after the other and cold.
//
// Work is dealt out as for few rows: the steps of all (tile pair, head) tasks stand in one line, every CTA takes an equal
// part, and tasks that this cuts are joined by a second launch.  A first launch lists the tile pairs.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "serving.hpp"
#include "serving_kv8.cuh"
#include "tc_common.cuh"

namespace ptowsp::dev {

namespace {

using namespace tc;

constexpr int kRows = 256;               // of a task: two tiles of 128
constexpr int kKeys = 128;               // per step
constexpr int kSoftmaxWarps = 16;        // eight per tile: two threads per row
constexpr int kConvertWarp = kSoftmaxWarps, kMmaWarp = kConvertWarp + 4, kLoadWarp = kMmaWarp + 1;
constexpr int kThreads = (kMmaWarp + 4) * 32;
// Registers of a thread: 80 at launch, dealt out anew by role: 4 * 128 * 88 + 128 * 72 + 128 * 56 = 768 * 80.
constexpr int kListThreads = 1024;
constexpr float kNone = -1.7e38f;        // M before the first visible key
constexpr float kLeast = 1e-30f;         // of a score's factor: positive whatever the scales, and nothing to a finite score

// One pair of row tiles of a request, and the steps before its first one.
struct Pair {
    int token0, row0, rows;  // the request's first q token; the pair's first row and its number of rows
    int base;                // row j's last key: base + (row0 + j) / group
    int lo, hi;              // keys to walk, lo a multiple of 16
    int seen;                // the first key that any row sees
    int units;               // steps per head
    int64_t before;
    int request, pad[1];
};
static_assert(sizeof(Pair) == 48, "three 16-byte loads");

struct PrefillArgs {
    AttendArgs a;
    Pair* pairs;        // the list, in the workspace
    int64_t* total;     // [0] steps, [1] pairs
    float* parts;       // two partial results per CTA: [rows][M, l], then [rows][D]
    int threshold;      // requests with more rows than this are taken
};

__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
// With its wait: the values may be used at once.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}

// S = Q.K^T over D dims: D / 16 MMAs of K = 16 in one asm block, so that the issuing thread spends one addition per
// operand.  Both are K-major, 128-byte swizzle: +32 bytes per 16 dims, +16 KB per 64 (descriptors count 16 bytes).
template <int D>
__device__ __forceinline__ void mma_scores(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 x, y;\n\t"
        "setp.ne.b32 p, %3, %3;\n\tsetp.eq.b32 q, %3, %3;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "add.s64 x, %1, 2;\n\tadd.s64 y, %2, 2;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, q;\n\t"
        "add.s64 x, %1, 4;\n\tadd.s64 y, %2, 4;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, q;\n\t"
        "add.s64 x, %1, 6;\n\tadd.s64 y, %2, 6;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, q;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc)
        : "memory");
    if constexpr (D == 128)
        asm volatile(
            "{\n\t.reg .pred q;\n\t.reg .b64 x, y;\n\t"
            "setp.eq.b32 q, %3, %3;\n\t"
            "add.s64 x, %1, 1024;\n\tadd.s64 y, %2, 1024;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, q;\n\t"
            "add.s64 x, %1, 1026;\n\tadd.s64 y, %2, 1026;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, q;\n\t"
            "add.s64 x, %1, 1028;\n\tadd.s64 y, %2, 1028;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, q;\n\t"
            "add.s64 x, %1, 1030;\n\tadd.s64 y, %2, 1030;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, q;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc)
            : "memory");
}
// O (+)= P.V over 128 tokens: P from TMEM (two tokens per column, 8 columns per MMA, the second 64 tokens 64 columns on),
// V MN-major (+2 KB per 16 tokens).
__device__ __forceinline__ void mma_values(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 y;\n\t.reg .b32 x;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 q, %4, %4;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "add.u32 x, %1, 8;\n\tadd.s64 y, %2, 128;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [x], y, %3, q;\n\t"
        "add.u32 x, %1, 16;\n\tadd.s64 y, %2, 256;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [x], y, %3, q;\n\t"
        "add.u32 x, %1, 24;\n\tadd.s64 y, %2, 384;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [x], y, %3, q;\n\t"
        "add.u32 x, %1, 64;\n\tadd.s64 y, %2, 512;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [x], y, %3, q;\n\t"
        "add.u32 x, %1, 72;\n\tadd.s64 y, %2, 640;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [x], y, %3, q;\n\t"
        "add.u32 x, %1, 80;\n\tadd.s64 y, %2, 768;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [x], y, %3, q;\n\t"
        "add.u32 x, %1, 88;\n\tadd.s64 y, %2, 896;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [x], y, %3, q;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accum)
        : "memory");
}

// One arrival for the warp, after what all its lanes did (arrivals on one barrier go one by one).
__device__ __forceinline__ void arrive_warp(uint32_t bar) {
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// A bounded wait: false when another role gave up or this one does.
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity, volatile int* abort_flag, int32_t* status) {
    uint64_t start = 0;
    for (uint32_t it = 0;; ++it) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((it & 255u) == 255u) {
            if (*abort_flag) return false;
            const uint64_t now = globaltimer();
            if (start == 0) {
                start = now;
            } else if (now - start > kTimeoutNs) {
                if (status) atomicOr(status, PTOWSP_SERVING_TIMEOUT);
                *abort_flag = 1;
                return false;
            }
        }
    }
}

// ---------------------------------------------------------------------------
// The list of tile pairs
// ---------------------------------------------------------------------------

__device__ __forceinline__ int64_t block_inclusive(int64_t v, int64_t* part, int64_t* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t o = __shfl_up_sync(~0u, v, d);
        if (lane >= d) v += o;
    }
    __syncthreads();
    if (lane == 31) part[warp] = v;
    __syncthreads();
    int64_t p = part[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t o = __shfl_up_sync(~0u, p, d);
        if (lane >= d) p += o;
    }
    *total = __shfl_sync(~0u, p, 31);
    const int64_t before = __shfl_sync(~0u, p, warp ? warp - 1 : 0);
    return v + (warp ? before : 0);
}

struct Ask {  // a request as this kernel sees it
    int token0, nq, len, pairs;
};
__device__ __forceinline__ Ask ask_of(const PrefillArgs& g, int r, int* flags) {
    const AttendArgs& a = g.a;
    Ask q;
    q.token0 = a.q_start ? a.q_start[r] : r;
    q.nq = (a.q_start ? a.q_start[r + 1] : r + 1) - q.token0;
    if (q.token0 < 0 || q.nq < 0 || q.token0 + static_cast<int64_t>(q.nq) > a.tokens || q.nq > a.max_q) {
        *flags |= PTOWSP_SERVING_LENGTH;
        q.nq = 0;
    }
    q.len = a.kv_len[r];
    const int64_t room = static_cast<int64_t>(a.max_pages) << a.cache.page_shift;
    if (q.len < 0 || q.len > room) {
        *flags |= PTOWSP_SERVING_LENGTH;
        q.len = q.len < 0 ? 0 : static_cast<int>(room);
    }
    const int64_t rows = static_cast<int64_t>(q.nq) * a.group;
    q.pairs = rows > g.threshold ? static_cast<int>((rows + kRows - 1) / kRows) : 0;
    return q;
}

__global__ void __launch_bounds__(kListThreads) list_kernel(const __grid_constant__ PrefillArgs g, int max_pairs) {
    __shared__ int64_t part[32];
    const AttendArgs& a = g.a;
    int flags = 0;
    int64_t pairs = 0;
    // each request's pairs, one thread per request, into their places
    for (int r0 = 0; r0 < a.requests; r0 += kListThreads) {
        const int r = r0 + threadIdx.x;
        Ask q{};
        if (r < a.requests) q = ask_of(g, r, &flags);
        int64_t all;
        const int64_t end = pairs + block_inclusive(q.pairs, part, &all);
        pairs += all;
        for (int i = 0; i < q.pairs; ++i) {  // only who they are: the rest is computed in parallel below
            const int64_t at = end - q.pairs + i;
            if (at < max_pairs) {
                g.pairs[at].request = r;
                g.pairs[at].row0 = i * kRows;
            }
        }
    }
    if (pairs > max_pairs) {  // the lengths ask for more rows than there are tokens
        flags |= PTOWSP_SERVING_LENGTH;
        pairs = max_pairs;
    }
    if (flags && a.status) atomicOr(a.status, flags);
    __syncthreads();
    int64_t steps = 0;
    for (int64_t p0 = 0; p0 < pairs; p0 += kListThreads) {
        const int64_t p = p0 + threadIdx.x;
        int64_t mine = 0;
        Pair t{};
        if (p < pairs) {
            int ignore = 0;
            t.request = g.pairs[p].request;
            t.row0 = g.pairs[p].row0;
            const Ask q = ask_of(g, t.request, &ignore);
            t.token0 = q.token0;
            t.rows = static_cast<int>(min(static_cast<int64_t>(kRows), static_cast<int64_t>(q.nq) * a.group - t.row0));
            t.base = q.len - q.nq;
            const int first = t.base + t.row0 / a.group, last = t.base + (t.row0 + t.rows - 1) / a.group;
            t.hi = max(0, min(q.len, last + 1));
            if (a.window > 0 && first >= a.window) t.seen = first - a.window + 1;  // first may be far below zero
            t.lo = t.seen & ~15;
            t.units = t.hi > t.lo ? (t.hi - t.lo + kKeys - 1) / kKeys : 1;  // a task without keys writes its zeros
            mine = static_cast<int64_t>(t.units) * a.cache.kv_heads;
        }
        int64_t all;
        const int64_t end = steps + block_inclusive(mine, part, &all);
        steps += all;
        if (p < pairs) {
            t.before = end - mine;
            g.pairs[p] = t;
        }
    }
    if (threadIdx.x == 0) {
        g.total[0] = steps;
        g.total[1] = pairs;
    }
}

// The share of CTA c of n in `total` steps.
__device__ __forceinline__ int64_t share_start(int64_t total, int n, int64_t c) {
    const int64_t q = total / n, r = total - q * n;
    return c * q + (c < r ? c : r);
}
__device__ __forceinline__ int64_t share_owner(int64_t total, int n, int64_t i) {
    const int64_t q = total / n, r = total - q * n, big = r * (q + 1);
    return i < big ? i / (q + 1) : r + (i - big) / q;
}

// The last pair whose first step is at or before `at`; the whole warp looks.
__device__ __forceinline__ int find_pair(const Pair* pairs, int n, int64_t at) {
    const int lane = threadIdx.x & 31;
    int lo = 0, len = n;  // in [lo, lo + len)
    while (len > 1) {
        const int stride = (len + 31) / 32;
        const int i = lo + lane * stride;
        const bool ok = lane * stride < len && pairs[i].before <= at;
        const int k = 31 - __clz(static_cast<int>(__ballot_sync(~0u, ok)));
        lo += k * stride;
        len = min(stride, len - k * stride);
    }
    return lo;
}

// ---------------------------------------------------------------------------
// The attention
// ---------------------------------------------------------------------------

template <int D>
struct Smem {
    static constexpr int kBox = 128 * 128;               // 128 rows of 64 f16
    static constexpr int kBoxes = D / 64;
    static constexpr int kTile = kBoxes * kBox;
    static constexpr int kQ = 0;                         // two tiles
    static constexpr int kK = kQ + 2 * kTile;            // two stages
    static constexpr int kV = kK + 2 * kTile;            // two stages
    static constexpr int kLand = kV + 2 * kTile;         // codes of K, of V as they come: [128][D]
    static constexpr int kScales = kLand + 2 * kKeys * D;  // [4][3][8]: k scale, log2 of v scale, 1 / v scale of the groups
    static constexpr int kLive = kScales + 4 * 3 * 8 * 4;  // [2][8]: tokens of a landed group that are there
    static constexpr int kMeet = kLive + 2 * 8 * 4;      // [2 tiles][2 halves][128]: what a row's threads tell each other
    static constexpr int kBars = kMeet + 2 * 2 * 128 * 4;
    static constexpr int kBytes = kBars + 256;           // dynamic shared memory begins at a multiple of 1024
};
static_assert(Smem<128>::kBytes <= 232448, "227 KB of shared memory per CTA");

// The segments of a CTA's share, one after the other; every role walks them alike.
struct Walk {
    int64_t at, stop;
    int pair, head, unit;  // next segment's
    Pair p;
    int n;                 // steps of the present segment
    int unit0, head0;
    bool whole;

    __device__ bool next(const PrefillArgs& g) {
        if (at >= stop) return false;
        p = g.pairs[pair];
        unit0 = unit;
        head0 = head;
        const int64_t left = p.units - unit;
        n = static_cast<int>(left < stop - at ? left : stop - at);
        whole = n == p.units;
        at += n;
        unit = 0;
        if (++head == g.a.cache.kv_heads) {
            head = 0;
            ++pair;
        }
        return true;
    }
};

template <int FMT, int D>
__global__ void __launch_bounds__(kThreads, 1) prefill_kernel(const __grid_constant__ PrefillArgs g, const __grid_constant__ CUtensorMap k_map,
                   const __grid_constant__ CUtensorMap v_map) {
    using S = Smem<D>;
    constexpr int CH = D / 16;               // 16-byte chunks of a row of codes
    extern __shared__ __align__(1024) uint8_t smem[];
    const AttendArgs& a = g.a;
    float* scales = reinterpret_cast<float*>(smem + S::kScales);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
    const uint32_t bar0 = smem_u32(bars);
    const uint32_t q_full = bar0, k_full = bar0 + 16, k_empty = bar0 + 32, v_full = bar0 + 48, v_empty = bar0 + 64,
                   s_full = bar0 + 80, p_full = bar0 + 96, o_full = bar0 + 112, drain = bar0 + 128, l_full = bar0 + 136,
                   l_empty = bar0 + 152;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 21);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 22);
    volatile int* live = reinterpret_cast<volatile int*>(smem + S::kLive);
    volatile int* first_pair = reinterpret_cast<volatile int*>(bars + 23);
    const uint32_t meet_full = bar0 + 192;  // [2][4]: of a tile, by the row's quarter
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    const int64_t total = g.total[0];
    Walk w{};
    w.at = share_start(total, gridDim.x, blockIdx.x);
    w.stop = share_start(total, gridDim.x, blockIdx.x + 1);
    if (w.at >= w.stop) return;  // the whole CTA: nothing is set up yet
    if (smem_u32(smem) & 1023) {  // the swizzled layouts need it
        if (threadIdx.x == 0 && a.status) atomicOr(a.status, PTOWSP_SERVING_TIMEOUT);
        return;
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(q_full + 8 * i, 8);
            mbar_init(k_full + 8 * i, 4);
            mbar_init(k_empty + 8 * i, 1);
            mbar_init(v_full + 8 * i, 4);
            mbar_init(v_empty + 8 * i, 1);
            mbar_init(s_full + 8 * i, 1);
            mbar_init(p_full + 8 * i, 8);
            mbar_init(o_full + 8 * i, 1);
            mbar_init(l_full + 8 * i, 1);
            mbar_init(l_empty + 8 * i, 4);
        }
        for (int i = 0; i < 8; ++i) mbar_init(meet_full + 8 * i, 2);
        mbar_init(drain, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        const int p = find_pair(g.pairs, static_cast<int>(g.total[1]), w.at);
        if (lane == 0) *first_pair = p;
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot))
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    w.pair = *first_pair;
    {
        const Pair p = g.pairs[w.pair];
        const int64_t in = w.at - p.before;
        w.head = static_cast<int>(in / p.units);
        w.unit = static_cast<int>(in - static_cast<int64_t>(w.head) * p.units);
    }
    const uint32_t sQ = smem_u32(smem + S::kQ), sK = smem_u32(smem + S::kK), sV = smem_u32(smem + S::kV);

    if (warp < kSoftmaxWarps) {
        // ---------------- softmax: two threads per row ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 88;");
        const int x = warp >> 3;          // tile A or B
        const int half = warp >> 2 & 1;   // keys 64 half .. 64 half + 63 of a step, and as large a part of the dims
        const int row = (warp & 3) * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_cols = tmem + lanes + x * 128 + half * 64, o_cols = tmem + lanes + 256 + x * 128 + half * (D / 2);
        float* mine = reinterpret_cast<float*>(smem + S::kMeet) + (x * 2 + half) * 128 + row;
        const float* other = reinterpret_cast<float*>(smem + S::kMeet) + (x * 2 + (half ^ 1)) * 128 + row;
        const uint32_t meet_bar = meet_full + 8 * (x * 4 + (warp & 3));
        uint32_t tiles = 0, steps = 0, segments = 0, meets = 0;  // of this tile; of the CTA; of this tile; of these warps
        bool ok = true;
        // Rows of q and of the output go between memory and this tile's place in shared memory with kRowLanes lanes side by
        // side in a row; two warps share 32 rows, 16 each.  These loops and the converters' are rolled up on purpose: the
        // roles' code has to stay in the instruction cache together.  For chunks of 1100-1500 rows over 2800-6200 keys
        // (21864 steps) both rolled take 543 us; the converters unrolled over K and V 596, these loops unrolled as well 616.
        // The softmax's inner loops lose when rolled up (558), and so does the MMA thread's over the two tiles (569).
        constexpr int kRowLanes = D / 8, kRowsRead = 32 / kRowLanes;
        const auto io_lane = []() {  // read anew at either use: what follows from it would hold registers across the steps
            int i;
            asm volatile("mov.u32 %0, %%laneid;" : "=r"(i));
            return i;
        };
        const auto io_at = [&](int r, int unit) {
            return reinterpret_cast<uint4*>(smem + S::kQ + x * S::kTile + (unit >> 3) * S::kBox + r * 128 +
                                            (((unit & 7) ^ (r & 7)) << 4));
        };
        // waits for the row's other thread; both warps come here alike
        const auto meet = [&]() {
            arrive_warp(meet_bar);
            ok = __all_sync(~0u, wait_for(meet_bar, meets & 1, abort_flag, a.status));
            ++meets;
        };
        while (ok && w.next(g)) {
            const bool live = w.p.rows > x * 128;  // the whole tile
            if (!live) {
                steps += w.n;
                continue;
            }
            const int flat = w.p.row0 + x * 128 + row;
            const bool real = x * 128 + row < w.p.rows;
            const int pos = real ? w.p.base + flat / a.group : -1;
            // -- q as f16 times a power of two that brings the row's largest below 2^15: this warp's 16 rows --
            {
                const int io = io_lane(), io_unit = io % kRowLanes, io_row = (warp & 3) * 32 + half * 16 + io / kRowLanes;
                const int f0 = w.p.row0 + x * 128 + io_row;
                int j = f0 / a.group, gq = f0 - j * a.group;
#pragma unroll 1
                for (int i = 0; i < 16; i += kRowsRead) {
                    const bool there = x * 128 + io_row + i < w.p.rows;
                    const uint16_t* src = static_cast<const uint16_t*>(a.q);
                    if (there)
                        src += (w.p.token0 + static_cast<int64_t>(j)) * a.q_token_stride +
                               static_cast<int64_t>(w.head0 * a.group + gq) * a.q_head_stride + io_unit * 8;
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(io_at(io_row + i, io_unit))),
                                 "l"(src), "r"(there ? 16 : 0)
                                 : "memory");
                    for (gq += kRowsRead; gq >= a.group; gq -= a.group) ++j;
                }
                asm volatile("cp.async.wait_all;" ::: "memory");  // a lane works on what it copied itself
                const bool f16 = a.dtype == PTOWSP_F16;
                float* factors = reinterpret_cast<float*>(smem + S::kMeet) + x * 2 * 128;
#pragma unroll 1
                for (int i = 0; i < 16; i += kRowsRead) {
                    uint4* at = io_at(io_row + i, io_unit);
                    const uint4 raw = *at;
                    const uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
                    float v[8];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if (f16) {
                            const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&u[k]));
                            v[2 * k] = t.x;
                            v[2 * k + 1] = t.y;
                        } else {
                            v[2 * k] = __uint_as_float(u[k] << 16);
                            v[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
                        }
                    }
                    float m = 0.f;
#pragma unroll
                    for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(v[k]));
#pragma unroll
                    for (int d = 1; d < kRowLanes; d <<= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
                    int e = 0;
                    if (m > 0.f && m < INFINITY)
                        e = min(max(14 - (static_cast<int>(__float_as_uint(m) >> 23) - 127), -120), 120);
                    float f = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
                    if (io_unit == 0)
                        factors[io_row + i] =
                            fabsf(a.scale) * 1.4426950408889634f * __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
                    // The factor of the scores is positive, so a group's maximum is theirs and a masked score of -inf
                    // stays one: q takes the sign of the scale, or is zero with it.
                    if (a.scale < 0.f) f = -f;
                    if (a.scale == 0.f) f = 0.f;
                    *at = make_uint4(pack2(v[0] * f, v[1] * f), pack2(v[2] * f, v[3] * f), pack2(v[4] * f, v[5] * f),
                                     pack2(v[6] * f, v[7] * f));
                }
            }
            meet();
            if (!ok) break;
            const float factor = reinterpret_cast<const float*>(smem + S::kMeet)[x * 2 * 128 + row];
            fence_proxy_async_smem();
            arrive_warp(q_full + 8 * x);

            // steps of this tile that need no mask: every row sees all 128 keys
            const int tile_rows = min(128, w.p.rows - x * 128);
            const int low = w.p.base + (w.p.row0 + x * 128) / a.group;
            const int high = w.p.base + (w.p.row0 + x * 128 + tile_rows - 1) / a.group;
            const int plain0 = a.window > 0 && high >= a.window ? high - a.window + 1 : 0;
            float M = kNone, l = 0.f;  // l: of this thread's keys
            int key0 = w.p.lo + w.unit0 * kKeys;
            for (int j = 0; j < w.n; ++j, key0 += kKeys) {
                const bool plain = key0 + kKeys <= min(low + 1, w.p.hi) && key0 >= plain0;
                const float* sc = scales + (steps & 3) * 24 + half * 4;
                // The scores being there, the step's scales are.  The TMEM loads are the whole warp's.
                ok = __all_sync(~0u, wait_for(s_full + 8 * x, tiles & 1, abort_flag, a.status));
                if (!ok) break;
                tc_fence_after();
                ++steps;
                ++tiles;
                if (!plain) {  // -inf over what the row does not see
                    const int k0 = key0 + half * 64, c1 = min(pos, w.p.hi - 1) - k0;
                    const int c0 = a.window > 0 ? max(pos - k0, 0) - a.window + 1 : -64;  // c1 < 0 hides all of it anyway
#pragma unroll 1
                    for (int h = 0; h < 4; ++h) {
                        uint32_t r[16];
                        tmem_ld16(s_cols + h * 16, r);
#pragma unroll
                        for (int c = 0; c < 16; ++c)
                            if (h * 16 + c > c1 || h * 16 + c < c0) r[c] = 0xff800000u;
                        tmem_st16(s_cols + h * 16, r);
                    }
                    tmem_wait_st();
                }
                // the largest exponent
                float top = -INFINITY;
                {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t r[32];
                        tmem_ld32_async(s_cols + h * 32, r);
                        tmem_wait_ld();
                        reg_fence(r);
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const uint32_t* v = &r[q * 16];
                            float m0 = __uint_as_float(v[0]), m1 = __uint_as_float(v[1]);
#pragma unroll
                            for (int c = 2; c < 16; c += 4) {
                                m0 = fmaxf(fmaxf(m0, __uint_as_float(v[c])), __uint_as_float(v[c + 1]));
                                if (c + 2 < 16) m1 = fmaxf(fmaxf(m1, __uint_as_float(v[c + 2])), __uint_as_float(v[c + 3]));
                            }
                            // a group without a page has a log2 of -inf
                            top = fmaxf(top, fmaf(fmaxf(m0, m1), fmaxf(factor * sc[h * 2 + q], kLeast), sc[8 + h * 2 + q]));
                        }
                    }
                }
                // What a thread posts here its partner has read before the next time: the next scores wait for PV, and
                // that for both threads' weights.
                *mine = top;
                meet();
                if (!ok) break;
                top = fmaxf(top, *other);
                const bool grow = top > M + 15.f;
                if (__any_sync(~0u, grow)) {
                    const float m = grow ? top - 7.f : M;
                    const float f = ex2(M - m);
                    M = m;
                    l *= f;
                    if (j > 0) {  // O holds the steps before this one: PV of step j - 1 came before S of this one
#pragma unroll 1
                        for (int c = 0; c < D / 32; ++c) {
                            uint32_t o[16];
                            tmem_ld16(o_cols + c * 16, o);
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            tmem_st16(o_cols + c * 16, o);
                        }
                        tmem_wait_st();
                    }
                }
                // the weights, as f16 over the first half of this thread's scores; those of the second half are read
                // before anything is written over them
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    uint32_t r[32], p[16];
                    tmem_ld32_async(s_cols + h * 32, r);
                    tmem_wait_ld();
                    reg_fence(r);
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const uint32_t* v = &r[q * 16];
                        const float f = fmaxf(factor * sc[h * 2 + q], kLeast), c = sc[8 + h * 2 + q] - M;
                        float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float w0 = ex2(fmaf(__uint_as_float(v[2 * i]), f, c));
                            const float w1 = ex2(fmaf(__uint_as_float(v[2 * i + 1]), f, c));
                            sum0 += w0;
                            sum1 += w1;
                            p[q * 8 + i] = pack2(w0, w1);
                        }
                        l = fmaf(sum0 + sum1, sc[16 + h * 2 + q], l);
                    }
                    tmem_st16(s_cols + h * 16, p);
                }
                tmem_wait_st();
                tc_fence_before();
                arrive_warp(p_full + 8 * x);
            }
            if (!ok) break;
            ok = __all_sync(~0u, wait_for(o_full + 8 * x, segments & 1, abort_flag, a.status));
            if (!ok) break;
            ++segments;
            tc_fence_after();
            *mine = l;
            meet();
            if (!ok) break;
            l += *other;
            meet();  // both have read: the next segment's first post may come
            if (!ok) break;
            const bool any = l > 0.f || l != l;  // NaN goes through; a row that saw no key is zero
            const float inv = any ? 1.f / l : 0.f;
            float* part = g.parts + (static_cast<int64_t>(blockIdx.x) * 2 + (w.unit0 > 0 ? 0 : 1)) * kRows * (D + 2);
            // Every MMA of this tile is done: O takes the place of Q on its way out, whole as 16 bits, in parts as f32 in
            // two passes.
#pragma unroll 1
            for (int c = 0; c < 2; ++c) {
#pragma unroll 1
                for (int d = 0; d < D / 4; d += 16) {
                    uint32_t r[16];
                    tmem_ld16(o_cols + c * (D / 4) + d, r);
                    if (w.whole) {
                        uint32_t h[8];
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float v0 = any ? __uint_as_float(r[2 * k]) * inv : 0.f;
                            const float v1 = any ? __uint_as_float(r[2 * k + 1]) * inv : 0.f;
                            if (a.dtype == PTOWSP_F16) {
                                h[k] = pack2(v0, v1);
                            } else {
                                const __nv_bfloat162 b = __floats2bfloat162_rn(v0, v1);
                                h[k] = *reinterpret_cast<const uint32_t*>(&b);
                            }
                        }
                        const int unit = half * (D / 16) + c * (D / 32) + d / 8;
                        *io_at(row, unit) = make_uint4(h[0], h[1], h[2], h[3]);
                        *io_at(row, unit + 1) = make_uint4(h[4], h[5], h[6], h[7]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            *io_at(row, half * (D / 16) + d / 4 + i) =
                                make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
                    }
                }
                if (w.whole && c == 0) continue;
                meet();
                if (!ok) break;
                const int io = io_lane(), io_unit = io % kRowLanes, io_row = (warp & 3) * 32 + half * 16 + io / kRowLanes;
                const int f0 = w.p.row0 + x * 128 + io_row;
                int j = f0 / a.group, gq = f0 - j * a.group;
#pragma unroll 1
                for (int r = io_row; r < (warp & 3) * 32 + half * 16 + 16 && x * 128 + r < w.p.rows; r += kRowsRead) {
                    const uint4 v = *io_at(r, io_unit);
                    if (w.whole) {
                        *reinterpret_cast<uint4*>(
                            static_cast<uint16_t*>(a.out) + (w.p.token0 + static_cast<int64_t>(j)) * a.out_token_stride +
                            static_cast<int64_t>(w.head0 * a.group + gq) * a.out_head_stride + io_unit * 8) = v;
                        for (gq += kRowsRead; gq >= a.group; gq -= a.group) ++j;
                    } else {
                        const int dim = io_unit / (D / 16) * (D / 2) + c * (D / 4) + io_unit % (D / 16) * 4;
                        *reinterpret_cast<uint4*>(part + 2 * kRows + (x * 128 + r) * D + dim) = v;
                    }
                }
                if (!w.whole && c == 0) {
                    meet();  // both have read what the second pass writes over
                    if (!ok) break;
                }
            }
            if (!ok) break;
            tc_fence_before();  // O has been read: the next segment's first PV comes after this thread's next P
            if (real && half == 0) {
                if (!w.whole) {
                    part[(x * 128 + row) * 2] = M;
                    part[(x * 128 + row) * 2 + 1] = l;
                } else if (a.lse) {
                    const int j = flat / a.group;
                    a.lse[(w.p.token0 + static_cast<int64_t>(j)) * a.heads + w.head0 * a.group + flat - j * a.group] = any ? (M + log2f(l)) * 0.6931471805599453f : -INFINITY;
                }
            }
        }
    } else if (warp < kMmaWarp) {
        // ---------------- conversion ----------------
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        constexpr int RPL = 128 / CH;            // rows that all 128 threads read at once
        constexpr int NL = kKeys / RPL;          // reads per tile and thread
        const int t = threadIdx.x - kConvertWarp * 32;
        const int chunk = t % CH, row0 = t / CH;
        const int box = chunk >> 2, unit = (chunk & 3) * 2;
        const int steps = static_cast<int>(w.stop - w.at);
        bool ok = true;
        // one side's tile of step s from its landing place into its stage
        const auto convert = [&](int side, int s, uint32_t full, uint32_t empty, uint8_t* tiles) {
            ok = wait_for(l_full + 8 * side, s & 1, abort_flag, a.status);
            if (!__all_sync(~0u, ok)) return;
            uint4 x[NL];
            const uint8_t* from = smem + S::kLand + side * kKeys * D + row0 * D + chunk * 16;
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const int row = row0 + i * RPL;
                x[i] = *reinterpret_cast<const uint4*>(from + i * RPL * D);
                if ((row & 15) >= live[side * 8 + (row >> 4)]) x[i] = make_uint4(0, 0, 0, 0);  // stale codes could be NaN
            }
            // The reads are done, not only issued, before the next copy may write here: an arrival can overtake loads
            // that stand in a queue.
            fence_proxy_async_smem();
            arrive_warp(l_empty + 8 * side);
            if (s >= 2) ok = wait_for(empty + 8 * (s & 1), ((s >> 1) & 1) ^ 1u, abort_flag, a.status);
            if (!__all_sync(~0u, ok)) return;
            // both 16-byte halves of a chunk's f16; the boxes' lanes take them in turn, so that no two meet in a bank
            uint8_t* to = tiles + (s & 1) * S::kTile + box * S::kBox + row0 * 128;
            const bool swap = box & 1;
            const int ua = ((unit + (swap ? 1 : 0)) ^ (row0 & 7)) << 4, ub = ((unit + (swap ? 0 : 1)) ^ (row0 & 7)) << 4;
#pragma unroll
            for (int i = 0; i < NL; ++i) {  // RPL is a multiple of 8: the swizzle is the same in every row
                uint32_t h[8];
                codes_f16<FMT>(x[i].x, h[0], h[1]);
                codes_f16<FMT>(x[i].y, h[2], h[3]);
                codes_f16<FMT>(x[i].z, h[4], h[5]);
                codes_f16<FMT>(x[i].w, h[6], h[7]);
                *reinterpret_cast<uint4*>(to + i * RPL * 128 + ua) =
                    swap ? make_uint4(h[4], h[5], h[6], h[7]) : make_uint4(h[0], h[1], h[2], h[3]);
                *reinterpret_cast<uint4*>(to + i * RPL * 128 + ub) =
                    swap ? make_uint4(h[0], h[1], h[2], h[3]) : make_uint4(h[4], h[5], h[6], h[7]);
            }
            fence_proxy_async_smem();
            arrive_warp(full + 8 * (s & 1));
        };
        for (int s = 0; s < steps && __all_sync(~0u, ok); ++s) {
#pragma unroll 1
            for (int side = 0; side < 2 && __all_sync(~0u, ok); ++side)  // one copy of the code
                convert(side, s, k_full + 32 * side, k_empty + 32 * side, smem + S::kK + side * (S::kV - S::kK));
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    }
    if (warp == kLoadWarp) {
        // ---------------- loads ----------------
        const int pmask = a.cache.page_size - 1;
        int64_t pair = w.pair;
        int head = w.head, unit = w.unit;
        Pair p = g.pairs[pair];
        int64_t at = w.at;
        // group lane & 7 of the present step: its page (-1: no row sees a token) and how many of its tokens are there
        const auto look = [&](int* tokens) -> int {
            const int tok = p.lo + unit * kKeys + (lane & 7) * 16;
            int id = -1;
            *tokens = 0;
            if (at < w.stop && tok < p.hi && tok + 16 > p.seen) {
                id = a.page_table[p.request * a.table_stride + (tok >> a.cache.page_shift)];
                if (static_cast<uint32_t>(id) >= a.cache.pages) {
                    id = -1;
                    if (a.status && lane < 8) atomicOr(a.status, PTOWSP_SERVING_PAGE);
                } else {
                    *tokens = min(16, p.hi - tok);
                }
            }
            return id;
        };
        const auto scale_of = [&](const Kv8Side& side, int id) -> float {
            return lane < 8 && id >= 0 ? side.scale[static_cast<int64_t>(id) * a.cache.kv_heads + head] : 0.f;
        };
        const int steps = static_cast<int>(w.stop - w.at);
        bool ok = true;
        int tokens, id = look(&tokens);
        float ks = scale_of(a.cache.k, id), vs = scale_of(a.cache.v, id);
        int asked = 0;
        for (int s = 0; ok && s < steps; ++s) {
            const int tok = (p.lo + unit * kKeys + (lane & 7) * 16) & pmask, h = head, here = id, count = tokens;
            const uint32_t there = __ballot_sync(~0u, lane < 8 && here >= 0);
            for (int side = 0; side < 2; ++side) {
                if (s > 0) ok = __all_sync(~0u, wait_for(l_empty + 8 * side, (s - 1) & 1, abort_flag, a.status));
                if (!ok) break;
                if (lane < 8) live[side * 8 + lane] = count;
                if (side == 0 && lane < 8) {
                    // The scales go before K's arrival: whoever has this step's scores has its scales by the chain
                    // landed - converted - multiplied.  (A barrier of their own would not do: a tile that sits out short
                    // pairs comes to it any number of phases early, where the parity of an old phase lets it pass.)
                    // Slot s & 3 was last read in step s - 4: K of step s - 1 has been read, so V of step s - 2 has been
                    // converted, for which PV of step s - 4 had to be done, and with it both tiles' softmax.
                    float* to = scales + (s & 3) * 24 + lane;
                    const bool any = here >= 0 && ks > 0.f;  // a group without a page: log2 -inf, nothing to the sum
                    to[0] = any ? ks : 0.f;
                    to[8] = any ? log2f(vs) : -INFINITY;
                    to[16] = any ? 1.f / vs : 0.f;
                }
                __syncwarp();
                if (lane == 0) mbar_expect_tx(l_full + 8 * side, __popc(there) * 16 * D);
                __syncwarp();
                if (lane < 8 && here >= 0)
                    tma_load_page(sQ - S::kQ + S::kLand + side * kKeys * D + lane * 16 * D, side ? &v_map : &k_map, h, tok,
                                  here, l_full + 8 * side);
                asked = 2 * s + side + 1;
                if (side == 0) {  // the next step's page and scales
                    ++at;
                    if (++unit == p.units && at < w.stop) {
                        unit = 0;
                        if (++head == a.cache.kv_heads) {
                            head = 0;
                            p = g.pairs[++pair];
                        }
                    }
                    id = look(&tokens);
                    ks = scale_of(a.cache.k, id);
                    vs = scale_of(a.cache.v, id);
                }
            }
        }
        // every copy asked for has landed before shared memory goes away
        const uint64_t start = globaltimer();
        for (int side = 0; side < 2; ++side) {
            const int fills = (asked + 1 - side) / 2;
            while (fills > 0 && !mbar_try_wait(l_full + 8 * side, (fills - 1) & 1))
                if (globaltimer() - start > kTimeoutNs) {
                    if (a.status) atomicOr(a.status, PTOWSP_SERVING_TIMEOUT);
                    break;
                }
        }
    }
    if (warp == kMmaWarp && lane == 0) {
        // ---------------- MMAs ----------------
        constexpr uint32_t idesc_s = idesc_f16(128, kKeys, 0), idesc_o = idesc_f16(128, D, 1);
        const uint64_t q_desc = smem_desc(sQ, 16, 1024), k_desc = smem_desc(sK, 16, 1024);
        const uint64_t v_desc = smem_desc(sV, S::kBox, 1024);
        uint32_t steps = 0, seg[2] = {0, 0}, tiles[2] = {0, 0};
        bool ok = true, issued = false;
        while (ok && w.next(g)) {
            const int nx = w.p.rows > 128 ? 2 : 1;
            const auto scores = [&](int x, uint32_t step) {
                mma_scores<D>(tmem + x * 128, q_desc + x * (S::kTile >> 4), k_desc + (step & 1) * (S::kTile >> 4), idesc_s);
                mma_commit(s_full + 8 * x);
                issued = true;
            };
            for (int x = 0; ok && x < nx; ++x) {
                ok = wait_for(q_full + 8 * x, seg[x] & 1, abort_flag, a.status);
                ++seg[x];
            }
            if (ok) ok = wait_for(k_full + 8 * (steps & 1), (steps >> 1) & 1, abort_flag, a.status);
            if (!ok) break;
            tc_fence_after();
            for (int x = 0; x < nx; ++x) scores(x, steps);
            mma_commit(k_empty + 8 * (steps & 1));
            for (int j = 0; ok && j < w.n; ++j, ++steps) {
                const uint32_t stage = steps & 1;
                const bool last = j + 1 == w.n;
                for (int x = 0; ok && x < nx; ++x) {
                    if (x == 0) ok = wait_for(v_full + 8 * stage, (steps >> 1) & 1, abort_flag, a.status);
                    if (ok) ok = wait_for(p_full + 8 * x, tiles[x] & 1, abort_flag, a.status);
                    if (!ok) break;
                    ++tiles[x];
                    tc_fence_after();
                    mma_values(tmem + 256 + x * 128, tmem + x * 128, v_desc + stage * (S::kTile >> 4), idesc_o, j > 0);
                    if (last) mma_commit(o_full + 8 * x);
                    if (x + 1 == nx) mma_commit(v_empty + 8 * stage);
                    if (!last) {
                        if (x == 0) {
                            ok = wait_for(k_full + 8 * (stage ^ 1), ((steps + 1) >> 1) & 1, abort_flag, a.status);
                            if (!ok) break;
                            tc_fence_after();
                        }
                        scores(x, steps + 1);
                        if (x + 1 == nx) mma_commit(k_empty + 8 * (stage ^ 1));
                    }
                }
            }
        }
        if (issued) {  // every MMA issued has completed before TMEM is freed
            mma_commit(drain);
            const uint64_t start = globaltimer();
            while (!mbar_try_wait(drain, 0))
                if (globaltimer() - start > kTimeoutNs) {
                    if (a.status) atomicOr(a.status, PTOWSP_SERVING_TIMEOUT);
                    break;
                }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kMmaWarp) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

// ---------------------------------------------------------------------------
// Joining the tasks that the deal cut: one CTA column per cut, a warp per row, few pieces per task.
// ---------------------------------------------------------------------------

constexpr int kJoinThreads = 256;

template <int D>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ PrefillArgs g, int ctas) {
    const AttendArgs& a = g.a;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t total = g.total[0];
    const int64_t c = blockIdx.x + 1;
    const int64_t at = share_start(total, ctas, c);
    if (at >= total) return;
    const int pair = find_pair(g.pairs, static_cast<int>(g.total[1]), at);
    const Pair p = g.pairs[pair];
    const int64_t in = at - p.before;
    const int head = static_cast<int>(in / p.units);
    const int64_t begin = p.before + static_cast<int64_t>(head) * p.units, end = begin + p.units;
    if (at == begin || share_start(total, ctas, c - 1) > begin) return;  // no cut in a task, or not its first one
    const int pieces = static_cast<int>(share_owner(total, ctas, end - 1) - c) + 2;
    constexpr int64_t kPiece = static_cast<int64_t>(kRows) * (D + 2);
    constexpr int V = D / 32;
    const float* first = g.parts + ((c - 1) * 2 + 1) * kPiece;
    const auto piece = [&](int i) { return first + (i == 0 ? 0 : (2 * i - 1) * kPiece); };
    for (int row = blockIdx.y * (kJoinThreads / 32) + warp; row < p.rows; row += gridDim.y * (kJoinThreads / 32)) {
        float m = kNone;
        for (int i = lane; i < pieces; i += 32) m = fmaxf(m, piece(i)[row * 2]);
#pragma unroll
        for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
        float x[V], sum = 0.f;
#pragma unroll
        for (int k = 0; k < V; ++k) x[k] = 0.f;
#pragma unroll 4
        for (int i = 0; i < pieces; ++i) {
            const float* o = piece(i);
            const float li = o[row * 2 + 1];
            const float f = li == 0.f ? 0.f : ex2(o[row * 2] - m);  // a piece without a key may hold no O
            sum = fmaf(f, li, sum);
#pragma unroll
            for (int k = 0; k < V; ++k) x[k] = f == 0.f ? x[k] : fmaf(f, o[2 * kRows + row * D + lane * V + k], x[k]);
        }
        const int flat = p.row0 + row;
        const int64_t tok = p.token0 + flat / a.group;
        const int hq = head * a.group + flat % a.group;
        const bool any = sum > 0.f || sum != sum;
        const float r = any ? 1.f / sum : 0.f;
        const int64_t off = tok * a.out_token_stride + hq * a.out_head_stride + lane * V;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            if (a.dtype == PTOWSP_F16) static_cast<__half*>(a.out)[off + k] = __float2half_rn(x[k] * r);
            else static_cast<__nv_bfloat16*>(a.out)[off + k] = __float2bfloat16_rn(x[k] * r);
        }
        if (lane == 0 && a.lse) a.lse[tok * a.heads + hq] = any ? (m + log2f(sum)) * 0.6931471805599453f : -INFINITY;
    }
}

int64_t most_pairs(const AttendArgs& a) {
    return std::min<int64_t>(a.tokens * a.group / kRows + a.requests,
                             (static_cast<int64_t>(a.max_q) * a.group + kRows - 1) / kRows * a.requests);
}
size_t list_bytes(const AttendArgs& a) { return (256 + static_cast<size_t>(most_pairs(a)) * sizeof(Pair) + 255) / 256 * 256; }

template <int FMT, int D>
cudaError_t launch(const PrefillArgs& g, int sms, cudaStream_t s) {
    static SmemOptIn opt_in;
    cudaError_t e = opt_in.once(reinterpret_cast<const void*>(prefill_kernel<FMT, D>), Smem<D>::kBytes);
    if (e != cudaSuccess) return e;
    const int64_t pairs = most_pairs(g.a);
    if (pairs > INT32_MAX) return cudaErrorInvalidValue;
    CUtensorMap k_map, v_map;
    if (!kv8_map(&k_map, g.a.cache, g.a.cache.k, 16, false) || !kv8_map(&v_map, g.a.cache, g.a.cache.v, 16, false))
        return cudaErrorInvalidValue;
    list_kernel<<<1, kListThreads, 0, s>>>(g, static_cast<int>(pairs));
    prefill_kernel<FMT, D><<<sms, kThreads, Smem<D>::kBytes, s>>>(g, k_map, v_map);
    if (sms > 1) join_kernel<D><<<dim3(sms - 1, 8), kJoinThreads, 0, s>>>(g, sms);
    return cudaGetLastError();
}

}  // namespace

size_t prefill_workspace_bytes(const AttendArgs& a, int sms) {
    return list_bytes(a) + static_cast<size_t>(sms) * 2 * kRows * (a.cache.head_dim + 2) * sizeof(float);
}

cudaError_t launch_prefill(const AttendArgs& a, int threshold, char* workspace, int sms, cudaStream_t s) {
    PrefillArgs g{};
    g.a = a;
    g.total = reinterpret_cast<int64_t*>(workspace);
    g.pairs = reinterpret_cast<Pair*>(workspace + 256);
    g.parts = reinterpret_cast<float*>(workspace + list_bytes(a));
    g.threshold = threshold;
    if (a.cache.format == PTOWSP_KV8_E4M3)
        return a.cache.head_dim == 64 ? launch<PTOWSP_KV8_E4M3, 64>(g, sms, s) : launch<PTOWSP_KV8_E4M3, 128>(g, sms, s);
    return a.cache.head_dim == 64 ? launch<PTOWSP_KV8_INT8, 64>(g, sms, s) : launch<PTOWSP_KV8_INT8, 128>(g, sms, s);
}

}  // namespace ptowsp::dev

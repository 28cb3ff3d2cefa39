// Attention over a paged KV cache held in 8 bits, for few query rows per request (decoding, verification).
//
// With code c, page scale s (one per page and head): k = s_k c_k, v = s_v c_v, so
//   out = sum_t e^(a s_k(t) q.c_k(t)) s_v(t) c_v(t) / sum_t e^(a s_k(t) q.c_k(t)).
// The scales fold into the exponent: w_t = 2^(a' s_k q.c_k + log2 s_v - M) weighs the V codes and w_t / s_v the
// denominator, with M following the largest exponent.  That bounds what is summed whatever the pages' scales are: the
// largest w is between 2^7 and 2^15, so w fits f16 for the second product, and a weight too small for f16's 11 bits
// is off by at most 2^-32 of the largest.
//
// Codes become f16 exactly (e4m3 and int8 are subsets of it).  A row of q enters as f16 times a power of two that
// brings its largest element below 2^15, which is exact for f16 and for bf16 elements down to 2^-29 of the row's
// largest; below that the lost part is under 2^-39 of it.  Sums are f32 in the MMA and in registers.
//
// Bound by HBM: every code is read once.  64 requests of one token over 512-8192 keys (8 KV heads of 128, groups of four:
// 582 MB) take 108 us as a whole call, 5.4 TB/s; the copy rate would take 89.  Three requests over 100,000-200,000 keys:
// 115 us for 599 MB.  What is left is the second launch and the CTAs' ends, some 8 us, and the warps' waits for boxes of
// 2 to 4 KB, which 16 bytes per thread by cp.async (118 us) and plain loads (128) served worse.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "serving.hpp"
#include "serving_kv8.cuh"
#include "tc_common.cuh"

namespace ptowsp::dev {

namespace {

constexpr int kWarps = 4;
constexpr int kTile = 32;                 // tokens per warp and step
constexpr int kUnit = kWarps * kTile;     // tokens per CTA and step: the grain in which work is dealt out
constexpr int kSlots = 3;                  // tiles of K or V that a warp's ring holds
constexpr int kThreads = kWarps * 32;
constexpr float kNone = -1.7e38f;         // M before the first visible key: below every exponent, yet finite

// CTAs per SM.  With one fragment of q rows four (128 registers) spill: 120 us against 109 over the 64-request decode
// workload; rings of four tiles instead of three took 112.
__host__ __device__ constexpr int ctas_per_sm(int nb) { return nb <= 2 ? 3 : 2; }

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float log2_approx(float x) {
    float r;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// ---------------------------------------------------------------------------
// Dealing out the work.  A request has `tiles` tiles of q rows for each KV head, and every one of these tasks takes
// `units` steps of kUnit tokens.  The steps of all tasks stand in one line (request, tile, head, step), and CTA c of n
// takes the c-th n-th of it, so all CTAs read the same amount whatever the lengths are.  A task that this cuts leaves
// one partial result in each CTA it touches; the CTA with the first one writes down what a second launch has to join.
// ---------------------------------------------------------------------------

struct Request {
    int row0, nq;         // q rows (tokens)
    int lo, hi;           // tokens to walk: [lo, hi), lo a multiple of kTile
    int seen;             // the first token that any row sees, lo <= seen
    int len;              // tokens in the cache
    int64_t tasks, units;
};

template <int ROWS>
__device__ __forceinline__ Request request_at(const AttendArgs& a, int r, int* flags) {
    Request q;
    q.row0 = a.q_start ? a.q_start[r] : r;
    const int end = a.q_start ? a.q_start[r + 1] : r + 1;
    q.nq = end - q.row0;
    if (q.row0 < 0 || q.nq < 0 || end > a.tokens || q.nq > a.max_q) {
        if (flags) *flags |= PTOWSP_SERVING_LENGTH;
        q.nq = 0;
    }
    q.len = a.kv_len[r];
    const int64_t room = static_cast<int64_t>(a.max_pages) << a.cache.page_shift;
    if (q.len < 0 || q.len > room) {
        if (flags) *flags |= PTOWSP_SERVING_LENGTH;
        q.len = q.len < 0 ? 0 : static_cast<int>(room);
    }
    q.hi = q.len;
    q.lo = q.seen = 0;
    if (a.window > 0) {  // row 0 sees from len - nq + 1 - window on
        const int64_t lo = static_cast<int64_t>(q.len) - q.nq + 1 - a.window;
        if (lo > 0) {
            q.seen = static_cast<int>(lo);
            q.lo = q.seen & ~(kTile - 1);
        }
    }
    if (a.few && static_cast<int64_t>(q.nq) * a.group > a.few) q.nq = 0;
    q.tasks = static_cast<int64_t>((static_cast<int64_t>(q.nq) * a.group + ROWS - 1) / ROWS) * a.cache.kv_heads;
    const int64_t span = q.hi - q.lo;
    q.units = span > 0 ? (span + kUnit - 1) / kUnit : 1;  // a task without keys still writes its zeros
    return q;
}

// a / b for a >= 0, b > 0: 64-bit division is a long routine, and what is divided here nearly always fits 32 bits.
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
    return a / b;
}

// The steps of all requests, and for a place in their line the request that holds it and the steps before that.
struct Deal {
    int64_t total;        // steps in all
    int64_t ctas;         // CTAs that share them
    int64_t share, rest;  // steps of each, and the first CTAs that have one more
    int per;              // requests per thread of the scan
    bool left_out;        // a request may have been left out
    bool loose;           // that, or rows before the first request's or behind the last one's

    __device__ __forceinline__ int64_t start(int64_t c) const { return c * share + (c < rest ? c : rest); }
    // the CTA that has step i
    __device__ __forceinline__ int64_t owner(int64_t i) const {
        const int64_t big = rest * (share + 1);
        return i < big ? quotient(i, share + 1) : rest + quotient(i - big, share);
    }
};

template <int ROWS>
__device__ Deal deal_out(const AttendArgs& a, int ctas, int64_t* sums, int* flags) {
    Deal d;
    d.per = (a.requests + kThreads - 1) / kThreads;
    const bool ends = a.q_start && threadIdx.x == 0 && (a.q_start[0] != 0 || a.q_start[a.requests] < a.tokens);
    int64_t mine = 0;
    for (int i = 0; i < d.per; ++i) {
        const int r = threadIdx.x * d.per + i;
        if (r >= a.requests) break;
        const Request q = request_at<ROWS>(a, r, flags);
        mine += q.tasks * q.units;
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t v = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t t = __shfl_up_sync(~0u, v, o);
        if (lane >= o) v += t;
    }
    __shared__ int64_t warp_sum[kWarps];
    if (lane == 31) warp_sum[warp] = v;
    __syncthreads();
    for (int w = 0; w < warp; ++w) v += warp_sum[w];
    sums[threadIdx.x] = v;  // inclusive
    d.loose = __syncthreads_or(*flags || ends);
    d.left_out = d.loose && __syncthreads_or(*flags);
    d.total = sums[kThreads - 1];
    d.ctas = d.total < ctas ? (d.total > 0 ? d.total : 1) : ctas;
    d.share = quotient(d.total, d.ctas);
    d.rest = d.total - d.share * d.ctas;
    return d;
}

struct Place {
    int r;             // request
    Request q;
    int64_t task;      // of the request: tile * kv_heads + head
    int64_t unit;      // of the task
};

template <int ROWS>
__device__ Place find_place(const AttendArgs& a, const Deal& d, const int64_t* sums, int64_t at) {
    int lo = 0, hi = kThreads - 1;  // first thread whose inclusive sum passes `at`
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sums[mid] > at) hi = mid;
        else lo = mid + 1;
    }
    int64_t before = lo ? sums[lo - 1] : 0;
    Place p;
    for (p.r = lo * d.per;; ++p.r) {
        p.q = request_at<ROWS>(a, p.r, nullptr);
        const int64_t n = p.q.tasks * p.q.units;
        if (at < before + n) break;
        before += n;
    }
    p.task = quotient(at - before, p.q.units);
    p.unit = at - before - p.task * p.q.units;
    return p;
}

// The workspace: a record per CTA, then two partial results per CTA.
struct Cut {      // the task whose first piece is the CTA's last share
    int pieces;   // 0: there is none
    int row0, head, row_base, rows;
    int pad[3];
};
constexpr int kMaxSms = 512;
constexpr size_t kCuts = kMaxSms * 4 * sizeof(Cut);
// A partial result: [rows][M, l], then [rows][D] of O.
template <int D, int NB>
constexpr size_t partial_floats() { return static_cast<size_t>(8 * NB) * (D + 2); }

// Divides V dims of a finished row by its sum and stores them, and the row's lse where `first`.
template <int V>
__device__ __forceinline__ void store_row(const AttendArgs& a, int row0, int head, int flat, int dim,
                                          const float (&x)[V], float m, float sum, bool first) {
    const int64_t tok = row0 + flat / a.group;
    const int hq = head * a.group + flat % a.group;
    const bool any = sum > 0.f || sum != sum;  // NaN goes through; a row that saw no key is zero
    const float r = any ? 1.f / sum : 0.f;
    const int64_t off = tok * a.out_token_stride + hq * a.out_head_stride + dim;
#pragma unroll
    for (int k = 0; k < V; ++k) {
        if (a.dtype == PTOWSP_F16) static_cast<__half*>(a.out)[off + k] = __float2half_rn(x[k] * r);
        else static_cast<__nv_bfloat16*>(a.out)[off + k] = __float2bfloat16_rn(x[k] * r);
    }
    if (first && a.lse) a.lse[tok * a.heads + hq] = any ? (m + log2f(sum)) * 0.6931471805599453f : -INFINITY;
}

// Rows of q that no request has -- before the first one's or behind the last one's, as where the rows are padded to a
// fixed number, and those of a request that was left out -- get zeros and lse = -inf.  `some`: a request may have been
// left out, so every row is looked up; else only the ends are.  A warp per row.
template <int D>
__device__ __noinline__ void clear_rows(const AttendArgs& a, bool some) {
    const int lane = threadIdx.x & 31;
    const int begin = a.q_start[0], end = a.q_start[a.requests];
    const int64_t skip = !some && begin == 0 ? end : 0;
    for (int64_t t = skip + blockIdx.x * kWarps + (threadIdx.x >> 5); t < a.tokens; t += gridDim.x * kWarps) {
        if (t >= begin && t < end) {
            int lo = 0, hi = a.requests - 1;  // the request whose rows these are: the first that ends behind t
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if (a.q_start[mid + 1] > t) hi = mid;
                else lo = mid + 1;
            }
            const int row0 = a.q_start[lo], row1 = a.q_start[lo + 1];
            if (row0 >= 0 && row1 <= a.tokens && row1 - row0 <= a.max_q) continue;
        }
        for (int h = 0; h < a.heads; ++h) {
            char* to = static_cast<char*>(a.out) + (t * a.out_token_stride + h * a.out_head_stride) * 2;
            if (lane < D / 8) reinterpret_cast<uint4*>(to)[lane] = make_uint4(0, 0, 0, 0);
            if (lane == 0 && a.lse) a.lse[t * a.heads + h] = -INFINITY;
        }
    }
}

template <int D, int NB>
struct Layout {
    static constexpr int ROWS = 8 * NB;
    static constexpr int kSlot = kTile * D;               // bytes of a tile of K or of V
    static constexpr int QP = 2 * D + 32;                 // bytes between q rows: their 8-byte fragment loads hit all banks
    static constexpr int kRing = kWarps * kSlots * kSlot;
    static constexpr int kQ = kRing;                      // [ROWS] rows of QP bytes
    static constexpr int kRow = kQ + ROWS * QP;           // [ROWS] factor, [ROWS] last visible key
    static constexpr int kStat = kRow + ROWS * 8;         // [kWarps][ROWS][2] M and l
    static constexpr int kBars = kStat + kWarps * ROWS * 8;  // [kWarps][kSlots] mbarriers
    static constexpr int kBytes = kBars + kWarps * kSlots * 8 + 1024;  // the ring begins at a multiple of 1024
    // the warps' O meet in the ring; where it is too small for all of D, half of D at a time
    static constexpr int kParts = kWarps * ROWS * (D + 4) * 4 <= kRing ? 1 : 2;
    static constexpr int OP = D / kParts + 4;             // floats between rows there
};

// One tile of q rows of one head against its share of the tokens.  S^T = K.Q^T and O^T = V^T.P^T on
// mma.m16n8k16: 16 tokens (then 16 dims) x 8 q rows, so a group of 8 or fewer rows wastes at most half of the MMA, and
// the converted codes of a step serve 8 * NB rows.  tcgen05's 64 or 128 rows would be mostly padding here.
//
// Bound by HBM (4 FLOP per byte and q row).  Each warp runs on its own: its ring of three tiles takes K and V in turn,
// a tile's place is asked for again as soon as it is read, and no barrier joins the warps before the end of the share.
template <int FMT, int D, int NB>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(NB)) attend_kernel(const __grid_constant__ AttendArgs a, const __grid_constant__ CUtensorMap k_map,
              const __grid_constant__ CUtensorMap v_map) {
    using L = Layout<D, NB>;
    constexpr int ROWS = L::ROWS;
    constexpr int CH = D / 16;                // 16-byte chunks of a row of codes
    extern __shared__ char raw_smem[];
    char* smem = raw_smem + (1024 - (tc::smem_u32(raw_smem) & 1023)) % 1024;
    char* q_smem = smem + L::kQ;
    float* q_scale = reinterpret_cast<float*>(smem + L::kRow);  // [ROWS] a' = scale * log2(e) / row's power of two
    int* q_pos = reinterpret_cast<int*>(q_scale + ROWS);        // [ROWS] last key the row sees; -1: none, or no row
    float* stat = reinterpret_cast<float*>(smem + L::kStat);
    __shared__ int64_t sums[kThreads];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t4 = lane & 3;
    Cut* cut = reinterpret_cast<Cut*>(a.workspace) + blockIdx.x;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    int flags = 0;
    const Deal deal = deal_out<ROWS>(a, gridDim.x, sums, &flags);
    if (blockIdx.x == 0 && flags && a.status) atomicOr(a.status, flags);
    if (a.q_start && deal.loose) clear_rows<D>(a, deal.left_out);
    if (deal.total == 0 || blockIdx.x >= deal.ctas) {
        if (threadIdx.x == 0) cut->pieces = 0;
        return;
    }
    int64_t at = deal.start(blockIdx.x);
    const int64_t stop = deal.start(blockIdx.x + 1);
    Place p = find_place<ROWS>(a, deal, sums, at);

    const uint32_t ring = tc::smem_u32(smem) + warp * kSlots * L::kSlot;
    const uint32_t bars = tc::smem_u32(smem + L::kBars) + warp * kSlots * 8;
    if (lane == 0) {
        for (int i = 0; i < kSlots; ++i) tc::mbar_init(bars + i * 8, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    const int pshift = a.cache.page_shift, pmask = a.cache.page_size - 1;
    uint32_t phases = 0;  // bit i: parity of slot i's next fill
    bool dead = false;    // a wait gave up: nothing is asked for any more
    // the fill of a slot, bounded; all lanes see the same outcome
    const auto wait = [&](int slot) {
        const uint32_t bar = bars + slot * 8, parity = phases >> slot & 1u;
        phases ^= 1u << slot;
        if (__all_sync(~0u, tc::mbar_try_wait(bar, parity)) || dead) return;
        const uint64_t start = tc::globaltimer();
        do {
            if (__all_sync(~0u, tc::mbar_try_wait(bar, parity))) return;
            dead = __any_sync(~0u, tc::globaltimer() - start > tc::kTimeoutNs);
        } while (!dead);
        if (a.status) atomicOr(a.status, PTOWSP_SERVING_TIMEOUT);
    };
    // swizzled places of the fragments' 16-byte chunks: rows (lane & 15), chunks c + (lane >> 4)
    const int frow = lane & 15, fsw = D == 128 ? frow & 7 : (frow >> 1) & 3;

    while (at < stop) {
        const int head = static_cast<int>(p.task % a.cache.kv_heads);
        const int row_base = static_cast<int>(p.task / a.cache.kv_heads) * ROWS;
        const int64_t left = p.q.units - p.unit;
        const int64_t take = left < stop - at ? left : stop - at;
        const bool whole = take == p.q.units;
        const int tok0 = p.q.lo + static_cast<int>(p.unit) * kUnit;
        const int tok1 = min(p.q.hi, tok0 + static_cast<int>(take) * kUnit);
        const int32_t* table = a.page_table + p.r * a.table_stride;
        const int rows = min(ROWS, p.q.nq * a.group - row_base);

        // -- the warp's tiles: first + i * kUnit --
        const int first = tok0 + warp * kTile;
        const int ntiles = tok1 > first ? (tok1 - first + kUnit - 1) / kUnit : 0;
        // page ids of the two 16-token halves of tile i, in lanes 0 and 1 (-1: no token there)
        const int seen = p.q.seen;
        auto page_of = [&](int i) -> int {
            int id = -1;
            const int tok = first + i * kUnit + lane * 16;
            if (lane < 2 && tok < tok1 && tok + 16 > seen) {
                id = table[tok >> pshift];
                if (static_cast<uint32_t>(id) >= a.cache.pages) {
                    id = -1;
                    if (a.status) atomicOr(a.status, PTOWSP_SERVING_PAGE);
                }
            }
            return id;
        };
        // asks for tile i of one side: one box where the pages hold 32 tokens or more, else one per half
        auto ask = [&](const CUtensorMap* map, int i, int ids, int slot) {
            if (i >= ntiles || dead) return;
            const int id0 = __shfl_sync(~0u, ids, 0), id1 = __shfl_sync(~0u, ids, 1);
            if (lane == 0) {
                const int tok = (first + i * kUnit) & pmask;
                const uint32_t dst = ring + slot * L::kSlot, bar = bars + slot * 8;
                if (pmask == 15) {
                    tc::mbar_expect_tx(bar, ((id0 >= 0) + (id1 >= 0)) * (L::kSlot / 2));
                    if (id0 >= 0) tma_load_page(dst, map, head, 0, id0, bar);
                    if (id1 >= 0) tma_load_page(dst + L::kSlot / 2, map, head, 0, id1, bar);
                } else {  // both halves are in one page; the first may lie before the window
                    const int id = id0 >= 0 ? id0 : id1;
                    tc::mbar_expect_tx(bar, id >= 0 ? L::kSlot : 0);
                    if (id >= 0) tma_load_page(dst, map, head, tok, id, bar);
                }
            }
        };
        // k scale of half 0 and 1 of a tile, then v's, in lanes 0 .. 3; 0 where there is no page
        auto scale_of = [&](int ids) -> float {
            const int id = __shfl_sync(~0u, ids, lane & 1);
            if (lane >= 4 || id < 0) return 0.f;
            const float* s = lane < 2 ? a.cache.k.scale : a.cache.v.scale;
            return s[static_cast<int64_t>(id) * a.cache.kv_heads + head];
        };
        // rows of a slot that hold no token become zeros: what stands there could be NaN
        auto clear = [&](uint32_t slot_addr, int i, float sc0, float sc1) {
            const int tile = first + i * kUnit;
#pragma unroll
            for (int j = 0; j < kTile / 8; ++j) {
                const int row = j * 8 + (lane >> 2);
                if (tile + row >= tok1 || !((row < 16 ? sc0 : sc1) > 0.f)) {
#pragma unroll
                    for (int c = 0; c < CH / 4; ++c)
                        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(slot_addr + row * D +
                                                                                     ((lane & 3) + c * 4) * 16),
                                     "r"(0)
                                     : "memory");
                }
            }
            tc::fence_proxy_async_smem();
            __syncwarp();
        };
        int ids1, ids2;  // of the tile after the present one, and of the one after that
        float scales;    // of the present tile
        {
            const int ids0 = page_of(0);
            ids1 = page_of(1);
            ids2 = page_of(2);
            ask(&k_map, 0, ids0, 0);
            ask(&v_map, 0, ids0, 1);
            ask(&k_map, 1, ids1, 2);
            scales = scale_of(ids0);
        }

        // -- q rows, as f16 times a power of two; one warp per row --
        for (int row = warp; row < ROWS; row += kWarps) {
            const int flat = row_base + row;
            const bool real = row < rows;
            const int j = flat / a.group, gq = flat % a.group;
            float x[D / 32];
            if (real) {
                const int64_t off = static_cast<int64_t>(p.q.row0 + j) * a.q_token_stride +
                                    static_cast<int64_t>(head * a.group + gq) * a.q_head_stride + lane * (D / 32);
#pragma unroll
                for (int k = 0; k < D / 32; ++k)
                    x[k] = a.dtype == PTOWSP_F16 ? __half2float(static_cast<const __half*>(a.q)[off + k])
                                                 : __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[off + k]);
            } else {
#pragma unroll
                for (int k = 0; k < D / 32; ++k) x[k] = 0.f;
            }
            float m = 0.f;
#pragma unroll
            for (int k = 0; k < D / 32; ++k) m = fmaxf(m, fabsf(x[k]));
            m = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(m)));
            // 2^e with m * 2^e in [2^14, 2^15); the exponent is kept where 2^e and 2^-e are normal numbers
            int e = 0;
            if (m > 0.f && m < INFINITY) e = min(max(14 - (static_cast<int>(__float_as_uint(m) >> 23) - 127), -120), 120);
            const float f = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
            __half* to = reinterpret_cast<__half*>(q_smem + row * L::QP) + lane * (D / 32);
#pragma unroll
            for (int k = 0; k < D / 32; ++k) to[k] = __float2half_rn(x[k] * f);
            if (lane == 0) {
                q_scale[row] = a.scale * 1.4426950408889634f * __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
                q_pos[row] = real ? p.q.len - p.q.nq + j : -1;
            }
        }
        __syncthreads();

        float qs[NB][2];
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) qs[n][c] = q_scale[n * 8 + 2 * t4 + c];
        // tiles [plain0, plain0 + plains) need no mask: their 32 tokens exist and every row sees them
        int plain0 = 0, plains;
        {
            const int low = p.q.len - p.q.nq + row_base / a.group;               // the first row's last key
            const int high = p.q.len - p.q.nq + (row_base + rows - 1) / a.group;  // the last row's
            const int end = min(tok1, low + 1);
            plains = end - kTile >= first ? (end - kTile - first) / kUnit + 1 : 0;
            if (a.window > 0 && high >= a.window && high - a.window >= first) {
                plain0 = (high - a.window - first) / kUnit + 1;
                plains = max(plains - plain0, 0);
            }
        }
        uint32_t qf[NB == 1 ? CH : 1][2];
        if constexpr (NB == 1) {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const uint2 w = *reinterpret_cast<const uint2*>(q_smem + g * L::QP + c * 32 + t4 * 8);
                qf[c][0] = w.x;
                qf[c][1] = w.y;
            }
        }

        float M[NB][2], l[NB][2], o[NB][CH][4];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            M[n][0] = M[n][1] = kNone;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int c = 0; c < CH; ++c) o[n][c][0] = o[n][c][1] = o[n][c][2] = o[n][c][3] = 0.f;
        }

        int kslot = 0, vslot = 1;  // of the present tile
        for (int i = 0; i < ntiles && !dead; ++i) {
            const int ids3 = page_of(i + 3);
            const float next_scales = scale_of(ids1);
            const float sc[4] = {__shfl_sync(~0u, scales, 0), __shfl_sync(~0u, scales, 1), __shfl_sync(~0u, scales, 2),
                                 __shfl_sync(~0u, scales, 3)};
            scales = next_scales;
            // no mask, and no row without a token
            const bool plain = static_cast<unsigned>(i - plain0) < static_cast<unsigned>(plains) && sc[0] > 0.f && sc[1] > 0.f;
            wait(kslot);
            if (!plain) clear(ring + kslot * L::kSlot, i, sc[0], sc[1]);

            // S^T: two blocks of 16 tokens
            float s[2][NB][4];
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int n = 0; n < NB; ++n) s[b][n][0] = s[b][n][1] = s[b][n][2] = s[b][n][3] = 0.f;
            const uint32_t krow = ring + kslot * L::kSlot + frow * D;
#pragma unroll
            for (int c = 0; c < CH; c += 2) {
                const uint32_t at_c = krow + ((c + (lane >> 4)) ^ fsw) * 16;
                uint32_t qv[NB][2][2];
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        if constexpr (NB == 1) {
                            qv[n][k][0] = qf[c + k][0];
                            qv[n][k][1] = qf[c + k][1];
                        } else {
                            const uint2 w =
                                *reinterpret_cast<const uint2*>(q_smem + (n * 8 + g) * L::QP + (c + k) * 32 + t4 * 8);
                            qv[n][k][0] = w.x;
                            qv[n][k][1] = w.y;
                        }
                    }
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    uint32_t w[4];
                    ldmatrix4(at_c + b * 16 * D, w);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        uint32_t a0, a1, a2, a3;
                        codes_f16<FMT>(w[2 * k], a0, a2);
                        codes_f16<FMT>(w[2 * k + 1], a1, a3);
#pragma unroll
                        for (int n = 0; n < NB; ++n) mma16816(s[b][n], a0, a1, a2, a3, qv[n][k][0], qv[n][k][1]);
                    }
                }
            }
            tc::fence_proxy_async_smem();  // reads that are still queued come before the copy's writes
            __syncwarp();
            ask(&v_map, i + 1, ids1, kslot);  // K's place is free

            // exponents t = a' s_k S + log2 s_v
            const float lv[2] = {log2_approx(sc[2]), log2_approx(sc[3])};
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float f0 = qs[n][c] * sc[0], f1 = qs[n][c] * sc[1];
                    s[0][n][c] = fmaf(s[0][n][c], f0, lv[0]);
                    s[0][n][c + 2] = fmaf(s[0][n][c + 2], f0, lv[0]);
                    s[1][n][c] = fmaf(s[1][n][c], f1, lv[1]);
                    s[1][n][c + 2] = fmaf(s[1][n][c + 2], f1, lv[1]);
                }
            if (!plain) {
                const int tile = first + i * kUnit;
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int n = 0; n < NB; ++n)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int tok = tile + b * 16 + g + (k >> 1) * 8;
                            const int last = q_pos[n * 8 + 2 * t4 + (k & 1)];
                            const bool see = sc[b] > 0.f && tok < tok1 && tok <= last &&
                                             !(a.window > 0 && tok <= last - a.window);
                            if (!see) s[b][n][k] = -INFINITY;
                        }
            }
            // M follows only when a weight would pass 2^15, and then leaves the largest at 2^7
            float top[NB][2];
            bool grow = false;
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    top[n][c] = fmaxf(fmaxf(s[0][n][c], s[0][n][c + 2]), fmaxf(s[1][n][c], s[1][n][c + 2]));
                    grow |= top[n][c] > M[n][c] + 15.f;
                }
            if (__any_sync(~0u, grow)) {
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float m = top[n][c];
                        m = fmaxf(m, __shfl_xor_sync(~0u, m, 4));
                        m = fmaxf(m, __shfl_xor_sync(~0u, m, 8));
                        m = fmaxf(m, __shfl_xor_sync(~0u, m, 16));
                        m = fmaxf(m - 7.f, M[n][c]);
                        const float f = exp2_approx(M[n][c] - m);
                        M[n][c] = m;
                        l[n][c] *= f;
#pragma unroll
                        for (int d = 0; d < CH; ++d) {
                            o[n][d][c] *= f;
                            o[n][d][c + 2] *= f;
                        }
                    }
            }
            const float inv[2] = {sc[2] > 0.f ? rcp_approx(sc[2]) : 0.f, sc[3] > 0.f ? rcp_approx(sc[3]) : 0.f};
            uint32_t pb[2][NB][2];
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    const float w0 = exp2_approx(s[b][n][0] - M[n][0]), w1 = exp2_approx(s[b][n][1] - M[n][1]);
                    const float w2 = exp2_approx(s[b][n][2] - M[n][0]), w3 = exp2_approx(s[b][n][3] - M[n][1]);
                    l[n][0] = fmaf(w0 + w2, inv[b], l[n][0]);
                    l[n][1] = fmaf(w1 + w3, inv[b], l[n][1]);
                    pb[b][n][0] = transpose8x8(pack_f16(w0, w1));
                    pb[b][n][1] = transpose8x8(pack_f16(w2, w3));
                }

            wait(vslot);
            if (!plain) clear(ring + vslot * L::kSlot, i, sc[0], sc[1]);
            // O^T += V^T.P^T
            const uint32_t vrow = ring + vslot * L::kSlot + frow * D;
#pragma unroll
            for (int c = 0; c < CH; c += 2) {
                const uint32_t at_c = vrow + ((c + (lane >> 4)) ^ fsw) * 16;
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    uint32_t w[4];
                    ldmatrix4_trans(at_c + b * 16 * D, w);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        // bytes (token 2t, dims 2g and 2g + 1), (token 2t + 1, the same): pair the tokens
                        uint32_t a0, a1, a2, a3;
                        codes_f16<FMT>(__byte_perm(w[2 * k], 0, 0x3120), a0, a1);
                        codes_f16<FMT>(__byte_perm(w[2 * k + 1], 0, 0x3120), a2, a3);
#pragma unroll
                        for (int n = 0; n < NB; ++n) mma16816(o[n][c + k], a0, a1, a2, a3, pb[b][n][0], pb[b][n][1]);
                    }
                }
            }
            tc::fence_proxy_async_smem();
            __syncwarp();
            ask(&k_map, i + 2, ids2, vslot);  // V's place is free
            ids1 = ids2;
            ids2 = ids3;
            // K of i + 1 stands behind V of i, V of i + 1 where K of i was
            const int next = vslot == kSlots - 1 ? 0 : vslot + 1;
            vslot = kslot;
            kslot = next;
        }

        // One warp gave up: the CTA leaves, so that no further wait of its share can run out as well.  The copies that this
        // warp asked for get the time to land first, and the join finds no task written down.
        if (dead) {
            const uint64_t start = tc::globaltimer();
            while (tc::globaltimer() - start < tc::kTimeoutNs) {
            }
        }
        if (__syncthreads_or(dead)) {
            if (threadIdx.x == 0) cut->pieces = 0;
            return;
        }

        // -- join the warps: M and l first, then O through the ring, which every warp is done with --
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float v = l[n][c];
                v += __shfl_xor_sync(~0u, v, 4);
                v += __shfl_xor_sync(~0u, v, 8);
                v += __shfl_xor_sync(~0u, v, 16);
                if (g == 0) {
                    const int row = n * 8 + 2 * t4 + c;
                    stat[(warp * ROWS + row) * 2] = M[n][c];
                    stat[(warp * ROWS + row) * 2 + 1] = v;
                }
            }
        float* o_smem = reinterpret_cast<float*>(smem);
        float* parts = reinterpret_cast<float*>(a.workspace + kCuts);
        float* part = parts + (static_cast<int64_t>(blockIdx.x) * 2 + (p.unit > 0 ? 0 : 1)) * partial_floats<D, NB>();
        constexpr int DP = D / L::kParts;    // dims at a time
        constexpr int V = DP / 32;           // per lane
#pragma unroll
        for (int h = 0; h < L::kParts; ++h) {
            if (h > 0) __syncthreads();
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int c = 0; c < CH / L::kParts; ++c)
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        *reinterpret_cast<float2*>(&o_smem[(warp * ROWS + n * 8 + 2 * t4 + k) * L::OP + c * 16 + 2 * g]) =
                            make_float2(o[n][h * (CH / L::kParts) + c][k], o[n][h * (CH / L::kParts) + c][k + 2]);
            __syncthreads();
            for (int row = warp; row < rows; row += kWarps) {
                float m = kNone, sum = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) m = fmaxf(m, stat[(w * ROWS + row) * 2]);
                float x[V];
#pragma unroll
                for (int k = 0; k < V; ++k) x[k] = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float f = exp2_approx(stat[(w * ROWS + row) * 2] - m);
                    sum = fmaf(f, stat[(w * ROWS + row) * 2 + 1], sum);
#pragma unroll
                    for (int k = 0; k < V; ++k) x[k] = fmaf(f, o_smem[(w * ROWS + row) * L::OP + lane * V + k], x[k]);
                }
                if (whole) {
                    store_row<V>(a, p.q.row0, head, row_base + row, h * DP + lane * V, x, m, sum, h == 0 && lane == 0);
                } else {
#pragma unroll
                    for (int k = 0; k < V; ++k) part[2 * ROWS + row * D + h * DP + lane * V + k] = x[k];
                    if (h == 0 && lane == 0) {
                        part[row * 2] = m;
                        part[row * 2 + 1] = sum;
                    }
                }
            }
        }
        if (at + take == stop && threadIdx.x == 0) {  // the share ends here: is this the first piece of a cut task?
            Cut c{};
            if (!whole && p.unit == 0) {
                c.pieces = static_cast<int>(deal.owner(at + p.q.units - 1)) - static_cast<int>(blockIdx.x) + 1;
                c.row0 = p.q.row0;
                c.head = head;
                c.row_base = row_base;
                c.rows = rows;
            }
            *cut = c;
        }
        tc::fence_proxy_async_smem();  // what was written to the ring here is ordered before the next share's copies
        __syncthreads();

        at += take;
        if (at < stop) {  // the next task, or the next request that has any
            p.unit = 0;
            if (++p.task == p.q.tasks) {
                p.task = 0;
                do {
                    p.q = request_at<ROWS>(a, ++p.r, nullptr);
                } while (p.q.tasks == 0);
            }
        }
    }
}

// Joins the pieces of the tasks that the deal cut: CTA (c, y) those of the task that CTA c wrote down, the second place
// of c and the first ones of the CTAs behind it.  Few pieces: y = 0 takes all rows, a warp each; many (a long history of
// one request): four rows per CTA and two warps per row, so that enough loads are under way.
constexpr int kJoinWarps = 8;
template <int D, int NB>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const __grid_constant__ AttendArgs a) {
    constexpr int ROWS = 8 * NB, V = D / 32;
    constexpr int64_t kPiece = partial_floats<D, NB>();
    __shared__ float x_smem[kJoinWarps][D + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Cut cut = reinterpret_cast<const Cut*>(a.workspace)[blockIdx.x];
    const int pieces = cut.pieces;
    if (pieces == 0) return;
    const float* first =
        reinterpret_cast<const float*>(a.workspace + kCuts) + (static_cast<int64_t>(blockIdx.x) * 2 + 1) * kPiece;
    const auto piece = [&](int i) { return first + (i == 0 ? 0 : (2 * i - 1) * kPiece); };
    const bool shared = pieces > 2 * kJoinWarps;
    if (!shared && blockIdx.y > 0) return;
    const int step = shared ? 4 * gridDim.y : kJoinWarps;
    for (int row0 = shared ? blockIdx.y * 4 : 0; row0 < cut.rows; row0 += step) {
        const int row = row0 + (shared ? warp >> 1 : warp), part = shared ? warp & 1 : 0;
        const bool real = row < cut.rows;
        float m = kNone, x[V], sum = 0.f;
#pragma unroll
        for (int k = 0; k < V; ++k) x[k] = 0.f;
        if (real) {
            for (int i = lane; i < pieces; i += 32) m = fmaxf(m, __ldcg(piece(i) + row * 2));
#pragma unroll
            for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
#pragma unroll 8
            for (int i = part; i < pieces; i += shared ? 2 : 1) {
                const float* o = piece(i);
                const float f = exp2_approx(__ldcg(o + row * 2) - m);
                sum = fmaf(f, __ldcg(o + row * 2 + 1), sum);
#pragma unroll
                for (int k = 0; k < V; ++k) x[k] = fmaf(f, __ldcg(o + 2 * ROWS + row * D + lane * V + k), x[k]);
            }
        }
        if (shared) {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < V; ++k) x_smem[warp][lane * V + k] = x[k];
            if (lane == 0) x_smem[warp][D] = sum;
            __syncthreads();
            if (part == 0) {
                sum += x_smem[warp + 1][D];
#pragma unroll
                for (int k = 0; k < V; ++k) x[k] += x_smem[warp + 1][lane * V + k];
            }
        }
        if (real && part == 0) store_row<V>(a, cut.row0, cut.head, cut.row_base + row, lane * V, x, m, sum, lane == 0);
    }
}

template <int FMT, int D, int NB>
cudaError_t launch_rows(const AttendArgs& a, int sms, cudaStream_t s) {
    constexpr int smem = Layout<D, NB>::kBytes;
    static SmemOptIn opt_in;
    cudaError_t e = opt_in.once(reinterpret_cast<const void*>(attend_kernel<FMT, D, NB>), smem);
    if (e != cudaSuccess) return e;
    const int ctas = sms * ctas_per_sm(NB);
    CUtensorMap k_map, v_map;
    const int box = a.cache.page_size < kTile ? a.cache.page_size : kTile;
    if (!kv8_map(&k_map, a.cache, a.cache.k, box, true) || !kv8_map(&v_map, a.cache, a.cache.v, box, true))
        return cudaErrorInvalidValue;
    attend_kernel<FMT, D, NB><<<ctas, kThreads, smem, s>>>(a, k_map, v_map);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    // the join's CTAs come in as the last ones leave, and wait for them before they read
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas, 2);
    cfg.blockDim = dim3(kJoinWarps * 32);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, join_kernel<D, NB>, a);
}

// Fragments of 8 q rows per tile: as many as the largest request needs, but where the large ones are left to the other
// kernel, as many as one token does.  That is right where the rest have one token, and wrong where they have several, whose
// cache is then read once per tile; the lengths are on the device, so the rule cannot tell.  Whole calls with tiles of
// one token / of up to 32 rows, 4096 keys, D = 128: two chunks and 30 single tokens, groups of four, 245 / 259 us; one of 10
// tokens and 63 single ones 161 / 200; a chunk and 31 of 2-8 tokens 228 / 218; up to 9 tokens each 181 / 159.
int fragments(const AttendArgs& a) {
    const int64_t rows = a.few ? a.group : static_cast<int64_t>(a.max_q) * a.group;
    return rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
}

template <int FMT, int D>
cudaError_t launch_d(const AttendArgs& a, int sms, cudaStream_t s) {
    switch (fragments(a)) {
        case 1: return launch_rows<FMT, D, 1>(a, sms, s);
        case 2: return launch_rows<FMT, D, 2>(a, sms, s);
        default: return launch_rows<FMT, D, 4>(a, sms, s);
    }
}

// Above so many q rows of a request and KV head the tcgen05 kernel is faster although it pads them to 128: the warp MMAs
// read the codes once per 32 rows.  Here / there in us, 4096 keys each: 32 requests of 8 KV heads, D = 128, int8 or e4m3: 32
// rows 114-122 / 169-171, 40 rows 193-208 / 169-173; 8 requests of 2 heads: 46 / 52, then 52 / 52 up to 64 rows; four of 8
// heads over 32768 keys: 116 / 161, then 181 / 159.  With D = 64 the rows between 33 and 64 would still be faster
// here (32 requests of 4 heads: 32 rows 63 / 91, 40 rows 81 / 91, 64 rows 85 / 93), which the rule gives away.
constexpr int kFew = 32;

size_t few_bytes(const AttendArgs& a, int sms) {
    const int nb = fragments(a);
    return (kCuts + static_cast<size_t>(sms) * ctas_per_sm(nb) * 2 * (8 * nb) * (a.cache.head_dim + 2) * sizeof(float) +
            255) / 256 * 256;
}

AttendArgs split(const AttendArgs& a) {
    AttendArgs b = a;
    b.few = static_cast<int64_t>(a.max_q) * a.group > kFew ? kFew : 0;
    return b;
}

}  // namespace

bool kv8_map(CUtensorMap* m, const Kv8& c, const Kv8Side& side, int tokens, bool swizzle) {
    const uint64_t dims[4] = {static_cast<uint64_t>(c.head_dim), static_cast<uint64_t>(c.kv_heads),
                              static_cast<uint64_t>(c.page_size), static_cast<uint64_t>(c.pages)};
    // a dimension of one element has no stride that matters
    const uint64_t strides[3] = {c.kv_heads > 1 ? static_cast<uint64_t>(side.head_stride) : dims[0],
                                 static_cast<uint64_t>(side.token_stride),
                                 c.pages > 1 ? static_cast<uint64_t>(side.page_stride) : dims[0]};
    const uint32_t box[4] = {static_cast<uint32_t>(c.head_dim), 1, static_cast<uint32_t>(tokens), 1};
    return tc::make_map_u8_4d(m, side.codes, dims, strides, box, swizzle);
}

size_t attend_workspace_bytes(const AttendArgs& args, int sms) {
    const AttendArgs a = split(args);
    return few_bytes(a, sms) + (a.few ? prefill_workspace_bytes(a, sms) : 0);
}

cudaError_t launch_attend(const AttendArgs& args, int sms, cudaStream_t s) {
    if (args.tokens == 0) return cudaSuccess;
    const AttendArgs a = split(args);
    cudaError_t e = cudaSuccess;
    if (a.few && a.requests > 0) e = launch_prefill(a, kFew, a.workspace + few_bytes(a, sms), sms, s);
    if (e != cudaSuccess) return e;
    if (a.cache.format == PTOWSP_KV8_E4M3)
        return a.cache.head_dim == 64 ? launch_d<PTOWSP_KV8_E4M3, 64>(a, sms, s) : launch_d<PTOWSP_KV8_E4M3, 128>(a, sms, s);
    return a.cache.head_dim == 64 ? launch_d<PTOWSP_KV8_INT8, 64>(a, sms, s) : launch_d<PTOWSP_KV8_INT8, 128>(a, sms, s);
}

}  // namespace ptowsp::dev

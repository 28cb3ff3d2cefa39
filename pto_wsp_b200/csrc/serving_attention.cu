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
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "serving.hpp"
#include "serving_kv8.cuh"

namespace ptowsp::dev {

namespace {

constexpr int kWarps = 4;
constexpr int kTile = 32;                 // tokens per warp and step
constexpr int kUnit = kWarps * kTile;     // tokens per CTA and step: the grain in which work is dealt out
constexpr int kStages = 3;
constexpr int kThreads = kWarps * 32;
constexpr int kCtasPerSm = 2;

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
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
// one partial result in each CTA it touches, which a second launch joins.
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
    q.tasks = static_cast<int64_t>((static_cast<int64_t>(q.nq) * a.group + ROWS - 1) / ROWS) * a.cache.kv_heads;
    const int64_t span = q.hi - q.lo;
    q.units = span > 0 ? (span + kUnit - 1) / kUnit : 1;  // a task without keys still writes its zeros
    return q;
}

// The steps of all requests, and for a place in their line the request that holds it and the steps before that.
struct Deal {
    int64_t total;   // steps in all
    int64_t ctas;    // CTAs that share them
    int per;         // requests per thread of the scan
};

template <int ROWS>
__device__ Deal deal_out(const AttendArgs& a, int ctas, int64_t* sums, int* flags) {
    Deal d;
    d.per = (a.requests + kThreads - 1) / kThreads;
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
    __syncthreads();
    d.total = sums[kThreads - 1];
    d.ctas = d.total < ctas ? (d.total > 0 ? d.total : 1) : ctas;
    return d;
}

// First step of CTA c.
__device__ __forceinline__ int64_t deal_start(const Deal& d, int64_t c) {
    return c * (d.total / d.ctas) + (c < d.total % d.ctas ? c : d.total % d.ctas);
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
    p.task = (at - before) / p.q.units;
    p.unit = (at - before) % p.q.units;
    return p;
}

template <int D, int NB>
constexpr size_t partial_floats() { return static_cast<size_t>(8 * NB) * (D + 2); }

template <int D, int NB>
constexpr int attend_smem() {
    const int stage = kTile * D * 2 + 32;  // K and V codes, 4 scales
    const int ring = kWarps * kStages * stage;
    const int q = 8 * NB * (2 * D + 32);
    return ring + q + 8 * NB * 8 + kWarps * 8 * NB * 8;
}

// One tile of q rows of one head against its share of the tokens.  S^T = K.Q^T and O^T = V^T.P^T on
// mma.m16n8k16: 16 tokens (then 16 dims) x 8 q rows, so a group of 8 or fewer rows wastes at most half of the MMA, and
// the converted codes of a step serve 8 * NB rows.
template <int FMT, int D, int NB>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) attend_kernel(AttendArgs a) {
    constexpr int ROWS = 8 * NB;
    constexpr int CH = D / 16;                // 16-byte chunks of a row of codes
    constexpr int kSide = kTile * D;          // bytes of one side's tile
    constexpr int kStage = kSide * 2 + 32;
    constexpr int QP = 2 * D + 32;            // bytes between q rows: the fragments' 8-byte loads hit all banks
    extern __shared__ __align__(128) char smem[];
    char* q_smem = smem + kWarps * kStages * kStage;
    float* q_scale = reinterpret_cast<float*>(q_smem + ROWS * QP);   // [ROWS] a' = scale * log2(e) / row's power of two
    int* q_pos = reinterpret_cast<int*>(q_scale + ROWS);             // [ROWS] last key the row sees; -1: none, no row
    float* stat = reinterpret_cast<float*>(q_pos + ROWS);            // [kWarps][ROWS][2] M, l of the warps
    __shared__ int64_t sums[kThreads];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t4 = lane & 3;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    int flags = 0;
    const Deal deal = deal_out<ROWS>(a, gridDim.x, sums, &flags);
    if (blockIdx.x == 0 && flags && a.status) atomicOr(a.status, flags);
    if (deal.total == 0 || blockIdx.x >= deal.ctas) return;
    int64_t at = deal_start(deal, blockIdx.x);
    const int64_t stop = deal_start(deal, blockIdx.x + 1);
    Place p = find_place<ROWS>(a, deal, sums, at);

    char* ring = smem + warp * kStages * kStage;
    const uint32_t ring_u32 = smem_addr(ring);
    const int pshift = a.cache.page_shift, pmask = a.cache.page_size - 1;
    const int crow = lane / CH, cchunk = lane % CH;   // this lane's row and chunk of a 16-byte copy
    constexpr int RPC = 32 / CH;                      // rows per copy instruction

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

        // -- the warp's tiles: tok0 + (warp + 4 i) * 32 --
        const int first = tok0 + warp * kTile;
        const int ntiles = tok1 > first ? (tok1 - first + kUnit - 1) / kUnit : 0;
        // page ids of the two 16-token halves of tile i, lane 0 and 1 (-1: no token there)
        auto page_of = [&](int i) -> int {
            int id = -1;
            const int tok = first + i * kUnit + lane * 16;
            if (lane < 2 && i < ntiles && tok < tok1 && tok + 16 > p.q.seen) {
                id = table[tok >> pshift];
                if (id < 0 || id >= a.cache.pages) {
                    id = -1;
                    if (a.status) atomicOr(a.status, PTOWSP_SERVING_PAGE);
                }
            }
            return id;
        };
        auto issue = [&](int i, int ids) {
            if (i < ntiles) {
                const int tile = first + i * kUnit;
                const uint32_t dst = ring_u32 + (i % kStages) * kStage;
#pragma unroll
                for (int j = 0; j < kTile / RPC; ++j) {
                    const int row = j * RPC + crow;
                    const int id = __shfl_sync(~0u, ids, row >> 4);
                    const int tok = tile + row;
                    const bool live = id >= 0 && tok < tok1;
                    const int sw = D == 128 ? (cchunk ^ (row & 7)) : (cchunk ^ ((row >> 1) & 3));
                    const uint32_t to = dst + row * D + sw * 16;
                    const int64_t page = live ? id : 0;
                    const int64_t off = live ? (tok & pmask) : 0;
                    cp_async16(to, a.cache.k.codes + page * a.cache.k.page_stride + off * a.cache.k.token_stride +
                                       head * a.cache.k.head_stride + cchunk * 16, live);
                    cp_async16(to + kSide, a.cache.v.codes + page * a.cache.v.page_stride +
                                               off * a.cache.v.token_stride + head * a.cache.v.head_stride + cchunk * 16,
                               live);
                }
                const int id = __shfl_sync(~0u, ids, lane & 1);
                if (lane < 4) {  // k scale of half 0, 1, then v scale of half 0, 1; 0 where there is no page
                    const float* s = lane < 2 ? a.cache.k.scale : a.cache.v.scale;
                    cp_async4(dst + 2 * kSide + lane * 4,
                              s + static_cast<int64_t>(id < 0 ? 0 : id) * a.cache.kv_heads + head, id >= 0);
                }
            }
            cp_async_commit();
        };
        int ids = page_of(0);
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) {
            const int next = page_of(i + 1);
            issue(i, ids);
            ids = next;
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
            __half* to = reinterpret_cast<__half*>(q_smem + row * QP) + lane * (D / 32);
#pragma unroll
            for (int k = 0; k < D / 32; ++k) to[k] = __float2half_rn(x[k] * f);
            if (lane == 0) {
                q_scale[row] = a.scale * 1.4426950408889634f * __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
                q_pos[row] = real ? p.q.len - p.q.nq + j : -1;
            }
        }
        __syncthreads();

        float qs[NB][2];
        int pos[NB][2];
        int min_pos = INT32_MAX, max_pos = -1;
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                qs[n][c] = q_scale[n * 8 + 2 * t4 + c];
                pos[n][c] = q_pos[n * 8 + 2 * t4 + c];
            }
        for (int i = 0; i < rows; ++i) {  // of the real rows: which tiles need no mask
            min_pos = min(min_pos, q_pos[i]);
            max_pos = max(max_pos, q_pos[i]);
        }
        uint32_t qf[NB <= 2 ? NB : 1][CH][2];
        if constexpr (NB <= 2) {
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int c = 0; c < CH; ++c) {
                    const uint2 w = *reinterpret_cast<const uint2*>(q_smem + (n * 8 + g) * QP + c * 32 + t4 * 8);
                    qf[n][c][0] = w.x;
                    qf[n][c][1] = w.y;
                }
        }

        float M[NB][2], l[NB][2], o[NB][CH][4];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            M[n][0] = M[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
#pragma unroll
            for (int c = 0; c < CH; ++c) o[n][c][0] = o[n][c][1] = o[n][c][2] = o[n][c][3] = 0.f;
        }

        for (int i = 0; i < ntiles; ++i) {
            const int next = page_of(i + kStages);
            issue(i + kStages - 1, ids);
            ids = next;
            cp_async_wait<kStages - 1>();
            __syncwarp();
            const int tile = first + i * kUnit;
            const char* st = ring + (i % kStages) * kStage;
            const uint32_t st_u32 = ring_u32 + (i % kStages) * kStage;

            // S^T: two blocks of 16 tokens
            float s[2][NB][4];
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int n = 0; n < NB; ++n) s[b][n][0] = s[b][n][1] = s[b][n][2] = s[b][n][3] = 0.f;
#pragma unroll
            for (int c = 0; c < CH; c += 2) {
                uint32_t qv[NB][2][2];
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        if constexpr (NB <= 2) {
                            qv[n][k][0] = qf[n][c + k][0];
                            qv[n][k][1] = qf[n][c + k][1];
                        } else {
                            const uint2 w =
                                *reinterpret_cast<const uint2*>(q_smem + (n * 8 + g) * QP + (c + k) * 32 + t4 * 8);
                            qv[n][k][0] = w.x;
                            qv[n][k][1] = w.y;
                        }
                    }
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const int row = b * 16 + (lane & 15), ch = c + (lane >> 4);
                    const int sw = D == 128 ? (ch ^ (row & 7)) : (ch ^ ((row >> 1) & 3));
                    uint32_t w[4];
                    ldmatrix4(st_u32 + row * D + sw * 16, w);
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

            // exponents t = a' s_k S + log2 s_v
            const float* sc = reinterpret_cast<const float*>(st + 2 * kSide);
            const bool plain = tile + kTile <= min(tok1, min_pos + 1) && sc[0] > 0.f && sc[1] > 0.f &&
                               !(a.window > 0 && tile <= max_pos - a.window);
            float inv[2];
            bool grow = false;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const float ks = sc[b], vs = sc[2 + b];
                const float lv = log2_approx(vs);
                inv[b] = 1.f / vs;
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        float x = fmaf(s[b][n][k], qs[n][k & 1] * ks, lv);
                        if (!plain) {
                            const int tok = tile + b * 16 + g + (k >> 1) * 8;
                            const int last = pos[n][k & 1];
                            const bool seen = ks > 0.f && tok < tok1 && tok <= last &&
                                              !(a.window > 0 && tok <= last - a.window);
                            if (!seen) x = -INFINITY;
                        }
                        s[b][n][k] = x;
                        grow |= x > M[n][k & 1] + 15.f;
                    }
                if (!(vs > 0.f)) inv[b] = 0.f;
            }
            // M follows only when a weight would pass 2^15, and then leaves the largest at 2^7
            if (__any_sync(~0u, grow)) {
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        float m = fmaxf(fmaxf(s[0][n][c], s[0][n][c + 2]), fmaxf(s[1][n][c], s[1][n][c + 2]));
                        m = fmaxf(m, __shfl_xor_sync(~0u, m, 4));
                        m = fmaxf(m, __shfl_xor_sync(~0u, m, 8));
                        m = fmaxf(m, __shfl_xor_sync(~0u, m, 16));
                        m = fmaxf(m - 7.f, M[n][c]);
                        const float f = M[n][c] == -INFINITY ? 0.f : exp2_approx(M[n][c] - m);
                        M[n][c] = m;
                        l[n][c] *= f;
#pragma unroll
                        for (int d = 0; d < CH; ++d) {
                            o[n][d][c] *= f;
                            o[n][d][c + 2] *= f;
                        }
                    }
            }
            uint32_t pb[2][NB][2];
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    const float m0 = M[n][0] == -INFINITY ? 0.f : M[n][0], m1 = M[n][1] == -INFINITY ? 0.f : M[n][1];
                    const float w0 = exp2_approx(s[b][n][0] - m0), w1 = exp2_approx(s[b][n][1] - m1);
                    const float w2 = exp2_approx(s[b][n][2] - m0), w3 = exp2_approx(s[b][n][3] - m1);
                    l[n][0] = fmaf(w0 + w2, inv[b], l[n][0]);
                    l[n][1] = fmaf(w1 + w3, inv[b], l[n][1]);
                    pb[b][n][0] = transpose8x8(pack_f16(w0, w1));
                    pb[b][n][1] = transpose8x8(pack_f16(w2, w3));
                }
            // O^T += V^T.P^T
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int c = 0; c < CH; c += 2) {
                    const int row = b * 16 + (lane & 15), ch = c + (lane >> 4);
                    const int sw = D == 128 ? (ch ^ (row & 7)) : (ch ^ ((row >> 1) & 3));
                    uint32_t w[4];
                    ldmatrix4_trans(st_u32 + kSide + row * D + sw * 16, w);
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
            __syncwarp();
        }
        cp_async_wait<0>();

        // -- join the warps: O through the ring (every warp is done with it), M and l beside it --
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
        __syncthreads();
        constexpr int OP = D + 4;  // floats between rows
        float* o_smem = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    *reinterpret_cast<float2*>(&o_smem[(warp * ROWS + n * 8 + 2 * t4 + k) * OP + c * 16 + 2 * g]) =
                        make_float2(o[n][c][k], o[n][c][k + 2]);
        __syncthreads();
        float* part = reinterpret_cast<float*>(a.workspace) +
                      (static_cast<int64_t>(blockIdx.x) * 2 + (p.unit > 0 ? 0 : 1)) * partial_floats<D, NB>();
        for (int row = warp; row < rows; row += kWarps) {
            float m = -INFINITY, sum = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) m = fmaxf(m, stat[(w * ROWS + row) * 2]);
            float f[kWarps];
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float mw = stat[(w * ROWS + row) * 2];
                f[w] = mw == -INFINITY ? 0.f : exp2_approx(mw - m);
                sum += f[w] * stat[(w * ROWS + row) * 2 + 1];
            }
            float x[D / 32];
#pragma unroll
            for (int k = 0; k < D / 32; ++k) x[k] = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w)
#pragma unroll
                for (int k = 0; k < D / 32; ++k)
                    x[k] = fmaf(f[w], o_smem[(w * ROWS + row) * OP + lane * (D / 32) + k], x[k]);
            if (whole) {
                const int flat = row_base + row;
                const int64_t tok = p.q.row0 + flat / a.group;
                const int hq = head * a.group + flat % a.group;
                const float r = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
                const int64_t off = tok * a.out_token_stride + hq * a.out_head_stride + lane * (D / 32);
#pragma unroll
                for (int k = 0; k < D / 32; k += 2) {
                    if (a.dtype == PTOWSP_F16)
                        *reinterpret_cast<__half2*>(static_cast<__half*>(a.out) + off + k) =
                            __floats2half2_rn(x[k] * r, x[k + 1] * r);
                    else
                        *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(a.out) + off + k) =
                            __floats2bfloat162_rn(x[k] * r, x[k + 1] * r);
                }
                if (lane == 0 && a.lse)
                    a.lse[tok * a.heads + hq] = sum > 0.f || sum != sum ? (m + log2f(sum)) * 0.6931471805599453f : -INFINITY;
            } else {
#pragma unroll
                for (int k = 0; k < D / 32; ++k) part[2 * ROWS + row * D + lane * (D / 32) + k] = x[k];
                if (lane == 0) {
                    part[row * 2] = m;
                    part[row * 2 + 1] = sum;
                }
            }
        }
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

// Joins the partial results of the tasks that the deal cut.  CTA c looks at the cut before CTA c's share and does the
// work where that is its task's first cut: the pieces are the last one of CTA c - 1 and the first ones of the CTAs
// from c to the task's end.  One warp per row, its lanes over the dims, warps over the rows.
template <int D, int NB>
__global__ void __launch_bounds__(kThreads) join_kernel(AttendArgs a, int ctas) {
    constexpr int ROWS = 8 * NB;
    __shared__ int64_t sums[kThreads];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Deal deal = deal_out<ROWS>(a, ctas, sums, nullptr);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t c = blockIdx.x + 1;
    if (c >= deal.ctas) return;
    const int64_t at = deal_start(deal, c);
    const Place p = find_place<ROWS>(a, deal, sums, at);
    if (p.unit == 0) return;  // a cut between tasks
    const int64_t begin = at - p.unit, end = begin + p.q.units;
    if (deal_start(deal, c - 1) > begin) return;  // an earlier cut of this task has it
    int64_t last = c;
    while (last + 1 < deal.ctas && deal_start(deal, last + 1) < end) ++last;
    const int pieces = static_cast<int>(last - c) + 2;
    const int head = static_cast<int>(p.task % a.cache.kv_heads);
    const int row_base = static_cast<int>(p.task / a.cache.kv_heads) * ROWS;
    const int rows = min(ROWS, p.q.nq * a.group - row_base);
    const float* ws = reinterpret_cast<const float*>(a.workspace);
    auto piece = [&](int i) {
        return ws + (i == 0 ? (c - 1) * 2 + 1 : (c + i - 1) * 2) * static_cast<int64_t>(partial_floats<D, NB>());
    };
    for (int row = blockIdx.y * kWarps + warp; row < rows; row += gridDim.y * kWarps) {
        float m = -INFINITY;
        for (int i = lane; i < pieces; i += 32) m = fmaxf(m, __ldcg(piece(i) + row * 2));
#pragma unroll
        for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
        float x[D / 32], sum = 0.f;
#pragma unroll
        for (int k = 0; k < D / 32; ++k) x[k] = 0.f;
#pragma unroll 8
        for (int i = 0; i < pieces; ++i) {
            const float* q = piece(i);
            const float mi = __ldcg(q + row * 2), li = __ldcg(q + row * 2 + 1);
            const float f = mi == -INFINITY ? 0.f : exp2_approx(mi - m);
            sum = fmaf(f, li, sum);
#pragma unroll
            for (int k = 0; k < D / 32; ++k)
                x[k] = fmaf(f, __ldcg(q + 2 * ROWS + row * D + lane * (D / 32) + k), x[k]);
        }
        const int flat = row_base + row;
        const int64_t tok = p.q.row0 + flat / a.group;
        const int hq = head * a.group + flat % a.group;
        const float r = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
        const int64_t off = tok * a.out_token_stride + hq * a.out_head_stride + lane * (D / 32);
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
            if (a.dtype == PTOWSP_F16) static_cast<__half*>(a.out)[off + k] = __float2half_rn(x[k] * r);
            else static_cast<__nv_bfloat16*>(a.out)[off + k] = __float2bfloat16_rn(x[k] * r);
        }
        if (lane == 0 && a.lse)
            a.lse[tok * a.heads + hq] = sum > 0.f || sum != sum ? (m + log2f(sum)) * 0.6931471805599453f : -INFINITY;
    }
}

template <int FMT, int D, int NB>
cudaError_t launch_rows(const AttendArgs& a, int sms, cudaStream_t s) {
    constexpr int smem = attend_smem<D, NB>();
    cudaError_t e = cudaFuncSetAttribute(attend_kernel<FMT, D, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    const int ctas = sms * kCtasPerSm;
    attend_kernel<FMT, D, NB><<<ctas, kThreads, smem, s>>>(a);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    // the join starts while the last CTAs finish; it waits for them before it reads
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(ctas - 1, 2 * NB);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, join_kernel<D, NB>, a, ctas);
}

template <int FMT, int D>
cudaError_t launch_d(const AttendArgs& a, int sms, cudaStream_t s) {
    const int64_t rows = static_cast<int64_t>(a.max_q) * a.group;
    if (rows <= 8) return launch_rows<FMT, D, 1>(a, sms, s);
    if (rows <= 16) return launch_rows<FMT, D, 2>(a, sms, s);
    return launch_rows<FMT, D, 4>(a, sms, s);
}

}  // namespace

size_t attend_workspace_bytes(const AttendArgs& a, int sms) {
    const int64_t rows = static_cast<int64_t>(a.max_q) * a.group;
    const int nb = rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
    return static_cast<size_t>(sms) * kCtasPerSm * 2 * (8 * nb) * (a.cache.head_dim + 2) * sizeof(float);
}

cudaError_t launch_attend(const AttendArgs& a, int sms, cudaStream_t s) {
    if (a.requests == 0 || a.tokens == 0) return cudaSuccess;
    if (a.cache.format == PTOWSP_KV8_E4M3)
        return a.cache.head_dim == 64 ? launch_d<PTOWSP_KV8_E4M3, 64>(a, sms, s) : launch_d<PTOWSP_KV8_E4M3, 128>(a, sms, s);
    return a.cache.head_dim == 64 ? launch_d<PTOWSP_KV8_INT8, 64>(a, sms, s) : launch_d<PTOWSP_KV8_INT8, 128>(a, sms, s);
}

}  // namespace ptowsp::dev

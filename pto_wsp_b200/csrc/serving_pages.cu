// Page reservation (block tables and slot maps from request lengths) and the writer of the 8-bit paged KV cache.
#include <cuda_fp8.h>

#include <algorithm>

#include "serving.hpp"
#include "serving_kv8.cuh"

namespace ptowsp::dev {

namespace {

// ---------------------------------------------------------------------------
// Reservation.  Per request r: have = ceil(len / page), need = ceil((len + new) / page) - have; the new pages are the
// ring entries head + (sum of need before r) + j, the new tokens the list entries q_start[r] + j.  Everything follows
// from prefix sums over the requests: tokens, needed pages, returned pages, and the pages in fact given, four block scans
// of three barriers each per 1024 requests.  Every CTA runs the sums for itself -- a thousand requests are one round of
// the scans, cheaper than a second launch -- keeps the two that the token list needs in shared memory and then fills its
// share of the outputs; CTA 0 writes the per-request ones.
//
// Bound by latency: 5.5 us on the device for 64 requests of one token, 12 for 1001 requests with 0-511 each, of a whole
// call of 18 us in which the host allocates six results.
// ---------------------------------------------------------------------------

constexpr int kRsvThreads = 1024;

__device__ __forceinline__ int64_t warp_inclusive(int64_t v, int lane) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t o = __shfl_up_sync(~0u, v, d);
        if (lane >= d) v += o;
    }
    return v;
}

// Inclusive scan over the block; *total: the block's sum.  `part`: 32 words that nothing else uses.
__device__ __forceinline__ int64_t block_inclusive(int64_t v, int64_t* part, int64_t* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    v = warp_inclusive(v, lane);
    __syncthreads();
    if (lane == 31) part[warp] = v;
    __syncthreads();
    if (warp == 0) part[lane] = warp_inclusive(part[lane], lane);
    __syncthreads();
    *total = part[31];
    return v + (warp ? part[warp - 1] : 0);
}

struct RsvRequest {
    int64_t len, want, have, need, back;
    bool fits;
};

__global__ void __launch_bounds__(kRsvThreads) reserve_kernel(ReserveArgs a) {
    extern __shared__ int32_t rsv_smem[];
    int32_t* q_end = rsv_smem;               // [requests], saturated
    int32_t* taken = rsv_smem + a.requests;  // [requests]: ring pages taken before r, -1: refused or ended
    __shared__ int64_t part[32];
    const int64_t page = a.page_size;
    const int shift = 31 - __clz(a.page_size);
    const int64_t head = a.free_state[0], tail = a.free_state[1];
    int64_t avail = tail - head;
    int flags = 0;
    // such a ring gives no page and takes none; the last comparison keeps the places behind the tail countable
    const bool broken = head < 0 || tail < head || avail > a.ring_size || tail > INT64_MAX - a.ring_size;
    if (broken) {
        avail = 0;
        flags |= PTOWSP_SERVING_RING;
    }
    int64_t q_before = 0, need_before = 0, back_before = 0, used = 0;
    const bool first = blockIdx.x == 0;
    for (int r0 = 0; r0 < a.requests; r0 += kRsvThreads) {
        const int r = r0 + threadIdx.x;
        RsvRequest t{};
        int64_t fresh = 0;
        if (r < a.requests) {
            t.len = a.kv_len[r];
            fresh = a.new_tokens[r];
            t.want = fresh > 0 ? fresh : 0;
            const bool bad = t.len < 0;
            if (bad) flags |= PTOWSP_SERVING_LENGTH;
            t.have = bad ? 0 : (t.len + page - 1) >> shift;
            if (t.have > a.max_pages) {
                flags |= PTOWSP_SERVING_LENGTH;
                t.have = a.max_pages;
                t.fits = false;
            } else {
                t.fits = !bad && fresh >= 0;
            }
            t.back = fresh < 0 ? t.have : 0;
        }
        int64_t total;
        const int64_t qe = q_before + block_inclusive(t.want, part, &total);
        q_before += total;
        const int64_t after = (t.len + t.want + page - 1) >> shift;
        t.fits = t.fits && after <= a.max_pages && qe <= a.max_tokens;
        t.need = t.fits ? after - t.have : 0;
        const int64_t ne = need_before + block_inclusive(t.need, part, &total);
        need_before += total;
        const int64_t be = back_before + block_inclusive(t.back, part, &total);
        back_before += total;
        const bool granted = t.fits && (t.need == 0 || ne <= avail);
        int64_t got = granted ? t.need : 0;
        block_inclusive(got, part, &total);
        used += total;
        if (r < a.requests) {
            q_end[r] = static_cast<int32_t>(qe < INT32_MAX ? qe : INT32_MAX);
            taken[r] = granted ? static_cast<int32_t>(ne - t.need) : -1;
            if (fresh >= 0 && !granted) flags |= PTOWSP_SERVING_REFUSED;
            if (first) {
                a.q_start[r + 1] = q_end[r];
                a.kv_len_out[r] = static_cast<int32_t>(fresh < 0 ? 0 : t.len + (granted ? t.want : 0));
                a.granted[r] = granted;
            }
            if (t.back) taken[r] = -2 - static_cast<int32_t>(be - t.back < INT32_MAX - 2 ? be - t.back : INT32_MAX - 2);
        }
    }
    const bool overflow = broken || avail + back_before > a.ring_size;  // more pages than the ring has places
    if (overflow) flags |= PTOWSP_SERVING_RING;
    if (first && threadIdx.x == 0) {
        a.q_start[0] = 0;
        a.free_state_out[0] = head + used;
        a.free_state_out[1] = tail + (overflow ? 0 : back_before);
    }
    if (first && flags && a.status) atomicOr(a.status, flags);
    __syncthreads();

    // page-table rows of granted requests and ring places of ended ones: a warp per request
    const int lane = threadIdx.x & 31;
    const int warps = gridDim.x * (kRsvThreads / 32);
    for (int r = blockIdx.x * (kRsvThreads / 32) + (threadIdx.x >> 5); r < a.requests; r += warps) {
        const int64_t len = a.kv_len[r], fresh = a.new_tokens[r];
        int64_t have = (len + page - 1) >> shift;
        int32_t* row = a.page_table + r * a.table_stride;
        if (taken[r] >= 0) {
            const int64_t after = (len + fresh + page - 1) >> shift;
            for (int64_t j = have + lane; j < after; j += 32)
                row[j] = a.free_ring[(head + taken[r] + j - have) % a.ring_size];
        } else if (taken[r] <= -2 && !overflow) {
            if (have > a.max_pages) have = a.max_pages;
            const int64_t to = tail - 2 - static_cast<int64_t>(taken[r]);
            for (int64_t j = lane; j < have; j += 32) a.free_ring[(to + j) % a.ring_size] = row[j];
        }
    }
    // the token list: a binary search for the request, then its page from the table or straight from the ring
    const int64_t threads = static_cast<int64_t>(gridDim.x) * kRsvThreads;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kRsvThreads + threadIdx.x; i < a.max_tokens; i += threads) {
        int lo = 0, hi = a.requests;  // first r with q_end[r] > i
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (q_end[mid] > i) hi = mid;
            else lo = mid + 1;
        }
        int64_t slot = -1, pos = -1;
        if (lo < a.requests && taken[lo] >= 0) {
            const int64_t len = a.kv_len[lo], have = (len + page - 1) >> shift;
            pos = len + i - (lo ? q_end[lo - 1] : 0);
            const int64_t j = pos >> shift;
            const int32_t id = j < have ? a.page_table[lo * a.table_stride + j]
                                        : a.free_ring[(head + taken[lo] + j - have) % a.ring_size];
            slot = static_cast<int64_t>(id) * page + (pos & (page - 1));
        }
        a.slots[i] = slot;
        a.positions[i] = static_cast<int32_t>(pos);
    }
}

// ---------------------------------------------------------------------------
// Append.  A run -- the new tokens of one page -- of one head of K or of V belongs to one team of 1, 2 or 4 warps: it takes
// the largest |x|, settles the page's scale and writes the codes, so no two teams share a scale and no atomic is
// needed.  A CTA looks at `chunk` consecutive tokens of one head; a token whose predecessor is in another page begins a
// run, which the CTA that holds its first token writes to its end (at most a page).  Many short runs (decoding): a warp
// each; few long ones (prefill): the warps share each, so that its rows are all under way at once and are read once.
//
// Bound by HBM in principle, 2 or 4 bytes in and 1 out per element; in fact by instructions and the runs' fixed parts:
// 16,001 tokens of 8 heads of 128 in f16 to int8 (98 MB) take 45 us, 2.2 TB/s, and 31 million warp instructions.  Without
// the encoding it would be 23 million and a sixth less time: the rest is addresses, slots, bookkeeping, and warps that wait at
// the barrier while the first one looks for runs.  One warp per run took 128 us there.  64 single tokens take 8.5 us, 4.4 of them on the device.
// ---------------------------------------------------------------------------

constexpr int kAppWarps = 8;
constexpr int kAppMaxChunk = 32;

template <typename T>
__device__ __forceinline__ void unpack16(const uint4& w, float (&x)[16 / sizeof(T)]);
template <>
__device__ __forceinline__ void unpack16<float>(const uint4& w, float (&x)[4]) {
    x[0] = __uint_as_float(w.x);
    x[1] = __uint_as_float(w.y);
    x[2] = __uint_as_float(w.z);
    x[3] = __uint_as_float(w.w);
}
template <>
__device__ __forceinline__ void unpack16<__half>(const uint4& w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
template <>
__device__ __forceinline__ void unpack16<__nv_bfloat16>(const uint4& w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(u[i] << 16);
        x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}

// The largest |x| of 16-byte loads as a bit pattern, which orders like the magnitude, infinity and NaN above all.
template <typename T>
struct Largest {  // 16-bit types: two at a time
    uint32_t bits = 0;
    __device__ __forceinline__ void add(const uint4& w) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (sizeof(T) == 4) bits = max(bits, u[i] & 0x7fffffffu);
            else asm("max.u16x2 %0, %0, %1;" : "+r"(bits) : "r"(u[i] & 0x7fff7fffu));
        }
    }
    // over the warp, as f32; *finite: no infinity and no NaN among them
    __device__ __forceinline__ float of_warp(bool* finite) const;
};
template <>
__device__ __forceinline__ float Largest<float>::of_warp(bool* finite) const {
    const uint32_t m = __reduce_max_sync(~0u, bits);
    *finite = m < 0x7f800000u;
    return __uint_as_float(m);
}
template <>
__device__ __forceinline__ float Largest<__half>::of_warp(bool* finite) const {
    const uint32_t m = __reduce_max_sync(~0u, max(bits & 0xffffu, bits >> 16));
    *finite = m < 0x7c00u;
    return __half2float(__ushort_as_half(static_cast<unsigned short>(m)));
}
template <>
__device__ __forceinline__ float Largest<__nv_bfloat16>::of_warp(bool* finite) const {
    const uint32_t m = __reduce_max_sync(~0u, max(bits & 0xffffu, bits >> 16));
    *finite = m < 0x7f80u;
    return __uint_as_float(m << 16);
}

// Codes of 4 values x / scale, x not NaN; inv = RN(1 / scale), `exact` where that is exact (a power of two).  int8: the
// product is within 2^-16 of the quotient, so it rounds to the same integer unless it is that near to a half; only
// there the quotient itself is taken.  Adding 1.5 * 2^23 rounds to the nearest even integer and leaves it in the low bits
// (the conversion instructions have a quarter of an addition's rate).
__device__ __noinline__ uint32_t divide4(float x0, float x1, float x2, float x3, float scale) {
    const float v[4] = {x0, x1, x2, x3};
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float q = fminf(fmaxf(__fdiv_rn(v[i], scale), -127.f), 127.f);
        r |= (__float_as_uint(q + 12582912.f) & 0xffu) << (8 * i);
    }
    return r;
}
__device__ __noinline__ uint32_t divide4_e4m3(float x0, float x1, float x2, float x3, float scale) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(x0, scale), __fdiv_rn(x1, scale)), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(__fdiv_rn(x2, scale), __fdiv_rn(x3, scale)), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
}
template <int FMT>
__device__ __forceinline__ uint32_t encode4(float x0, float x1, float x2, float x3, float scale, float inv, bool exact) {
    const float v[4] = {x0, x1, x2, x3};
    if (FMT == PTOWSP_KV8_E4M3) {
        if (!exact) return divide4_e4m3(x0, x1, x2, x3, scale);
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x0 * inv, x1 * inv), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x2 * inv, x3 * inv), __NV_SATFINITE, __NV_E4M3);
        return lo | (hi << 16);
    }
    constexpr float kMagic = 12582912.f;
    uint32_t t[4];
    float far = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float q = fminf(fmaxf(v[i] * inv, -127.f), 127.f);
        const float r = q + kMagic;
        t[i] = __float_as_uint(r);
        far = fmaxf(far, fabsf(q - (r - kMagic)));
    }
    if (far > 0.49997f) return divide4(x0, x1, x2, x3, scale);
    return __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
}

template <int FMT>
__device__ __forceinline__ float scale_for(float amax) {
    if (FMT == PTOWSP_KV8_INT8) return fminf(fmaxf(amax * (1.f / 127.f), kKv8MinScale), kKv8MaxScale);
    if (!(amax > 0.f)) return kKv8MinScale;
    int e;
    const float m = frexpf(amax, &e);  // amax = m * 2^e with m in [0.5, 1); 448 = 0.875 * 2^9
    e = m <= 0.875f ? e - 9 : e - 8;
    return ldexpf(1.f, min(max(e, -60), 60));
}

// Warp `sub` of a team of `team` on one run.  `part`: a float per warp of the block.  Every warp of the block comes here
// (with run 0 where it has none) when the team is more than one warp, for the barriers.
template <typename T, int FMT, int D>
__device__ __forceinline__ void append_run(const Kv8Side& c, int64_t page, int head, int heads, int page_size, const char* x,
                                           int64_t token_stride, const int64_t* slots, int64_t i0, int run, int sub,
                                           int team, float* part) {
    constexpr int V = 16 / sizeof(T);       // elements per 16-byte load
    constexpr int LPT = D / V;              // lanes per token
    constexpr int TPW = 32 / LPT;           // tokens per warp load
    constexpr int U = 8;                    // loads in flight
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int el = (lane % LPT) * V;
    const T* src = reinterpret_cast<const T*>(x) + el + (i0 + sub * TPW + lane / LPT) * token_stride;
    const int64_t step = static_cast<int64_t>(team) * TPW * token_stride;  // between this lane's loads
    // token of load s of this lane
    const auto token = [&](int s) { return (s * team + sub) * TPW + lane / LPT; };
    const int steps = (run + TPW * team - 1) / (TPW * team);
    uint4 raw[U];
    Largest<T> largest;
    for (int s0 = 0; s0 < steps; s0 += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = token(s0 + u);
            raw[u] = make_uint4(0, 0, 0, 0);
            if (j < run) raw[u] = *reinterpret_cast<const uint4*>(src + (s0 + u) * step);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) largest.add(raw[u]);
    }
    bool finite;
    float amax = largest.of_warp(&finite);
    if (!finite) {  // look again, at the finite ones
        amax = 0.f;
        for (int s = 0; s < steps; ++s) {
            const int j = token(s);
            uint4 w = make_uint4(0, 0, 0, 0);
            if (j < run) w = *reinterpret_cast<const uint4*>(src + s * step);
            float f[V];
            unpack16<T>(w, f);
#pragma unroll
            for (int k = 0; k < V; ++k) amax = fabsf(f[k]) < INFINITY ? fmaxf(amax, fabsf(f[k])) : amax;
        }
        amax = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(amax)));  // ordered: not negative
    }
    float* scale_at = c.scale + page * heads + head;
    const float old = run ? *scale_at : 1.f;
    if (team > 1) {
        if (lane == 0) part[warp] = amax;
        __syncthreads();
        for (int w = warp - sub; w < warp - sub + team; ++w) amax = fmaxf(amax, part[w]);
    }
    if (!run) return;
    // a run's slots ascend, so its first one tells whether it holds the page's token 0
    const bool fresh = (slots[i0] & (page_size - 1)) == 0;
    const float need = scale_for<FMT>(amax);
    const float scale = fresh ? need : fmaxf(old, need);
    const float inv = __frcp_rn(scale);
    const bool exact = (__float_as_uint(scale) & 0x007fffffu) == 0;
    uint8_t* base = c.codes + page * c.page_stride + head * c.head_stride;
    if (!fresh && scale > old) {  // round the page's other codes to the new scale
        uint32_t mask[4] = {0, 0, 0, 0};  // offsets that the run writes
        for (int j = lane; j < run; j += 32) {
            const int off = static_cast<int>(slots[i0 + j] & (page_size - 1));
            mask[off >> 5] |= 1u << (off & 31);
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) mask[w] = __reduce_or_sync(~0u, mask[w]);
        constexpr int LPR = D / 16, RPW = 32 / LPR;  // lanes per row of codes, rows per warp
        for (int off = sub * RPW + lane / LPR; off < page_size; off += team * RPW) {
            const uint32_t word = off < 32 ? mask[0] : off < 64 ? mask[1] : off < 96 ? mask[2] : mask[3];
            if (word >> (off & 31) & 1u) continue;
            uint4* p = reinterpret_cast<uint4*>(base + off * c.token_stride + (lane % LPR) * 16);
            uint4 w = *p;
            uint32_t* u = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float f[4];
                decode4<FMT>(u[k], f);
                u[k] = encode4<FMT>(f[0] * old, f[1] * old, f[2] * old, f[3] * old, scale, inv, exact);
            }
            *p = w;
        }
    }
    __syncwarp();  // the old scale has been read, by the team's other warps before the barrier above
    if (sub == 0 && lane == 0) *scale_at = scale;
    for (int s0 = 0; s0 < steps; s0 += U) {
        if (steps > U) {  // a share of more than U loads is read again (it is in the cache); else it is in registers
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = token(s0 + u);
                raw[u] = make_uint4(0, 0, 0, 0);
                if (j < run) raw[u] = *reinterpret_cast<const uint4*>(src + (s0 + u) * step);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = token(s0 + u);
            if (j >= run) continue;
            float f[V];
            unpack16<T>(raw[u], f);
            if (!finite) {
#pragma unroll
                for (int k = 0; k < V; ++k) f[k] = f[k] == f[k] ? f[k] : 0.f;
            }
            uint32_t out[V / 4];
#pragma unroll
            for (int k = 0; k < V / 4; ++k)
                out[k] = encode4<FMT>(f[4 * k], f[4 * k + 1], f[4 * k + 2], f[4 * k + 3], scale, inv, exact);
            const int off = static_cast<int>(slots[i0 + j] & (page_size - 1));
            uint8_t* to = base + off * c.token_stride + el;
            if constexpr (V == 8) *reinterpret_cast<uint2*>(to) = make_uint2(out[0], out[1]);
            else *reinterpret_cast<uint32_t*>(to) = out[0];
        }
    }
}

template <typename T, int FMT, int D>
__global__ void __launch_bounds__(kAppWarps * 32, 4) append_kernel(const __grid_constant__ AppendArgs a, int chunk) {
    __shared__ int first[kAppMaxChunk], length[kAppMaxChunk], page_of[kAppMaxChunk];
    __shared__ int runs;
    __shared__ float part[kAppWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int heads = a.cache.kv_heads, shift = a.cache.page_shift, page_size = a.cache.page_size;
    // the heads of a token stand side by side in memory: their CTAs run at the same time
    const int head = static_cast<int>(blockIdx.x % static_cast<unsigned>(heads));
    const int64_t c0 = static_cast<int64_t>(blockIdx.x / static_cast<unsigned>(heads)) * chunk;
    if (warp == 0) {
        const int64_t limit = a.cache.pages << shift;
        // whether token i goes on with the run of token i - 1, and its slot
        const auto look = [&](int64_t i, bool* goes_on) -> int64_t {
            const int64_t s = i < a.tokens ? a.slots[i] : -1;
            const int64_t before = i > 0 && i <= a.tokens ? a.slots[i - 1] : -1;
            const bool ok = s >= 0 && s < limit;
            *goes_on = ok && before >= 0 && before < s && (before >> shift) == (s >> shift);
            return ok ? s : s == -1 ? -1 : -2;
        };
        bool goes_on;
        const int64_t s = look(c0 + lane, &goes_on);
        const bool here = lane < chunk;
        if (here && s == -2 && a.status) atomicOr(a.status, PTOWSP_SERVING_PAGE);
        const uint32_t begins = __ballot_sync(~0u, here && s >= 0 && !goes_on);
        const uint32_t breaks = __ballot_sync(~0u, here && !goes_on);
        if (begins >> lane & 1u) {
            const int k = __popc(begins & ((1u << lane) - 1u));
            const uint32_t later = lane == 31 ? 0u : breaks >> (lane + 1) << (lane + 1);
            first[k] = lane;
            page_of[k] = static_cast<int>(s >> shift);
            length[k] = (later ? __ffs(later) - 1 : chunk) - lane;
        }
        if (lane == 0) runs = __popc(begins);
        // the run that holds the chunk's last token may go on behind it, to the end of its page at most
        const bool open = begins && __clz(static_cast<int>(breaks)) == __clz(static_cast<int>(begins));
        __syncwarp();
        if (open) {
            int more = 0;
            for (int64_t i = c0 + chunk;; i += 32) {
                look(i + lane, &goes_on);
                const uint32_t stop = __ballot_sync(~0u, !goes_on);
                if (stop) {
                    more += __ffs(stop) - 1;
                    break;
                }
                more += 32;
            }
            if (lane == 0) length[__popc(begins) - 1] += more;
        }
    }
    __syncthreads();
    const int items = runs * 2;
    const int team = items > kAppWarps / 2 ? 1 : items > kAppWarps / 4 ? 2 : 4;
    const int teams = kAppWarps / team;
    for (int it0 = 0; it0 < items; it0 += teams) {
        const int it = it0 + warp / team;
        const bool live = it < items;
        const int which = it & 1, k = live ? it >> 1 : 0;
        const int64_t i0 = c0 + first[k];
        const char* x = static_cast<const char*>(which ? a.v : a.k) +
                        head * (which ? a.v_head_stride : a.k_head_stride) * static_cast<int64_t>(sizeof(T));
        append_run<T, FMT, D>(which ? a.cache.v : a.cache.k, page_of[k], head, heads, page_size, x,
                              which ? a.v_token_stride : a.k_token_stride, a.slots, i0, live ? length[k] : 0, warp % team,
                              team, part);
        if (team > 1) __syncthreads();  // `part` has been read
    }
}

template <typename T, int FMT>
cudaError_t append_d(const AppendArgs& a, dim3 grid, int chunk, cudaStream_t s) {
    if (a.cache.head_dim == 64) append_kernel<T, FMT, 64><<<grid, kAppWarps * 32, 0, s>>>(a, chunk);
    else append_kernel<T, FMT, 128><<<grid, kAppWarps * 32, 0, s>>>(a, chunk);
    return cudaGetLastError();
}

template <typename T>
cudaError_t append_t(const AppendArgs& a, dim3 grid, int chunk, cudaStream_t s) {
    return a.cache.format == PTOWSP_KV8_E4M3 ? append_d<T, PTOWSP_KV8_E4M3>(a, grid, chunk, s)
                                             : append_d<T, PTOWSP_KV8_INT8>(a, grid, chunk, s);
}

}  // namespace

cudaError_t launch_reserve(const ReserveArgs& a, cudaStream_t s) {
    const int smem = std::max(1, a.requests) * 8;
    if (smem > 47 * 1024) {  // with the kernel's static words more than 48 KB
        static SmemOptIn opt_in;  // for the most requests at once: a limit of this call's size would be another thread's too
        const cudaError_t e = opt_in.once(reinterpret_cast<const void*>(reserve_kernel), kReserveMaxRequests * 8);
        if (e != cudaSuccess) return e;
    }
    // one CTA per 4096 tokens or 256 requests: below that the extra CTAs' own prefix sums cost more than they save
    const int64_t want = std::max<int64_t>((a.max_tokens + 4095) / 4096, (a.requests + 255) / 256);
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(want, 1), 148));
    reserve_kernel<<<grid, kRsvThreads, smem, s>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_append(const AppendArgs& a, cudaStream_t s) {
    if (a.tokens == 0) return cudaSuccess;
    // few tokens: two per CTA and head; many: 32
    int chunk = 2;
    while (chunk < kAppMaxChunk && a.tokens * a.cache.kv_heads > 592 * static_cast<int64_t>(chunk)) chunk *= 2;
    const int64_t blocks = (a.tokens + chunk - 1) / chunk * a.cache.kv_heads;
    if (blocks > INT32_MAX) return cudaErrorInvalidValue;
    const dim3 grid(static_cast<unsigned>(blocks));
    switch (a.dtype) {
        case PTOWSP_F32: return append_t<float>(a, grid, chunk, s);
        case PTOWSP_F16: return append_t<__half>(a, grid, chunk, s);
        default: return append_t<__nv_bfloat16>(a, grid, chunk, s);
    }
}

}  // namespace ptowsp::dev

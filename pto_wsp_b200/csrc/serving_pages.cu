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
// from three prefix sums over the requests (tokens, needed pages, returned pages).  Every CTA runs the sums for
// itself -- a thousand requests are one round of a block scan, cheaper than a second launch -- keeps the two that the
// token list needs in shared memory and then fills its share of the outputs; CTA 0 writes the per-request ones.
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

// Inclusive scan over the block; *total: the block's sum.  `part`: 33 words that nothing else uses.
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
    if (avail < 0 || avail > a.ring_size || head < 0) {
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
    const bool overflow = avail + back_before > a.ring_size;  // more pages than the ring has places
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
// Append.  One warp owns one run -- the new tokens of one page -- of one head of K or of V: it takes the largest |x|,
// settles the page's scale and writes the codes, so no two warps share a scale and no atomic is needed.  A CTA looks
// at `chunk` consecutive tokens; a token whose predecessor is in another page begins a run, which the CTA that holds
// its first token writes to its end (at most a page).
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

// Codes of 4 values x / scale, x not NaN.  `inv` is the reciprocal of a power of two (the product is then the exact
// quotient), or 0: divide.
template <int FMT>
__device__ __forceinline__ uint32_t encode4(float x0, float x1, float x2, float x3, float scale, float inv) {
    float v[4] = {x0, x1, x2, x3};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = inv != 0.f ? v[i] * inv : __fdiv_rn(v[i], scale);
    if (FMT == PTOWSP_KV8_E4M3) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[0], v[1]), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[2], v[3]), __NV_SATFINITE, __NV_E4M3);
        return lo | (hi << 16);
    }
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = static_cast<int>(rintf(fminf(fmaxf(v[i], -127.f), 127.f)));
        r |= (static_cast<uint32_t>(c) & 0xffu) << (8 * i);
    }
    return r;
}

// 1 / s for a power of two, else 0.
__device__ __forceinline__ float exact_inverse(float s) {
    return (__float_as_uint(s) & 0x007fffffu) == 0 ? __fdiv_rn(1.f, s) : 0.f;
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

template <typename T, int FMT, int D>
__device__ void append_run(const Kv8Side& c, int64_t page, int head, int heads, int page_size, const char* x,
                           int64_t token_stride, const int64_t* slots, int64_t i0, int run, int lane) {
    constexpr int V = 16 / sizeof(T);       // elements per 16-byte load
    constexpr int LPT = D / V;              // lanes per token
    constexpr int TPW = 32 / LPT;           // tokens per warp load
    constexpr int U = 8;                    // loads in flight
    const int sub = lane / LPT, el = (lane % LPT) * V;
    const T* src = reinterpret_cast<const T*>(x) + el;
    // offsets that the run writes, and its largest finite |x|
    uint32_t mask[4] = {0, 0, 0, 0};
    for (int j = lane; j < run; j += 32) {
        const int off = static_cast<int>(slots[i0 + j] & (page_size - 1));
        mask[off >> 5] |= 1u << (off & 31);
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) mask[w] = __reduce_or_sync(~0u, mask[w]);
    float amax = 0.f;
    uint4 raw[U];
    const int steps = (run + TPW - 1) / TPW;
    for (int s0 = 0; s0 < steps; s0 += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = (s0 + u) * TPW + sub;
            raw[u] = make_uint4(0, 0, 0, 0);
            if (j < run) raw[u] = *reinterpret_cast<const uint4*>(src + (i0 + j) * token_stride);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float f[V];
            unpack16<T>(raw[u], f);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float m = fabsf(f[k]);
                amax = m < INFINITY ? fmaxf(amax, m) : amax;
            }
        }
    }
    amax = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(amax)));  // ordered: not negative
    float* scale_at = c.scale + page * heads + head;
    const bool fresh = mask[0] & 1u;
    const float old = *scale_at;
    const float need = scale_for<FMT>(amax);
    const float scale = fresh ? need : fmaxf(old, need);
    const float inv = exact_inverse(scale);
    uint8_t* base = c.codes + page * c.page_stride + head * c.head_stride;
    if (!fresh && scale > old) {  // round the page's other codes to the new scale
        constexpr int LPR = D / 16;  // lanes per row of codes
        for (int off = lane / LPR; off < page_size; off += 32 / LPR) {
            if (mask[off >> 5] >> (off & 31) & 1u) continue;
            uint4* p = reinterpret_cast<uint4*>(base + off * c.token_stride + (lane % LPR) * 16);
            uint4 w = *p;
            uint32_t* u = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float f[4];
                decode4<FMT>(u[k], f);
                u[k] = encode4<FMT>(f[0] * old, f[1] * old, f[2] * old, f[3] * old, scale, inv);
            }
            *p = w;
        }
    }
    __syncwarp();
    if (lane == 0) *scale_at = scale;
    for (int s0 = 0; s0 < steps; s0 += U) {
        if (steps > U) {  // a long run is read again (it is in the cache); a short one is still in registers
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = (s0 + u) * TPW + sub;
                raw[u] = make_uint4(0, 0, 0, 0);
                if (j < run) raw[u] = *reinterpret_cast<const uint4*>(src + (i0 + j) * token_stride);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = (s0 + u) * TPW + sub;
            if (j >= run) continue;
            float f[V];
            unpack16<T>(raw[u], f);
#pragma unroll
            for (int k = 0; k < V; ++k) f[k] = f[k] == f[k] ? f[k] : 0.f;
            uint32_t out[V / 4];
#pragma unroll
            for (int k = 0; k < V / 4; ++k)
                out[k] = encode4<FMT>(f[4 * k], f[4 * k + 1], f[4 * k + 2], f[4 * k + 3], scale, inv);
            const int off = static_cast<int>(slots[i0 + j] & (page_size - 1));
            uint8_t* to = base + off * c.token_stride + el;
            if constexpr (V == 8) *reinterpret_cast<uint2*>(to) = make_uint2(out[0], out[1]);
            else *reinterpret_cast<uint32_t*>(to) = out[0];
        }
    }
}

template <typename T, int FMT, int D>
__global__ void __launch_bounds__(kAppWarps * 32) append_kernel(AppendArgs a, int chunk) {
    __shared__ int first[kAppMaxChunk], length[kAppMaxChunk];
    __shared__ int runs;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c0 = static_cast<int64_t>(blockIdx.x) * chunk;
    const int heads = a.cache.kv_heads, shift = a.cache.page_shift, page_size = a.cache.page_size;
    const int64_t limit = a.cache.pages << shift;
    if (warp == 0) {
        const int64_t i = c0 + lane;
        bool begins = false;
        int len = 0;
        if (lane < chunk && i < a.tokens) {
            const int64_t s = a.slots[i];
            const bool ok = s >= 0 && s < limit;
            if (!ok && s != -1 && a.status) atomicOr(a.status, PTOWSP_SERVING_PAGE);
            const int64_t before = i ? a.slots[i - 1] : -1;
            begins = ok && (before < 0 || (before >> shift) != (s >> shift) || before >= s);
            if (begins) {
                int64_t last = s;
                for (len = 1; i + len < a.tokens; ++len) {
                    const int64_t n = a.slots[i + len];
                    if (n <= last || (n >> shift) != (s >> shift)) break;
                    last = n;
                }
            }
        }
        const uint32_t all = __ballot_sync(~0u, begins);
        if (begins) {
            const int k = __popc(all & ((1u << lane) - 1u));
            first[k] = lane;
            length[k] = len;
        }
        if (lane == 0) runs = __popc(all);
    }
    __syncthreads();
    const int head = blockIdx.y;
    for (int it = warp; it < runs * 2; it += kAppWarps) {
        const int which = it & 1, k = it >> 1;
        const int64_t i0 = c0 + first[k];
        const int64_t page = a.slots[i0] >> shift;
        const char* x = static_cast<const char*>(which ? a.v : a.k) +
                        head * (which ? a.v_head_stride : a.k_head_stride) * static_cast<int64_t>(sizeof(T));
        append_run<T, FMT, D>(which ? a.cache.v : a.cache.k, page, head, heads, page_size, x,
                              which ? a.v_token_stride : a.k_token_stride, a.slots, i0, length[k], lane);
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
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(reserve_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
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
    const int64_t blocks = (a.tokens + chunk - 1) / chunk;
    if (blocks > INT32_MAX) return cudaErrorInvalidValue;
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(a.cache.kv_heads));
    switch (a.dtype) {
        case PTOWSP_F32: return append_t<float>(a, grid, chunk, s);
        case PTOWSP_F16: return append_t<__half>(a, grid, chunk, s);
        default: return append_t<__nv_bfloat16>(a, grid, chunk, s);
    }
}

}  // namespace ptowsp::dev

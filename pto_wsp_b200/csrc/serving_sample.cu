// Token sampling: temperature, top-k, min-p and top-p over one row of logits per CTA.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "serving.hpp"

namespace ptowsp::dev {

namespace {

constexpr int kThreads = 1024;

template <typename T>
__device__ __forceinline__ float logit(const T* row, int i);
template <>
__device__ __forceinline__ float logit<float>(const float* row, int i) { return row[i]; }
template <>
__device__ __forceinline__ float logit<__half>(const __half* row, int i) { return __half2float(row[i]); }
template <>
__device__ __forceinline__ float logit<__nv_bfloat16>(const __nv_bfloat16* row, int i) { return __bfloat162float(row[i]); }

// Order-preserving keys: NaN as -inf, -0 as +0.
__device__ __forceinline__ uint32_t key_of(float x) {
    x = x == x ? x + 0.f : -INFINITY;
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// Weight of a logit below the row's largest, in f32.
__device__ __forceinline__ float weight_of(float x, float top, float temperature) {
    if (x == top) return 1.f;
    const float w = expf(__fdiv_rn(x - top, temperature));
    return w == w && x > -INFINITY ? w : 0.f;
}
__device__ __forceinline__ int64_t whole_of(float w) { return static_cast<int64_t>(w * 1099511627776.f); }

template <typename V, typename F>
__device__ V block_reduce(V v, F op, V* part) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v = op(v, __shfl_xor_sync(~0u, v, d));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = part[threadIdx.x & 31];
#pragma unroll
    for (int d = 16; d; d >>= 1) v = op(v, __shfl_xor_sync(~0u, v, d));
    return v;
}

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

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(SampleArgs a) {
    __shared__ int64_t part[32];
    __shared__ uint32_t part32[32];
    __shared__ int picked;
    const int r = blockIdx.x;
    const T* row = static_cast<const T*>(a.logits) + r * a.row_stride;
    const float temperature = a.temperature ? a.temperature[r] : 1.f;
    const bool greedy = !(temperature > 0.f);
    const float t = greedy ? 1.f : temperature;
    const float min_p = a.min_p ? fminf(a.min_p[r], 1.f) : 0.f;
    const float top_p = a.top_p ? a.top_p[r] : 1.f;
    int64_t k = greedy ? 1 : a.top_k ? a.top_k[r] : 0;
    const auto add = [](int64_t x, int64_t y) { return x + y; };

    uint32_t best = 0;
    for (int i = threadIdx.x; i < a.vocab; i += kThreads) best = max(best, key_of(logit(row, i)));
    best = block_reduce(best, [](uint32_t x, uint32_t y) { return max(x, y); }, part32);
    const float top = value_of(best);
    if (top == -INFINITY || a.vocab == 0) {
        if (threadIdx.x == 0) {
            a.token[r] = -1;
            if (a.logprob) a.logprob[r] = -INFINITY;
        }
        return;
    }
    const auto whole_at = [&](uint32_t key) -> int64_t {
        const float x = value_of(key);
        const float w = weight_of(x, top, t);
        return w >= min_p ? whole_of(w) : 0;
    };
    // top-k: the largest key that k elements reach, and how many of that key are in
    uint32_t cut = 0;
    int64_t ties = INT64_MAX;
    if (k > 0 && k < a.vocab) {
        for (int b = 31; b >= 0; --b) {
            const uint32_t c = cut | (1u << b);
            int64_t n = 0;
            for (int i = threadIdx.x; i < a.vocab; i += kThreads) n += key_of(logit(row, i)) >= c;
            if (block_reduce(n, add, part) >= k) cut = c;
        }
        int64_t n = 0;
        for (int i = threadIdx.x; i < a.vocab; i += kThreads) n += key_of(logit(row, i)) > cut;
        ties = k - block_reduce(n, add, part);
    }
    // mass of the candidates with a key above c
    const auto above = [&](uint32_t c) {
        int64_t n = 0;
        for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
            const uint32_t key = key_of(logit(row, i));
            if (key > c) n += whole_at(key);
        }
        return block_reduce(n, add, part);
    };
    const auto count_of = [&](uint32_t c) {
        int64_t n = 0;
        for (int i = threadIdx.x; i < a.vocab; i += kThreads) n += key_of(logit(row, i)) == c;
        return block_reduce(n, add, part);
    };
    int64_t total = above(cut);
    if (cut) {
        const int64_t n = count_of(cut);
        total += whole_at(cut) * (ties < n ? ties : n);
    }
    if (top_p < 1.f) {
        int64_t limit = static_cast<int64_t>(ceil(static_cast<double>(top_p) * static_cast<double>(total)));
        if (limit < 1) limit = 1;
        // the largest key c with mass(key >= c) >= limit: mass(key > c - 1)
        if (limit < total) {
            uint32_t c2 = 0;
            for (int b = 31; b >= 0; --b) {
                const uint32_t c = c2 | (1u << b);
                int64_t m = 0;
                if (c > cut) m = above(c - 1);
                else m = total;
                if (m >= limit) c2 = c;
            }
            const int64_t m = above(c2);
            const int64_t w = whole_at(c2);
            int64_t need = w > 0 ? (limit - m + w - 1) / w : 0;
            const int64_t n = count_of(c2);
            if (need > n) need = n;
            if (c2 == cut && ties < need) need = ties;
            cut = c2;
            ties = need;
            total = m + w * need;
        }
    }
    int64_t pick = static_cast<int64_t>(static_cast<double>(a.u[r]) * static_cast<double>(total));
    if (pick < 0) pick = 0;
    if (pick > total - 1) pick = total - 1;
    int64_t mass = 0, seen_ties = 0;
    if (threadIdx.x == 0) picked = -1;
    __syncthreads();
    for (int i0 = 0; i0 < a.vocab; i0 += kThreads) {
        const int i = i0 + threadIdx.x;
        const uint32_t key = i < a.vocab ? key_of(logit(row, i)) : 0;
        const bool tie = i < a.vocab && key == cut;
        int64_t n, all;
        n = seen_ties + block_inclusive(tie, part, &all);
        seen_ties += all;
        int64_t w = 0;
        if (i < a.vocab && (key > cut || (tie && n <= ties))) w = whole_at(key);
        const int64_t end = mass + block_inclusive(w, part, &all);
        mass += all;
        if (w > 0 && end > pick && end - w <= pick) {
            a.token[r] = i;
            if (a.logprob) a.logprob[r] = logf(static_cast<float>(w) / static_cast<float>(total));
            picked = i;
        }
        __syncthreads();
        if (picked >= 0) break;
    }
}

}  // namespace

cudaError_t launch_sample(const SampleArgs& a, int sms, cudaStream_t s) {
    (void)sms;
    if (a.rows == 0) return cudaSuccess;
    switch (a.dtype) {
        case PTOWSP_F32: sample_kernel<float><<<a.rows, kThreads, 0, s>>>(a); break;
        case PTOWSP_F16: sample_kernel<__half><<<a.rows, kThreads, 0, s>>>(a); break;
        default: sample_kernel<__nv_bfloat16><<<a.rows, kThreads, 0, s>>>(a); break;
    }
    return cudaGetLastError();
}

}  // namespace ptowsp::dev

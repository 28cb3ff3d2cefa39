// Launchers of the serving operators: page reservation, the writer and the attention of an 8-bit paged KV cache,
// token sampling.  The C entry points (serving_api.cpp) check arguments; these launch on the current device.
#pragma once

#include <cuda_runtime_api.h>

#include <atomic>
#include <cstdint>

#include "../../include/ptowsp_cuda.h"

namespace ptowsp::dev {

constexpr int kReserveMaxRequests = 16384;  // two words of shared memory each
constexpr float kKv8MinScale = 8.673617379884035e-19f;  // 2^-60
constexpr float kKv8MaxScale = 1152921504606846976.f;   // 2^60

// A kernel's opt-in to more than 48 KB of dynamic shared memory, asked for once per device.
class SmemOptIn {
    std::atomic<uint64_t> done_{0};

public:
    cudaError_t once(const void* kernel, int bytes) {
        int device = 0;
        cudaError_t e = cudaGetDevice(&device);
        if (e != cudaSuccess) return e;
        const uint64_t bit = uint64_t{1} << (device & 63);
        if (device < 64 && (done_.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess && device < 64) done_.fetch_or(bit, std::memory_order_relaxed);
        return e;
    }
};

struct ReserveArgs {
    int32_t* page_table;
    int64_t table_stride;
    int max_pages, page_size, requests;
    const int32_t* kv_len;
    const int32_t* new_tokens;
    int32_t* free_ring;
    int64_t ring_size;
    const int64_t* free_state;
    int64_t* slots;
    int32_t* positions;
    int64_t max_tokens;
    int32_t* q_start;
    int32_t* kv_len_out;
    int64_t* free_state_out;
    uint8_t* granted;
    int32_t* status;
};
cudaError_t launch_reserve(const ReserveArgs& a, cudaStream_t s);

// One of K and V: codes, scales and the element strides of the cache.
struct Kv8Side {
    uint8_t* codes;
    float* scale;
    int64_t page_stride, token_stride, head_stride;
};
struct Kv8 {
    Kv8Side k, v;
    int64_t pages;
    int page_size, page_shift, kv_heads, head_dim, format;
};

struct AppendArgs {
    Kv8 cache;
    const void* k;
    const void* v;
    int64_t k_token_stride, k_head_stride, v_token_stride, v_head_stride;
    int dtype;
    const int64_t* slots;
    int64_t tokens;
    int32_t* status;
};
cudaError_t launch_append(const AppendArgs& a, cudaStream_t s);

struct AttendArgs {
    Kv8 cache;
    const void* q;
    void* out;
    float* lse;
    int64_t q_token_stride, q_head_stride, out_token_stride, out_head_stride;
    int dtype;
    const int32_t* page_table;
    int64_t table_stride;
    int max_pages;
    const int32_t* kv_len;
    const int32_t* q_start;  // nullptr: one token per request
    int requests, heads, group, max_q, window;
    int few;  // requests with more q rows (tokens x group) are left to launch_prefill; 0: none are
    int64_t tokens;
    float scale;
    char* workspace;
    int32_t* status;
};
size_t attend_workspace_bytes(const AttendArgs& a, int sms);
cudaError_t launch_attend(const AttendArgs& a, int sms, cudaStream_t s);

constexpr int kSampleMaxSmem = 224 << 10;  // of a CTA: its slice of the row, histograms and lists
constexpr int kSampleMaxVocab = 393216;    // eight slices of 192 KB of f32
// Requests of more than `threshold` q rows, on tcgen05 (serving_prefill.cu).
size_t prefill_workspace_bytes(const AttendArgs& a, int sms);
cudaError_t launch_prefill(const AttendArgs& a, int threshold, char* workspace, int sms, cudaStream_t s);

struct SampleArgs {
    const void* logits;
    int64_t row_stride;
    int dtype;
    int rows, vocab;
    const float* u;
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    int32_t* token;
    float* logprob;
};
cudaError_t launch_sample(const SampleArgs& a, int sms, cudaStream_t s);

}  // namespace ptowsp::dev

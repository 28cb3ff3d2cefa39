// C entry points of the serving operators (declared in include/ptowsp_cuda.h): argument checks and launches.
#include <cuda_runtime_api.h>

#include <atomic>
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "runtime.hpp"
#include "serving.hpp"

namespace {

using namespace ptowsp::dev;

// A fixed buffer: these entry points must not throw.
int fail(int code, const char* fmt, ...) noexcept {
    char text[256];
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(text, sizeof text, fmt, ap);
    va_end(ap);
    try {
        ptowsp::set_error(text);
    } catch (...) {
    }
    return code;
}

int launched(cudaError_t e, const char* what) noexcept {
    if (e == cudaSuccess) return PTOWSP_OK;
    cudaGetLastError();  // a refused launch is not left for the next call to find
    return fail(PTOWSP_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

bool aligned(const void* p, uintptr_t n) noexcept { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// Whether a dimension of `n` elements may have this stride: a multiple of `unit`, or any where no second element is.
bool steps_by(int64_t n, int64_t stride, int64_t unit) noexcept { return n <= 1 || stride % unit == 0; }

bool power_of_two(int64_t v) noexcept { return v > 0 && (v & (v - 1)) == 0; }

// SMs of the current device, asked once per device.
int sm_count(int* sms) noexcept {
    static std::atomic<int> known[64];
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return launched(e, "cudaGetDevice");
    if (device >= 0 && device < 64) {
        *sms = known[device].load(std::memory_order_relaxed);
        if (*sms > 0) return PTOWSP_OK;
    }
    e = cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, device);
    if (e != cudaSuccess) return launched(e, "cudaDeviceGetAttribute");
    if (device >= 0 && device < 64) known[device].store(*sms, std::memory_order_relaxed);
    return PTOWSP_OK;
}

int kv8_of(const ptowsp_kv8_cache* c, Kv8* out, const char* what) noexcept {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return fail(PTOWSP_ERR_ARG, "%s: null cache pointer", what);
    if (c->format != PTOWSP_KV8_E4M3 && c->format != PTOWSP_KV8_INT8)
        return fail(PTOWSP_ERR_ARG, "%s: unknown cache format %d", what, c->format);
    if (c->head_dim != 64 && c->head_dim != 128)
        return fail(PTOWSP_ERR_UNSUPPORTED, "%s: head_dim must be 64 or 128 (got %d)", what, c->head_dim);
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
        return fail(PTOWSP_ERR_UNSUPPORTED, "%s: page_size must be 16, 32, 64 or 128 (got %d)", what, c->page_size);
    if (c->num_kv_heads <= 0 || c->num_kv_heads > 65535 || c->num_pages <= 0 || c->num_pages > INT32_MAX)
        return fail(PTOWSP_ERR_ARG, "%s: num_kv_heads must be 1 .. 65535 and num_pages 1 .. 2^31 - 1", what);
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4))
        return fail(PTOWSP_ERR_ARG, "%s: cache codes must be 16-byte aligned, scales 4-byte", what);
    const struct {
        int64_t n, stride;
    } dims[] = {{c->num_pages, c->k_page_stride}, {c->page_size, c->k_token_stride}, {c->num_kv_heads, c->k_head_stride},
                {c->num_pages, c->v_page_stride}, {c->page_size, c->v_token_stride}, {c->num_kv_heads, c->v_head_stride}};
    for (const auto& d : dims)
        if (!steps_by(d.n, d.stride, 16) || (d.n > 1 && d.stride < 0))
            return fail(PTOWSP_ERR_ARG, "%s: cache strides must be multiples of 16, not negative", what);
    int shift = 4;
    while ((1 << shift) < c->page_size) ++shift;
    *out = Kv8{{static_cast<uint8_t*>(c->k), c->k_scale, c->k_page_stride, c->k_token_stride, c->k_head_stride},
               {static_cast<uint8_t*>(c->v), c->v_scale, c->v_page_stride, c->v_token_stride, c->v_head_stride},
               c->num_pages, c->page_size, shift, c->num_kv_heads, c->head_dim, c->format};
    return PTOWSP_OK;
}

int attend_of(const ptowsp_kv8_cache* cache, const ptowsp_kv8_attention_args* g, AttendArgs* a) noexcept {
    const char* what = "kv8_attention";
    if (!g) return fail(PTOWSP_ERR_ARG, "%s: null argument", what);
    *a = AttendArgs{};
    const int rc = kv8_of(cache, &a->cache, what);
    if (rc != PTOWSP_OK) return rc;
    if (g->requests < 0 || g->tokens < 0 || g->max_q < 0 || g->window < 0 || g->max_pages < 0 || g->tokens > INT32_MAX)
        return fail(PTOWSP_ERR_ARG, "%s: sizes must not be negative, tokens below 2^31", what);
    if (g->num_heads <= 0 || g->num_heads % a->cache.kv_heads)
        return fail(PTOWSP_ERR_ARG, "%s: num_heads (%d) must be a multiple of num_kv_heads (%d)", what, g->num_heads,
                    a->cache.kv_heads);
    if (g->dtype != PTOWSP_F16 && g->dtype != PTOWSP_BF16)
        return fail(PTOWSP_ERR_UNSUPPORTED, "%s: q and out must be f16 or bf16", what);
    if (static_cast<int64_t>(g->max_pages) * a->cache.page_size > (int64_t{1} << 30) * 2 - 1 - 65536)
        return fail(PTOWSP_ERR_LIMIT, "%s: max_pages * page_size must stay below 2^31 - 65536", what);
    if (static_cast<int64_t>(g->max_q) * (g->num_heads / a->cache.kv_heads) > (1 << 30))
        return fail(PTOWSP_ERR_LIMIT, "%s: max_q times the head group must be at most 2^30", what);
    if (!std::isfinite(g->scale)) return fail(PTOWSP_ERR_ARG, "%s: scale must be finite", what);
    a->q = g->q;
    a->out = g->out;
    a->lse = g->lse;
    a->q_token_stride = g->q_token_stride;
    a->q_head_stride = g->q_head_stride;
    a->out_token_stride = g->out_token_stride;
    a->out_head_stride = g->out_head_stride;
    a->dtype = g->dtype;
    a->page_table = g->page_table;
    a->table_stride = g->table_stride;
    a->max_pages = g->max_pages;
    a->kv_len = g->kv_len;
    a->q_start = g->q_start;
    a->requests = g->requests;
    a->heads = g->num_heads;
    a->group = g->num_heads / a->cache.kv_heads;
    a->max_q = g->max_q;
    // a window as long as the table hides nothing
    a->window = g->window < static_cast<int64_t>(g->max_pages) * a->cache.page_size ? g->window : 0;
    a->tokens = g->tokens;
    a->scale = g->scale;
    a->workspace = static_cast<char*>(g->workspace);
    a->status = g->status;
    return PTOWSP_OK;
}

}  // namespace

extern "C" {

int ptowsp_cuda_reserve_pages(const ptowsp_reserve_args* g, void* stream) {
    const char* what = "reserve_pages";
    if (!g) return fail(PTOWSP_ERR_ARG, "%s: null argument", what);
    if (g->requests < 0 || g->max_tokens < 0 || g->max_pages < 0 || g->ring_size < 0 || g->table_stride < g->max_pages)
        return fail(PTOWSP_ERR_ARG, "%s: sizes must not be negative, table rows not overlap", what);
    if (g->requests > kReserveMaxRequests)
        return fail(PTOWSP_ERR_LIMIT, "%s: at most %d requests (got %d)", what, kReserveMaxRequests, g->requests);
    if (!power_of_two(g->page_size) || g->page_size > 65536)
        return fail(PTOWSP_ERR_ARG, "%s: page_size must be a power of two up to 65536 (got %d)", what, g->page_size);
    if (static_cast<int64_t>(g->max_pages) * g->page_size > INT32_MAX || g->max_tokens > INT32_MAX ||
        g->ring_size > INT32_MAX)
        return fail(PTOWSP_ERR_LIMIT, "%s: max_pages * page_size, max_tokens and ring_size must stay below 2^31", what);
    if (!g->free_state || !g->free_state_out || !g->q_start ||
        (g->requests && (!g->kv_len || !g->new_tokens || !g->kv_len_out || !g->granted)) ||
        (g->requests && g->max_pages && !g->page_table) || (g->ring_size && !g->free_ring) ||
        (g->max_tokens && (!g->slots || !g->positions)))
        return fail(PTOWSP_ERR_ARG, "%s: null pointer", what);
    if (g->kv_len == g->kv_len_out && g->requests)
        return fail(PTOWSP_ERR_ARG, "%s: kv_len_out must not be kv_len", what);
    if (g->free_state == g->free_state_out) return fail(PTOWSP_ERR_ARG, "%s: free_state_out must not be free_state", what);
    ReserveArgs a{g->page_table, g->table_stride, g->max_pages,  g->page_size, g->requests,   g->kv_len,
                  g->new_tokens, g->free_ring,    g->ring_size,  g->free_state, g->slots,     g->positions,
                  g->max_tokens, g->q_start,      g->kv_len_out, g->free_state_out, g->granted, g->status};
    return launched(launch_reserve(a, static_cast<cudaStream_t>(stream)), what);
}

int ptowsp_cuda_kv8_append(const ptowsp_kv8_cache* cache, const ptowsp_kv8_append_args* g, void* stream) {
    const char* what = "kv8_append";
    if (!g) return fail(PTOWSP_ERR_ARG, "%s: null argument", what);
    AppendArgs a{};
    const int rc = kv8_of(cache, &a.cache, what);
    if (rc != PTOWSP_OK) return rc;
    if (g->dtype != PTOWSP_F32 && g->dtype != PTOWSP_F16 && g->dtype != PTOWSP_BF16)
        return fail(PTOWSP_ERR_UNSUPPORTED, "%s: k and v must be f32, f16 or bf16", what);
    if (g->tokens < 0 || g->tokens > INT32_MAX) return fail(PTOWSP_ERR_ARG, "%s: tokens must be 0 .. 2^31 - 1", what);
    if (g->tokens == 0) return PTOWSP_OK;
    if (!g->k || !g->v || !g->slots) return fail(PTOWSP_ERR_ARG, "%s: null pointer", what);
    const int64_t unit = g->dtype == PTOWSP_F32 ? 4 : 8;  // elements in 16 bytes
    const int64_t heads = a.cache.kv_heads;
    if (!aligned(g->k, 16) || !aligned(g->v, 16) || !steps_by(g->tokens, g->k_token_stride, unit) ||
        !steps_by(heads, g->k_head_stride, unit) || !steps_by(g->tokens, g->v_token_stride, unit) ||
        !steps_by(heads, g->v_head_stride, unit))
        return fail(PTOWSP_ERR_ARG, "%s: rows of k and v must be 16-byte aligned", what);
    a.k = g->k;
    a.v = g->v;
    a.k_token_stride = g->k_token_stride;
    a.k_head_stride = g->k_head_stride;
    a.v_token_stride = g->v_token_stride;
    a.v_head_stride = g->v_head_stride;
    a.dtype = g->dtype;
    a.slots = g->slots;
    a.tokens = g->tokens;
    a.status = g->status;
    return launched(launch_append(a, static_cast<cudaStream_t>(stream)), what);
}

size_t ptowsp_cuda_kv8_attention_workspace(const ptowsp_kv8_cache* cache, const ptowsp_kv8_attention_args* g) {
    AttendArgs a{};
    int sms = 0;
    if (attend_of(cache, g, &a) != PTOWSP_OK || sm_count(&sms) != PTOWSP_OK) return 0;
    return attend_workspace_bytes(a, sms);
}

int ptowsp_cuda_kv8_attention(const ptowsp_kv8_cache* cache, const ptowsp_kv8_attention_args* g, void* stream) {
    const char* what = "kv8_attention";
    AttendArgs a{};
    int rc = attend_of(cache, g, &a);
    if (rc != PTOWSP_OK) return rc;
    if (a.tokens == 0) return PTOWSP_OK;
    if (!a.q || !a.out || (a.requests && (!a.kv_len || (a.max_pages && !a.page_table))))
        return fail(PTOWSP_ERR_ARG, "%s: null pointer", what);
    if (!a.q_start && (a.tokens != a.requests || a.max_q != 1))
        return fail(PTOWSP_ERR_ARG, "%s: without q_start every request has one token (max_q 1)", what);
    if (!aligned(a.q, 16) || !aligned(a.out, 16) || !steps_by(a.tokens, a.q_token_stride, 8) ||
        !steps_by(a.heads, a.q_head_stride, 8) || !steps_by(a.tokens, a.out_token_stride, 8) ||
        !steps_by(a.heads, a.out_head_stride, 8))
        return fail(PTOWSP_ERR_ARG, "%s: rows of q and out must be 16-byte aligned", what);
    int sms = 0;
    rc = sm_count(&sms);
    if (rc != PTOWSP_OK) return rc;
    const size_t need = attend_workspace_bytes(a, sms);
    if (g->workspace_bytes < need || !a.workspace || !aligned(a.workspace, 256))
        return fail(PTOWSP_ERR_ARG, "%s: the workspace must have %zu bytes, 256-byte aligned", what, need);
    return launched(launch_attend(a, sms, static_cast<cudaStream_t>(stream)), what);
}

int ptowsp_cuda_sample_tokens(const ptowsp_sample_args* g, void* stream) {
    const char* what = "sample_tokens";
    if (!g) return fail(PTOWSP_ERR_ARG, "%s: null argument", what);
    if (g->rows < 0 || g->vocab < 1) return fail(PTOWSP_ERR_ARG, "%s: rows must be >= 0 and vocab >= 1", what);
    if (g->vocab > kSampleMaxVocab)
        return fail(PTOWSP_ERR_LIMIT, "%s: vocab must be at most %d (got %d)", what, kSampleMaxVocab, g->vocab);
    if (g->dtype != PTOWSP_F32 && g->dtype != PTOWSP_F16 && g->dtype != PTOWSP_BF16)
        return fail(PTOWSP_ERR_UNSUPPORTED, "%s: logits must be f32, f16 or bf16", what);
    if (g->rows == 0) return PTOWSP_OK;
    if (!g->logits || !g->u || !g->token) return fail(PTOWSP_ERR_ARG, "%s: null pointer", what);
    if (!aligned(g->logits, g->dtype == PTOWSP_F32 ? 4 : 2))
        return fail(PTOWSP_ERR_ARG, "%s: logits are not aligned to their type", what);
    int sms = 0;
    const int rc = sm_count(&sms);
    if (rc != PTOWSP_OK) return rc;
    SampleArgs a{g->logits, g->row_stride, g->dtype, g->rows,  g->vocab, g->u,
                 g->temperature, g->top_k, g->top_p, g->min_p, g->token, g->logprob};
    return launched(launch_sample(a, sms, static_cast<cudaStream_t>(stream)), what);
}

}  // extern "C"

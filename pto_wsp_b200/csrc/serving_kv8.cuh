// Conversions of the 8-bit cache codes, shared by its writer and its readers.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "serving.hpp"

namespace ptowsp::dev {

// Bytes 0, 1 -> lo and bytes 2, 3 -> hi as f16 pairs, exactly.  int8: the byte with its sign flipped is the low
// mantissa byte of 1024 + (code + 128), from which 1152 is taken.
template <int FMT>
__device__ __forceinline__ void codes_f16(uint32_t w, uint32_t& lo, uint32_t& hi) {
    if (FMT == PTOWSP_KV8_E4M3) {
        asm("{\n\t.reg .b16 x, y;\n\tmov.b32 {x, y}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, x;\n\tcvt.rn.f16x2.e4m3x2 %1, y;\n\t}"
            : "=r"(lo), "=r"(hi)
            : "r"(w));
    } else {
        w ^= 0x80808080u;
        lo = __byte_perm(w, 0x64646464u, 0x4140);
        hi = __byte_perm(w, 0x64646464u, 0x4342);
        const __half2 bias = __floats2half2_rn(1152.f, 1152.f);
        *reinterpret_cast<__half2*>(&lo) = __hsub2(*reinterpret_cast<__half2*>(&lo), bias);
        *reinterpret_cast<__half2*>(&hi) = __hsub2(*reinterpret_cast<__half2*>(&hi), bias);
    }
}

// A box of a page's codes (a head's dims of some tokens) into shared memory; its bytes count on `bar`.
__device__ __forceinline__ void tma_load_page(uint32_t dst, const CUtensorMap* map, int head, int token, int page,
                                              uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(head), "r"(token), "r"(page), "r"(bar)
        : "memory");
}

// Host: one side's codes as a tensor [pages][page_size][heads][head_dim] whose box is one head's dims of `tokens` tokens
// of a page, with the 64- or 128-byte swizzle of the row's length or none.
bool kv8_map(CUtensorMap* m, const Kv8& c, const Kv8Side& side, int tokens, bool swizzle);

template <int FMT>
__device__ __forceinline__ void decode4(uint32_t w, float (&f)[4]) {
    uint32_t lo, hi;
    codes_f16<FMT>(w, lo, hi);
    const float2 a = __half22float2(*reinterpret_cast<__half2*>(&lo));
    const float2 b = __half22float2(*reinterpret_cast<__half2*>(&hi));
    f[0] = a.x;
    f[1] = a.y;
    f[2] = b.x;
    f[3] = b.y;
}

}  // namespace ptowsp::dev

// What both attention kernels over a 4-bit cache make numbers of nibbles with, and how their warps wait.
#pragma once

#include "attention4.h"
#include "tcgen05.cuh"

#include <cuda_fp16.h>

namespace lb_a4 {
namespace {

// 2^n, n in -126 .. 127.
__device__ __forceinline__ float pow2(int n) { return __uint_as_float((uint32_t)(127 + n) << 23); }
__device__ __forceinline__ uint32_t h2(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
__device__ __forceinline__ __half2 as_h2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
// bfloat16 number i of a run of words.
__device__ __forceinline__ float number(const uint32_t* w, int i) { return __uint_as_float((i & 1) != 0 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16); }
template <int BYTES>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t* w) {
    if constexpr (BYTES == 16) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else if constexpr (BYTES == 8) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        w[0] = u.x; w[1] = u.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
}

// A word's values as four float16 pairs: r[i] = nibbles (i, i + 4) less 8.
__device__ __forceinline__ void pairs_of(uint32_t w, __half2 (&r)[4]) {
    const __half2 offset = __float2half2_rn(-1032.0f), sixteenth = __float2half2_rn(0.0625f), offset16 = __float2half2_rn(-72.0f);
    const uint32_t hi = w >> 8;
    r[0] = __hadd2(as_h2((w & 0x000f000fu) | 0x64006400u), offset);
    r[1] = __hfma2(as_h2((w & 0x00f000f0u) | 0x64006400u), sixteenth, offset16);         // (1024 + 16 n) / 16 - 72
    r[2] = __hadd2(as_h2((hi & 0x000f000fu) | 0x64006400u), offset);
    r[3] = __hfma2(as_h2((hi & 0x00f000f0u) | 0x64006400u), sixteenth, offset16);
}

// A bounded wait, one answer for the warp.  Most find the phase done: one question then (mbar_wait's loop is 90 cycles of a warp that has the SM for itself, this 30).
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "vote.sync.all.pred q, p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(ok) : "r"(lb_tc::smem_u32(bar)), "r"(parity) : "memory");
    if (ok != 0) return true;
    return __all_sync(0xffffffffu, lb_tc::mbar_wait(bar, parity, abort_flag));
}

}  // namespace
}  // namespace lb_a4

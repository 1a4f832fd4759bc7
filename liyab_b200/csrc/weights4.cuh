// 4-bit weights as the products read them (the layout: api.h, lb_weights4) and what their kernels share: nibbles to halves of a register,
// 8-bit floats, and the epilogue.
//
// w[n, k] = q s r with q in -8 .. 7 (at most three significant bits), s in e4m3 (four) and r in 32 bits.  q, and q s as well (at most seven
// significant bits), are bfloat16 and float16 numbers without rounding, and so are the activations (bfloat16 as they are, e4m3 as float16):
// the tensor cores multiply exactly, sums are 32-bit, and r and the activations' scale a row meet the finished sum.
#pragma once

#include "api.h"
#include "common.cuh"

#include <cuda_fp16.h>

namespace lb_w4 {

constexpr int kTileRows = 16, kTileK = 128, kTileBytes = kTileRows * kTileK / 2;

// Where a row's 16 bytes of an octet of every 32 lie in a tile, in units of 16 bytes: [row / 4][t / 2][row % 4][t % 2], so that eight neighbouring threads of either kernel (two
// rows by four t, or eight rows of one t) touch two lines of 128 bytes.  With [t][row] the first touch four: 41 MB of weights for one token took 12.1 us in place of 10.7.
__host__ __device__ __forceinline__ constexpr int piece_at(int row, int t) { return (row >> 2) * 16 + (t >> 1) * 8 + (row & 3) * 2 + (t & 1); }

// (x & mask) | bits in one instruction: with both numbers as literals it becomes two.
__device__ __forceinline__ uint32_t masked_or(uint32_t x, uint32_t mask, uint32_t bits) {
    uint32_t v;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(x), "r"(mask), "r"(bits));
    return v;
}

// The operand type of the tensor cores: bfloat16 activations go with bfloat16 weights, e4m3 ones with float16.
struct Bf16 {
    static constexpr bool kHalf = false;
};
struct F16 {
    static constexpr bool kHalf = true;
};

template <typename V>
__device__ __forceinline__ uint32_t minus2(uint32_t v, uint32_t c) {
    const V d = __hsub2(*reinterpret_cast<const V*>(&v), *reinterpret_cast<const V*>(&c));
    return *reinterpret_cast<const uint32_t*>(&d);
}

// Nibbles q + 8 to q.  bfloat16 has room for a nibble in one place only: 0x4300 | u is 128 + u, three shifts a word.  float16 has two: 0x6400 | u is 1024 + u and 0x5400 | u << 4
// is 64 + u, and one shift a word does (a product of one token reads 5.1 TB/s of weights so, 4.1 in bfloat16; bfloat16 rows as float16 times a power of two of their
// own made up 7 % of that and lost more to finding it).  The masks and the exponent bits are kept in registers, hidden from constant folding.
template <typename T>
struct Unpack {
    uint32_t mask, bits, mask4, bits4;
    __device__ __forceinline__ Unpack() {
        asm volatile("mov.b32 %0, 0x000F000F;\n\tmov.b32 %1, %4;\n\tmov.b32 %2, 0x00F000F0;\n\tmov.b32 %3, 0x54005400;"
                     : "=r"(mask), "=r"(bits), "=r"(mask4), "=r"(bits4) : "n"(T::kHalf ? 0x64006400 : 0x43004300));
    }
    // Weights 2p and 2p + 1 of a word of eight, in the halves of a register.
    __device__ __forceinline__ uint32_t operator()(uint32_t word, int p) const {
        if constexpr (T::kHalf) {
            const uint32_t w = p < 2 ? word : word >> 8;
            return p & 1 ? minus2<__half2>(masked_or(w, mask4, bits4), 0x54805480u) : minus2<__half2>(masked_or(w, mask, bits), 0x64086408u);
        } else {
            return minus2<__nv_bfloat162>(masked_or(word >> (4 * p), mask, bits), 0x43084308u);
        }
    }
};

// Two e4m3 numbers (16 bits) -> float16.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
    uint32_t out;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(out) : "h"((uint16_t)two));
    return out;
}
__device__ __forceinline__ float e4m3_to_float(uint32_t byte) {
    const uint32_t v = e4m3x2_to_f16x2(byte & 0xffu);
    return __low2float(*reinterpret_cast<const __half2*>(&v));
}
// Two floats -> e4m3, rounded to the nearest even, values beyond 448 to 448; `lo` in the low byte.
__device__ __forceinline__ uint32_t floats_to_e4m3x2(float lo, float hi) {
    uint16_t out;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(out) : "f"(hi), "f"(lo));
    return out;
}

// The accumulator's 16 x 8 tile += weights (rows) x activations (columns).
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (T::kHalf)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight e4m3 of a row from column k on, zeros past K.  `wide`: rows are aligned so that eight come by one load.
__device__ __forceinline__ void load_eight_bytes(uint32_t& lo, uint32_t& hi, const void* a, int64_t row_at, int k, int K, bool wide) {
    const uint8_t* p = static_cast<const uint8_t*>(a) + row_at;
    lo = hi = 0;
    if (wide && k + 8 <= K) {
        const uint2 two = *reinterpret_cast<const uint2*>(p + k);
        lo = two.x;
        hi = two.y;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (k + i < K) lo |= (uint32_t)p[k + i] << (8 * i);
            if (k + 4 + i < K) hi |= (uint32_t)p[k + 4 + i] << (8 * i);
        }
    }
}

// Eight activations of a row from column k on as four registers of two (bfloat16 as they are, e4m3 as float16), zeros past K.  `wide`: rows are aligned so that eight come by one load.
template <bool EIGHT>
__device__ __forceinline__ void load_eight(uint32_t (&v)[4], const void* a, int64_t row_at, int k, int K, bool wide) {
    if constexpr (EIGHT) {
        uint32_t lo, hi;
        load_eight_bytes(lo, hi, a, row_at, k, K, wide);
        v[0] = e4m3x2_to_f16x2(lo & 0xffffu);
        v[1] = e4m3x2_to_f16x2(lo >> 16);
        v[2] = e4m3x2_to_f16x2(hi & 0xffffu);
        v[3] = e4m3x2_to_f16x2(hi >> 16);
    } else {
        const uint16_t* p = static_cast<const uint16_t*>(a) + row_at;
        if (wide && k + 8 <= K) {
            const uint4 four = *reinterpret_cast<const uint4*>(p + k);
            v[0] = four.x;
            v[1] = four.y;
            v[2] = four.z;
            v[3] = four.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t lo = k + 2 * i < K ? p[k + 2 * i] : 0u, hi = k + 2 * i + 1 < K ? p[k + 2 * i + 1] : 0u;
                v[i] = lo | hi << 16;
            }
        }
    }
}

// What happens to a finished sum.  Of paired weights a feature's two sums (already times r and the activations' scale) become one value.
struct Epilogue {
    const float* a_scale;        // [M] or null
    const float* bias;           // [n] or null
    const float* residual;
    void* out;
    int64_t ldr, ldo;
    int M, n;                    // n: columns of out
    int act, gate;               // gate: only of paired weights
    float alpha, limit;
    bool out_f32;
};

// The weights' factor of a row as one between 2^-60 and 2^60 (left in `factor`) and a power of two, for sums that meet a scale of the activations too: the sum is multiplied by the
// first and then by the second times the scale, of which no product leaves float32's range before the result does (the product of two small factors would).
__device__ __forceinline__ float split_factor(float& factor) {
    const float size = fabsf(factor);
    const float rest = size < 8.6736174e-19f ? 5.4210109e-20f : size > 1.1529215e18f && size < __int_as_float(0x7f800000) ? 1.8446744e19f : 1.0f;        // 2^-64, 2^64
    factor *= size < 8.6736174e-19f ? 1.8446744e19f : rest > 1.0f ? 5.4210109e-20f : 1.0f;
    return rest;
}

// The larger and the smaller of two numbers; a NaN stays, which fmaxf and fminf would drop.
__device__ __forceinline__ float at_least(float v, float least) {
    float out;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(out) : "f"(v), "f"(least));
    return out;
}
__device__ __forceinline__ float at_most(float v, float most) {
    float out;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(out) : "f"(v), "f"(most));
    return out;
}

// lb_activate, but relu2 keeps a NaN as the others do.
__device__ __forceinline__ float relu2(float v) {
    const float some = at_least(v, 0.0f);
    return some * some;
}
__device__ __forceinline__ float activated(float v, int act, const lb_act_pair& pair) { return act == LB_ACT_RELU2 ? relu2(v) : lb_activate(v, act, pair); }

// lb_gated_pair, but a NaN in either half makes the result one under every gate.
__device__ __forceinline__ float gated_pair(float g, float u, int kind, float alpha, float limit) {
    if (kind == LB_GATE_RELU) return at_least(g, 0.0f) * u;
    if (kind == LB_GATE_CAPPED) {
        g = at_most(g, limit);
        u = at_most(at_least(u, -limit), limit);
        return g * (1.0f / (1.0f + expf(-alpha * g))) * (u + 1.0f);
    }
    return lb_gated_pair(g, u, kind, alpha, limit);
}

__device__ __forceinline__ void store_out(const Epilogue& e, int m, int col, float v) {
    if (e.out_f32) static_cast<float*>(e.out)[(int64_t)m * e.ldo + col] = v;
    else static_cast<__nv_bfloat16*>(e.out)[(int64_t)m * e.ldo + col] = __float2bfloat16_rn(v);
}

}  // namespace lb_w4

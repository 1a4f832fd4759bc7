// The states of one query row over parts of its keys become its result: what both attention kernels over a 4-bit cache end with.
#pragma once

#include "attention4.h"

#include <float.h>
#include <math_constants.h>

namespace lb_a4 {
namespace {

constexpr float kLowest = -FLT_MAX;            // a reference before any score; finite, so that differences with it are numbers

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A state: [reference m, sum, unit f, a place, HD values], the sum relative to 2^m, the values to 2^(m + f).  A team of warps (a power of two of the block's, 32 at most) has a row, a lane HD / 32 neighbouring values; the warps
// take the states in turn, and their sums meet in their order.  All threads of the block call it; state is null for rows that are not there.
template <int HD>
__device__ __forceinline__ void join_row(const Call& c, const Portion& part, int seq, int kvh, int r, const float* state, int64_t step, int runs, int team_shift, float (*joined)[HD + 3]) {
    constexpr int V = HD / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, team = 1 << team_shift, mine = warp & (team - 1);
    float m = kLowest, l = 0.0f, f = kLowest, v[V] = {};
    if (state != nullptr) {
        // Thirty-two at a time: a lane has a state's reference, sum and unit, and its factors once the largest are known.  The values come eight states at a time, the first eight before the factors.
        for (int i0 = mine; i0 < runs; i0 += 32 * team) {
            constexpr int kAhead = 8;
            const int n = min(32, (runs - i0 + team - 1) >> team_shift);
            const float* at = state + i0 * step + 4 + V * lane;
            float4 mlf = make_float4(kLowest, 0.0f, kLowest, 0.0f);
            if (lane < n) mlf = *reinterpret_cast<const float4*>(state + (i0 + lane * team) * step);
            float o[kAhead][V];
            auto load = [&](int x0) {
#pragma unroll
                for (int x = 0; x < kAhead; ++x) {
#pragma unroll
                    for (int e = 0; e < V; ++e) o[x][e] = 0.0f;
                    if (x0 + x < n) {
                        const float* p = at + (x0 + x) * team * step;
                        if constexpr (V == 4) *reinterpret_cast<float4*>(o[x]) = *reinterpret_cast<const float4*>(p);
                        else *reinterpret_cast<float2*>(o[x]) = *reinterpret_cast<const float2*>(p);
                    }
                }
            };
            load(0);
            const bool some = mlf.y != 0.0f;                // (a NaN is some)
            float high = some ? mlf.x : kLowest, unit = some ? mlf.z : kLowest;
#pragma unroll
            for (int x = 16; x > 0; x /= 2) {
                high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, x));
                unit = fmaxf(unit, __shfl_xor_sync(0xffffffffu, unit, x));
            }
            high = fmaxf(high, m);
            unit = fmaxf(unit, f);
            const float w = some ? ex2((mlf.x - high) + (mlf.z - unit)) : 0.0f, keep = ex2((m - high) + (f - unit));
            l = fmaf(l, ex2(m - high), lb_warp_sum(some ? mlf.y * ex2(mlf.x - high) : 0.0f));
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] *= keep;
            m = high;
            f = unit;
            for (int x0 = 0; x0 < n; x0 += kAhead) {
                if (x0 > 0) load(x0);
#pragma unroll
                for (int x = 0; x < kAhead; ++x) {
                    const float factor = __shfl_sync(0xffffffffu, w, (x0 + x) & 31);
#pragma unroll
                    for (int e = 0; e < V; ++e) v[e] = fmaf(o[x][e], factor, v[e]);
                }
            }
        }
    }
    if (team > 1) {
#pragma unroll
        for (int e = 0; e < V; ++e) joined[warp][3 + V * lane + e] = v[e];
        if (lane == 0) {
            joined[warp][0] = m;
            joined[warp][1] = l;
            joined[warp][2] = f;
        }
        __syncthreads();
        if (mine > 0) return;
        // A lane has a warp's reference, sum and unit.
        const float mi = lane < team ? joined[warp + lane][0] : kLowest, li = lane < team ? joined[warp + lane][1] : 0.0f, fi = lane < team ? joined[warp + lane][2] : kLowest;
        const bool some = li != 0.0f;
        float high = some ? mi : kLowest, unit = some ? fi : kLowest;
#pragma unroll
        for (int x = 16; x > 0; x /= 2) {
            high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, x));
            unit = fmaxf(unit, __shfl_xor_sync(0xffffffffu, unit, x));
        }
        const float w = some ? ex2((mi - high) + (fi - unit)) : 0.0f;
        l = lb_warp_sum(some ? li * ex2(mi - high) : 0.0f);
        m = high;
        f = unit;
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = 0.0f;
#pragma unroll 4
        for (int i = 0; i < team; ++i) {
            const float factor = __shfl_sync(0xffffffffu, w, i);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = fmaf(joined[warp + i][3 + V * lane + e], factor, v[e]);
        }
    }
    if (state == nullptr) return;
    const int token = part.count == 1 ? 0 : r / c.per, head = kvh * c.per + r - token * c.per;
    float top = m, factor = 1.0f;
    if (c.sink != nullptr) {
        const float sink = c.sink[head] * kLbLog2e;
        top = fmaxf(m, sink);
        factor = lb_sink_join_exp2(sink, m, l);
    }
    factor = l == 0.0f ? 0.0f : __fdividef(factor, l);
    const float unit_size = ex2(f);
    __nv_bfloat16* out = c.out + (int64_t)(part.first + token) * c.out_stride + head * HD + V * lane;
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = __float2bfloat16_rn(v[e] * factor * unit_size);
    if (lane == 0 && c.log_sums != nullptr) c.log_sums[((int64_t)seq * c.pages.n_kv_head + kvh) * c.max_rows + r] = l == 0.0f ? CUDART_INF_F : top + log2f(l);
}

}  // namespace
}  // namespace lb_a4

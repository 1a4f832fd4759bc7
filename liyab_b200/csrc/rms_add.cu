// A sublayer's output joins the residual stream and is normed for the next one: t = x + delta, h = t / sqrt(mean(t^2) + eps) * gain, left in bfloat16 or in
// e4m3 with a scale a row.
//
// Bound by memory: one pass, x and delta in, the sum and the result out.  A row stays in registers as t (gain_offset + gain), up to 32 values a thread, between its sum of
// squares, its largest value and its results, which 1 / sqrt and the scale meet as one factor (a value whose t (gain_offset + gain) is past float32's range counts as not finite).  From 296 rows
// on a warp has a row of up to 512 values (no barrier); else a block has a row (one barrier).  24 instructions a value at 2.3 a cycle stay below what memory takes: 4096 bfloat16 rows of 8192
// 44 us, 0.83 of the measured copy bandwidth (69 with the divisions, selections and comparisons of a first version).  Rows of more than 8192 values have 32 a thread, of which the 64 registers of
// two blocks an SM spill 8 to 24 (2048 bfloat16 rows of 16384 58 us, 0.63 of the copy bandwidth).
// Rows off the 16 bytes, and of more than 16384 values, go through shared memory, one or two values at a time and neighbours by neighbouring threads.
#include "linear4.h"

namespace {

using namespace lb_w4;

constexpr int kMaxWidth = 56 * 1024;
constexpr float kSmallest = 6.018531e-36f;      // 2^-117: 448 / it is still finite
constexpr uint32_t kInfinity = 0x7f800000u;

using Rows = lb_rms_add_args;

// The larger size; a NaN stays.
__device__ __forceinline__ float largest(float top, float v) {
    float out;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(out) : "f"(top), "f"(fabsf(v)));
    return out;
}

// What a row's largest |h| makes of the row: the factor on h (0: the row becomes zeros) and the scale.
__device__ __forceinline__ float row_factor(float top, float* scale) {
    const bool some = __float_as_uint(top) < kInfinity && top >= kSmallest;
    *scale = some ? top * (1.0f / 448.0f) : __float_as_uint(top) < kInfinity ? 0.0f : __int_as_float(0x7fc00000);
    return some ? __fdividef(448.0f / 256.0f, top * (1.0f / 256.0f)) : 0.0f;         // (the fast division makes 0 of divisors above 2^126)
}

// 8 values from 16 or 32 bytes.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(u[i] << 16);
            v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    }
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    }
}

// V: eights a thread.  WARP: a warp a row.
template <typename TX, typename TD, int V, bool WARP>
__global__ void __launch_bounds__(512, V == 4 ? 2 : 3)
rms_add_kernel(const Rows p) {
    __shared__ float sums[32];
    __shared__ uint32_t tops[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n_warps = blockDim.x >> 5;
    const int tid = WARP ? lane : (int)threadIdx.x, threads = WARP ? 32 : (int)blockDim.x;
    const int r = WARP ? (int)blockIdx.x * n_warps + warp : (int)blockIdx.x;
    lb_wait_for_predecessor();
    lb_dependents_may_launch();
    if (WARP && r >= p.rows) return;
    float v[V][8], d[V][8];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int at = (j * threads + tid) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j][i] = d[j][i] = 0.0f;
        if (at < p.width) {
            load8(static_cast<const TX*>(p.x) + (int64_t)r * p.ldx + at, v[j]);
            if (p.delta != nullptr) load8(static_cast<const TD*>(p.delta) + (int64_t)r * p.ldd + at, d[j]);
        }
    }
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[j][i] += d[j][i];
            ss = fmaf(v[j][i], v[j][i], ss);
        }
    ss = lb_warp_sum(ss);
    if (!WARP && lane == 0) sums[warp] = ss;
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int at = (j * threads + tid) * 8;
        if (at >= p.width) break;
        if (p.total != nullptr) store8(static_cast<TX*>(p.total) + (int64_t)r * p.ldt + at, v[j]);
        if (p.gain != nullptr) {
            float g[8];
            load8(p.gain + at, g);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[j][i] *= p.gain_offset + g[i];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) top = largest(top, v[j][i]);
    }
    uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
    if (!WARP) {
        if (lane == 0) tops[warp] = bits;
        __syncthreads();
        ss = lb_warp_sum(lane < n_warps ? sums[lane] : 0.0f);
        bits = __reduce_max_sync(0xffffffffu, lane < n_warps ? tops[lane] : 0u);
    }
    // h = v inv; where the squares overflow, inv is 0 and the finite values' row becomes zeros.
    const float inv = rsqrtf(__fdividef(ss, (float)p.width) + p.eps);
    if (p.scale == nullptr) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int at = (j * threads + tid) * 8;
            if (at >= p.width) break;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[j][i] *= inv;
            store8(static_cast<__nv_bfloat16*>(p.out) + (int64_t)r * p.ldo + at, v[j]);
        }
        return;
    }
    float scale;
    float f = row_factor(__uint_as_float(bits) * inv, &scale);
    if (f * inv < __uint_as_float(kInfinity)) {
        f *= inv;
    } else if (f != 0.0f) {
        // Values so small that one factor for both would be an infinity: the root meets them first.
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[j][i] *= inv;
    }
    if (tid == 0) p.scale[r] = scale;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int at = (j * threads + tid) * 8;
        if (at >= p.width) break;
        uint2 eight = make_uint2(0u, 0u);
        if (f != 0.0f) {
            eight.x = floats_to_e4m3x2(v[j][0] * f, v[j][1] * f) | floats_to_e4m3x2(v[j][2] * f, v[j][3] * f) << 16;
            eight.y = floats_to_e4m3x2(v[j][4] * f, v[j][5] * f) | floats_to_e4m3x2(v[j][6] * f, v[j][7] * f) << 16;
        }
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(p.out) + (int64_t)r * p.ldo + at) = eight;
    }
}

// One value, or two neighbours.
template <int U, typename T>
__device__ __forceinline__ void load_unit(const T* p, float (&v)[U]) {
    if constexpr (U == 1) {
        v[0] = lb_to_float(*p);
    } else if constexpr (sizeof(T) == 4) {
        const float2 two = *reinterpret_cast<const float2*>(p);
        v[0] = two.x;
        v[1] = two.y;
    } else {
        const uint32_t two = *reinterpret_cast<const uint32_t*>(p);
        v[0] = __uint_as_float(two << 16);
        v[1] = __uint_as_float(two & 0xffff0000u);
    }
}
template <int U, typename T>
__device__ __forceinline__ void store_unit(T* p, const float (&v)[U]) {
    if constexpr (U == 1) *p = lb_from_float<T>(v[0]);
    else if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
    else *reinterpret_cast<uint32_t*>(p) = pack_bf16(v[0], v[1]);
}

// Rows of any place and length: units of two values where all rows allow it, else of one, eight values a thread on their way together (one after the other 19 float32 rows of
// 10925 took 9.8 us, so 6.4; 4096 bfloat16 rows of 8190 take 193 us by ones and 93 by twos).
constexpr int kBatch = 8;

template <typename TX, typename TD, int U>
__global__ void __launch_bounds__(1024)
rms_add_any_kernel(const Rows p) {
    extern __shared__ __align__(16) float row[];        // (read and written in twos)
    __shared__ float sums[33];
    __shared__ uint32_t tops[32];
    constexpr int kUnits = kBatch / U;
    lb_wait_for_predecessor();
    lb_dependents_may_launch();
    const int r = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n_warps = blockDim.x >> 5, step = U * (int)blockDim.x;
    const TX* x = static_cast<const TX*>(p.x) + (int64_t)r * p.ldx;
    const TD* delta = static_cast<const TD*>(p.delta) + (int64_t)r * p.ldd;
    TX* total = static_cast<TX*>(p.total) + (int64_t)r * p.ldt;
    float ss = 0.0f;
    for (int i0 = U * threadIdx.x; i0 < p.width; i0 += kUnits * step) {
        float t[kUnits][U] = {}, d[kUnits][U] = {};
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const int i = i0 + u * step;
            if (i < p.width) load_unit<U>(x + i, t[u]);
            if (i < p.width && p.delta != nullptr) load_unit<U>(delta + i, d[u]);
        }
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const int i = i0 + u * step;
            if (i >= p.width) break;
#pragma unroll
            for (int k = 0; k < U; ++k) {
                t[u][k] += d[u][k];
                ss = fmaf(t[u][k], t[u][k], ss);
            }
            if (p.total != nullptr) store_unit<U>(total + i, t[u]);
            store_unit<U>(row + i, t[u]);
        }
    }
    const float inv = rsqrtf(__fdividef(lb_block_sum(ss, sums), (float)p.width) + p.eps);
    float top = 0.0f;
    for (int i0 = U * threadIdx.x; i0 < p.width; i0 += kUnits * step) {
        float g[kUnits][U];
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const int i = i0 + u * step;
#pragma unroll
            for (int k = 0; k < U; ++k) g[u][k] = 1.0f - p.gain_offset;
            if (p.gain != nullptr && i < p.width) load_unit<U>(p.gain + i, g[u]);
        }
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const int i = i0 + u * step;
            if (i >= p.width) break;
            float h[U];
            load_unit<U>(row + i, h);
#pragma unroll
            for (int k = 0; k < U; ++k) h[k] *= p.gain != nullptr ? inv * (p.gain_offset + g[u][k]) : inv;
            if (p.scale == nullptr) {
                store_unit<U>(static_cast<__nv_bfloat16*>(p.out) + (int64_t)r * p.ldo + i, h);
            } else {
                store_unit<U>(row + i, h);
#pragma unroll
                for (int k = 0; k < U; ++k) top = largest(top, h[k]);
            }
        }
    }
    if (p.scale == nullptr) return;
    uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
    if (lane == 0) tops[warp] = bits;
    __syncthreads();
    bits = __reduce_max_sync(0xffffffffu, lane < n_warps ? tops[lane] : 0u);
    float scale;
    const float f = row_factor(__uint_as_float(bits), &scale);
    uint8_t* out = static_cast<uint8_t*>(p.out) + (int64_t)r * p.ldo;
    for (int i = U * threadIdx.x; i < p.width; i += step) {
        float h[U];
        load_unit<U>(row + i, h);
        const uint32_t bytes = f != 0.0f ? floats_to_e4m3x2(h[0] * f, h[U - 1] * f) : 0u;
        if constexpr (U == 1) out[i] = (uint8_t)bytes;
        else *reinterpret_cast<uint16_t*>(out + i) = (uint16_t)bytes;
    }
    if (threadIdx.x == 0) p.scale[r] = scale;
}

template <typename TX, typename TD>
int launch(const Rows& p) {
    const cudaStream_t s = static_cast<cudaStream_t>(p.stream);
    auto aligned = [](const void* q, int64_t ld, int bytes) { return q == nullptr || (reinterpret_cast<uintptr_t>(q) % 16 == 0 && ld * bytes % 16 == 0); };
    const bool eight = p.scale != nullptr;
    const bool wide = p.width % 8 == 0 && aligned(p.x, p.ldx, sizeof(TX)) && aligned(p.delta, p.ldd, sizeof(TD)) && aligned(p.total, p.ldt, sizeof(TX)) && aligned(p.gain, 0, 4) &&
                      (eight ? reinterpret_cast<uintptr_t>(p.out) % 8 == 0 && p.ldo % 8 == 0 : aligned(p.out, p.ldo, 2));
    const int eights = (p.width + 7) / 8;
    if (!wide || eights > 2048) {
        auto even = [](const void* q, int64_t ld, int bytes) { return q == nullptr || (reinterpret_cast<uintptr_t>(q) % (2 * bytes) == 0 && ld % 2 == 0); };
        const bool twos = p.width % 2 == 0 && even(p.x, p.ldx, sizeof(TX)) && even(p.delta, p.ldd, sizeof(TD)) && even(p.total, p.ldt, sizeof(TX)) && even(p.gain, 0, 4) &&
                          even(p.out, p.ldo, eight ? 1 : 2);
        auto kernel = twos ? rms_add_any_kernel<TX, TD, 2> : rms_add_any_kernel<TX, TD, 1>;
        const size_t smem = sizeof(float) * p.width;
        if (smem > 40 * 1024) LB_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxWidth * 4));
        const int share = (p.width + 32 * kBatch - 1) / (32 * kBatch) * 32, block = share < 128 ? 128 : share > 1024 ? 1024 : share;
        LB_CHECK_CUDA(lb_launch_overlapped(kernel, dim3(p.rows), dim3(block), smem, s, p));
        return LB_OK;
    }
#define LB_RMS(V_, WARP_, GRID_, BLOCK_)                                                                                                                \
    do {                                                                                                                                                \
        LB_CHECK_CUDA(lb_launch_overlapped(rms_add_kernel<TX, TD, V_, WARP_>, dim3(GRID_), dim3(BLOCK_), 0, s, p));                                     \
        return LB_OK;                                                                                                                                   \
    } while (0)
    const bool many = p.rows >= 296;
    if (many && eights <= 64) {
        if (eights <= 32) LB_RMS(1, true, (p.rows + 3) / 4, 128);
        LB_RMS(2, true, (p.rows + 3) / 4, 128);
    }
    const int v = eights > 1024 ? 4 : eights > 512 || (many && eights > 256) ? 2 : 1;
    const int block = ((eights + v - 1) / v + 31) / 32 * 32;
    if (v == 1) LB_RMS(1, false, p.rows, block);
    if (v == 2) LB_RMS(2, false, p.rows, block);
    LB_RMS(4, false, p.rows, block);
#undef LB_RMS
}

}  // namespace

extern "C" int lb_rms_add_rows(const lb_rms_add_args* args) {
    LB_CHECK_ARG(args != nullptr, "rms_add: no arguments");
    lb_rms_add_args p = *args;
    LB_CHECK_ARG(p.rows >= 0 && (p.rows == 0 || (p.x != nullptr && p.out != nullptr)), "rms_add: %d rows, or no memory for them", p.rows);
    LB_CHECK_ARG(p.width > 0 && p.width <= kMaxWidth, "rms_add: rows of %d values (1 to %d)", p.width, kMaxWidth);
    LB_CHECK_ARG((p.x_dtype == LB_F32 || p.x_dtype == LB_BF16) && (p.delta_dtype == LB_F32 || p.delta_dtype == LB_BF16), "rms_add: x and delta are float32 or bfloat16");
    LB_CHECK_ARG(p.out_dtype == LB_BF16 || p.out_dtype == LB_E4M3, "rms_add: the output is bfloat16 or e4m3");
    LB_CHECK_ARG((p.out_dtype == LB_E4M3) == (p.scale != nullptr), "rms_add: an e4m3 output has a scale a row, a bfloat16 one has none");
    if (p.rows == 1) p.ldx = p.ldd = p.ldt = p.ldo = p.width;         // a single row has no stride
    LB_CHECK_ARG(p.ldx >= p.width && p.ldo >= p.width && (p.delta == nullptr || p.ldd >= p.width) && (p.total == nullptr || p.ldt >= p.width), "rms_add: rows overlap");
    if (p.rows == 0) return LB_OK;
    if (int rc = device_check("rms_add", p.device)) return rc;
    if (p.x_dtype == LB_F32) return p.delta_dtype == LB_F32 ? launch<float, float>(p) : launch<float, __nv_bfloat16>(p);
    return p.delta_dtype == LB_F32 ? launch<__nv_bfloat16, float>(p) : launch<__nv_bfloat16, __nv_bfloat16>(p);
}

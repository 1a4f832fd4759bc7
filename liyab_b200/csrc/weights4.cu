// 4-bit weights: laying a matrix out, rounding one to 4 bits, reading one back.  Done once when a model is set up; the products are elsewhere.
#include "linear4.h"

namespace {

using namespace lb_w4;

struct Sizes {
    int rows, padded, k_tiles;
};

// Rows as they are laid out: of a paired matrix each half is filled up to a multiple of eight.
Sizes sizes_of(int n, int k, int paired) {
    Sizes s;
    s.rows = paired ? 2 * ((n / 2 + 7) / 8 * 8) : n;
    s.padded = (s.rows + 127) / 128 * 128;
    s.k_tiles = (k + kTileK - 1) / kTileK;
    return s;
}

// The matrix's row that lies at `row`, -1 where it is padding.
__device__ __forceinline__ int source_row(int row, int n, int paired) {
    if (!paired) return row < n ? row : -1;
    const int f = row / 16 * 8 + (row & 7), half = row >> 3 & 1;
    return f < n / 2 ? half * (n / 2) + f : -1;
}

// Weight i of a word is nibble i / 2 + 4 (i % 2).
__device__ __forceinline__ int nibble_shift(int i) { return 4 * ((i >> 1) + 4 * (i & 1)); }

__device__ __forceinline__ size_t word_at(int row, int kt, int t, int j, int k_tiles) {
    return ((size_t)(row >> 4) * k_tiles + kt) * (kTileBytes / 4) + piece_at(row & 15, t) * 4 + j;
}

// A row's scales of a k tile.
__device__ __forceinline__ uint8_t* scales_at(const lb_weights4& w, int row, int kt, int k_tiles) {
    return static_cast<uint8_t*>(w.scales) + (((size_t)(row >> 4) * k_tiles + kt) * kTileRows + (row & 15)) * (kTileK / w.group);
}

// A block a row: its words of eight weights, its scales and its factor.
__global__ void lay_out_kernel(const int8_t* __restrict__ q, int64_t ldq, const uint8_t* __restrict__ s, int64_t lds, const float* __restrict__ r,
                               const lb_weights4 w, int k_tiles) {
    const int row = blockIdx.x, from = source_row(row, w.n, w.paired), groups = (w.k + w.group - 1) / w.group;
    uint32_t* words = static_cast<uint32_t*>(w.nibbles);
    for (int i = threadIdx.x; i < 16 * k_tiles; i += blockDim.x) {
        const int kt = i >> 4, t = i >> 2 & 3, j = i & 3, k0 = kt * kTileK + 32 * j + 8 * t;
        uint32_t word = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int k = k0 + e, v = from >= 0 && k < w.k ? q[(int64_t)from * ldq + k] : 0;
            word |= (uint32_t)(min(7, max(-8, v)) + 8) << nibble_shift(e);
        }
        words[word_at(row, kt, t, j, k_tiles)] = word;
    }
    const int per_tile = kTileK / w.group;
    for (int g = threadIdx.x; g < k_tiles * per_tile; g += blockDim.x)
        scales_at(w, row, g / per_tile, k_tiles)[g % per_tile] = from >= 0 && g < groups ? s[(int64_t)from * lds + g] : 0;
    if (threadIdx.x == 0) w.rows[row] = from >= 0 ? r[from] : 0.0f;
}

// A block a row, a warp a piece of 128 weights, four neighbours a lane; a group is 8, 16 or 32 lanes.
template <typename T>
__global__ void quantise_kernel(const T* __restrict__ matrix, int64_t ldm, const lb_weights4 w, int k_tiles) {
    __shared__ float tops[32];
    const int row = blockIdx.x, from = source_row(row, w.n, w.paired), warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n_warps = blockDim.x >> 5;
    const T* in = matrix + (from >= 0 ? (int64_t)from * ldm : 0);
    const int lanes = w.group / 4;
    // The largest value of the row; a value that is not finite makes it a NaN.
    float top = 0.0f;
    bool finite = true;
    for (int k = threadIdx.x; from >= 0 && k < w.k; k += blockDim.x) {
        const float v = fabsf(lb_to_float(in[k]));
        finite &= v <= 3.402823466e38f;
        top = fmaxf(top, v);
    }
    top = lb_warp_max(top);
    finite = __all_sync(0xffffffffu, finite);
    if (lane == 0) tops[warp] = finite ? top : -1.0f;
    __syncthreads();
    top = 0.0f;
    for (int i = 0; i < n_warps; ++i) {
        finite &= tops[i] >= 0.0f;
        top = fmaxf(top, tops[i]);
    }
    float r = __fdiv_rn(__fdiv_rn(top, 7.0f), 448.0f);
    const bool some = r >= 1.17549435e-38f && finite;
    if (!some) r = finite ? 0.0f : __int_as_float(0x7fc00000);

    uint32_t* words = static_cast<uint32_t*>(w.nibbles);
    for (int kt = warp; kt < k_tiles; kt += n_warps) {
        float v[4], peak = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int k = kt * kTileK + 4 * lane + e;
            v[e] = from >= 0 && k < w.k && some ? lb_to_float(in[k]) : 0.0f;
            peak = fmaxf(peak, fabsf(v[e]));
        }
        for (int o = 1; o < lanes; o <<= 1) peak = fmaxf(peak, __shfl_xor_sync(0xffffffffu, peak, o));
        const uint32_t s = some ? floats_to_e4m3x2(__fdiv_rn(__fdiv_rn(peak, 7.0f), r), 0.0f) & 0xffu : 0u;
        const float step = e4m3_to_float(s) * r;
        uint32_t part = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float q = step > 0.0f ? fminf(7.0f, fmaxf(-8.0f, rintf(__fdiv_rn(v[e], step)))) : 0.0f;
            part |= (uint32_t)((int)q + 8) << nibble_shift(4 * (lane & 1) + e);
        }
        part |= __shfl_xor_sync(0xffffffffu, part, 1);
        if ((lane & 1) == 0) words[word_at(row, kt, lane >> 1 & 3, lane >> 3, k_tiles)] = part;
        if (lane % lanes == 0) scales_at(w, row, kt, k_tiles)[lane / lanes] = (uint8_t)s;
    }
    if (threadIdx.x == 0) w.rows[row] = r;
}

__global__ void values_kernel(const lb_weights4 w, float* __restrict__ out, int64_t ldo, int k_tiles) {
    const int row = blockIdx.x, to = source_row(row, w.n, w.paired);
    if (to < 0) return;
    const uint32_t* words = static_cast<const uint32_t*>(w.nibbles);
    for (int k = threadIdx.x; k < w.k; k += blockDim.x) {
        const int in = k % kTileK;
        const uint32_t word = words[word_at(row, k / kTileK, in >> 3 & 3, in >> 5, k_tiles)];
        const float q = (float)((int)(word >> nibble_shift(in & 7) & 15u) - 8);
        out[(int64_t)to * ldo + k] = q * e4m3_to_float(scales_at(w, row, k / kTileK, k_tiles)[in / w.group]) * w.rows[row];
    }
}

// The products ask for their weights before they wait for the kernel before them: what writes weights is finished when the call returns.
int finished(cudaStream_t stream) {
    LB_CHECK_LAUNCH();
    LB_CHECK_CUDA(cudaStreamSynchronize(stream));
    return LB_OK;
}

}  // namespace

int weights4_check(const lb_weights4* w, const char* what) {
    LB_CHECK_ARG(w != nullptr && w->nibbles != nullptr && w->scales != nullptr && w->rows != nullptr, "%s: weights without memory", what);
    LB_CHECK_ARG(w->group == 32 || w->group == 64 || w->group == 128, "%s: group is %d, not 32, 64 or 128", what, w->group);
    LB_CHECK_ARG(w->n > 0 && w->k > 0 && w->n <= (1 << 26) && w->k <= (1 << 26) && (!w->paired || w->n % 2 == 0), "%s: a matrix of %d x %d", what, w->n, w->k);
    LB_CHECK_ARG(((reinterpret_cast<uintptr_t>(w->nibbles) | reinterpret_cast<uintptr_t>(w->scales)) % 16 | reinterpret_cast<uintptr_t>(w->rows) % 4) == 0,
                 "%s: nibbles and scales are not 16-byte aligned, or rows not as floats are", what);
    return LB_OK;
}

extern "C" int lb_weights4_sizes(int n, int k, int group, int paired, int64_t* nibble_bytes, int64_t* scale_bytes, int* n_padded) {
    LB_CHECK_ARG(nibble_bytes != nullptr && scale_bytes != nullptr && n_padded != nullptr, "weights4: nowhere to write the sizes");
    LB_CHECK_ARG(group == 32 || group == 64 || group == 128, "weights4: group is %d, not 32, 64 or 128", group);
    LB_CHECK_ARG(n > 0 && k > 0 && n <= (1 << 26) && k <= (1 << 26) && (!paired || n % 2 == 0), "weights4: a matrix of %d x %d", n, k);
    const Sizes s = sizes_of(n, k, paired);
    *nibble_bytes = (int64_t)(s.padded / kTileRows) * s.k_tiles * kTileBytes;
    *n_padded = s.padded;
    *scale_bytes = (int64_t)s.padded * s.k_tiles * (kTileK / group);
    return LB_OK;
}

extern "C" int lb_weights4_lay_out(const int8_t* q, int64_t ldq, const void* s, int64_t lds, const float* r, const lb_weights4* w, void* stream) {
    if (int rc = weights4_check(w, "weights4_lay_out")) return rc;
    LB_CHECK_ARG(q != nullptr && s != nullptr && r != nullptr && (w->n == 1 || (ldq >= w->k && lds >= (w->k + w->group - 1) / w->group)), "weights4_lay_out: a part is missing or its rows overlap");
    const Sizes z = sizes_of(w->n, w->k, w->paired);
    lay_out_kernel<<<z.padded, 256, 0, static_cast<cudaStream_t>(stream)>>>(q, ldq, static_cast<const uint8_t*>(s), lds, r, *w, z.k_tiles);
    return finished(static_cast<cudaStream_t>(stream));
}

extern "C" int lb_weights4_quantise(int dtype, const void* matrix, int64_t ldm, const lb_weights4* w, void* stream) {
    if (int rc = weights4_check(w, "weights4_quantise")) return rc;
    LB_CHECK_ARG(matrix != nullptr && (w->n == 1 || ldm >= w->k), "weights4_quantise: no matrix, or its rows overlap");
    LB_CHECK_ARG(dtype == LB_F32 || dtype == LB_BF16, "weights4_quantise: a matrix is float32 or bfloat16");
    const Sizes z = sizes_of(w->n, w->k, w->paired);
    if (dtype == LB_F32) quantise_kernel<float><<<z.padded, 256, 0, static_cast<cudaStream_t>(stream)>>>(static_cast<const float*>(matrix), ldm, *w, z.k_tiles);
    else quantise_kernel<__nv_bfloat16><<<z.padded, 256, 0, static_cast<cudaStream_t>(stream)>>>(static_cast<const __nv_bfloat16*>(matrix), ldm, *w, z.k_tiles);
    return finished(static_cast<cudaStream_t>(stream));
}

extern "C" int lb_weights4_values(const lb_weights4* w, float* out, int64_t ldo, void* stream) {
    if (int rc = weights4_check(w, "weights4_values")) return rc;
    LB_CHECK_ARG(out != nullptr && (w->n == 1 || ldo >= w->k), "weights4_values: no output, or its rows overlap");
    const Sizes z = sizes_of(w->n, w->k, w->paired);
    values_kernel<<<z.padded, 256, 0, static_cast<cudaStream_t>(stream)>>>(*w, out, ldo, z.k_tiles);
    LB_CHECK_LAUNCH();
    return LB_OK;
}

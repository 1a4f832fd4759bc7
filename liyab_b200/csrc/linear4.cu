// Products with 4-bit weights: out = act(a w^T + bias) + residual, and gate(a w_gate^T) * (a w_up^T) over paired rows.
//
// A block takes a row tile of 16 weights' rows and eight tokens; warp i takes the k tiles i, i + 8, ...: a lane's words are the rows of an mma whose
// columns are the tokens.  A group's sum is made from the integers q, its scale meets it in 32 bits; the warps' sums meet in shared memory in order.
#include "weights4.cuh"

namespace {

using namespace lb_w4;

constexpr int kWarps = 8, kTokens = 8;

template <typename T, bool PAIRED>
__global__ void __launch_bounds__(32 * kWarps)
linear4_kernel(const lb_weights4 w, const void* __restrict__ a, int64_t lda, bool wide, const Epilogue e, int k_tiles) {
    __shared__ float sums[kWarps][kTileRows][kTokens + 1];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int row0 = blockIdx.x * kTileRows, m0 = blockIdx.y * kTokens, m = m0 + g;
    const uint4* tiles = static_cast<const uint4*>(w.nibbles) + (size_t)blockIdx.x * k_tiles * (kTileBytes / 16);
    const uint8_t* scales = static_cast<const uint8_t*>(w.scales) + (size_t)(row0 + g) * w.scale_stride;
    const int per_tile = kTileK / w.group, words_per_group = w.group / 32;
    lb_wait_for_predecessor();
    lb_dependents_may_launch();

    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int kt = warp; kt < k_tiles; kt += kWarps) {
        const uint4 top = tiles[kt * (kTileBytes / 16) + 4 * g + t], low = tiles[kt * (kTileBytes / 16) + 4 * (g + 8) + t];
        const uint32_t wt[4] = {top.x, top.y, top.z, top.w}, wl[4] = {low.x, low.y, low.z, low.w};
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t b[4] = {0u, 0u, 0u, 0u};
            if (m < e.M) load_eight<T>(b, a, (int64_t)m * lda, kt * kTileK + 32 * j + 8 * t, w.k, wide);
#pragma unroll
            for (int s = 0; s < 2; ++s)
                mma16816<T>(part, pair_of<T>(wt[j], 2 * s), pair_of<T>(wl[j], 2 * s), pair_of<T>(wt[j], 2 * s + 1), pair_of<T>(wl[j], 2 * s + 1), b[2 * s], b[2 * s + 1]);
            if ((j + 1) % words_per_group == 0) {
                const int group = kt * per_tile + j / words_per_group;
                const float st = e4m3_to_float(scales[group]), sl = e4m3_to_float(scales[(size_t)8 * w.scale_stride + group]);
                acc[0] = fmaf(part[0], st, acc[0]);
                acc[1] = fmaf(part[1], st, acc[1]);
                acc[2] = fmaf(part[2], sl, acc[2]);
                acc[3] = fmaf(part[3], sl, acc[3]);
                part[0] = part[1] = part[2] = part[3] = 0.0f;
            }
        }
    }
    sums[warp][g][2 * t] = acc[0];
    sums[warp][g][2 * t + 1] = acc[1];
    sums[warp][g + 8][2 * t] = acc[2];
    sums[warp][g + 8][2 * t + 1] = acc[3];
    __syncthreads();

    const int row = threadIdx.x & 15, token = threadIdx.x >> 4;
    if (token >= kTokens || m0 + token >= e.M || (PAIRED && row >= 8)) return;
    const float scale = e.a_scale != nullptr ? e.a_scale[m0 + token] : 1.0f;
    float v = 0.0f;
    for (int i = 0; i < kWarps; ++i) v += sums[i][row][token];
    v *= w.rows[row0 + row] * scale;
    if constexpr (PAIRED) {
        float up = 0.0f;
        for (int i = 0; i < kWarps; ++i) up += sums[i][row + 8][token];
        up *= w.rows[row0 + 8 + row] * scale;
        const int col = row0 / 2 + row;
        if (col < e.n) store_out(e, m0 + token, col, lb_gated_pair(v, up, e.gate, e.alpha, e.limit));
    } else if (row0 + row < e.n) {
        finish_one(e, lb_act_load(e.bias, e.n, e.act), m0 + token, row0 + row, v);
    }
}

template <bool PAIRED>
int launch(const lb_weights4* w, int a_dtype, const void* a, int64_t lda, const Epilogue& e, cudaStream_t stream) {
    const int k_tiles = (w->k + kTileK - 1) / kTileK, rows = PAIRED ? 2 * ((e.n + 7) / 8 * 8) : e.n;
    const dim3 grid((rows + kTileRows - 1) / kTileRows, (e.M + kTokens - 1) / kTokens);
    const bool half = a_dtype == LB_E4M3;
    const bool wide = half ? lda % 8 == 0 && reinterpret_cast<uintptr_t>(a) % 8 == 0 : lda % 8 == 0 && reinterpret_cast<uintptr_t>(a) % 16 == 0;
    if (half) LB_CHECK_CUDA(lb_launch_overlapped(linear4_kernel<F16, PAIRED>, grid, dim3(32 * kWarps), 0, stream, *w, a, lda, wide, e, k_tiles));
    else LB_CHECK_CUDA(lb_launch_overlapped(linear4_kernel<Bf16, PAIRED>, grid, dim3(32 * kWarps), 0, stream, *w, a, lda, wide, e, k_tiles));
    return LB_OK;
}

int check(const char* what, const lb_weights4* w, int a_dtype, const void* a, int64_t lda, const float* a_scale, int out_dtype, const void* out, int64_t ldo, int M, int n) {
    LB_CHECK_ARG(w != nullptr && w->nibbles != nullptr && w->scales != nullptr && w->rows != nullptr, "%s: weights without memory", what);
    LB_CHECK_ARG(w->group == 32 || w->group == 64 || w->group == 128, "%s: group is %d, not 32, 64 or 128", what, w->group);
    LB_CHECK_ARG(M >= 0 && (M == 0 || (a != nullptr && out != nullptr)), "%s: %d rows, or no memory for them", what, M);
    LB_CHECK_ARG(M <= 65535 * kTokens, "%s: %d rows are more than %d", what, M, 65535 * kTokens);
    LB_CHECK_ARG(lda >= w->k && ldo >= n, "%s: rows overlap", what);
    LB_CHECK_ARG(a_dtype == LB_BF16 || a_dtype == LB_E4M3, "%s: activations are bfloat16 or e4m3", what);
    LB_CHECK_ARG((a_dtype == LB_E4M3) == (a_scale != nullptr), "%s: e4m3 activations have a scale a row, bfloat16 ones have none", what);
    LB_CHECK_ARG(out_dtype == LB_BF16 || out_dtype == LB_F32, "%s: the output is bfloat16 or float32", what);
    return LB_OK;
}

}  // namespace

extern "C" int lb_linear4(const lb_weights4* w, int a_dtype, const void* a, int64_t lda, const float* a_scale, const float* bias, const float* residual, int64_t ldr,
                          int out_dtype, void* out, int64_t ldo, int M, int act, void* stream) {
    if (int rc = check("linear4", w, a_dtype, a, lda, a_scale, out_dtype, out, ldo, M, w != nullptr ? w->n : 0)) return rc;
    LB_CHECK_ARG(!w->paired, "linear4: paired weights are read by gated4");
    LB_CHECK_ARG(act >= LB_ACT_NONE && act <= LB_ACT_RELU2 && (act != LB_ACT_XIELU || bias != nullptr), "linear4: activation %d", act);
    LB_CHECK_ARG(residual == nullptr || ldr >= w->n, "linear4: the residual's rows overlap");
    if (M == 0) return LB_OK;
    const Epilogue e{a_scale, bias, residual, out, ldr, ldo, M, w->n, act, 0, 0.0f, 0.0f, out_dtype == LB_F32};
    return launch<false>(w, a_dtype, a, lda, e, static_cast<cudaStream_t>(stream));
}

extern "C" int lb_gated4(const lb_weights4* w, int a_dtype, const void* a, int64_t lda, const float* a_scale, int out_dtype, void* out, int64_t ldo, int M, int gate,
                         float alpha, float limit, void* stream) {
    if (int rc = check("gated4", w, a_dtype, a, lda, a_scale, out_dtype, out, ldo, M, w != nullptr ? w->n / 2 : 0)) return rc;
    LB_CHECK_ARG(w->paired, "gated4: the weights are not laid out in pairs");
    LB_CHECK_ARG(gate >= LB_GATE_SIGMOID && gate <= LB_GATE_CAPPED, "gated4: gate %d", gate);
    if (M == 0) return LB_OK;
    const Epilogue e{a_scale, nullptr, nullptr, out, 0, ldo, M, w->n / 2, LB_ACT_NONE, gate, alpha, limit, out_dtype == LB_F32};
    return launch<true>(w, a_dtype, a, lda, e, static_cast<cudaStream_t>(stream));
}

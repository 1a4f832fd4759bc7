// A sublayer's output joins the residual stream and is normed for the next one: t = x + delta, h = t / sqrt(mean(t^2) + eps) * gain, left in bfloat16 or in
// e4m3 with a scale a row.  A block a row; the row stays in shared memory between the passes over it (sum of squares, largest value, results).
#include "weights4.cuh"

namespace {

using namespace lb_w4;

constexpr int kMaxWidth = 56 * 1024;
constexpr float kSmallest = 6.018531e-36f;      // 2^-117: 448 / it is still finite

__device__ __forceinline__ float block_max(float v, float* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n_warps = blockDim.x >> 5;
    v = lb_warp_max(v);
    __syncthreads();
    if (lane == 0) scratch[warp] = v;
    __syncthreads();
    v = scratch[0];
    for (int i = 1; i < n_warps; ++i) v = fmaxf(v, scratch[i]);
    return v;
}

template <typename TX, typename TD>
__global__ void rms_add_kernel(const TX* x, int64_t ldx, const TD* delta, int64_t ldd, TX* total, int64_t ldt, const float* __restrict__ gain, float gain_offset, float eps,
                               void* out, int64_t ldo, float* scale, int width) {
    extern __shared__ float row[];
    __shared__ float scratch[33];
    lb_wait_for_predecessor();
    lb_dependents_may_launch();
    const int r = blockIdx.x;
    float ss = 0.0f;
    for (int i = threadIdx.x; i < width; i += blockDim.x) {
        float t = lb_to_float(x[(int64_t)r * ldx + i]);
        if (delta != nullptr) t += lb_to_float(delta[(int64_t)r * ldd + i]);
        if (total != nullptr) total[(int64_t)r * ldt + i] = lb_from_float<TX>(t);
        row[i] = t;
        ss = fmaf(t, t, ss);
    }
    const float inv = 1.0f / sqrtf(lb_block_sum(ss, scratch) / (float)width + eps);
    float top = 0.0f;
    bool finite = true;
    for (int i = threadIdx.x; i < width; i += blockDim.x) {
        const float h = row[i] * inv * (gain != nullptr ? gain_offset + gain[i] : 1.0f);
        row[i] = h;
        finite &= fabsf(h) <= 3.402823466e38f;
        top = fmaxf(top, fabsf(h));
    }
    if (scale == nullptr) {
        for (int i = threadIdx.x; i < width; i += blockDim.x) static_cast<__nv_bfloat16*>(out)[(int64_t)r * ldo + i] = __float2bfloat16_rn(row[i]);
        return;
    }
    finite = __syncthreads_and(finite);
    top = block_max(top, scratch);
    const bool some = finite && top >= kSmallest;
    const float f = some ? 448.0f / top : 0.0f;
    for (int i = threadIdx.x; i < width; i += blockDim.x)
        static_cast<uint8_t*>(out)[(int64_t)r * ldo + i] = some ? (uint8_t)floats_to_e4m3x2(row[i] * f, 0.0f) : 0;
    if (threadIdx.x == 0) scale[r] = some ? top / 448.0f : finite ? 0.0f : __int_as_float(0x7fc00000);
}

template <typename TX, typename TD>
int launch(const void* x, int64_t ldx, const void* delta, int64_t ldd, void* total, int64_t ldt, const float* gain, float gain_offset, float eps, void* out, int64_t ldo,
           float* scale, int rows, int width, cudaStream_t stream) {
    const size_t smem = sizeof(float) * width;
    auto kernel = rms_add_kernel<TX, TD>;
    if (smem > 48 * 1024) LB_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    LB_CHECK_CUDA(lb_launch_overlapped(kernel, dim3(rows), dim3(width >= 2048 ? 512 : 256), smem, stream, static_cast<const TX*>(x), ldx, static_cast<const TD*>(delta), ldd,
                                       static_cast<TX*>(total), ldt, gain, gain_offset, eps, out, ldo, scale, width));
    return LB_OK;
}

}  // namespace

extern "C" int lb_rms_add_rows(int x_dtype, const void* x, int64_t ldx, int delta_dtype, const void* delta, int64_t ldd, void* total, int64_t ldt, const float* gain,
                          float gain_offset, float eps, int out_dtype, void* out, int64_t ldo, float* scale, int rows, int width, void* stream) {
    LB_CHECK_ARG(rows >= 0 && (rows == 0 || (x != nullptr && out != nullptr)), "rms_add: %d rows, or no memory for them", rows);
    LB_CHECK_ARG(width > 0 && width <= kMaxWidth, "rms_add: rows of %d values (1 to %d)", width, kMaxWidth);
    LB_CHECK_ARG((x_dtype == LB_F32 || x_dtype == LB_BF16) && (delta_dtype == LB_F32 || delta_dtype == LB_BF16), "rms_add: x and delta are float32 or bfloat16");
    LB_CHECK_ARG(out_dtype == LB_BF16 || out_dtype == LB_E4M3, "rms_add: the output is bfloat16 or e4m3");
    LB_CHECK_ARG((out_dtype == LB_E4M3) == (scale != nullptr), "rms_add: an e4m3 output has a scale a row, a bfloat16 one has none");
    LB_CHECK_ARG(ldx >= width && ldo >= width && (delta == nullptr || ldd >= width) && (total == nullptr || ldt >= width), "rms_add: rows overlap");
    if (rows == 0) return LB_OK;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (x_dtype == LB_F32)
        return delta_dtype == LB_F32 ? launch<float, float>(x, ldx, delta, ldd, total, ldt, gain, gain_offset, eps, out, ldo, scale, rows, width, s)
                                     : launch<float, __nv_bfloat16>(x, ldx, delta, ldd, total, ldt, gain, gain_offset, eps, out, ldo, scale, rows, width, s);
    return delta_dtype == LB_F32 ? launch<__nv_bfloat16, float>(x, ldx, delta, ldd, total, ldt, gain, gain_offset, eps, out, ldo, scale, rows, width, s)
                                 : launch<__nv_bfloat16, __nv_bfloat16>(x, ldx, delta, ldd, total, ldt, gain, gain_offset, eps, out, ldo, scale, rows, width, s);
}

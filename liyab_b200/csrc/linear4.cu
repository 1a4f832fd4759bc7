// Products with 4-bit weights: what both entry points check, and which kernel takes a call.
#include "linear4.h"

int linear4_sm_count() {
    static const int count = [] {
        int dev = 0, n = 0;
        return cudaGetDevice(&dev) == cudaSuccess && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess ? n : 148;
    }();
    return count;
}

namespace {

using namespace lb_w4;

int launch(const lb_weights4* w, int a_dtype, const void* a, int64_t lda, const Epilogue& e, int rows, void* scratch, cudaStream_t stream) {
    const FewPlan p = few_plan(e.M, rows, w->k, w->group, linear4_sm_count());
    return p.warps > 0 ? few_tokens(w, a_dtype, a, lda, e, p, stream) : many_tokens(w, a_dtype, a, lda, e, scratch, stream);
}

int check(const char* what, const lb_weights4* w, int a_dtype, const void* a, int64_t lda, const float* a_scale, int out_dtype, const void* out, int64_t ldo, int M, int n) {
    LB_CHECK_ARG(w != nullptr && w->nibbles != nullptr && w->scales != nullptr && w->rows != nullptr, "%s: weights without memory", what);
    LB_CHECK_ARG(w->group == 32 || w->group == 64 || w->group == 128, "%s: group is %d, not 32, 64 or 128", what, w->group);
    LB_CHECK_ARG(M >= 0 && (M == 0 || (a != nullptr && out != nullptr)), "%s: %d rows, or no memory for them", what, M);
    LB_CHECK_ARG(M <= 65535 * 16, "%s: %d rows are more than %d", what, M, 65535 * 16);
    LB_CHECK_ARG(lda >= w->k && ldo >= n, "%s: rows overlap", what);
    LB_CHECK_ARG(a_dtype == LB_BF16 || a_dtype == LB_E4M3, "%s: activations are bfloat16 or e4m3", what);
    LB_CHECK_ARG((a_dtype == LB_E4M3) == (a_scale != nullptr), "%s: e4m3 activations have a scale a row, bfloat16 ones have none", what);
    LB_CHECK_ARG(out_dtype == LB_BF16 || out_dtype == LB_F32, "%s: the output is bfloat16 or float32", what);
    return LB_OK;
}

}  // namespace

extern "C" int lb_linear4(const lb_weights4* w, int a_dtype, const void* a, int64_t lda, const float* a_scale, const float* bias, const float* residual, int64_t ldr,
                          int out_dtype, void* out, int64_t ldo, int M, int act, void* scratch, void* stream) {
    if (int rc = check("linear4", w, a_dtype, a, lda, a_scale, out_dtype, out, ldo, M, w != nullptr ? w->n : 0)) return rc;
    LB_CHECK_ARG(!w->paired, "linear4: paired weights are read by gated4");
    LB_CHECK_ARG(act >= LB_ACT_NONE && act <= LB_ACT_RELU2 && (act != LB_ACT_XIELU || bias != nullptr), "linear4: activation %d", act);
    LB_CHECK_ARG(residual == nullptr || ldr >= w->n, "linear4: the residual's rows overlap");
    if (M == 0) return LB_OK;
    const Epilogue e{a_scale, bias, residual, out, ldr, ldo, M, w->n, act, 0, 0.0f, 0.0f, out_dtype == LB_F32};
    return launch(w, a_dtype, a, lda, e, w->n, scratch, static_cast<cudaStream_t>(stream));
}

extern "C" int lb_gated4(const lb_weights4* w, int a_dtype, const void* a, int64_t lda, const float* a_scale, int out_dtype, void* out, int64_t ldo, int M, int gate,
                         float alpha, float limit, void* scratch, void* stream) {
    if (int rc = check("gated4", w, a_dtype, a, lda, a_scale, out_dtype, out, ldo, M, w != nullptr ? w->n / 2 : 0)) return rc;
    LB_CHECK_ARG(w->paired, "gated4: the weights are not laid out in pairs");
    LB_CHECK_ARG(gate >= LB_GATE_SIGMOID && gate <= LB_GATE_CAPPED, "gated4: gate %d", gate);
    if (M == 0) return LB_OK;
    const Epilogue e{a_scale, nullptr, nullptr, out, 0, ldo, M, w->n / 2, LB_ACT_NONE, gate, alpha, limit, out_dtype == LB_F32};
    return launch(w, a_dtype, a, lda, e, 2 * ((e.n + 7) / 8 * 8), scratch, static_cast<cudaStream_t>(stream));
}

extern "C" int64_t lb_linear4_scratch(const lb_weights4* w, int a_dtype, const void* a, int64_t lda, int M) {
    if (w == nullptr || M <= 0) return 0;
    const int rows = w->paired ? 2 * ((w->n / 2 + 7) / 8 * 8) : w->n;
    return few_plan(M, rows, w->k, w->group, linear4_sm_count()).warps > 0 ? 0 : many_scratch_bytes(w, a_dtype, a, lda, M);
}

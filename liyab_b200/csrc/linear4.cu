// Products with 4-bit weights: what both entry points check, and which kernel takes a call.
#include "linear4.h"

int linear4_sm_count() {
    static const int count = [] {
        int dev = 0, n = 0;
        return cudaGetDevice(&dev) == cudaSuccess && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess ? n : 148;
    }();
    return count;
}

int device_check(const char* what, int device) {
    if (device <= 0) return LB_OK;
    int current = 0;
    LB_CHECK_CUDA(cudaGetDevice(&current));
    LB_CHECK_ARG(current == device - 1, "%s: the tensors are on cuda:%d, the current device is cuda:%d", what, device - 1, current);
    return LB_OK;
}

namespace {

using namespace lb_w4;

int launch(const lb_weights4* w, int a_dtype, const void* a, int64_t lda, const Epilogue& e, int rows, void* scratch, cudaStream_t stream) {
    const FewPlan p = few_plan(e.M, rows, w->k, w->group, linear4_sm_count());
    return p.warps > 0 ? few_tokens(w, a_dtype, a, lda, e, p, stream) : many_tokens(w, a_dtype, a, lda, e, scratch, stream);
}

int check(const char* what, const lb_linear4_args* p, bool paired) {
    LB_CHECK_ARG(p != nullptr, "%s: no arguments", what);
    const lb_weights4* w = p->w;
    if (int rc = weights4_check(w, what)) return rc;
    LB_CHECK_ARG((w->paired != 0) == paired, "%s: the weights are %slaid out in pairs", what, paired ? "not " : "");
    LB_CHECK_ARG(p->M >= 0 && (p->M == 0 || (p->a != nullptr && p->out != nullptr)), "%s: %d rows, or no memory for them", what, p->M);
    LB_CHECK_ARG(p->M <= 65535 * 16, "%s: %d rows are more than %d", what, p->M, 65535 * 16);
    LB_CHECK_ARG(p->M == 1 || (p->lda >= w->k && p->ldo >= (paired ? w->n / 2 : w->n) && (p->residual == nullptr || p->ldr >= w->n)), "%s: rows overlap", what);
    LB_CHECK_ARG(p->a_dtype == LB_BF16 || p->a_dtype == LB_E4M3, "%s: activations are bfloat16 or e4m3", what);
    LB_CHECK_ARG((p->a_dtype == LB_E4M3) == (p->a_scale != nullptr), "%s: e4m3 activations have a scale a row, bfloat16 ones have none", what);
    LB_CHECK_ARG(p->out_dtype == LB_BF16 || p->out_dtype == LB_F32, "%s: the output is bfloat16 or float32", what);
    auto at = [](const void* q) { return reinterpret_cast<uintptr_t>(q); };
    LB_CHECK_ARG((at(p->a) % (p->a_dtype == LB_BF16 ? 2 : 1) | at(p->out) % (p->out_dtype == LB_BF16 ? 2 : 4) | (at(p->a_scale) | at(p->bias) | at(p->residual)) % 4) == 0,
                 "%s: a pointer is not aligned to its type", what);
    return p->M > 0 ? device_check(what, w->device) : LB_OK;
}

// A single row has no stride.
int64_t stride_of(const lb_linear4_args* p) { return p->M > 1 ? p->lda : 0; }

}  // namespace

extern "C" int lb_linear4(const lb_linear4_args* p) {
    if (int rc = check("linear4", p, false)) return rc;
    LB_CHECK_ARG(p->act >= LB_ACT_NONE && p->act <= LB_ACT_RELU2 && (p->act != LB_ACT_XIELU || p->bias != nullptr), "linear4: activation %d", p->act);
    if (p->M == 0) return LB_OK;
    const Epilogue e{p->a_scale, p->bias, p->residual, p->out, p->ldr, p->ldo, p->M, p->w->n, p->act, 0, 0.0f, 0.0f, p->out_dtype == LB_F32};
    return launch(p->w, p->a_dtype, p->a, stride_of(p), e, p->w->n, p->scratch, static_cast<cudaStream_t>(p->stream));
}

extern "C" int lb_gated4(const lb_linear4_args* p) {
    if (int rc = check("gated4", p, true)) return rc;
    LB_CHECK_ARG(p->act >= LB_GATE_SIGMOID && p->act <= LB_GATE_CAPPED, "gated4: gate %d", p->act);
    LB_CHECK_ARG(p->bias == nullptr && p->residual == nullptr, "gated4: neither a bias nor a residual is added");
    if (p->M == 0) return LB_OK;
    const Epilogue e{p->a_scale, nullptr, nullptr, p->out, 0, p->ldo, p->M, p->w->n / 2, LB_ACT_NONE, p->act, p->alpha, p->limit, p->out_dtype == LB_F32};
    return launch(p->w, p->a_dtype, p->a, stride_of(p), e, 2 * ((e.n + 7) / 8 * 8), p->scratch, static_cast<cudaStream_t>(p->stream));
}

extern "C" int lb_linear4_plan(const lb_weights4* w, int M, int out_dtype, int* plan) {
    if (int rc = weights4_check(w, "linear4_plan")) return rc;
    LB_CHECK_ARG(plan != nullptr && M > 0 && (out_dtype == LB_BF16 || out_dtype == LB_F32), "linear4_plan: no rows, no such result, or no place for the answer");
    const int rows = w->paired ? 2 * ((w->n / 2 + 7) / 8 * 8) : w->n;
    const FewPlan f = few_plan(M, rows, w->k, w->group, linear4_sm_count());
    if (f.warps > 0) {
        plan[0] = 0;
        plan[1] = M;
        plan[2] = f.splits;
        plan[3] = f.clusters;
        return LB_OK;
    }
    const ManyPlan m = many_plan(M, rows, w->k, out_dtype == LB_F32, linear4_sm_count());
    plan[0] = m.walk ? 2 : 1;
    plan[1] = m.tokens;
    plan[2] = m.splits;
    plan[3] = (M + m.tokens - 1) / m.tokens * ((rows + 127) / 128);
    return LB_OK;
}

extern "C" int64_t lb_linear4_scratch(const lb_weights4* w, int a_dtype, const void* a, int64_t lda, int M) {
    if (M <= 0 || weights4_check(w, "linear4_scratch") != LB_OK) return 0;      // (the product refuses such weights)
    const int rows = w->paired ? 2 * ((w->n / 2 + 7) / 8 * 8) : w->n;
    return few_plan(M, rows, w->k, w->group, linear4_sm_count()).warps > 0 ? 0 : many_scratch_bytes(w, a_dtype, a, lda, M);
}

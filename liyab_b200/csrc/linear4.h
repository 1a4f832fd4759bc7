// What the kernels behind lb_linear4 and lb_gated4 share on the host.
#pragma once

#include "weights4.cuh"

int linear4_sm_count();

// Whether a kernel can read these weights: memory, alignment, sizes (every entry point that is given weights asks first).
int weights4_check(const lb_weights4* w, const char* what);

// Whether the device with this number, less 1, is the current one (0: anyone): kernels run there.
int device_check(const char* what, int device);

// How few_tokens cuts a product: warps a block, blocks a cluster (along k), clusters, row tiles a round, bytes of shared memory.
// warps 0: it does not take it.
struct FewPlan {
    int warps, splits, clusters, round, smem;
};
FewPlan few_plan(int M, int rows, int k, int group, int n_sm);
int few_tokens(const lb_weights4* w, int a_dtype, const void* a, int64_t lda, const lb_w4::Epilogue& e, const FewPlan& p, cudaStream_t stream);

// How many_tokens cuts one: whether a block an SM walks the tiles, tokens a tile, blocks a cluster (along k), stages, columns of tensor memory for the sums and in all, bytes of shared memory; k tiles a
// chain of the accumulator's additions, chains of a block, columns between accumulators, whether the chains take turns between two; warps that make weights.
struct ManyPlan {
    int walk, tokens, splits, stages, d_columns, tmem_columns, smem, chain, chains, chain_columns, turn, makers;
};
ManyPlan many_plan(int M, int rows, int k, bool out_f32, int n_sm);
// Activations that TMA does not take as they are (e4m3, rows off the 16 bytes) go through scratch memory.
int64_t many_scratch_bytes(const lb_weights4* w, int a_dtype, const void* a, int64_t lda, int M);
int many_tokens(const lb_weights4* w, int a_dtype, const void* a, int64_t lda, const lb_w4::Epilogue& e, void* scratch, cudaStream_t stream);

// What the kernels behind lb_attention4 share.
#pragma once

#include "cache4.cuh"

#include <atomic>

namespace lb_a4 {

// A call, checked (host) and as the kernels get it.
struct Call {
    lb_c4::Pages pages;
    const __nv_bfloat16* q;
    const int32_t* q_start;
    const int32_t* last;
    const int32_t* table;
    __nv_bfloat16* out;
    const float* distance;
    const float* sink;
    float* scores;                  // [request][key/value head][row][score_keys]: scores (base 2) for the keys' weights, or null
    float* log_sums;                // [request][key/value head][row]: base-2 logarithm of the softmax's divisor, or null
    float* partial;                 // states of runs: [launch row][warp + unit][row][reference, sum, values]
    int* starts;                    // [launch row][request + 1]: where a request's tiles start in the row's order
    int64_t q_stride, out_stride;
    int table_stride, n_seq, n_tokens, n_head, per, max_rows, score_keys, max_keys, window;
    float scale, soft_cap;
    int withhold;                   // a test's launch, in which what the kernels wait for does not come
};

// The tokens of request s, [first, first + count), and the place of its first: decode calls have a token a request.
struct Portion {
    int first, count, place;
};
__device__ __forceinline__ Portion portion_of(const Call& c, int s) {
    Portion p;
    if (c.q_start == nullptr) {
        p.first = s;
        p.count = 1;
    } else {
        p.first = max(c.q_start[s], 0);
        p.count = min(min(c.q_start[s + 1], c.n_tokens) - p.first, c.max_rows / c.per);       // no more than the call names
    }
    p.place = c.last[s];
    return p;
}

// Rows of weights in memory: [n][heads][width] floats, `row` and `head` from one to the next (host).
struct WeightRows {
    const float* at;
    int64_t row, head, n, heads, width;
};
// Whether no two of the rows overlap: one of the strides has the rows of the other between two of its own.
bool rows_apart(const WeightRows& a);
// Whether no number is in both.  (Rows of the same strides may lie between each other's; of other strides they do not share a stretch of memory.)
bool rows_disjoint(const WeightRows& a, const WeightRows& b);

// Lets a kernel have this much dynamic shared memory: asked once a device (a question costs as much as half a launch).
template <typename Kernel>
int allow_shared(Kernel kernel, int bytes, std::atomic<uint64_t>& asked) {
    int device = 0;
    LB_CHECK_CUDA(cudaGetDevice(&device));
    const uint64_t bit = device < 64 ? (uint64_t)1 << device : 0;
    if ((asked.load(std::memory_order_relaxed) & bit) != 0) return LB_OK;
    LB_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    asked.fetch_or(bit, std::memory_order_relaxed);
    return LB_OK;
}

// How the kernel for few rows cuts a call: rows a tile (4 or 8), row tiles a request and key/value head, requests a launch row, blocks of a row, warps that join a row's
// states, bytes of the states and of the requests' starts.
struct RowsPlan {
    int rows, tiles, per_row, blocks, join_team;
    bool fits;                      // whether it can run at all
    bool whole;                     // a block for each request's row tiles and key/value heads
    double us;                      // about how long it takes
    int64_t states, starts;
};
RowsPlan rows_plan(int n_seq, int n_kv_head, int max_rows, int max_keys, int head_dim, int n_sm);
// Portions of many rows, on tcgen05: blocks that may share a row tile's keys, tiles of 128 keys each has at most, bytes of their states, about how long it takes.
struct TilesPlan {
    int splits, share;
    int64_t states;
    double us;
};
TilesPlan tiles_plan(int n_seq, int n_kv_head, int per, int max_rows, int max_keys, int window, int head_dim, int n_sm);
int many_rows(const Call& c, int head_dim, const TilesPlan& p, cudaStream_t stream);
int few_rows(const Call& c, int head_dim, const RowsPlan& p, cudaStream_t stream);

}  // namespace lb_a4

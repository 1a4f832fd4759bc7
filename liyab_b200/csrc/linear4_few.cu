// Products with 4-bit weights for few tokens: out = act(a w^T + bias) + residual, and gate(a w_gate^T) * (a w_up^T) over paired rows.
//
// The weights are the rows of mma.sync (16 of them by 16 k), the tokens, eight at most, its columns.  A block owns a stretch of row tiles; its activations
// lie in shared memory in the order of the operand.  Row tiles by k tiles of 128 are one sequence that the block's warps cut into equal parts, whatever
// the two sizes are: a warp streams its part (a kilobyte a k tile, 16 bytes a lane twice, three or four tiles on the way), makes a register of two weights of a shift, a mask and a
// subtraction, and a group's sum of the integers, which meets its scale in 32 bits, and leaves the sum of every row tile that it touched in a slot of shared memory.
// After one barrier the slots of a row tile (neighbouring warps) are added in order.  The blocks of a cluster share a long reduction and read one another's sums, in order.
// Between two bounds: the weights' bytes (4 x 50257 x 1600 6.5 us of 11.5; 8 x 4096 x 16384 5.4 of 14.8) and the instructions that make operands of nibbles (165 a warp and k tile of 16 x 128 weights, 180 with
// the ends, at 2.2 and 1.6 a cycle and SM; a form with a fifth fewer took the same time), with some 4 us of launch, first weights and barrier (1 x 1600 x 1600 3.0 us).  With the products and the unpacking left out
// 1 x 40960 x 8192 takes 27 us, with them 34.  More than eight tokens
// would cost a second product and its sums for every operand; the tensor core of linear4_many.cu is then faster (16 x 4096 x 4096 6.6 us there, 7.6 here; 8 x 8192 x 8192 16.3 there, 12.1 here).
#include "linear4.h"
#include "tcgen05.cuh"

namespace {

using namespace lb_w4;
using lb_tc::smem_u32;

constexpr int kMostWarps = 16, kTwoWarps = 12;     // of a block alone on its SM, of one of two
constexpr int kTwoFrom = 12;             // row tiles an SM from which two blocks share it
constexpr int kRound = 32;               // row tiles between two barriers
constexpr int kTokens = 8;
constexpr int kSlot = 16 * kTokens;      // a row tile's sums

__device__ __forceinline__ uint4 load_weights(const uint4* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// The scales of a row's k tile (1, 2 or 4 of them) in the low bytes.
template <int GROUP>
__device__ __forceinline__ uint32_t load_scales(const uint8_t* p) {
    if constexpr (GROUP == 128) return __ldg(p);
    else if constexpr (GROUP == 64) return __ldg(reinterpret_cast<const uint16_t*>(p));
    else return __ldg(reinterpret_cast<const uint32_t*>(p));
}

__device__ __forceinline__ float load_remote(uint32_t local, uint32_t rank) {
    float v;
    asm volatile("{\n\t.reg .u32 r;\n\tmapa.shared::cluster.u32 r, %1, %2;\n\tld.shared::cluster.f32 %0, [r];\n\t}" : "=f"(v) : "r"(local), "r"(rank) : "memory");
    return v;
}
__device__ __forceinline__ int load_remote_int(uint32_t local, uint32_t rank) { return __float_as_int(load_remote(local, rank)); }

// Shared memory: activations [k tile][token][j ^ (token & 1)][t] of 16 bytes (the exclusive or keeps eight lanes' reads off one another's banks) behind a line of zeros
// for the columns without a token; the slots [slot][16][8].
struct Layout {
    int rows_at, slots_at, total;
    __host__ __device__ Layout(int M, int n_kt, int tiles, int warps) {
        rows_at = 256;
        slots_at = rows_at + n_kt * M * 256;
        total = slots_at + 4 * kSlot * (tiles + warps);
    }
};

// SPLIT: the cluster's blocks share the reduction.  TWO: two blocks an SM with fewer registers each, so that one's sums and results hide under the other's products; for many row
// tiles, whose ends cost what the shorter way ahead loses (4 x 50257 x 1600 12.3 -> 11.5 us, 1 x 32000 x 2048 9.3 -> 9.1, but 1 x 14336 x 4096 9.0 -> 9.2).
template <typename T, int GROUP, bool SPLIT, bool TWO>
__global__ void __launch_bounds__(32 * (TWO ? kTwoWarps : kMostWarps), TWO ? 2 : 1)
few_tokens_kernel(const lb_weights4 w, const void* __restrict__ a, int64_t lda, bool wide, const Epilogue e, int n_tiles, int k_tiles, int splits, int round_tiles) {
    constexpr int kPerTile = kTileK / GROUP, kScaleBytes = kTileRows * kPerTile, kAhead = TWO ? 3 : 4;      // (k tiles on the way a warp)
    extern __shared__ __align__(128) uint8_t shared[];
    __shared__ float factors[kRound * 16], biases[kRound * 16], a_scales[kTokens];                       // of the rows between two barriers, of the tokens
    __shared__ int parts_of[kRound][2];                                                               // the first and the last warp of a row tile
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, n_warps = blockDim.x >> 5;
    const int rank = SPLIT ? (int)blockIdx.x % splits : 0, cluster = SPLIT ? (int)blockIdx.x / splits : (int)blockIdx.x, clusters = SPLIT ? (int)gridDim.x / splits : (int)gridDim.x;
    const int per_rank = SPLIT ? (k_tiles + splits - 1) / splits : k_tiles, kt0 = rank * per_rank, n_kt = min(k_tiles, kt0 + per_rank) - kt0;   // the host leaves no rank without one
    const int first = (int)((int64_t)cluster * n_tiles / clusters), last = (int)((int64_t)(cluster + 1) * n_tiles / clusters);
    const Layout at_of(e.M, per_rank, round_tiles, n_warps);
    float* slots = reinterpret_cast<float*>(shared + at_of.slots_at);

    // This warp's part of a round: k tiles x0 .. x1 of the round's sequence, in memory one stretch, but for a rank of several, whose stretch of every row tile ends before
    // that of the next begins.
    int x0 = 0, x1 = 0, start = 0, kt = 0, left = 0;
    const uint4* from = nullptr;                 // of the tile that is computed next (SPLIT: of the one that is fetched next)
    const uint8_t* scales_from = nullptr;
    uint4 words[kAhead][2];
    uint32_t steps[kAhead][2];
    auto fetch = [&](int i, int at) {
        words[i][0] = load_weights(from + at * (kTileBytes / 16));
        words[i][1] = load_weights(from + at * (kTileBytes / 16) + kTileBytes / 32);
        steps[i][0] = load_scales<GROUP>(scales_from + at * kScaleBytes);
        steps[i][1] = load_scales<GROUP>(scales_from + at * kScaleBytes + 8 * kPerTile);
        if (SPLIT) {
            const int skip = --left == 0 ? k_tiles - n_kt + 1 : 1;
            if (left == 0) left = n_kt;
            from += (size_t)skip * (kTileBytes / 16);
            scales_from += (size_t)skip * kScaleBytes;
        }
    };
    auto begin_round = [&](int base) {
        const int length = min(round_tiles, last - base) * n_kt, parts = min(n_warps, length);        // no warp between two others is without a k tile
        x0 = warp < parts ? (int)((int64_t)warp * length / parts) : 0;
        x1 = warp < parts ? (int)((int64_t)(warp + 1) * length / parts) : 0;
        start = base + x0 / n_kt;
        kt = x0 % n_kt;
        left = n_kt - kt;
        const size_t tile0 = (size_t)start * k_tiles + kt0 + kt;
        from = static_cast<const uint4*>(w.nibbles) + tile0 * (kTileBytes / 16) + piece_at(g, t);
        scales_from = static_cast<const uint8_t*>(w.scales) + tile0 * kScaleBytes + g * kPerTile;
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (x0 + i < x1) fetch(i, SPLIT ? 0 : i);
    };
    if (first < last) begin_round(first);
    const Unpack<T> unpack;
    lb_wait_for_predecessor();
    lb_dependents_may_launch();
    if (threadIdx.x < 16) reinterpret_cast<uint4*>(shared)[threadIdx.x] = make_uint4(0u, 0u, 0u, 0u);
    // Pieces of eight k by four tokens, the four on their way together.
    const int pieces = n_kt * 16;
    for (int q = threadIdx.x; q < pieces * ((e.M + 3) / 4); q += blockDim.x) {
        const int m0 = q / pieces * 4, c = q - m0 / 4 * pieces, at = c & 3, j = c >> 2 & 3, k_tile = c >> 4;
        uint4* to = reinterpret_cast<uint4*>(shared + at_of.rows_at) + (k_tile * e.M + m0) * 16 + at;
        uint32_t v[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (m0 + i < e.M) {
                // (e4m3 becomes float16 when all four are there.)
                if constexpr (T::kHalf) load_eight_bytes(v[i][0], v[i][1], a, (int64_t)(m0 + i) * lda, (kt0 + k_tile) * kTileK + 32 * j + 8 * at, w.k, wide);
                else load_eight<false>(v[i], a, (int64_t)(m0 + i) * lda, (kt0 + k_tile) * kTileK + 32 * j + 8 * at, w.k, wide);
            }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (m0 + i < e.M) {
                uint4 eight;
                if constexpr (T::kHalf)
                    eight = make_uint4(e4m3x2_to_f16x2(v[i][0] & 0xffffu), e4m3x2_to_f16x2(v[i][0] >> 16), e4m3x2_to_f16x2(v[i][1] & 0xffffu), e4m3x2_to_f16x2(v[i][1] >> 16));
                else eight = make_uint4(v[i][0], v[i][1], v[i][2], v[i][3]);
                to[i * 16 + (j ^ (i & 1)) * 4] = eight;
            }
    }
    if (threadIdx.x < kTokens) a_scales[threadIdx.x] = e.a_scale != nullptr && (int)threadIdx.x < e.M ? e.a_scale[threadIdx.x] : 1.0f;

    // This lane's activations: of a token, or the line of zeros; words of even and of odd j lie `swap` bytes further and nearer.
    const bool there = g < e.M;
    const uint32_t columns = smem_u32(shared) + (there ? at_of.rows_at + g * 256 : 0) + 16 * t;
    const int column_step = there ? 256 * e.M : 0;
    const int swap = (g & 1) * 64;
    for (int base = first; base < last; base += round_tiles) {
        __syncthreads();                    // the activations are there; the last round's slots have been read
        const int tiles = min(round_tiles, last - base);
        // What the sums will meet is asked for now: the rows' factors and biases, and the residual of this thread's first unit (a token and the rows `row` and `row` + 8).
        const int unit0 = rank * (int)blockDim.x + (int)threadIdx.x, units = tiles * 8 * e.M;
        float add[2] = {0.0f, 0.0f};
        if (e.residual != nullptr && unit0 < units) {
            const int i = (unit0 >> 3) / e.M, token = (unit0 >> 3) - i * e.M, col = (base + i) * 16 + (unit0 & 7);
            if (col < e.n) add[0] = e.residual[(int64_t)token * e.ldr + col];
            if (col + 8 < e.n) add[1] = e.residual[(int64_t)token * e.ldr + col + 8];
        }
        for (int i = threadIdx.x; i < tiles * 16; i += blockDim.x) {
            factors[i] = w.rows[base * 16 + i];
            biases[i] = e.bias != nullptr && base * 16 + i < e.n ? __ldg(e.bias + base * 16 + i) : 0.0f;
        }
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        uint32_t column = columns + kt * column_step;
        const bool ends_tile = (x1 - x0 + kt) % n_kt == 0;                                            // whether this part ends where a row tile does
        int of = start - base;
        float* slot = slots + (of + warp) * kSlot;
        if (x0 < x1 && kt == 0) parts_of[of][0] = warp;
        // Counted from the group of kAhead k tiles that is at hand: those to be computed, those to be fetched, and where the row tile (or this warp's part) ends.
        int todo = x1 - x0, to_fetch = todo - kAhead, end = min(n_kt - kt, todo);
        while (todo > 0) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const uint4 top = words[i][0], low = words[i][1];
                const uint32_t st = steps[i][0], sl = steps[i][1];
                const uint32_t wt[4] = {top.x, top.y, top.z, top.w}, wl[4] = {low.x, low.y, low.z, low.w};
                float part[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint4 b;
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w) : "r"((j & 1 ? column - swap : column + swap) + 64 * j));
                    if ((j * 32) % GROUP == 0) part[0] = part[1] = part[2] = part[3] = 0.0f;
                    mma16816<T>(part, unpack(wt[j], 0), unpack(wl[j], 0), unpack(wt[j], 1), unpack(wl[j], 1), b.x, b.y);
                    mma16816<T>(part, unpack(wt[j], 2), unpack(wl[j], 2), unpack(wt[j], 3), unpack(wl[j], 3), b.z, b.w);
                    if ((j * 32 + 32) % GROUP == 0) {
                        const uint32_t both = e4m3x2_to_f16x2(__byte_perm(st, sl, 0x0040 + (j * 32 / GROUP) * 0x11));
                        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&both));
                        acc[0] = fmaf(part[0], f.x, acc[0]);
                        acc[1] = fmaf(part[1], f.x, acc[1]);
                        acc[2] = fmaf(part[2], f.y, acc[2]);
                        acc[3] = fmaf(part[3], f.y, acc[3]);
                    }
                }
                column += column_step;
                if (i < to_fetch) fetch(i, SPLIT ? 0 : i + kAhead);
                if (end == i + 1) {
                    *reinterpret_cast<float2*>(slot + g * kTokens + 2 * t) = make_float2(acc[0], acc[1]);
                    *reinterpret_cast<float2*>(slot + (g + 8) * kTokens + 2 * t) = make_float2(acc[2], acc[3]);
                    acc[0] = acc[1] = acc[2] = acc[3] = 0.0f;
                    column = columns;
                    slot += kSlot;
                    const bool last_tile = todo == i + 1;
                    if (!last_tile || ends_tile) parts_of[of][1] = warp;
                    if (last_tile) goto done;
                    parts_of[++of][0] = warp;
                    end = i + 1 + min(n_kt, todo - (i + 1));
                }
            }
            todo -= kAhead;
            to_fetch -= kAhead;
            end -= kAhead;
            if (!SPLIT) {
                from += kAhead * (kTileBytes / 16);
                scales_from += kAhead * kScaleBytes;
            }
        }
    done:
        if (base + round_tiles < last) begin_round(base + round_tiles);
        __syncthreads();

        if (SPLIT) {
            // Every row tile's sum into its first slot, where the other ranks read it.
            for (int u = threadIdx.x; u < tiles * kSlot; u += blockDim.x) {
                const int i = u / kSlot, at_slot = u % kSlot, lo = parts_of[i][0], hi = parts_of[i][1];
                float v = 0.0f;
                for (int q = lo; q <= hi; ++q) v += slots[(i + q) * kSlot + at_slot];
                slots[(i + lo) * kSlot + at_slot] = v;
            }
            __syncwarp();
            asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        }
        const lb_act_pair pair = w.paired ? lb_act_pair{0.0f, 0.0f} : lb_act_load(e.bias, e.n, e.act);
        for (int u = unit0; u < units; u += splits * (int)blockDim.x) {
            const int i = (u >> 3) / e.M, token = (u >> 3) - i * e.M, row = u & 7, tile = base + i;
            float factor[2] = {factors[i * 16 + row], factors[i * 16 + row + 8]};
            float v[2] = {0.0f, 0.0f};
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at_slot = (row + 8 * h) * kTokens + token;
                if (!SPLIT) {
                    const int hi = parts_of[i][1];
                    for (int q = parts_of[i][0]; q <= hi; ++q) v[h] += slots[(i + q) * kSlot + at_slot];
                } else {
                    for (int r = 0; r < splits; ++r) {
                        const int lo = load_remote_int(smem_u32(&parts_of[i][0]), r);
                        v[h] += load_remote(smem_u32(slots + (i + lo) * kSlot + at_slot), r);
                    }
                }
            }
            if constexpr (T::kHalf) {
                const float a_scale = a_scales[token];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float rest = split_factor(factor[h]);
                    v[h] *= factor[h];
                    factor[h] = rest * a_scale;
                }
            }
            if (w.paired) {
                const int col = tile * 8 + row;
                if (col < e.n) store_out(e, token, col, gated_pair(v[0] * factor[0], v[1] * factor[1], e.gate, e.alpha, e.limit));
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int col = tile * 16 + row + 8 * h;
                    if (col >= e.n) continue;
                    float y = activated(fmaf(v[h], factor[h], biases[i * 16 + row + 8 * h]), e.act, pair);
                    if (e.residual != nullptr) y += u == unit0 ? add[h] : e.residual[(int64_t)token * e.ldr + col];
                    store_out(e, token, col, y);
                }
            }
        }
        // No slot is written again, and no block leaves, while another may read these sums.
        if (SPLIT) {
            __syncwarp();                       // (lanes without a feature went past the others)
            asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
        }
    }
}

template <typename T, int GROUP>
int launch_group(const lb_weights4* w, const void* a, int64_t lda, bool wide, const Epilogue& e, const FewPlan& p, int n_tiles, int k_tiles, cudaStream_t s) {
    auto kernel = p.splits > 1 ? few_tokens_kernel<T, GROUP, true, false> : p.warps == kTwoWarps ? few_tokens_kernel<T, GROUP, false, true> : few_tokens_kernel<T, GROUP, false, false>;
    if (p.smem > 40 * 1024) LB_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 216 * 1024));
    LB_CHECK_CUDA(lb_launch_overlapped_cluster(0, p.splits, kernel, dim3(p.clusters * p.splits), dim3(32 * p.warps), p.smem, s, *w, a, lda, wide, e, n_tiles, k_tiles, p.splits,
                                               p.round));
    return LB_OK;
}

template <typename T>
int launch(const lb_weights4* w, const void* a, int64_t lda, const Epilogue& e, const FewPlan& p, int n_tiles, int k_tiles, cudaStream_t s) {
    const bool wide = lda % 8 == 0 && reinterpret_cast<uintptr_t>(a) % (T::kHalf ? 8 : 16) == 0;
    if (w->group == 32) return launch_group<T, 32>(w, a, lda, wide, e, p, n_tiles, k_tiles, s);
    if (w->group == 64) return launch_group<T, 64>(w, a, lda, wide, e, p, n_tiles, k_tiles, s);
    return launch_group<T, 128>(w, a, lda, wide, e, p, n_tiles, k_tiles, s);
}

}  // namespace

FewPlan few_plan(int M, int rows, int k, int group, int n_sm) {
    FewPlan p{};
    const int k_tiles = (k + kTileK - 1) / kTileK, n_tiles = (rows + kTileRows - 1) / kTileRows;
    if (M > kTokens) return p;
    if (n_tiles >= kTwoFrom * n_sm) {
        p.warps = kTwoWarps;
        p.splits = 1;
        p.clusters = 2 * n_sm;
        p.round = (n_tiles + p.clusters - 1) / p.clusters;
        if (p.round > kRound) p.round = kRound;
        p.smem = Layout(M, k_tiles, p.round, p.warps).total;
        if (p.smem <= 106 * 1024) return p;
        p.warps = 0;
    }
    for (p.splits = 1; p.splits <= 8; p.splits *= 2) {
        const int per_rank = (k_tiles + p.splits - 1) / p.splits;
        if (per_rank * (p.splits - 1) >= k_tiles) return p;
        p.clusters = n_tiles < n_sm / p.splits ? n_tiles : n_sm / p.splits;
        p.round = (n_tiles + p.clusters - 1) / p.clusters;
        if (p.round > kRound) p.round = kRound;
        const int length = p.round * per_rank, warps = length <= 96 ? 8 : 16;          // (1 x 12000 x 2048 6.1 and 6.5 us, gated 1 x 10240 x 4096 14.3 and 12.1)
        p.smem = Layout(M, per_rank, p.round, warps).total;
        if (p.smem <= 216 * 1024) {
            p.warps = warps;
            return p;
        }
    }
    return p;
}

int few_tokens(const lb_weights4* w, int a_dtype, const void* a, int64_t lda, const Epilogue& e, const FewPlan& p, cudaStream_t stream) {
    const int k_tiles = (w->k + kTileK - 1) / kTileK, rows = w->paired ? 2 * ((e.n + 7) / 8 * 8) : e.n, n_tiles = (rows + kTileRows - 1) / kTileRows;
    return a_dtype == LB_E4M3 ? launch<F16>(w, a, lda, e, p, n_tiles, k_tiles, stream) : launch<Bf16>(w, a, lda, e, p, n_tiles, k_tiles, stream);
}

// Products with 4-bit weights for more tokens than linear4_few.cu takes: out = act(a w^T + bias) + residual, and gate(a w_gate^T) * (a w_up^T) over paired rows.
//
// 128 rows of weights are the lanes of the accumulator, up to 256 tokens its columns.  The weights never pass through shared memory: a thread owns a row, makes
// q s of its nibbles in registers (a shift, a mask and one fused multiply-add for two: (16 + u) s - 24 s with u = q + 8, exact) and stores them into tensor memory, where
// tcgen05.mma reads its first operand; the activations come by TMA.  So the copies through shared memory are those of the tokens alone, and a k tile
// of 128 x 128 weights costs 860 instructions of a warp beside eight products, which take 512 cycles with 256 tokens.
// Where a product has too few tiles for the GPU the reduction is cut between the blocks of a cluster, which hand each other the sums of their share of the tokens through
// distributed shared memory and finish them in rank order.
//
// Roles: warp 0 copies the activations, warp 1 issues the products, warps 4 to 11 make weights (warp % 4 names the 32 lanes; the two warps of those take alternate k
// tiles) and finish the sums.  Handshakes and bounded waits as in the other tcgen05 products.
#include "gemm_tile.cuh"
#include "linear4.h"

namespace {

using namespace lb_tc;
using namespace lb_tile;
using namespace lb_w4;

constexpr int kMakers = 8, kFirstMaker = 4, kThreads = 32 * (kFirstMaker + kMakers), kGroups = kMakers / 4;
constexpr int kMaxStages = 6, kStageColumns = kTileK / 2;
constexpr int kLaneRows = 128;

struct Control {
    uint64_t a_full[kMaxStages];      // weights in tensor memory
    uint64_t b_full[kMaxStages];      // activations in shared memory
    uint64_t empty[kMaxStages];
    uint64_t acc_ready;
    uint32_t tmem_base;
    int abort_flag;
};

__device__ __forceinline__ void give_up(Control* c, int* status, int site, int detail) {
    atomicCAS(status, 0, (0xB << 12) | (site << 8) | (detail & 0xff));
    *(volatile int*)&c->abort_flag = 1;
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
                 "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// The product with its first operand in tensor memory (lane = row, two values of K to a column).
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint32_t b_lo, uint32_t desc_hi, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
        "mov.b64 db, {%2, %3};\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "r"(b_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate) : "memory");
}

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "r"(taddr) : "memory");
}

// Weights 2p and 2p + 1 of a word times their scale.  bfloat16: u in bits 3 to 6 under the exponent of 16 is 16 + u; float16: in bits 4 to 7 under that of 64 it is 64 + u.
template <typename T>
__device__ __forceinline__ uint32_t scaled_pair(uint32_t word, int p, uint32_t mask, uint32_t magic, uint32_t s, uint32_t minus) {
    constexpr int kAt = T::kHalf ? 4 : 3;
    const uint32_t v = masked_or(4 * p < kAt ? word << (kAt - 4 * p) : word >> (4 * p - kAt), mask, magic);
    uint32_t out;
    if constexpr (T::kHalf) asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(out) : "r"(v), "r"(s), "r"(minus));
    else asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(out) : "r"(v), "r"(s), "r"(minus));
    return out;
}

// An e4m3 scale in both halves of a register, and -24 (bfloat16) or -72 (float16) times it; both are exact.
template <typename T>
__device__ __forceinline__ void scale_pair(uint32_t byte, uint32_t& s, uint32_t& minus) {
    const uint32_t h = e4m3x2_to_f16x2(__byte_perm(byte, 0, 0x0000));
    if constexpr (T::kHalf) {
        s = h;
        const __half2 m = __hmul2(*reinterpret_cast<const __half2*>(&h), __float2half2_rn(-72.0f));
        minus = *reinterpret_cast<const uint32_t*>(&m);
    } else {
        const float f = __low2float(*reinterpret_cast<const __half2*>(&h));
        s = pack2(f, f);
        minus = pack2(-24.0f * f, -24.0f * f);
    }
}

template <int GROUP>
__device__ __forceinline__ uint32_t load_scales(const uint8_t* p) {
    if constexpr (GROUP == 128) return __ldg(p);
    else if constexpr (GROUP == 64) return __ldg(reinterpret_cast<const uint16_t*>(p));
    else return __ldg(reinterpret_cast<const uint32_t*>(p));
}

// gridDim.x = blocks of 128 rows x splits (a cluster), gridDim.y = tiles of `tokens` tokens (a multiple of 16).
template <typename T, int GROUP>
__global__ void __launch_bounds__(kThreads)
many_tokens_kernel(const __grid_constant__ CUtensorMap map_a, const lb_weights4 w, const Epilogue e, int k_tiles, int tokens, int splits, int n_stages, int d_columns,
                   int tmem_columns, int withhold, int* status) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const uint32_t atom_bytes = (uint32_t)tokens * 128u, stage_bytes = 2 * atom_bytes;
    Control* c = reinterpret_cast<Control*>(base + max((uint32_t)n_stages * stage_bytes, splits > 1 ? (uint32_t)tokens * 512u : 0u));
    float* inbox = reinterpret_cast<float*>(base);                     // [rank][share's tokens][128 rows], over the stages when their products are done
    volatile int* abort_flag = &c->abort_flag;
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rank = (int)blockIdx.x % splits, row0 = (int)blockIdx.x / splits * kLaneRows, m0 = (int)blockIdx.y * tokens;
    const int per = (k_tiles + splits - 1) / splits, kt0 = rank * per, n_kt = min(k_tiles, kt0 + per) - kt0;     // the host leaves no rank without one

    if (threadIdx.x == 0) {
        prefetch_tensormap(&map_a);
        for (int i = 0; i < n_stages; ++i) {
            mbar_init(&c->a_full[i], 4);
            mbar_init(&c->b_full[i], 1);
            mbar_init(&c->empty[i], 1);
        }
        mbar_init(&c->acc_ready, 1);
        c->abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        tmem_alloc(&c->tmem_base, tmem_columns);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, c->tmem_base, 0), tmem_a = tmem_base + d_columns;
    const uint32_t stages_u32 = smem_u32(base), a_full = smem_u32(&c->a_full[0]), b_full = smem_u32(&c->b_full[0]), empty = smem_u32(&c->empty[0]);
    const int quarter = warp & 3, group = (warp - kFirstMaker) >> 2, row = quarter * 32 + lane;
    bool ok = true;

    if (warp == 0) {
        lb_wait_for_predecessor();
        lb_dependents_may_launch();
        int issued = 0, st = 0;
        uint32_t parity = 1;                                           // a stage's first use waits for nothing
        for (int kt = 0; kt < n_kt; ++kt) {
            if (!__all_sync(0xffffffffu, wait_u32(empty + 8 * st, parity, abort_flag))) {
                give_up(c, status, 1, st);
                break;
            }
            if (elect_one()) {
                expect_tx_u32(b_full + 8 * st, stage_bytes);
                tma_load_u32(stages_u32 + st * stage_bytes, &map_a, b_full + 8 * st, (kt0 + kt) * kTileK, m0);
                tma_load_u32(stages_u32 + st * stage_bytes + atom_bytes, &map_a, b_full + 8 * st, (kt0 + kt) * kTileK + kBlockK, m0);
            }
            issued = kt + 1;
            if (++st == n_stages) {
                st = 0;
                parity ^= 1;
            }
        }
        // Leave no copy in flight: the barriers of the last loads complete when their bytes landed.
        if (*abort_flag != 0)
            for (int kt = max(0, issued - n_stages); kt < issued; ++kt) mbar_wait(&c->b_full[kt % n_stages], (kt / n_stages) & 1, nullptr);
    } else if (warp == 1) {
        const uint32_t columns = (uint32_t)min(tokens, (e.M - m0 + 15) / 16 * 16);
        const uint32_t idesc = T::kHalf ? umma_idesc(kLaneRows, (int)columns) & ~((1u << 7) | (1u << 10)) : umma_idesc(kLaneRows, (int)columns);
        const uint32_t desc_hi = (uint32_t)(1024 >> 4) | (1u << 14) | (2u << 29);
        const uint32_t lo0 = ((stages_u32 & 0x3FFFFu) >> 4) | (1u << 16);
        int st = 0;
        uint32_t parity = 0;
        for (int kt = 0; kt < n_kt; ++kt) {
            if (!__all_sync(0xffffffffu, wait_u32(b_full + 8 * st, parity, abort_flag) && wait_u32(a_full + 8 * st, parity, abort_flag))) {
                give_up(c, status, 2, st);
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t b_lo = lo0 + (uint32_t)st * (stage_bytes >> 4), ta = tmem_a + st * kStageColumns;
            if (elect_one()) {
#pragma unroll
                for (uint32_t k = 0; k < kTileK / kUmmaK; ++k)
                    umma_ts(tmem_base, ta + k * (kUmmaK / 2), b_lo + (k >> 2) * (atom_bytes >> 4) + 2 * (k & 3), desc_hi, idesc, kt + k != 0 ? 1u : 0u);
                commit_u32(empty + 8 * st);
            }
            if (++st == n_stages) {
                st = 0;
                parity ^= 1;
            }
        }
        // (`withhold`: a test's launch, whose epilogues find nothing and give up.)
        if (ok && withhold == 0 && elect_one()) umma_commit(&c->acc_ready);
        lb_wait_for_predecessor();
        lb_dependents_may_launch();
    } else if (warp >= kFirstMaker) {
        constexpr int kPerTile = kTileK / GROUP;
        const size_t tile0 = (size_t)((row0 + row) >> 4) * k_tiles + kt0;
        const uint4* from = static_cast<const uint4*>(w.nibbles) + tile0 * (kTileBytes / 16) + (row & 15);
        const uint8_t* scales = static_cast<const uint8_t*>(w.scales) + (tile0 * kTileRows + (row & 15)) * kPerTile;
        uint32_t mask, magic;
        asm volatile("mov.b32 %0, %2;\n\tmov.b32 %1, %3;" : "=r"(mask), "=r"(magic) : "n"(T::kHalf ? 0x00F000F0 : 0x00780078), "n"(T::kHalf ? 0x54005400 : 0x41804180));
        uint4 words[2][4];
        uint32_t steps[2];
        auto fetch = [&](int i, int kt) {
            if (kt < n_kt) {
#pragma unroll
                for (int t = 0; t < 4; ++t) words[i][t] = __ldg(from + kt * (kTileBytes / 16) + 16 * t);
                steps[i] = load_scales<GROUP>(scales + kt * kTileRows * kPerTile);
            }
        };
        fetch(0, group);
        fetch(1, group + kGroups);
        int st = group % n_stages;
        uint32_t parity = (group / n_stages & 1) ^ 1;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        for (int kt = group, i = 0; kt < n_kt; kt += kGroups, i ^= 1) {
            if (!__all_sync(0xffffffffu, wait_u32(empty + 8 * st, parity, abort_flag))) {
                give_up(c, status, 4, st);
                ok = false;
                break;
            }
            tc_fence_after();
            auto make = [&](int i) {
                uint32_t s = 0, minus = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (j * 32 % GROUP == 0) scale_pair<T>(steps[i] >> (8 * (j * 32 / GROUP)), s, minus);
                    uint32_t v[16];
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const uint32_t word = j == 0 ? words[i][t].x : j == 1 ? words[i][t].y : j == 2 ? words[i][t].z : words[i][t].w;
#pragma unroll
                        for (int p = 0; p < 4; ++p) v[4 * t + p] = scaled_pair<T>(word, p, mask, magic, s, minus);
                    }
                    tmem_st16(tmem_a + lanes + st * kStageColumns + 16 * j, v);
                }
                fetch(i, kt + 2 * kGroups);
            };
            if (i == 0) make(0);
            else make(1);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&c->a_full[st]);
            st += kGroups;
            if (st >= n_stages) {
                st -= n_stages;
                parity ^= 1;
            }
        }
        lb_wait_for_predecessor();           // before scales and residuals are read and anything is written
        lb_dependents_may_launch();
        ok = __all_sync(0xffffffffu, ok && mbar_wait(&c->acc_ready, 0, abort_flag));
        if (!ok) give_up(c, status, 3, quarter);
        tc_fence_after();
    }
    __syncwarp();
    // A row's factor; of paired rows lanes 8 apart hold a feature's two sums, and each of them finishes one of two tokens.
    const bool finishes = warp >= kFirstMaker && ok;
    const float factor = finishes ? w.rows[row0 + row] : 0.0f;
    const lb_act_pair pair = finishes && !w.paired ? lb_act_load(e.bias, e.n, e.act) : lb_act_pair{0.0f, 0.0f};
    const int up = lane >> 3 & 1, col = w.paired ? (row0 + row) / 16 * 8 + (row & 7) : row0 + row;
    auto finish_eight = [&](const float (&y)[8], int token) {
        if (w.paired) {
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float v0 = y[i] * factor, v1 = y[i + 1] * factor, other = __shfl_xor_sync(0xffffffffu, up ? v0 : v1, 8);
                const int m = token + i + up;
                if (m >= e.M || col >= e.n) continue;
                const float s = e.a_scale != nullptr ? e.a_scale[m] : 1.0f;
                store_out(e, m, col, lb_gated_pair((up ? other : v0) * s, (up ? v1 : other) * s, e.gate, e.alpha, e.limit));
            }
        } else if (col < e.n) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (token + i < e.M) finish_one(e, pair, token + i, col, y[i] * (factor * (e.a_scale != nullptr ? e.a_scale[token + i] : 1.0f)));
        }
    };
    const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16);
    const int here = min(tokens, e.M - m0);
    if (splits > 1) {
        // Every block's products are complete before their stages are written over.
        const int share = tokens / splits;
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (finishes) {
            for (int at = 8 * group; at < here; at += 8 * kGroups) {
                uint32_t v[8];
                tmem_ld8(t_row + at, v);
                const int to = at / share;
                uint32_t peer = peer_address(smem_u32(inbox + (size_t)(rank * share + at - to * share) * kLaneRows + row), (uint32_t)to);
#pragma unroll
                for (int i = 0; i < 8; ++i) asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(peer + i * kLaneRows * 4), "r"(v[i]) : "memory");
            }
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (finishes) {
            for (int at = 8 * group; at < share && rank * share + at < here; at += 8 * kGroups) {
                float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                for (int r = 0; r < splits; ++r)
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] += inbox[(size_t)(r * share + at + i) * kLaneRows + row];
                finish_eight(y, m0 + rank * share + at);
            }
        }
    } else if (finishes) {
        for (int at = 8 * group; at < here; at += 8 * kGroups) {
            uint32_t v[8];
            tmem_ld8(t_row + at, v);
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = __uint_as_float(v[i]);
            finish_eight(y, m0 + at);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, tmem_columns);
    }
}

// Activations as the copies need them: rows a multiple of 16 bytes apart; e4m3 as float16.
template <typename T>
__global__ void spread_rows_kernel(const void* __restrict__ a, int64_t lda, bool wide, uint4* __restrict__ to, int eights, int64_t all, int K) {
    lb_wait_for_predecessor();
    lb_dependents_may_launch();
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < all; i += (int64_t)gridDim.x * blockDim.x) {
        const int64_t m = i / eights;
        const int k = (int)(i - m * eights) * 8;
        uint32_t v[4];
        load_eight<T>(v, a, m * lda, k, K, wide);
        to[i] = make_uint4(v[0], v[1], v[2], v[3]);
    }
}

int g_withhold_next = 0;      // the next launch's blocks leave their accumulator-ready barriers unsignalled (tests)

template <typename T, int GROUP>
int launch(const CUtensorMap& map, const lb_weights4* w, const Epilogue& e, const ManyPlan& p, int row_blocks, int token_tiles, int k_tiles, cudaStream_t s) {
    static bool configured = false;
    if (!configured) {
        LB_CHECK_CUDA(cudaFuncSetAttribute(many_tokens_kernel<T, GROUP>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
        configured = true;
    }
    int* status = nullptr;
    if (int rc = lb_tc_status_word(&status)) return rc;
    LB_CHECK_CUDA(lb_launch_overlapped_cluster(1, p.splits, many_tokens_kernel<T, GROUP>, dim3(row_blocks * p.splits, token_tiles), dim3(kThreads), p.smem, s, map, *w, e,
                                               k_tiles, p.tokens, p.splits, p.stages, p.d_columns, p.tmem_columns, g_withhold_next, status));
    g_withhold_next = 0;
    return LB_OK;
}

template <typename T>
int run(const lb_weights4* w, const void* a, int64_t lda, const Epilogue& e, void* scratch, cudaStream_t s) {
    const int k_tiles = (w->k + kTileK - 1) / kTileK, rows = w->paired ? 2 * ((e.n + 7) / 8 * 8) : e.n, row_blocks = (rows + kLaneRows - 1) / kLaneRows;
    if (many_scratch_bytes(w, T::kHalf ? LB_E4M3 : LB_BF16, a, lda, e.M) > 0) {
        LB_CHECK_ARG(scratch != nullptr && reinterpret_cast<uintptr_t>(scratch) % 16 == 0, "linear4: these activations need scratch memory (lb_linear4_scratch)");
        const bool wide = lda % 8 == 0 && reinterpret_cast<uintptr_t>(a) % (T::kHalf ? 8 : 16) == 0;
        const int eights = (w->k + 7) / 8;
        const int64_t all = (int64_t)e.M * eights, blocks = (all + 255) / 256;
        LB_CHECK_CUDA(lb_launch_overlapped(spread_rows_kernel<T>, dim3((unsigned)(blocks < 2368 ? blocks : 2368)), dim3(256), 0, s, a, lda, wide,
                                           static_cast<uint4*>(scratch), eights, all, w->k));
        a = scratch;
        lda = 8 * (int64_t)eights;
    }
    const ManyPlan p = many_plan(e.M, rows, w->k, linear4_sm_count());
    CUtensorMap map;
    if (int rc = lb_tensor_map_2d_encode(&map, a, 2, e.M, w->k, lda, p.tokens)) return rc;
    const int token_tiles = (e.M + p.tokens - 1) / p.tokens;
    if (w->group == 32) return launch<T, 32>(map, w, e, p, row_blocks, token_tiles, k_tiles, s);
    if (w->group == 64) return launch<T, 64>(map, w, e, p, row_blocks, token_tiles, k_tiles, s);
    return launch<T, 128>(map, w, e, p, row_blocks, token_tiles, k_tiles, s);
}

}  // namespace

ManyPlan many_plan(int M, int rows, int k, int n_sm) {
    ManyPlan p{};
    const int k_tiles = (k + kTileK - 1) / kTileK, row_blocks = (rows + kLaneRows - 1) / kLaneRows, tiles = (M + 255) / 256;
    p.tokens = ((M + tiles - 1) / tiles + 15) / 16 * 16;
    p.splits = 1;
    while (p.splits < 8 && tiles * row_blocks * p.splits * 2 <= n_sm && k_tiles >= 4 * p.splits && (k_tiles + 2 * p.splits - 1) / (2 * p.splits) * (2 * p.splits - 1) < k_tiles)
        p.splits *= 2;
    // The tokens are shared out in eights between the ranks.
    if (p.splits > 1) p.tokens = (p.tokens + 8 * p.splits - 1) / (8 * p.splits) * (8 * p.splits);
    if (p.tokens > 256) p.tokens = 256;
    p.d_columns = p.tokens <= 64 ? 64 : p.tokens <= 128 ? 128 : 256;
    p.stages = p.d_columns == 128 ? 6 : 3;
    p.tmem_columns = p.d_columns == 64 ? 256 : 512;
    // The blocks of a cluster wait for one another while each holds its columns: as large a share of the shared memory as of the columns (see gemm_tcgen05_narrow.cu).
    const int needed = 1024 + p.stages * p.tokens * 256 + (p.splits > 1 && p.tokens * 512 > p.stages * p.tokens * 256 ? p.tokens * 512 - p.stages * p.tokens * 256 : 0) + (int)sizeof(Control);
    const int least = p.tmem_columns * (228 * 1024 / 512) - 1024;
    p.smem = needed < least ? least : needed;
    return p;
}

int64_t many_scratch_bytes(const lb_weights4* w, int a_dtype, const void* a, int64_t lda, int M) {
    if (a_dtype == LB_BF16 && lda % 8 == 0 && reinterpret_cast<uintptr_t>(a) % 16 == 0) return 0;
    return (int64_t)M * ((w->k + 7) / 8) * 16;
}

int many_tokens(const lb_weights4* w, int a_dtype, const void* a, int64_t lda, const Epilogue& e, void* scratch, cudaStream_t stream) {
    return a_dtype == LB_E4M3 ? run<F16>(w, a, lda, e, scratch, stream) : run<Bf16>(w, a, lda, e, scratch, stream);
}

// Tests: the next launch's sums are never announced.
extern "C" int lb_linear4_withhold_next(int on) {
    g_withhold_next = on;
    return LB_OK;
}

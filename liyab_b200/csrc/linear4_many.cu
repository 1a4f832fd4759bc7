// Products with 4-bit weights for more tokens than linear4_few.cu takes: out = act(a w^T + bias) + residual, and gate(a w_gate^T) * (a w_up^T) over paired rows.
//
// 128 rows of weights are the lanes of the accumulator, up to 256 tokens its columns.  The weights never pass through shared memory: a thread owns a row, makes
// q s of its nibbles in registers (a shift, a mask and one fused multiply-add for two: (16 + u) s - 24 s with u = q + 8, exact) and stores them into tensor memory, where
// tcgen05.mma reads its first operand; the activations come by TMA.  So the copies through shared memory are those of the tokens alone, and a k tile
// of 128 x 128 weights costs some 900 instructions of a warp beside eight products, which take 1,024 cycles with 256 tokens.
// Where a product has more tiles than the GPU has SMs, a block of each SM walks them and warps of their own finish a tile's sums under the next tile's products (the
// accumulator is free again when the last columns are in registers).  Where it has fewer, sixteen warps make weights and finish; the reduction is cut between the blocks of a
// cluster, which hand each other the sums of their share of the tokens through distributed shared memory and finish them in rank order.
//
// float32 results over more than 1,536 values of k are added up in several chains (many_plan says why): in accumulators of their own where tensor memory has the columns, else in two in turn, whose sums
// warps of their own add up in shared memory under the next chain's products.  Their tiles have 160 tokens at most, which cost more weights to make a product: 2048 x 8192 x 8192 218 us with float32 results,
// 186 with bfloat16 ones; 1024 x 4096 x 10240 84 and 62; up to some 300 tokens a few per cent.
//
// Roles: warp 0 copies the activations, warp 1 issues the products, warps 4 and up make weights (warp % 4 names the 32 lanes; the warps of those take k tiles in turn) and,
// in the same warps or in further ones, finish the sums.  Handshakes and bounded waits as in the other tcgen05 products:
//   a_full[s], b_full[s]   weights of stage s in tensor memory, activations in shared memory
//   empty[s]               the products have read both
//   acc_full, acc_empty    the sums of a tile, or of a chain, are complete, are in registers
#include "gemm_tile.cuh"
#include "linear4.h"

namespace {

using namespace lb_tc;
using namespace lb_tile;
using namespace lb_w4;

constexpr int kFirstMaker = 4;
constexpr int kMaxStages = 6, kStageColumns = kTileK / 2;
constexpr int kLaneRows = 128;
constexpr int kSpreadTokens = 32, kSpreadAhead = 4;      // e4m3 tokens that become float16 on their way: a tile's, k tiles of them in flight

struct Control {
    uint64_t a_full[kMaxStages];
    uint64_t b_full[kMaxStages];
    uint64_t empty[kMaxStages];
    uint64_t raw_full[kSpreadAhead], raw_empty[kSpreadAhead];
    uint64_t acc_full[2];
    uint64_t acc_empty[2];
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

// Asked for and waited for in one piece: until the wait nothing may touch the registers, and code between the two (calls above all) may move them.
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "r"(taddr) : "memory");
}

// A long wait that leaves the issue slots to others; bounded as mbar_wait is.
__device__ __forceinline__ bool wait_asleep(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    for (;;) {
        __nanosleep(200);
        if (mbar_try_wait(bar, parity)) return true;
        if (*abort_flag != 0 || clock64() - t0 > kWaitLimitCycles) return false;
    }
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

// The epilogue's activations on eight sums; results that are rounded to bfloat16 take the fast exponential and division (gemm_tile.cuh).  What is long stays out of line:
// the makers' loop and this code share the instruction cache.
// xIELU without a branch: the positive part feeds the square, the negative part exp(n) - 1 - n, which near 0 is the head of its series (the next term is below 5e-6 of it; the
// difference would keep nothing of numbers below 1e-7).
__device__ __forceinline__ float xielu_fast(float v, float a, float b) {
    const float pos = fmaxf(v, 0.0f), neg = fminf(v, 0.0f);
    const float series = neg * neg * fmaf(neg, fmaf(neg, 1.0f / 24.0f, 1.0f / 6.0f), 0.5f);
    return fmaf(a * pos, pos, fmaf(b, neg > -0.0625f ? series : __expf(neg) - 1.0f - neg, 0.5f * v));        // (a NaN comes through the last term)
}
__device__ __noinline__ float activate_long(float v, int act, bool exact, float a, float b) {
    if (exact) return activated(v, act, lb_act_pair{a, b});
    return xielu_fast(v, a, b);
}
__device__ __forceinline__ void activate_eight(float (&y)[8], int act, bool exact, const lb_act_pair& pair) {
    if (act == LB_ACT_RELU2) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = relu2(y[i]);
    } else if (act == LB_ACT_GELU_TANH && !exact) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = activate<LB_ACT_GELU_TANH, true>(y[i], pair);
    } else if (act == LB_ACT_GELU_ERF) {
        // (Out of line one by one 1776 x 12232 x 96 took 74 us, in fours 51, so 44.)
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = lb_gelu_erf(y[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = activate_long(y[i], act, exact, pair.a, pair.b);
    }
}
__device__ __noinline__ float gated_exact(float g, float u, int kind, float alpha, float limit) { return gated_pair(g, u, kind, alpha, limit); }
// gated_pair with the fast exponential and division (relative error about 1e-6), for results that are rounded to bfloat16; the gate is told apart once for four.
// An exponential that overflows makes 1 / infinity = 0 (what is below 2^-126 is 0), and a NaN stays one.
__device__ __forceinline__ float sigmoid_fast(float v) {
    float s;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.0f + __expf(-v)));
    return s;
}
__device__ __forceinline__ void gated_four(float (&z)[4], const float (&g)[4], const float (&u)[4], int kind, float alpha, float limit) {
    auto all = [&](auto f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) z[i] = f(g[i], u[i]);
    };
    if (kind == LB_GATE_SILU) all([](float x, float y) { return x * sigmoid_fast(x) * y; });
    else if (kind == LB_GATE_GELU_TANH) all([](float x, float y) { return x * sigmoid_fast(x * fmaf(0.07135481282553524f * x, x, 1.5957691216057308f)) * y; });
    else if (kind == LB_GATE_RELU) all([](float x, float y) { return at_least(x, 0.0f) * y; });
    else if (kind == LB_GATE_SIGMOID) all([](float x, float y) { return sigmoid_fast(x) * y; });
    else
        all([&](float x, float y) {
            x = at_most(x, limit);
            return x * sigmoid_fast(alpha * x) * (at_most(at_least(y, -limit), limit) + 1.0f);
        });
}

// What happens to the sums of a row (a lane) and eight tokens.  SCALED: the activations have a scale a row (and nothing waits for the row's factor before a sum meets it where they have not).  Of paired rows lanes 8 apart hold a feature's two sums, and each of them finishes one of two tokens.
template <bool SCALED>
struct RowEnd {
    int col, up;
    float factor, rest, bias;            // the row's factor: of moderate size, times a power of two (see split_factor)
    bool extreme;                        // some row of the warp's has one
    __device__ __forceinline__ RowEnd(const Epilogue& e, const lb_weights4& w, int row, int lane, bool used) {
        up = lane >> 3 & 1;
        col = w.paired ? row / 16 * 8 + (row & 7) : row;
        factor = used ? w.rows[row] : 0.0f;
        rest = 1.0f;
        extreme = false;
        if (SCALED) {
            rest = split_factor(factor);
            extreme = __any_sync(0xffffffffu, rest != 1.0f);
        }
        bias = used && e.bias != nullptr && col < e.n ? __ldg(e.bias + col) : 0.0f;
    }
    template <int COUNT, typename O>
    static __device__ __forceinline__ void put(O* o, int64_t step, const float (&y)[COUNT], int n) {
        if (n >= COUNT) {
#pragma unroll
            for (int i = 0; i < COUNT; ++i, o += step) *o = lb_from_float<O>(y[i]);
        } else {
#pragma unroll
            for (int i = 0; i < COUNT; ++i, o += step)
                if (i < n) *o = lb_from_float<O>(y[i]);
        }
    }
    __device__ __forceinline__ void finish(const Epilogue& e, bool paired, const lb_act_pair& pair, float (&y)[8], int token) const {
        const int n = e.M - token;               // at least one
        if (SCALED) {
            float s[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] = __ldg(e.a_scale + token + min(i, n - 1));
            if (extreme) {
#pragma unroll
                for (int i = 0; i < 8; ++i) s[i] *= rest;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = y[i] * factor * s[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] *= factor;
        }
        if (paired) {
            float g[4], u[4], z[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float other = __shfl_xor_sync(0xffffffffu, up ? y[2 * i] : y[2 * i + 1], 8);
                g[i] = up ? other : y[2 * i];
                u[i] = up ? y[2 * i + 1] : other;
            }
            if (!e.out_f32) {
                gated_four(z, g, u, e.gate, e.alpha, e.limit);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) z[i] = gated_exact(g[i], u[i], e.gate, e.alpha, e.limit);
            }
            if (col >= e.n) return;
            const int64_t at = (int64_t)(token + up) * e.ldo + col;
            const int rows = n >= 8 ? 4 : (n - up + 1) / 2;
            if (e.out_f32) put<4>(static_cast<float*>(e.out) + at, 2 * e.ldo, z, rows);
            else put<4>(static_cast<__nv_bfloat16*>(e.out) + at, 2 * e.ldo, z, rows);
            return;
        }
        if (col >= e.n) return;
        if (e.bias != nullptr) {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] += bias;
        }
        if (e.act != LB_ACT_NONE) activate_eight(y, e.act, e.out_f32, pair);
        if (e.residual != nullptr) {
            const float* r = e.residual + (int64_t)token * e.ldr + col;
            float add[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) add[i] = r[min(i, n - 1) * e.ldr];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] += add[i];
        }
        const int64_t at = (int64_t)token * e.ldo + col;
        if (e.out_f32) put<8>(static_cast<float*>(e.out) + at, e.ldo, y, n);
        else put<8>(static_cast<__nv_bfloat16*>(e.out) + at, e.ldo, y, n);
    }
};

// How the tiles lie: token tiles of a row block one after another.
struct Tiles {
    int tokens, token_tiles, total, k_tiles, splits, n_stages, d_columns;
    int spread;              // e4m3 rows become float16 on their way
    int chain, chain_columns;              // k tiles that one accumulator adds up; columns between accumulators
};

// Tokens of a tile that a rank of `splits` finishes, but for the last ones.
__host__ __device__ __forceinline__ int share_of(int tokens, int splits) { return ((tokens + splits - 1) / splits + 7) / 8 * 8; }

// WALK: a block walks the tiles blockIdx.x, blockIdx.x + gridDim.x, ..; else gridDim.x = tiles x splits, the splits of a tile a cluster.  FINISHERS: warps of their own that read the sums and
// finish; with none the makers do.  CHAINED: a tile's reduction is several chains of additions, which take turns between two accumulators (with finishing warps) or have one each.
template <typename T, int GROUP, int MAKERS, int FINISHERS, bool WALK, bool CHAINED>
__global__ void __launch_bounds__(32 * (kFirstMaker + MAKERS + FINISHERS))
many_tokens_kernel(const __grid_constant__ CUtensorMap map_a, const lb_weights4 w, const Epilogue e, const Tiles tiles, int tmem_columns, int withhold, int* status) {
    constexpr int kGroups = MAKERS / 4;
    constexpr int kTurn = CHAINED && FINISHERS > 0 ? 1 : 0;
    constexpr int kEnds = (FINISHERS > 0 ? FINISHERS : MAKERS) / 4;      // warps that share a quarter's sums
    constexpr bool kSpreads = T::kHalf && MAKERS == 8 && !WALK;        // where up to 32 e4m3 tokens may be a tile
    const bool spread = kSpreads && tiles.spread != 0;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int tokens = tiles.tokens, splits = WALK ? 1 : tiles.splits, n_stages = tiles.n_stages, k_tiles = tiles.k_tiles;
    const uint32_t atom_bytes = (uint32_t)tokens * 128u, stage_bytes = 2 * atom_bytes;
    Control* c = reinterpret_cast<Control*>(base + max((uint32_t)n_stages * stage_bytes, splits > 1 ? (uint32_t)(splits * share_of(tokens, splits)) * 512u : 0u));
    uint8_t* inbox = base;                                             // the ranks' sums, over the stages when their products are done
    volatile int* abort_flag = &c->abort_flag;
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rank = WALK ? 0 : (int)blockIdx.x % splits, first = WALK ? (int)blockIdx.x : (int)blockIdx.x / splits, stride = WALK ? (int)gridDim.x : tiles.total;
    const int per = (k_tiles + splits - 1) / splits, kt0 = rank * per, n_kt = min(k_tiles, kt0 + per) - kt0;     // the host leaves no rank without one
    const int chains = CHAINED ? (n_kt + tiles.chain - 1) / tiles.chain : 1;

    if (threadIdx.x == 0) {
        prefetch_tensormap(&map_a);
        for (int i = 0; i < n_stages; ++i) {
            mbar_init(&c->a_full[i], 4);
            mbar_init(&c->b_full[i], spread ? 2 : 1);
            mbar_init(&c->empty[i], 1);
        }
        if (spread)
            for (int i = 0; i < kSpreadAhead; ++i) {
                mbar_init(&c->raw_full[i], 1);
                mbar_init(&c->raw_empty[i], 2);
            }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&c->acc_full[i], 1);
            mbar_init(&c->acc_empty[i], FINISHERS > 0 ? FINISHERS : 1);
        }
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
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, c->tmem_base, 0), tmem_a = tmem_base + tiles.d_columns;
    const uint32_t stages_u32 = smem_u32(base), a_full = smem_u32(&c->a_full[0]), b_full = smem_u32(&c->b_full[0]), empty = smem_u32(&c->empty[0]);
    const int quarter = warp & 3, group = (warp - kFirstMaker) >> 2, row = quarter * 32 + lane;
    bool ok = true;

    const uint32_t raw_u32 = (smem_u32(c + 1) + 1023u) & ~1023u, raw_full = smem_u32(&c->raw_full[0]), raw_empty = smem_u32(&c->raw_empty[0]);
    if (warp == 0 && spread) {
        lb_wait_for_predecessor();
        lb_dependents_may_launch();
        int issued = 0;
        for (int kt = 0; kt < n_kt; ++kt, ++issued) {
            const int slot = kt & (kSpreadAhead - 1);
            if (!__all_sync(0xffffffffu, wait_u32(raw_empty + 8 * slot, (uint32_t)(kt / kSpreadAhead & 1) ^ 1u, abort_flag))) {
                give_up(c, status, 7, slot);
                break;
            }
            if (elect_one()) {
                expect_tx_u32(raw_full + 8 * slot, (uint32_t)tokens * kTileK);
                tma_load_u32(raw_u32 + slot * tokens * kTileK, &map_a, raw_full + 8 * slot, (kt0 + kt) * (kTileK / 2), first % tiles.token_tiles * tokens);
            }
        }
        if (*abort_flag != 0)
            for (int i = max(0, issued - kSpreadAhead); i < issued; ++i) mbar_wait(&c->raw_full[i & (kSpreadAhead - 1)], (uint32_t)(i / kSpreadAhead & 1), nullptr);
    } else if (warp == 0) {
        lb_wait_for_predecessor();
        lb_dependents_may_launch();
        int issued = 0, st = 0;
        uint32_t parity = 1;                                           // a stage's first use waits for nothing
        for (int tile = first; tile < tiles.total && ok; tile += stride) {
            const int m0 = tile % tiles.token_tiles * tokens;
            for (int kt = 0; kt < n_kt; ++kt) {
                if (!__all_sync(0xffffffffu, wait_u32(empty + 8 * st, parity, abort_flag))) {
                    give_up(c, status, 1, st);
                    ok = false;
                    break;
                }
                if (elect_one()) {
                    expect_tx_u32(b_full + 8 * st, stage_bytes);
                    tma_load_u32(stages_u32 + st * stage_bytes, &map_a, b_full + 8 * st, (kt0 + kt) * kTileK, m0);
                    tma_load_u32(stages_u32 + st * stage_bytes + atom_bytes, &map_a, b_full + 8 * st, (kt0 + kt) * kTileK + kBlockK, m0);
                }
                ++issued;
                if (++st == n_stages) {
                    st = 0;
                    parity ^= 1;
                }
            }
        }
        // Leave no copy in flight: the barriers of the last loads complete when their bytes landed.
        if (*abort_flag != 0)
            for (int i = max(0, issued - n_stages); i < issued; ++i) mbar_wait(&c->b_full[i % n_stages], (i / n_stages) & 1, nullptr);
    } else if (warp == 1) {
        const uint32_t desc_hi = (uint32_t)(1024 >> 4) | (1u << 14) | (2u << 29);
        const uint32_t lo0 = ((stages_u32 & 0x3FFFFu) >> 4) | (1u << 16);
        int st = 0;
        uint32_t parity = 0, unit = 0;                                 // chains so far
        for (int tile = first; tile < tiles.total && ok; tile += stride) {
            const int columns = min(tokens, (e.M - tile % tiles.token_tiles * tokens + 15) / 16 * 16);
            const uint32_t idesc = umma_idesc(kLaneRows, columns) & (T::kHalf ? ~((1u << 7) | (1u << 10)) : ~0u);
            // The sums of a tile, or of a chain, begin when the finishing warps have those that were there.
            auto begin = [&]() {
                if (FINISHERS == 0) return true;
                const bool free = __all_sync(0xffffffffu, wait_u32(smem_u32(&c->acc_empty[unit & kTurn]), (unit >> kTurn & 1) ^ 1, abort_flag));
                if (!free) give_up(c, status, 5, 0);
                tc_fence_after();
                return free;
            };
            uint32_t sums = tmem_base + (unit & kTurn) * tiles.chain_columns;
            int left = tiles.chain;
            ok = begin();
            for (int kt = 0; kt < n_kt && ok; ++kt) {
                if (CHAINED && left-- == 0) {
                    left = tiles.chain - 1;
                    if (FINISHERS > 0) {
                        if (withhold == 0 && elect_one()) umma_commit(&c->acc_full[unit & kTurn]);
                        ++unit;
                        sums = tmem_base + (unit & kTurn) * tiles.chain_columns;
                        ok = begin();
                        if (!ok) break;
                    } else {
                        sums += tiles.chain_columns;
                    }
                }
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
                        umma_ts(sums, ta + k * (kUmmaK / 2), b_lo + (k >> 2) * (atom_bytes >> 4) + 2 * (k & 3), desc_hi, idesc, (CHAINED ? left + 1 != tiles.chain : kt != 0) || k != 0 ? 1u : 0u);
                    commit_u32(empty + 8 * st);
                }
                if (++st == n_stages) {
                    st = 0;
                    parity ^= 1;
                }
            }
            // (`withhold`: a test's launch, whose epilogues find nothing and give up.)
            if (ok && withhold == 0 && elect_one()) umma_commit(&c->acc_full[unit & kTurn]);
            ++unit;
        }
        lb_wait_for_predecessor();
        lb_dependents_may_launch();
    } else if (spread && (warp == 2 || warp == 3)) {
        // Two warps make float16 of the e4m3 that warp 0 copies: sixteen of a token a lane and piece, from one 128-byte swizzle to the other.  (Loads of their own would be waited
        // for by the fence that shows the results to the tensor core: 0.7 us a k tile.)
        lb_wait_for_predecessor();
        lb_dependents_may_launch();
        const int pieces = min(tokens, e.M - first % tiles.token_tiles * tokens) * 8, q = (int)threadIdx.x - 64, piece = q & 7;
        int st = 0;
        uint32_t parity = 1;
        for (int kt = 0; kt < n_kt; ++kt) {
            const int slot = kt & (kSpreadAhead - 1);
            if (!__all_sync(0xffffffffu, wait_u32(raw_full + 8 * slot, (uint32_t)(kt / kSpreadAhead & 1), abort_flag) && wait_u32(empty + 8 * st, parity, abort_flag))) {
                give_up(c, status, 6, st);
                ok = false;
                break;
            }
            const uint32_t raw = raw_u32 + slot * tokens * kTileK, to = stages_u32 + st * stage_bytes + (piece >> 2) * atom_bytes;
#pragma unroll
            for (int i = 0; i < kSpreadTokens / 8; ++i)
                if (64 * i + q < pieces) {
                    const int r = 8 * i + (q >> 3), x = r & 7;
                    const float4 f = lds4(raw + r * 128 + ((piece ^ x) << 4));
                    const uint32_t v[4] = {__float_as_uint(f.x), __float_as_uint(f.y), __float_as_uint(f.z), __float_as_uint(f.w)};
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        sts4(to + r * 128 + (((2 * (piece & 3) + h) ^ x) << 4), make_uint4(e4m3x2_to_f16x2(v[2 * h] & 0xffffu), e4m3x2_to_f16x2(v[2 * h] >> 16),
                                                                                              e4m3x2_to_f16x2(v[2 * h + 1] & 0xffffu), e4m3x2_to_f16x2(v[2 * h + 1] >> 16)));
                }
            fence_async_shared();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&c->b_full[st]);
                mbar_arrive(&c->raw_empty[slot]);
            }
            if (++st == n_stages) {
                st = 0;
                parity ^= 1;
            }
        }
    } else if (warp >= kFirstMaker && group < kGroups) {
        constexpr int kPerTile = kTileK / GROUP;
        uint32_t mask, magic;
        asm volatile("mov.b32 %0, %2;\n\tmov.b32 %1, %3;" : "=r"(mask), "=r"(magic) : "n"(T::kHalf ? 0x00F000F0 : 0x00780078), "n"(T::kHalf ? 0x54005400 : 0x41804180));
        // No more warps take turns than there are stages: one that was a whole round of the stages ahead would take the parity of the round before for its own.
        const int turns = min(kGroups, n_stages);
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        constexpr int kDepth = FINISHERS > 0 ? 1 : 2;                               // k tiles on the way a warp (one where registers are short: the products take longer than the loads)
        uint4 words[kDepth][4];
        uint32_t steps[kDepth];
        // The k tiles of all of this block's tiles are one sequence, of which this warp takes every turns-th; `ahead` is where the next to be fetched lies.
        int ahead_tile = first, ahead_kt = group;
        const uint4* from = nullptr;
        const uint8_t* scales = nullptr;
        auto aim = [&]() {
            while (WALK && ahead_kt >= n_kt && ahead_tile < tiles.total) {
                ahead_kt -= n_kt;
                ahead_tile += stride;
            }
            const size_t at = (size_t)((ahead_tile / tiles.token_tiles * kLaneRows + row) >> 4) * k_tiles + kt0 + ahead_kt;
            from = static_cast<const uint4*>(w.nibbles) + at * (kTileBytes / 16) + piece_at(row & 15, 0);
            scales = static_cast<const uint8_t*>(w.scales) + (at * kTileRows + (row & 15)) * kPerTile;
        };
        auto fetch = [&](int i) {
            if (ahead_tile < tiles.total && ahead_kt < n_kt) {
#pragma unroll
                for (int t = 0; t < 4; ++t) words[i][t] = __ldg(from + piece_at(0, t));
                if constexpr (GROUP == 128) steps[i] = __ldg(scales);
                else if constexpr (GROUP == 64) steps[i] = __ldg(reinterpret_cast<const uint16_t*>(scales));
                else steps[i] = __ldg(reinterpret_cast<const uint32_t*>(scales));
                ahead_kt += turns;
                from += turns * (kTileBytes / 16);
                scales += turns * kTileRows * kPerTile;
                if (ahead_kt >= n_kt && WALK) aim();
            }
        };
        if (group < turns) {
            aim();
            fetch(0);
            if (kDepth > 1) fetch(1);
        }
        int st = group, tile = first, kt = group;
        uint32_t parity = 1;
        auto make = [&](int i) {
            if (!__all_sync(0xffffffffu, wait_u32(empty + 8 * st, parity, abort_flag))) {
                give_up(c, status, 4, st);
                ok = false;
                return;
            }
            tc_fence_after();
            const uint32_t to = __shfl_sync(0xffffffffu, tmem_a + lanes + st * kStageColumns, 0);       // one number for the warp
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
                tmem_st16(to + 16 * j, v);
            }
            fetch(i);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&c->a_full[st]);
            st += turns;
            if (st >= n_stages) {
                st -= n_stages;
                parity ^= 1;
            }
            kt += turns;
            while (WALK && kt >= n_kt && tile < tiles.total) {
                kt -= n_kt;
                tile += stride;
            }
        };
        if (WALK)
            while (kt >= n_kt && tile < tiles.total) {
                kt -= n_kt;
                tile += stride;
            }
        while (group < turns && ok && tile < tiles.total && kt < n_kt) {
            make(0);
            if (kDepth == 1) continue;
            if (!(ok && tile < tiles.total && kt < n_kt)) break;
            make(kDepth - 1);
        }
    }
    __syncwarp();

    const bool finisher = warp >= kFirstMaker + (FINISHERS > 0 ? MAKERS : 0);
    const int part = (warp - kFirstMaker - (FINISHERS > 0 ? MAKERS : 0)) >> 2;        // this warp's eights of columns are every kEnds-th from here
    const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16);
    lb_act_pair pair{0.0f, 0.0f};
    // Scales, residuals and the learned numbers behind the bias are read, and results written, after this.
    if (finisher) {
        lb_wait_for_predecessor();
        lb_dependents_may_launch();
        if (!w.paired) pair = lb_act_load(e.bias, e.n, e.act);
    }
    // A thread's sums of the chains before wait in its own words of shared memory, [token][row].
    float* before = reinterpret_cast<float*>(c + 1) + row;
    uint32_t unit = 0;                           // chains that the finishing warps have seen
    auto wait_for_sums = [&]() {
        const bool there = __all_sync(0xffffffffu, WALK ? wait_asleep(&c->acc_full[unit & kTurn], unit >> kTurn & 1, abort_flag)
                                                                : mbar_wait(&c->acc_full[unit & kTurn], unit >> kTurn & 1, abort_flag));
        if (!there) give_up(c, status, 3, quarter);
        tc_fence_after();
        return there;
    };
    auto sums_read = [&]() {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&c->acc_empty[unit & kTurn]);
    };
    // Eight tokens' sums from column `at` on, the chains' added in order.
    auto sums_at = [&](int at, float (&y)[8]) {
        uint32_t v[8];
        __syncwarp();                                                   // (the results' code parts lanes; a warp loads as one)
        tmem_ld8(t_row + (unit & kTurn) * tiles.chain_columns + at, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = __uint_as_float(v[i]);
    };
    auto add_before = [&](int at, float (&y)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] += before[(at + i) * kLaneRows];
    };
    // All chains of a tile but the last: their sums to shared memory, under the next one's products.
    auto earlier_chains = [&](int here) {
#pragma unroll 1
        for (int chain = 1; chain < chains; ++chain, ++unit) {
            if (!wait_for_sums()) return false;
#pragma unroll 1
            for (int at = 8 * part; at < here; at += 8 * kEnds) {
                float y[8];
                sums_at(at, y);
                if (chain > 1) add_before(at, y);
#pragma unroll
                for (int i = 0; i < 8; ++i) before[(at + i) * kLaneRows] = y[i];
            }
            sums_read();
        }
        return true;
    };
    if (WALK) {
        if (finisher) {
            for (int tile = first; tile < tiles.total; tile += stride, ++unit) {
                const int m0 = tile % tiles.token_tiles * tokens, here = min(tokens, e.M - m0);
                const RowEnd<T::kHalf> end(e, w, tile / tiles.token_tiles * kLaneRows + row, lane, true);
                if ((CHAINED && !earlier_chains(here)) || !wait_for_sums()) break;
                // When the last eight is there the next tile's products may begin.
#pragma unroll 1
                for (int at = 8 * part; at < here || at == 8 * part; at += 8 * kEnds) {
                    float y[8];
                    if (at < here) sums_at(at, y);
                    if (at + 8 * kEnds >= here) sums_read();
                    if (at >= here) break;
                    if (CHAINED && chains > 1) add_before(at, y);
                    end.finish(e, w.paired, pair, y, m0 + at);
                }
            }
        }
    } else {
        const int m0 = first % tiles.token_tiles * tokens, here = min(tokens, e.M - m0);
        if (finisher) {
            if (FINISHERS > 0) {
                ok = (!CHAINED || earlier_chains(here)) && wait_for_sums();
            } else {
                ok = __all_sync(0xffffffffu, ok && (mbar_wait(&c->acc_full[0], 0, abort_flag)));
                if (!ok) give_up(c, status, 3, quarter);
                tc_fence_after();
            }
        }
        __syncwarp();
        const bool finishes = finisher && ok;
        const RowEnd<T::kHalf> end(e, w, first / tiles.token_tiles * kLaneRows + row, lane, finishes);
        auto all_sums_at = [&](int at, float (&y)[8]) {
            sums_at(at, y);
            if (FINISHERS > 0) {
                if (CHAINED && chains > 1) add_before(at, y);
            } else if (CHAINED) {
#pragma unroll 1
                for (int chain = 1; chain < chains; ++chain) {
                    uint32_t v[8];
                    tmem_ld8(t_row + chain * tiles.chain_columns + at, v);
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] += __uint_as_float(v[i]);
                }
            }
        };
        if (splits > 1) {
            // Every block's products are complete before their stages are written over.  A rank's share is a whole number of eights of tokens, the last ranks' may be none.
            const int share = share_of(tokens, splits), eights = share / 8;
            float4* box = reinterpret_cast<float4*>(inbox) + row;      // [rank][eight][half][128 rows] of four tokens: a warp's 16-byte stores lie side by side
            __syncwarp();
            asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
            if (finishes) {
                for (int piece = part; 8 * piece < here; piece += kEnds) {
                    float y[8];
                    all_sums_at(8 * piece, y);
                    const int to = piece / eights;
                    const uint32_t peer = peer_address(smem_u32(box + (rank * eights + piece - to * eights) * 2 * kLaneRows), (uint32_t)to);
                    store_at_peer(peer, __float_as_uint(y[0]), __float_as_uint(y[1]), __float_as_uint(y[2]), __float_as_uint(y[3]));
                    store_at_peer(peer + kLaneRows * 16, __float_as_uint(y[4]), __float_as_uint(y[5]), __float_as_uint(y[6]), __float_as_uint(y[7]));
                }
            }
            __syncwarp();
            asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
            if (finishes) {
                for (int piece = part; piece < eights && rank * share + 8 * piece < here; piece += kEnds) {
                    float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                    for (int r = 0; r < splits; ++r) {
                        const float4 lo = box[(r * eights + piece) * 2 * kLaneRows], hi = box[((r * eights + piece) * 2 + 1) * kLaneRows];
                        y[0] += lo.x; y[1] += lo.y; y[2] += lo.z; y[3] += lo.w;
                        y[4] += hi.x; y[5] += hi.y; y[6] += hi.z; y[7] += hi.w;
                    }
                    end.finish(e, w.paired, pair, y, m0 + rank * share + 8 * piece);
                }
            }
        } else if (finishes) {
#pragma unroll 1
            for (int at = 8 * part; at < here; at += 8 * kEnds) {
                float y[8];
                all_sums_at(at, y);
                end.finish(e, w.paired, pair, y, m0 + at);
            }
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
        load_eight<T::kHalf>(v, a, m * lda, k, K, wide);
        to[i] = make_uint4(v[0], v[1], v[2], v[3]);
    }
}

int g_withhold_next = 0;      // the next launch's blocks leave their accumulator-ready barriers unsignalled (tests)

template <typename T, int GROUP, int MAKERS, int FINISHERS, bool WALK, bool CHAINED>
int launch_kernel(const CUtensorMap& map, const lb_weights4* w, const Epilogue& e, const ManyPlan& p, const Tiles& tiles, int n_sm, cudaStream_t s) {
    auto kernel = many_tokens_kernel<T, GROUP, MAKERS, FINISHERS, WALK, CHAINED>;
    static bool configured = false;
    if (!configured) {
        LB_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
        configured = true;
    }
    int* status = nullptr;
    if (int rc = lb_tc_status_word(&status)) return rc;
    const int blocks = WALK ? (tiles.total < n_sm ? tiles.total : n_sm) : tiles.total * p.splits;
    LB_CHECK_CUDA(lb_launch_overlapped_cluster(1, p.splits, kernel, dim3(blocks), dim3(32 * (kFirstMaker + MAKERS + FINISHERS)), p.smem, s, map, *w, e, tiles, p.tmem_columns, g_withhold_next,
                                               status));
    g_withhold_next = 0;
    return LB_OK;
}

template <typename T, int GROUP>
int launch(const CUtensorMap& map, const lb_weights4* w, const Epilogue& e, const ManyPlan& p, const Tiles& tiles, int n_sm, cudaStream_t s) {
    if (p.makers == 12)
        return p.walk ? launch_kernel<T, GROUP, 12, 12, true, true>(map, w, e, p, tiles, n_sm, s) : launch_kernel<T, GROUP, 12, 12, false, true>(map, w, e, p, tiles, n_sm, s);
    if (p.walk) return launch_kernel<T, GROUP, 8, 16, true, false>(map, w, e, p, tiles, n_sm, s);
    if (p.makers == 8)
        return p.chains > 1 ? launch_kernel<T, GROUP, 8, 0, false, true>(map, w, e, p, tiles, n_sm, s) : launch_kernel<T, GROUP, 8, 0, false, false>(map, w, e, p, tiles, n_sm, s);
    return p.chains > 1 ? launch_kernel<T, GROUP, 16, 0, false, true>(map, w, e, p, tiles, n_sm, s) : launch_kernel<T, GROUP, 16, 0, false, false>(map, w, e, p, tiles, n_sm, s);
}

// Whether e4m3 rows become float16 on their way, in a small tile's block: rows that TMA takes (24 x 8000 x 3008 9.5 us).  With more tokens, whose
// copies the two warps do not keep up with (60 x 8000 x 3008 14.4 us), or other rows a launch of its own comes first (10.3 and 11.8 us for the same).
bool spreads(const ManyPlan& p, const lb_weights4* w, const void* a, int64_t lda) {
    return p.tmem_columns == 256 && !p.walk && p.tokens <= kSpreadTokens && w->k % 2 == 0 && lda % 16 == 0 && reinterpret_cast<uintptr_t>(a) % 16 == 0;
}

bool copied_as_they_are(const void* a, int64_t lda) { return lda % 8 == 0 && reinterpret_cast<uintptr_t>(a) % 16 == 0; }       // bfloat16 rows that TMA takes

template <typename T>
int run(const lb_weights4* w, const void* a, int64_t lda, const Epilogue& e, void* scratch, cudaStream_t s) {
    const int k_tiles = (w->k + kTileK - 1) / kTileK, rows = w->paired ? 2 * ((e.n + 7) / 8 * 8) : e.n, row_blocks = (rows + kLaneRows - 1) / kLaneRows, n_sm = linear4_sm_count();
    const ManyPlan p = many_plan(e.M, rows, w->k, e.out_f32, n_sm);
    const bool spread = T::kHalf && spreads(p, w, a, lda);
    if (!spread && (T::kHalf || !copied_as_they_are(a, lda))) {
        LB_CHECK_ARG(scratch != nullptr && reinterpret_cast<uintptr_t>(scratch) % 16 == 0, "linear4: these activations need scratch memory (lb_linear4_scratch)");
        const bool wide = lda % 8 == 0 && reinterpret_cast<uintptr_t>(a) % (T::kHalf ? 8 : 16) == 0;
        const int eights = (w->k + 7) / 8;
        const int64_t all = (int64_t)e.M * eights, blocks = (all + 255) / 256;
        LB_CHECK_CUDA(lb_launch_overlapped(spread_rows_kernel<T>, dim3((unsigned)(blocks < 16 * n_sm ? blocks : 16 * n_sm)), dim3(256), 0, s, a, lda, wide,
                                           static_cast<uint4*>(scratch), eights, all, w->k));
        a = scratch;
        lda = 8 * (int64_t)eights;
    }
    // (Two e4m3 are copied as one value of two bytes.)
    CUtensorMap map;
    if (int rc = spread ? lb_tensor_map_2d_encode(&map, a, 2, e.M, w->k / 2, lda / 2, p.tokens) : lb_tensor_map_2d_encode(&map, a, 2, e.M, w->k, lda, p.tokens)) return rc;
    const int token_tiles = (e.M + p.tokens - 1) / p.tokens;
    LB_CHECK_ARG((int64_t)token_tiles * row_blocks * p.splits < (1ll << 30), "linear4: %d rows by %d features are too many tiles", e.M, rows);
    const Tiles tiles{p.tokens, token_tiles, token_tiles * row_blocks, k_tiles, p.splits, p.stages, p.d_columns, spread, p.chain, p.chain_columns};
    if (w->group == 32) return launch<T, 32>(map, w, e, p, tiles, n_sm, s);
    if (w->group == 64) return launch<T, 64>(map, w, e, p, tiles, n_sm, s);
    return launch<T, 128>(map, w, e, p, tiles, n_sm, s);
}

}  // namespace

// The cheapest cut by an estimate in us (a fit to some 150 launches of 24 to 2,048 tokens): 2.8 for the launch and the first weights; a k tile takes what its eight products take, which is no
// less than it takes the tensor core to load 128 x 128 weights (0.34, up to some 150 tokens; 0.57 for each of two blocks that share an SM); a token's column of sums 0.0115;
// the exchange of a cluster grows with its ranks and their tokens.
// The tensor core truncates the sum at each of its additions, which adds up along a chain: 3.4e-7 of the results at 2,048 values of k, 8e-7 at 4,096, 2.0e-6 at 8,192, 5.1e-6 at 16,384 (the
// additions of a product in 32 bits 1.1e-7 to 4.4e-7).  So float32 results have chains of kChain k tiles, whose sums are added in 32 bits; bfloat16's rounding hides either.  Where there are
// columns, a chain has an accumulator of its own in tensor memory; else twelve warps move its sums to shared memory under the products of the next, which has another accumulator.
ManyPlan many_plan(int M, int rows, int k, bool out_f32, int n_sm) {
    constexpr int kChain = 12;
    ManyPlan best{};
    const int k_tiles = (k + kTileK - 1) / kTileK, row_blocks = (rows + kLaneRows - 1) / kLaneRows, fewest = (M + 255) / 256;
    const bool deep = out_f32 && k_tiles > kChain;
    double least_us = 1e30;
    for (int token_tiles = fewest; token_tiles <= 2 * fewest + 2; ++token_tiles) {
        const int tokens = ((M + token_tiles - 1) / token_tiles + 15) / 16 * 16;
        if (token_tiles > fewest && tokens < 32) break;
        const long total = (long)((M + tokens - 1) / tokens) * row_blocks;
        const double stage = 0.55 * tokens / 256 > 0.34 ? 0.55 * tokens / 256 : 0.34, sums = 0.0115 * tokens;
        // (Each cut once, but for deep products that no cluster shares: by blocks of a tile each and by blocks that walk.)
        for (int way = 1; way <= (deep ? 9 : 8); ++way) {
            const int splits = way < 9 ? way : 1;
            ManyPlan p{};
            const int per = (k_tiles + splits - 1) / splits;
            if (splits > 1 && (per < 3 || per * (splits - 1) >= k_tiles)) continue;      // short parts, or a rank without one
            p.tokens = tokens;
            p.splits = splits;
            p.chains = deep ? (per + kChain - 1) / kChain : 1;
            p.chain = (per + p.chains - 1) / p.chains;
            p.chain_columns = (tokens + 31) / 32 * 32;
            p.turn = p.chains > 1 && (way == 9 || p.chains * p.chain_columns > 320);
            const int columns = p.chains == 1 ? tokens : p.chain_columns * (p.turn ? 2 : p.chains);
            if (columns > 320) continue;
            const bool two = way < 9 && !p.turn && columns <= 64;     // two blocks an SM, whose starts and ends hide under one another
            p.walk = deep ? way == 9 : splits == 1 && !two && total > n_sm;
            p.makers = p.turn ? 12 : two || p.walk ? 8 : 16;
            p.d_columns = two ? 64 : columns <= 128 ? 128 : columns <= 256 ? 256 : 320;
            p.stages = two || p.d_columns >= 256 ? 3 : 6;
            p.tmem_columns = two ? 256 : 512;
            const int before = p.turn ? tokens * kLaneRows * 4 : 0;                      // the sums of the chains before
            while (p.stages > 3 && 1024 + p.stages * tokens * 256 + (int)sizeof(Control) + before > 227 * 1024) --p.stages;
            // The blocks of a cluster wait for one another while each holds its columns: as large a share of the shared memory as of the columns (see gemm_tcgen05_narrow.cu).
            const int in_stages = p.stages * tokens * 256, inbox = splits > 1 ? splits * share_of(tokens, splits) * 512 : 0;
            const int needed = 1024 + (in_stages > inbox ? in_stages : inbox) + (int)sizeof(Control) + before + (two && tokens <= kSpreadTokens ? 1024 + kSpreadAhead * tokens * kTileK : 0);
            const int least = p.tmem_columns * (228 * 1024 / 512) - 1024;
            p.smem = needed < least ? least : needed;
            if (p.smem > 227 * 1024) continue;
            // Clusters lie within one group of SMs, which those of more than two blocks do not fill; a second wave of blocks is worth no split, unless for the chains' sake.
            const long blocks = total * splits, at_once = (long)n_sm * (splits <= 2 ? 148 : splits == 3 ? 144 : splits == 4 ? 132 : 104) / 148;
            if (!deep && splits > 1 && blocks > (two && splits == 2 ? 2 * at_once : at_once)) continue;
            const double exchange = splits > 1 ? 0.8 + (0.005 * splits + 0.004) * tokens : 0.0;
            double us = 2.8;
            if (p.walk) {
                us += (double)((total + n_sm - 1) / n_sm) * (per * (p.turn && stage < 0.4 ? 0.4 : stage) + 0.4 + sums);
            } else if (deep) {
                const long fit = two ? 2 * at_once : at_once, waves = (blocks + fit - 1) / fit;
                us += waves * (per * (two && blocks > at_once ? 0.57 : p.turn && stage < 0.4 ? 0.4 : stage) + sums / splits + exchange) + (waves - 1) * 4.0;
            } else {
                us += (double)((blocks + 2 * n_sm - 1) / (2 * n_sm)) * per * (two && blocks > n_sm ? 0.57 : stage) + sums / splits + exchange;
            }
            if (us < least_us) {
                least_us = us;
                best = p;
            }
        }
    }
    return best;
}

int64_t many_scratch_bytes(const lb_weights4* w, int a_dtype, const void* a, int64_t lda, int M) {
    if (a_dtype == LB_BF16 && copied_as_they_are(a, lda)) return 0;
    const int rows = w->paired ? 2 * ((w->n / 2 + 7) / 8 * 8) : w->n;
    // (Enough for either type of result.  Of more rows than this no tile is small enough.)
    if (a_dtype == LB_E4M3 && M <= 4 * kSpreadTokens && spreads(many_plan(M, rows, w->k, false, linear4_sm_count()), w, a, lda) &&
        spreads(many_plan(M, rows, w->k, true, linear4_sm_count()), w, a, lda))
        return 0;
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

// Attention over a 4-bit cache for many query rows: portions of prompts, on the fifth-generation tensor cores.
//
// The query rows of a request that share a key/value head (its tokens' heads, in the order of the tokens) are cut into tiles of 256; a block has a tile, as two groups of 128 rows, and walks the
// keys 128 at a time.  Both groups read the same keys and values, which eight warps make from the cache's nibbles:
//   warps 0..15   softmax, two threads a row: p = 2^(S - m + 7) as float16 back into tensor memory over the scores it came from, and O rescaled where m moved.
//   warps 16..23  makers: a warp has a block of sixteen keys.  The nibbles of the next tile are on their way while this one's become n s as float16, in the 128-byte swizzle that tcgen05 reads.
//   warps 24, 25  issue tcgen05.mma, one for each group: S = Q K^T (128 x 128), O += P V (64 values at a time, V as it lies, [key][dim]: the "MN-major" form).
// Tensor memory: the groups' scores (and p, in the first half of their columns), then the groups' O.  A group's next scores are asked for once its update has read p; meanwhile the other group is at
// its exponentials, so the two take turns at the tensor cores and at the special-function units (a tile's 2 x 16,384 exponentials take those 2,048 cycles, its products for heads of 128 the tensor
// cores 2,048).
// Numbers: a row of queries is float16 after a power of two that puts its largest at 2^14; n s after one for the block of sixteen keys that puts its largest scale at 2^8, which the scores, and p, are
// multiplied by again (for p relative to the largest block's so far, F, which O is in units of).  So K, V and p are rounded to float16 (2^-12, p of weights below 2^-21 of
// the row's largest to 2^-32 of it; without the factor of 2^7 it would be 2^-25, which 131,072 keys beside one that takes most of the weight made 2 % of the rest), and bfloat16's range is kept.
// A value scale that is NaN would meet p = 0 of rows that do not see its key in the products: such groups are made zeros, and the rows that see them take a note (a bit a group) and end as NaN.
// Every wait is bounded; one that runs out records a code in the device status word, and the block ends without results, once the products that it asked for are through.
// What bounds it.  A block alone on an SM (204 KB) gets through 256 rows by 64 keys in 1.46 us for heads of 128 (838 TFLOP/s over 148 SMs; 0.51 of cuBLAS's burst) and 1.30 for heads of 64 (469): its
// schedulers issue in 71 % of all cycles, exponentials, conversions and the largest score of a row above all (16 softmax warps), the makers' nibbles after them.  Leaving the makers' work out, or the
// exponentials, saved less than a tenth, as did turns that keep the groups half a unit apart: no one part is the bound.  A soft cap adds 36 % (4 x 512 tokens behind 8,192 keys, 32 heads over 8 of 128,
// capped: 514 us; the tangent by its series of four terms in scores of their own scale 583).  With one thread a row and the products of all groups issued by one warp 742, as a row's maximum, exponentials and sum are
// twice as long a chain.  A block takes 9 us to start (queries, first keys, tensor memory) and end; 2 x 1,024 tokens, 12 heads of 64: 28 us, of which 16 units of keys are 20.
#include "attention4.h"
#include "attention4_join.cuh"
#include "attention4_parts.cuh"

#include <float.h>
#include <math_constants.h>

#include <algorithm>

namespace lb_a4 {
namespace {

using namespace lb_c4;
using namespace lb_tc;

constexpr int kGroups = 2, kBM = 128, kBN = 128, kTileRows = kGroups * kBM;
constexpr int kUnit = 64;                      // keys of a score tile: half of what the makers make at a time
constexpr int kStages = 2;                     // tiles of keys, and of values, in shared memory
constexpr int kNotes = 4;                      // what the softmax reads of a tile, longer than a stage holds
constexpr int kSoftmaxWarps = 16, kMakers = 8, kMaker = kSoftmaxWarps, kIssuer = kMaker + kMakers;
constexpr int kManyThreads = 32 * (kIssuer + 4);         // (the last two warps are there because registers are dealt to four warps at a time)
// Registers a thread after the roles part: 4 x 80 + 2 x 72 + 40, the 7 x 72 that the block starts with.
constexpr int kSoftmaxRegs = 80, kMakerRegs = 72, kIssuerRegs = 40;
constexpr int kSub = 128 * 128;                // [128 rows][128 bytes]: 64 values of a tile
constexpr uint32_t kTmemCols = 512, kOCol = 256;
constexpr float kSlack = 8.0f, kLeastExponent = -100.0f;
constexpr float kUp = 7.0f;                    // p is 2^(S - m + kUp), up to 2^(kUp + kSlack) of float16's 2^16

struct Control {
    uint64_t q_full;
    uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
    uint64_t s_full[kGroups][2], p_full[kGroups][2], o_done[kGroups][2];       // of units in turn: what waits may be a unit behind, and a parity tells no more than two phases apart
    uint64_t drained[kGroups];                                             // of a group that gave up: the products under way are through
    uint32_t tmem_base;
    int abort_flag, whole;                                                 // whole: the block has all keys of its rows
    float k_factor[kNotes][kMakers], v_exponent[kNotes][kMakers];          // of a tile's blocks of sixteen keys
    uint8_t gone[kNotes][kMakers], nans[kNotes][kMakers];                  // on no page; values with scales that are NaN
    uint8_t nan_groups[kNotes][kBN];                                       // a bit a group
    float row_scale[kTileRows];                                            // of the scores, in base 2
    float row_high[kGroups][2][kBM], row_sum[kGroups][2][kBM];             // what the two threads of a row tell each other
    uint8_t row_nans[kGroups][2][kBM];
};

__device__ __forceinline__ void give_up(Control* c, int* status, int site) {
    atomicCAS(status, 0, (0xC << 12) | site);
    *(volatile int*)&c->abort_flag = 1;
}
template <int N>
__device__ __forceinline__ void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
// A word's values times s as four float16 pairs: nibbles (i, i + 4).
__device__ __forceinline__ void scaled_pairs(uint32_t w, __half2 s, uint32_t (&r)[4]) {
    __half2 n[4];
    pairs_of(w, n);
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = h2(__hmul2(n[i], s));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
          "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// The wait for a load, tied to its registers so that nothing is made of them before it.
__device__ __forceinline__ void tmem_ld_wait32(uint32_t (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]),
                   "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]),
                   "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
                 :: "memory");
}
// The product with its first operand in tensor memory (lane = row, two float16 values of K to a column).
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Descriptor of a tile [64 values][key][64 values] as the second operand in its MN-major form: rows of 128 bytes, eight keys to a 1024-byte group (the stride offset), the next 64 values
// behind all keys (the leading offset).
__device__ __forceinline__ uint64_t umma_desc_mn(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)(kSub >> 4) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
// Instruction descriptors: float16 operands (0 in both format fields), 32-bit sums; the second with the second operand MN-major (bit 16).
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }

// The largest finite bfloat16 number among the words' (0 where none is above it), over the warp.
template <int N>
__device__ __forceinline__ uint32_t largest(const uint32_t* w) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) top = __vmaxu2(top, w[i]);
    top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
    if (top < 0x7f80u) return top;
    top = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t lo = w[i] & 0xffffu, hi = w[i] >> 16;
        top = max(top, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
    }
    return __reduce_max_sync(0xffffffffu, top);
}

__device__ __forceinline__ void tmem_ld_wait16(uint32_t (&v)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]), "+r"(v[10]),
                   "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15])
                 :: "memory");
}

// Two multiply-adds, two additions, and the largest of three in one instruction each.
__device__ __forceinline__ void fma2(float& d0, float& d1, uint32_t a0, uint32_t a1, float b, float c) {
    asm("{\n\t.reg .b64 a, b, c, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %4};\n\tmov.b64 c, {%5, %5};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\t"
        "mov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d0), "=f"(d1) : "r"(a0), "r"(a1), "f"(b), "f"(c));
}
__device__ __forceinline__ void add2(float& d0, float& d1, float a0, float a1) {
    asm("{\n\t.reg .b64 a, d;\n\t"
        "mov.b64 a, {%2, %3};\n\tmov.b64 d, {%0, %1};\n\t"
        "add.rn.f32x2 d, d, a;\n\t"
        "mov.b64 {%0, %1}, d;\n\t}"
        : "+f"(d0), "+f"(d1) : "f"(a0), "f"(a1));
}
// Numbers in twos: the pair, a number twice, products and multiply-adds.
typedef unsigned long long Two;
__device__ __forceinline__ Two two(float a, float b) {
    Two d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
    Two d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
    Two d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ void of_two(Two a, uint32_t& lo, uint32_t& hi) { asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(a)); }
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Whether any of 64 threads says so; a barrier among them.
__device__ __forceinline__ bool any_of_pair(int barrier, bool mine) {
    uint32_t any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %2, 0;\n\t"
        "barrier.cta.red.or.pred q, %1, 64, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(any) : "r"(barrier), "r"((uint32_t)mine) : "memory");
    return any != 0;
}

// The keys that a tile of rows sees: the first (the start of a tile of keys), and tiles.
__device__ __forceinline__ void keys_of_rows(const Call& c, const Portion& part, int row0, int* lo, int* tiles) {
    const int n_rows = part.count * c.per, limit = min(c.max_keys, c.table_stride << c.pages.page_shift) - 1;
    auto place_of = [&](int row) { return min(part.place + min(row, n_rows - 1) / c.per, limit); };
    const int last = place_of(row0 + kTileRows - 1);
    *lo = 0;
    if (c.window != 0) {
        const int first = place_of(row0);
        *lo = first < 0 ? 0 : lb_first_visible(first, c.window) / kBN * kBN;
    }
    *tiles = last >= 0 ? (last - *lo) / kBN + 1 : 0;
}

// `n_splits` blocks share a row tile's keys, `share` tiles of keys each, the last what is left.
template <int HD, int NG, bool PLAIN>
__global__ void __launch_bounds__(kManyThreads, 1)
attention4_many_kernel(const Call c, int n_splits, int share, int* status) {
    using L = Layout<HD>;
    constexpr int SUBS = HD / 64, JK = HD / 32, JV = HD / 64;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* q_s = base;                                            // [group][64 values][128 rows]
    uint8_t* k_s = q_s + kGroups * SUBS * kSub;                     // [stage][64 values][128 keys]
    uint8_t* v_s = k_s + kStages * SUBS * kSub;
    Control* ctl = reinterpret_cast<Control*>(v_s + kStages * SUBS * kSub);
    volatile int* abort_flag = &ctl->abort_flag;

    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    lb_wait_for_predecessor();
    lb_dependents_may_launch();
    const int seq = blockIdx.z, kvh = blockIdx.y, kv = c.pages.n_kv_head;
    const Portion part = portion_of(c, seq);
    // The last tiles first, which see the most keys.
    const int split = (int)blockIdx.x % n_splits;
    const int n_rows = part.count * c.per, row0 = ((n_rows + kTileRows - 1) / kTileRows - 1 - (int)blockIdx.x / n_splits) * kTileRows;
    if (row0 < 0 || n_rows <= 0) return;
    const int limit = min(c.max_keys, c.table_stride << c.pages.page_shift) - 1;          // no key past this place is read
    auto place_of = [&](int row) { return min(part.place + min(row, n_rows - 1) / c.per, limit); };
    auto first_of = [&](int place) { return place < 0 ? 0 : lb_first_visible(place, c.window); };
    int all_lo, all_tiles;
    keys_of_rows(c, part, row0, &all_lo, &all_tiles);
    if (split > 0 && split * share >= all_tiles) return;
    const int last = place_of(row0 + kTileRows - 1), kv_lo = all_lo + split * share * kBN;
    const int n_tiles = split == n_splits - 1 ? all_tiles - split * share : min(share, all_tiles - split * share), p_hi = min(last, kv_lo + n_tiles * kBN - 1);
    // Whether rows of group g see keys of unit u.
    int g_lo[kGroups], g_hi[kGroups];                               // units
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
        const int from = row0 + g * kBM, hi = min(place_of(from + kBM - 1), p_hi), first = max(first_of(place_of(from)), kv_lo);
        const bool some = from < n_rows && hi >= first && n_tiles > 0;
        g_lo[g] = some ? (first - kv_lo) / kUnit : 0;
        g_hi[g] = some ? (hi - kv_lo) / kUnit + 1 : 0;
    }
    auto active = [&](int g, int u) { return u >= g_lo[g] && u < g_hi[g]; };

    if (threadIdx.x == 0) {
        mbar_init(&ctl->q_full, kSoftmaxWarps);
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&ctl->k_full[i], kMakers);
            mbar_init(&ctl->k_empty[i], kGroups);
            mbar_init(&ctl->v_full[i], kMakers);
            mbar_init(&ctl->v_empty[i], kGroups);
        }
        for (int i = 0; i < 2 * kGroups; ++i) {
            mbar_init(&ctl->s_full[i / 2][i % 2], 1);
            mbar_init(&ctl->p_full[i / 2][i % 2], kSoftmaxWarps / kGroups);
            mbar_init(&ctl->o_done[i / 2][i % 2], 1);
        }
        for (int i = 0; i < kGroups; ++i) mbar_init(&ctl->drained[i], 1);
        ctl->abort_flag = 0;
        ctl->whole = all_tiles <= share;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kIssuer) {
        tmem_alloc(&ctl->tmem_base, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, ctl->tmem_base, 0);

    if (warp >= kIssuer) registers_down<kIssuerRegs>();
    else if (warp >= kMaker) registers_down<kMakerRegs>();
    else registers_up<kSoftmaxRegs>();
    if (warp >= kIssuer + kGroups) {
        // (nothing)
    } else if (warp >= kIssuer) {
        // ---- products, a warp a group.  A group's scores of unit u + 1 are asked for ahead of its update of unit u, when its update of unit u - 1, whose p lay where they go, is done.
        constexpr uint32_t idesc_s = idesc_f16(kBM, kUnit), idesc_o = idesc_f16(kBM, HD) | (1u << 16);
        const int g = warp - kIssuer, lo = g == 0 ? g_lo[0] : g_lo[1], hi = g == 0 ? g_hi[0] : g_hi[1], n_units = 2 * n_tiles;
        const uint64_t dq = umma_desc(smem_u32(q_s + g * SUBS * kSub)), dk = umma_desc(smem_u32(k_s)), dv = umma_desc_mn(smem_u32(v_s));
        const uint32_t s_at = tmem_base + g * kBN, o_at = tmem_base + kOCol + g * HD;
        bool ok = wait(&ctl->q_full, 0, abort_flag);
        if (!ok) give_up(ctl, status, 2);
        auto scores = [&](int u) {
            const int st = (u >> 1) % kStages;
            // The values too, which are made a little later: what their makers note is the softmax's by the time it has the scores.
            if ((u & 1) == 0) ok = wait(&ctl->k_full[st], (u >> 1) / kStages & 1, abort_flag) && wait(&ctl->v_full[st], (u >> 1) / kStages & 1, abort_flag);
            if (u >= lo && u < hi) {
                if (u - 2 >= lo) ok = ok && wait(&ctl->o_done[g][u & 1], (uint32_t)((u - 2 - lo) >> 1) & 1u, abort_flag);
                if (!ok) return;
                tc_fence_after();
                const uint64_t db = dk + (uint64_t)((st * SUBS * kSub + (u & 1) * kUnit * 128) >> 4);
                if (elect_one()) {
#pragma unroll
                    for (int i = 0; i < HD / kUmmaK; ++i)
                        umma_bf16(s_at + (u & 1) * kUnit, dq + (uint64_t)(((i / 4) * kSub + i % 4 * 32) >> 4), db + (uint64_t)(((i / 4) * kSub + i % 4 * 32) >> 4), idesc_s, i != 0 ? 1u : 0u);
                    if (c.withhold == 0) umma_commit(&ctl->s_full[g][u & 1]);
                }
                __syncwarp();
            }
            if (ok && (u & 1) == 1 && elect_one()) umma_commit(&ctl->k_empty[st]);
            __syncwarp();
        };
        if (ok && n_units > 0) scores(0);
        for (int u = 0; u < n_units && ok; ++u) {
            const int st = (u >> 1) % kStages;
            if (u + 1 < n_units) scores(u + 1);
            if (!ok) break;
            if (u >= lo && u < hi) {
                ok = wait(&ctl->p_full[g][u & 1], (uint32_t)((u - lo) >> 1) & 1u, abort_flag);
                if (!ok) break;
                tc_fence_after();
                const uint64_t db = dv + (uint64_t)((st * SUBS * kSub + (u & 1) * kUnit * 128) >> 4);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < kUnit / kUmmaK; ++k)              // sixteen keys: eight columns of p, 2048 bytes of values
                        umma_ts(o_at, s_at + (u & 1) * kUnit + k * 8, db + (uint64_t)((k * 2048) >> 4), idesc_o, u > lo || k != 0 ? 1u : 0u);
                    umma_commit(&ctl->o_done[g][u & 1]);           // O holds unit u, and p has been read
                }
                __syncwarp();
            }
            if (ok && (u & 1) == 1 && elect_one()) umma_commit(&ctl->v_empty[st]);
            __syncwarp();
        }
        if (!ok) {
            // Products that are under way read shared memory and write tensor memory: they end (bounded as well) before the block gives either back.
            give_up(ctl, status, 3);
            if (elect_one()) umma_commit(&ctl->drained[g]);
            __syncwarp();
            mbar_wait(&ctl->drained[g], 0, nullptr);
        }
    } else if (warp >= kMaker) {
        // ---- makers
        const int b = warp - kMaker, g = lane >> 2, t = lane & 3;
        const int32_t* table = c.table + (int64_t)seq * c.table_stride;
        const int kb = block_bytes(HD, NG);
        int block_at = -1;                                   // lane i: the cache's block of this warp's keys in tile i of this 32; -1: on no page, -2: past the keys
        struct Raw {
            uint32_t k[2][JK], v[2][2 * JV], ks[NG], vs[2][NG];
        };
        auto load = [&](int j, Raw& r, int* where) {
            if ((j & 31) == 0) {
                const int key = kv_lo + (j + lane) * kBN + b * kBlockKeys;
                block_at = -2;
                if (key <= p_hi) {
                    const int page = table[key >> c.pages.page_shift];
                    block_at = (unsigned)page < (unsigned)c.pages.n_pages
                                   ? ((page * kv + kvh) << (c.pages.page_shift - 4)) + ((key & ((1 << c.pages.page_shift) - 1)) >> 4) : -1;
                }
            }
            *where = __shfl_sync(0xffffffffu, block_at, j & 31);
            if (*where < 0) return;
            const uint8_t* block = c.pages.memory + (int64_t)*where * kb;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                load_words<L::kPiece>(block + (32 * i + lane) * L::kPiece, r.k[i]);
                load_words<L::kPiece>(block + L::kV + (32 * i + t * 8 + L::v_turn(g, t)) * L::kPiece, r.v[i]);
                load_words<4 * NG>(block + L::kScales + 32 * NG + (2 * t + i) * 4 * NG, r.vs[i]);
            }
            load_words<4 * NG>(block + L::kScales + g * 4 * NG, r.ks);
        };
        Raw raw = {}, next = {};
        int where = -2, next_where = -2;
        bool ok = true;
        if (n_tiles > 0) load(0, raw, &where);
        for (int j = 0; j < n_tiles; ++j) {
            const int st = j % kStages, note = j % kNotes, key0 = kv_lo + j * kBN + b * kBlockKeys;
            const uint32_t empty = ((uint32_t)(j / kStages) & 1u) ^ 1u;
            if (j + 1 < n_tiles) load(j + 1, next, &next_where);
            if (where < 0) raw = Raw{};
            // Keys past the last row's: whatever the memory holds, their scales are 0.
            if (key0 + kBlockKeys - 1 > p_hi) {
                auto clear = [&](uint32_t* w, int key, int second) {
                    if (key <= p_hi) return;
                    if constexpr (NG == 1) {
                        w[0] &= second != 0 ? 0x0000ffffu : 0xffff0000u;
                    } else {
#pragma unroll
                        for (int i = 0; i < NG / 2; ++i) w[second * NG / 2 + i] = 0;
                    }
                };
#pragma unroll
                for (int second = 0; second < 2; ++second) {
                    clear(raw.ks, key0 + g + 8 * second, second);
                    clear(raw.vs[0], key0 + 2 * t + 8 * second, second);
                    clear(raw.vs[1], key0 + 2 * t + 1 + 8 * second, second);
                }
            }
            ok = wait(&ctl->k_empty[st], empty, abort_flag);
            if (!ok) break;
            {
                const uint32_t top = largest<NG>(raw.ks);
                const int e = max((int)(top >> 7) - 127, (int)kLeastExponent);
                const float up = pow2(8 - e);
                uint8_t* to = k_s + st * SUBS * kSub;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int key = b * kBlockKeys + g + 8 * i;
#pragma unroll
                    for (int jj = 0; jj < JK; ++jj) {
                        const int chunk = 4 * jj + t;
                        uint4 w;
                        uint32_t r[4];
                        scaled_pairs(raw.k[i][jj], __float2half2_rn(number(raw.ks, i * NG + jj * NG / JK) * up), r);
                        w.x = r[0]; w.y = r[1]; w.z = r[2]; w.w = r[3];
                        *reinterpret_cast<uint4*>(to + (chunk >> 3) * kSub + key * 128 + (((chunk & 7) ^ (key & 7)) << 4)) = w;
                    }
                }
                if (lane == 0) {
                    ctl->k_factor[note][b] = pow2(e - 8);
                    ctl->gone[note][b] = where == -1;
                }
            }
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctl->k_full[st]);
            ok = wait(&ctl->v_empty[st], empty, abort_flag);
            if (!ok) break;
            {
                const uint32_t top = max(largest<NG>(raw.vs[0]), largest<NG>(raw.vs[1]));
                const int e = max((int)(top >> 7) - 127, (int)kLeastExponent);
                const float up = pow2(8 - e);
                uint8_t* to = v_s + st * SUBS * kSub;
                bool nans = false;
#pragma unroll
                for (int i = 0; i < 2; ++i)                  // the keys 2 t, 2 t + 1, and those plus 8
#pragma unroll
                    for (int a = 0; a < 2; ++a) {
                        const int key = b * kBlockKeys + 8 * i + 2 * t + a;
                        float s[NG];
                        uint32_t bits = 0;
#pragma unroll
                        for (int x = 0; x < NG; ++x) {
                            s[x] = number(raw.vs[a], i * NG + x);
                            if (!(s[x] < CUDART_INF_F)) {
                                s[x] = 0.0f;
                                bits |= 1u << x;
                            }
                        }
                        if (g == 0) ctl->nan_groups[note][key] = (uint8_t)bits;
                        nans = nans || bits != 0;
#pragma unroll
                        for (int jj = 0; jj < JV; ++jj) {
                            uint32_t r[4], r2[4];
                            const uint32_t w = raw.v[i][a * JV + jj];
                            const __half2 s0 = __float2half2_rn(s[64 * jj / (HD / NG)] * up), s1 = __float2half2_rn(s[(64 * jj + 32) / (HD / NG)] * up);
                            scaled_pairs(w, s0, r);
                            if (NG * 32 == HD) scaled_pairs(w, s1, r2);
                            uint8_t* row = to + jj * kSub + key * 128 + (g & 1) * 8;
                            *reinterpret_cast<uint2*>(row + (((g >> 1) ^ (key & 7)) << 4)) = make_uint2(r[0], r[1]);
                            *reinterpret_cast<uint2*>(row + (((4 + (g >> 1)) ^ (key & 7)) << 4)) = NG * 32 == HD ? make_uint2(r2[2], r2[3]) : make_uint2(r[2], r[3]);
                        }
                    }
                nans = __any_sync(0xffffffffu, nans);
                if (lane == 0) {
                    ctl->v_exponent[note][b] = (float)e;
                    ctl->nans[note][b] = nans;
                }
            }
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctl->v_full[st]);
            raw = next;
            where = next_where;
        }
        if (!ok) give_up(ctl, status, 4);
    } else {
        // ---- softmax, two threads a row (warps w and w + 4): each has 32 of a unit's keys.
        const int g = warp >> 3, x = warp >> 2 & 1, quarter = warp & 3, row = row0 + g * kBM + quarter * 32 + lane;
        const uint32_t t_s = tmem_base + g * kBN + ((uint32_t)(quarter * 32) << 16), t_o = tmem_base + kOCol + g * HD + x * (HD / 2) + ((uint32_t)(quarter * 32) << 16);
        const int pair_barrier = 1 + g * 4 + quarter, all_barrier = 1 + 4 * kGroups;
        {
            // Sixteen rows a warp as float16 into shared memory, HD / 8 lanes a row, and the factors that bring their scores back.
            constexpr int LANES = HD / 8, AT_ONCE = 32 / LANES, STEPS = 4;
            const bool q_wide = reinterpret_cast<uintptr_t>(c.q) % 16 == 0 && c.q_stride % 8 == 0;
            const int chunk = lane % LANES;
#pragma unroll 1
            for (int from_row = warp * 16; from_row < warp * 16 + 16; from_row += STEPS * AT_ONCE) {         // (code that runs once costs its fetching)
            uint32_t u[STEPS][4];
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                const int r = row0 + from_row + i * AT_ONCE + lane / LANES, token = r / c.per;
                const __nv_bfloat16* from = c.q + (int64_t)(part.first + token) * c.q_stride + (int64_t)(kvh * c.per + r - token * c.per) * HD + 8 * chunk;
#pragma unroll
                for (int e = 0; e < 4; ++e) u[i][e] = 0;
                if (r < n_rows && q_wide) {
                    load_words<16>(reinterpret_cast<const uint8_t*>(from), u[i]);
                } else if (r < n_rows) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) u[i][e] = __bfloat16_as_ushort(from[2 * e]) | (uint32_t)__bfloat16_as_ushort(from[2 * e + 1]) << 16;
                }
            }
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                const int r = from_row + i * AT_ONCE + lane / LANES;
                uint32_t top = __vmaxu2(__vmaxu2(u[i][0] & 0x7fff7fffu, u[i][1] & 0x7fff7fffu), __vmaxu2(u[i][2] & 0x7fff7fffu, u[i][3] & 0x7fff7fffu));
                top = max(top & 0xffffu, top >> 16);
#pragma unroll
                for (int d = 1; d < LANES; d *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
                const bool finite = top < 0x7f80u;
                const int shift = top == 0 || !finite ? 0 : 14 - (max((int)(top >> 7), 1) - 127);
                const float up = copysignf(pow2(shift / 2), c.scale), up2 = pow2(shift - shift / 2);            // the scale's sign is the query's
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    w[e] = finite ? h2(__floats2half2_rn(__uint_as_float(u[i][e] << 16) * up * up2, __uint_as_float(u[i][e] & 0xffff0000u) * up * up2)) : 0u;
                *reinterpret_cast<uint4*>(q_s + ((r >> 7) * SUBS + (chunk >> 3)) * kSub + (r & 127) * 128 + (((chunk & 7) ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
                if (chunk == 0) ctl->row_scale[r] = !finite ? CUDART_NAN_F : fabsf(c.scale) * kLbLog2e * pow2(-shift / 2) * pow2(-shift - -shift / 2);
            }
            }
            fence_async_shared();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctl->q_full);
            named_barrier(all_barrier, 32 * kSoftmaxWarps);
        }
        const float row_scale = ctl->row_scale[row - row0];
        const bool there = row < n_rows;
        const int token = min(row, n_rows - 1) / c.per, head = kvh * c.per + min(row, n_rows - 1) - token * c.per;
        const int place = place_of(row), first = first_of(place);
        const int w_row = row0 + g * kBM + quarter * 32;
        const int place_lo = place_of(w_row), first_hi = first_of(place_of(w_row + 31));            // of the warp's rows
        const float units_out = !PLAIN && c.soft_cap > 0.0f ? c.soft_cap * kLbLog2e : 1.0f, units_in = 1.0f / units_out;          // (scores are in base 2)
        const bool biased = !PLAIN && c.distance != nullptr;
        const float r1 = biased ? c.distance[head] : 0.0f, r2 = biased ? c.distance[c.n_head + head] : 0.0f;
        const int lo = g == 0 ? g_lo[0] : g_lo[1], hi = g == 0 ? g_hi[0] : g_hi[1];
        float m = kLowest, l = 0.0f, big = kLeastExponent;                    // big: F, the largest exponent of value scales so far
        uint32_t nan_bits = 0;
        bool ok = true, bad = false;
        for (int u = lo; u < hi; ++u) {
            const int note = (u >> 1) % kNotes, b0 = (u & 1) * (kUnit / kBlockKeys) + 2 * x, key0 = kv_lo + u * kUnit + 32 * x;
            const uint32_t t_u = t_s + (u & 1) * kUnit;
            // Both threads of a row give up, or neither: a wait that ran out is met at the barrier below.
            ok = wait(&ctl->s_full[g][u & 1], (uint32_t)((u - lo) >> 1) & 1u, abort_flag);
            tc_fence_after();
            uint32_t v[32];
            tmem_ld32(t_u + 32 * x, v);
            float f0 = row_scale * ctl->k_factor[note][b0], f1 = row_scale * ctl->k_factor[note][b0 + 1];
            const float e0 = ctl->v_exponent[note][b0], e1 = ctl->v_exponent[note][b0 + 1];
            const uint32_t gone0 = ctl->gone[note][b0], gone1 = ctl->gone[note][b0 + 1], nans = ctl->nans[note][b0] | ctl->nans[note][b0 + 1];
            const bool masked = key0 + 31 > place_lo || key0 < first_hi || (gone0 | gone1) != 0;
            tmem_ld_wait32(v);
            if (!PLAIN || masked) {
                if constexpr (!PLAIN) {
                    // Scores, or, capped, in units of the cap: z, and what brings them back, f0.
                    const float g0 = f0 * units_in, g1 = f1 * units_in;
#pragma unroll
                    for (int i = 0; i < 32; i += 2) of_two(mul2(two(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), i < 16 ? two(g0, g0) : two(g1, g1)), v[i], v[i + 1]);
                    f0 = f1 = units_out;
                    if (c.soft_cap > 0.0f) {
                        // Where no score of the warp passes a quarter of the cap, tanh z is z times the polynomial in z^2 that is nearest to tanh z / z on 0 .. 1/16 (within 5.1e-7 of it); else
                        // 1 - 2 / (1 + e^2z).
                        float size = 0.0f;
#pragma unroll
                        for (int i = 0; i < 32; i += 2) size = max3(size, fabsf(__uint_as_float(v[i])), fabsf(__uint_as_float(v[i + 1])));
                        if (__all_sync(0xffffffffu, size <= 0.25f)) {
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                const Two z = two(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), y = mul2(z, z);
                                of_two(mul2(z, fma2(y, fma2(y, two(0.128418818f, 0.128418818f), two(-0.333219707f, -0.333219707f)), two(0.999999642f, 0.999999642f))), v[i], v[i + 1]);
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(fmaf(-2.0f, __fdividef(1.0f, 1.0f + ex2(__uint_as_float(v[i]) * (2.0f * kLbLog2e))), 1.0f));
                        }
                    }
                    if (biased) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(fmaf(__uint_as_float(v[i]), units_out, -lb_distance_penalty_log2(r1, r2, max(place - (key0 + i), 0))));
                        f0 = f1 = 1.0f;
                    }
                }
                if (masked) {
                    // A bit a key that the row sees.
                    const int from = first - key0, to = place - key0;
                    uint32_t seen = (to >= 31 ? 0xffffffffu : to < 0 ? 0u : (2u << to) - 1u) & (from <= 0 ? 0xffffffffu : from > 31 ? 0u : ~((1u << from) - 1u));
                    if (gone0 != 0) seen &= 0xffff0000u;
                    if (gone1 != 0) seen &= 0x0000ffffu;
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = (seen >> i & 1u) != 0 ? v[i] : 0xff800000u;
                    // Times a factor that is 0 in 32 bits it would be NaN.  (What the least factor makes of a score is nothing beside 1; a NaN stays.)
                    f0 = f0 < 1e-37f ? 1e-37f : f0;
                    f1 = f1 < 1e-37f ? 1e-37f : f1;
                }
            }
            float h[2][2];
#pragma unroll
            for (int half = 0; half < 2; ++half)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    h[half][e] = __uint_as_float(v[16 * half + 8 * e]);
#pragma unroll
                    for (int i = 1; i < 7; i += 2) h[half][e] = max3(h[half][e], __uint_as_float(v[16 * half + 8 * e + i]), __uint_as_float(v[16 * half + 8 * e + i + 1]));
                    h[half][e] = fmaxf(h[half][e], __uint_as_float(v[16 * half + 8 * e + 7]));
                }
            // (A factor is not negative: a scale's sign is the query's.)
            float high = max3(fmaxf(h[0][0], h[0][1]) * f0, fmaxf(h[1][0], h[1][1]) * f1, kLowest), high_exponent = fmaxf(fmaxf(e0, e1), big);
            // O, the sum and p are relative to m, O in units of 2^big as well; where a score passes m by more than 2^8, or a block's exponent big, they move, for both threads of a row: the
            // two warps ask each other.  By then both have their scores in registers, whose place p takes.
            tc_fence_before();
            const bool moved = any_of_pair(pair_barrier, !ok || high > m + kSlack || high_exponent > big);
            tc_fence_after();
            if (moved) {
                ctl->row_high[g][x][quarter * 32 + lane] = ok ? high : CUDART_NAN_F;
                ctl->row_sum[g][x][quarter * 32 + lane] = high_exponent;
                named_barrier(pair_barrier, 64);
                const float other = ctl->row_high[g][x ^ 1][quarter * 32 + lane];
                high_exponent = fmaxf(high_exponent, ctl->row_sum[g][x ^ 1][quarter * 32 + lane]);
                if (__any_sync(0xffffffffu, isnan(other)) || !ok) {
                    ok = false;
                    break;
                }
                const float m_new = fmaxf(fmaxf(m, high), other), corr = ex2(m - m_new), corr_o = corr * ex2(big - high_exponent);
                l *= corr;
                m = m_new;
                big = high_exponent;
                if (u > lo) {
                    if (!wait(&ctl->o_done[g][(u - 1) & 1], (uint32_t)((u - 1 - lo) >> 1) & 1u, abort_flag)) {
                        give_up(ctl, status, 6);
                        bad = true;
                    }
                    tc_fence_after();
                    uint32_t w[16];
#pragma unroll 1
                    for (int i = 0; i < HD / 32; ++i) {                  // each thread half of O
                        tmem_ld16(t_o + i * 16, w);
                        tmem_ld_wait16(w);
#pragma unroll
                        for (int e = 0; e < 16; ++e) w[e] = __float_as_uint(__uint_as_float(w[e]) * corr_o);
                        tmem_st16(t_o + i * 16, w);
                    }
                }
                named_barrier(pair_barrier, 64);                         // both have read before the next are written
            }
            // p times 2^(a block's exponent less big) in one exponential; the sum of a block's is brought back.  (What lies 2^60 below the largest scale's is nothing beside it.)
            uint32_t pk[16];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const float less = fmaxf((half == 0 ? e0 : e1) - big, -60.0f), from = less - m + kUp, factor = half == 0 ? f0 : f1;
                float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    float p0, p1;
                    fma2(p0, p1, v[16 * half + i], v[16 * half + i + 1], factor, from);
                    p0 = ex2(p0);
                    p1 = ex2(p1);
                    add2(sum0, sum1, p0, p1);
                    pk[8 * half + i / 2] = h2(__floats2half2_rn(p0, p1));
                }
                l = fmaf(sum0 + sum1, ex2(-less), l);
            }
            tmem_st16(t_u + x * 16, pk);
            if (nans != 0)
                for (int i = 0; i < 32; ++i)
                    if (key0 + i <= place && key0 + i >= first) nan_bits |= ctl->nan_groups[note][(u & 1) * kUnit + 32 * x + i];
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctl->p_full[g][u & 1]);
        }
        ok = ok && !bad;
        // The last two updates may both be under way.
        if (ok && hi > lo + 1) ok = wait(&ctl->o_done[g][hi & 1], (uint32_t)((hi - 2 - lo) >> 1) & 1u, abort_flag);
        if (ok && hi > lo) ok = wait(&ctl->o_done[g][(hi - 1) & 1], (uint32_t)((hi - 1 - lo) >> 1) & 1u, abort_flag);
        if (!ok) give_up(ctl, status, 5);
        // The threads' sums meet (a thread that gave up is here too), and each has half of the row's values.
        ctl->row_sum[g][x][quarter * 32 + lane] = l;
        ctl->row_nans[g][x][quarter * 32 + lane] = (uint8_t)nan_bits;
        named_barrier(pair_barrier, 64);
        l += ctl->row_sum[g][x ^ 1][quarter * 32 + lane];
        nan_bits |= ctl->row_nans[g][x ^ 1][quarter * 32 + lane];
        if (ok && w_row < n_rows) {
            tc_fence_after();
            // A row's result; where blocks share its keys a state, normed so that its sum is 1.  (Rows whose keys are one block's share have none.)
            const bool none = l == 0.0f, whole = ctl->whole != 0;                          // no key seen: O may be what the memory held
            float* state = c.partial + ((((int64_t)seq * kv + kvh) * c.max_rows + row) * n_splits + split) * (HD + 4);
            if (!whole && there && x == 0) *reinterpret_cast<float4*>(state) = make_float4(none ? kLowest : m - kUp + log2f(l), none ? 0.0f : 1.0f, 0.0f, 0.0f);
            float factor = 1.0f;
            if (whole && c.sink != nullptr) factor = lb_sink_join_exp2(c.sink[head] * kLbLog2e, m - kUp, l);
            factor = factor / l * ex2(big * 0.5f);
            const float factor2 = ex2(big * 0.5f - 8.0f);                 // in two steps: big may be 2^127's exponent
            __nv_bfloat16* out = c.out + (int64_t)(part.first + token) * c.out_stride + (int64_t)head * HD + x * (HD / 2);
            const bool out_wide = reinterpret_cast<uintptr_t>(c.out) % 16 == 0 && c.out_stride % 8 == 0;
#pragma unroll 1
            for (int h = 0; h < HD / 64; ++h) {
                uint32_t v[32];
                tmem_ld32(t_o + h * 32, v);
                tmem_ld_wait32(v);
                const bool nan = (nan_bits >> ((x * (HD / 2) + 32 * h) / (HD / NG)) & 1u) != 0;
                auto value = [&](int i) { return none ? 0.0f : nan ? CUDART_NAN_F : __uint_as_float(v[i]) * factor * factor2; };
                if (!there) continue;
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<float4*>(state + 4 + x * (HD / 2) + 32 * h + i) = make_float4(value(i), value(i + 1), value(i + 2), value(i + 3));
                } else if (out_wide) {
#pragma unroll
                    for (int i = 0; i < 32; i += 8)
                        *reinterpret_cast<uint4*>(out + 32 * h + i) =
                            make_uint4(pack2(value(i), value(i + 1)), pack2(value(i + 2), value(i + 3)), pack2(value(i + 4), value(i + 5)), pack2(value(i + 6), value(i + 7)));
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) out[32 * h + i] = __float2bfloat16_rn(value(i));
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == kIssuer) {
        tc_fence_after();
        tmem_dealloc(tmem_base, kTmemCols);
    }
}

// The states of blocks that share a row's keys, a warp a row: bound by their bytes and by two trips to memory.
template <int HD>
__global__ void __launch_bounds__(128)
attention4_many_join_kernel(const Call c, int n_splits, int share) {
    __shared__ float joined[1][HD + 3];
    lb_wait_for_predecessor();
    lb_dependents_may_launch();
    const int seq = blockIdx.z, kvh = blockIdx.y, r = blockIdx.x * 4 + (threadIdx.x >> 5);
    const Portion part = portion_of(c, seq);
    const float* state = r < part.count * c.per ? c.partial + (((int64_t)seq * c.pages.n_kv_head + kvh) * c.max_rows + r) * n_splits * (HD + 4) : nullptr;
    int lo, all_tiles;
    keys_of_rows(c, part, r / kTileRows * kTileRows, &lo, &all_tiles);
    if (all_tiles <= share) return;                 // (a block had them all.  The rows of a thread block are of one tile, so all its threads leave.)
    join_row<HD>(c, part, seq, kvh, r, state, HD + 4, min(n_splits, max(1, (all_tiles + share - 1) / share)), 0, joined);
}

template <int HD, int NG, bool PLAIN>
int launch(const Call& c, const TilesPlan& p, cudaStream_t s) {
    int* status = nullptr;
    if (int rc = lb_tc_status_word(&status)) return rc;
    auto kernel = attention4_many_kernel<HD, NG, PLAIN>;
    constexpr int smem = 1024 + (kGroups + 2 * kStages) * (HD / 64) * kSub + (int)sizeof(Control);
    static std::atomic<uint64_t> asked{0};
    if (int rc = allow_shared(kernel, smem, asked)) return rc;
    LB_CHECK_CUDA(lb_launch_overlapped(kernel, dim3((c.max_rows + kTileRows - 1) / kTileRows * p.splits, c.pages.n_kv_head, c.n_seq), dim3(kManyThreads), smem, s, c, p.splits, p.share, status));
    if (p.splits > 1) LB_CHECK_CUDA(lb_launch_overlapped(attention4_many_join_kernel<HD>, dim3((c.max_rows + 3) / 4, c.pages.n_kv_head, c.n_seq), dim3(128), 0, s, c, p.splits, p.share));
    return LB_OK;
}

template <int HD, int NG>
int launch_for(const Call& c, const TilesPlan& p, cudaStream_t s) {
    return c.distance == nullptr && c.soft_cap <= 0.0f ? launch<HD, NG, true>(c, p, s) : launch<HD, NG, false>(c, p, s);
}

}  // namespace

TilesPlan tiles_plan(int n_seq, int n_kv_head, int per, int max_rows, int max_keys, int window, int head_dim, int n_sm) {
    const int64_t units = (int64_t)std::max(1, n_seq) * n_kv_head;
    const int tiles = (max_rows + kTileRows - 1) / kTileRows;
    // Tiles of keys that row tile i sees at most, where the rows are those of the last of max_keys tokens.
    auto keys_of = [&](int i) {
        const int last = std::max(1, max_keys - (max_rows - std::min((i + 1) * kTileRows, max_rows)) / per), all = (last + kBN - 1) / kBN;
        return window != 0 ? std::min(all, (int)std::min<int64_t>(std::abs((int64_t)window), max_keys) / kBN + (kTileRows / per + 1) / kBN + 3) : all;
    };
    const int most = keys_of(tiles - 1);
    // The time by an estimate, in microseconds: a start and an end, and what a block takes for 128 keys, little less where it has 128 rows or fewer.  Where blocks share a row tile's keys, with two tiles
    // each at least and all of them on an SM of their own, the states are written, read and joined.  (32 heads over 8 of 128, 64 tokens behind 16,384 keys: 134 us, shared 53.
    // 2 x 1,024 tokens, 12 heads of 64: 28.4 us; shared by 2, 33.8, as many rows' states take longer than the keys they save.)
    const double each = max_rows <= kBM ? (head_dim == 128 ? 2.5 : 1.9) : head_dim == 128 ? 2.9 : 2.6;
    TilesPlan p = {1, most, 0, 9.0 + std::ceil((double)(units * tiles) / n_sm) * most * each};
    const int first = units * tiles <= n_sm ? (int)std::min<int64_t>({2 * n_sm / (units * tiles) + 1, (most + 1) / 2, 32}) : 1;
    for (int s = first; s > 1; --s) {
        const int share = (most + s - 1) / s, splits = (most + share - 1) / share;
        int64_t blocks = 0, shared = 0;
        for (int i = 0; i < tiles; ++i) {
            const int n = (keys_of(i) + share - 1) / share;
            blocks += n;
            if (n > 1) shared += (int64_t)n * std::min(kTileRows, max_rows - i * kTileRows);
        }
        if (blocks * units > n_sm) continue;
        const double us = 12.0 + share * each + units * shared * (head_dim + 4) * 4 / 1.25e6;
        if (us < p.us - 3.0) p = {splits, share, units * max_rows * splits * (head_dim + 4) * 4, us};
    }
    return p;
}

int many_rows(const Call& c, int head_dim, const TilesPlan& p, cudaStream_t s) {
    if (head_dim == 64) return c.pages.groups == 1 ? launch_for<64, 1>(c, p, s) : launch_for<64, 2>(c, p, s);
    return c.pages.groups == 1 ? launch_for<128, 1>(c, p, s) : c.pages.groups == 2 ? launch_for<128, 2>(c, p, s) : launch_for<128, 4>(c, p, s);
}

}  // namespace lb_a4

// Attention over a 4-bit cache for few query rows: single tokens, drafts of a few, the last tokens of a prompt.
//
// The query rows of a request that share a key/value head (its tokens' heads, in the order of the tokens) are cut into tiles of 8 or 16.  A block serves (key range,
// key/value head and row tile, request); its warps take the range's blocks of sixteen keys in turn, each fetched by one bulk copy into a ring of the warp's own.  A
// lane finds its values there in the order of the operands (cache4.cuh) and makes float16 numbers of the nibbles: w & 0x000f000f | 0x6400 6400 is 1024 + n of two
// values, which less 1032 is n - 8, exactly.  Then
//   S^T = K q^T      mma.sync m16n8k16, rows are keys, columns query rows: sums over a group of the scales, each met by its key's scale in 32 bits;
//   p = 2^(S - m)    m a row's reference in 32 bits;
//   O^T += V^T p^T   rows are dims; p times the value's scale, rounded to float16, turned by movmatrix into the second operand, one such for each group.
// So the numbers that are multiplied are exact but for p s (2^-12, or 2^-31 of the warp's largest value scale) and queries far below their row's largest (below 2^-29 of it).  The queries come as bfloat16 and become float16
// after a power of two a row that puts their largest at 2^14; the values' scales have any size that bfloat16 has, so m is the row's largest score plus the exponent of the warp's
// largest value scale f (down to 2^-80), less 6: 2^(S - m) s is at most 2^14.  Everything is relative to m, so f leaves no trace in the result.  m moves when a score passes it by more than
// 2^8, or a scale f: the warp votes, which costs a few instructions a tile where searching the maximum cost thirty.
// The warps' states meet in shared memory in their order, the ranges' in the shared memory of a cluster (up to 16), or in memory in another launch.
#include "attention4.h"
#include "tcgen05.cuh"

#include <cuda_fp16.h>
#include <float.h>
#include <math_constants.h>

#include <algorithm>

namespace lb_a4 {
namespace {

using namespace lb_c4;

constexpr int kStages = 4;
constexpr float kLowest = -FLT_MAX;            // a reference before any score; finite, so that differences with it are numbers
constexpr float kSlack = 8.0f;                 // how far a score may pass its row's reference (base 2)
constexpr float kLeastScale = -80.0f;          // the exponent of the largest value scale, before any
constexpr float kRoom = 6.0f;                  // p s reaches 2^(kRoom + kSlack) = 2^14 of float16's 2^16; what lies 2^-30 below the largest scale loses bits

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 2^n, n in -126 .. 127.
__device__ __forceinline__ float pow2(int n) { return __uint_as_float((uint32_t)(127 + n) << 23); }
__device__ __forceinline__ uint32_t h2(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
__device__ __forceinline__ __half2 as_h2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }

// A word's values as four float16 pairs: r[i] = nibbles (i, i + 4) less 8.
__device__ __forceinline__ void pairs_of(uint32_t w, uint32_t (&r)[4]) {
    const __half2 offset = __float2half2_rn(-1032.0f), sixteenth = __float2half2_rn(0.0625f), offset16 = __float2half2_rn(-72.0f);
    const uint32_t hi = w >> 8;
    r[0] = h2(__hadd2(as_h2((w & 0x000f000fu) | 0x64006400u), offset));
    r[1] = h2(__hfma2(as_h2((w & 0x00f000f0u) | 0x64006400u), sixteenth, offset16));         // (1024 + 16 n) / 16 - 72
    r[2] = h2(__hadd2(as_h2((hi & 0x000f000fu) | 0x64006400u), offset));
    r[3] = h2(__hfma2(as_h2((hi & 0x00f000f0u) | 0x64006400u), sixteenth, offset16));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turned(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void copy_block(void* to, const void* from, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(lb_tc::smem_u32(to)), "l"(from), "r"(bytes), "r"(lb_tc::smem_u32(bar)) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t* w) {
    if constexpr (BYTES == 16) {
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else if constexpr (BYTES == 8) {
        const uint2 u = *reinterpret_cast<const uint2*>(p);
        w[0] = u.x; w[1] = u.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
}
// bfloat16 number i of a run of words.
__device__ __forceinline__ float number(const uint32_t* w, int i) { return __uint_as_float((i & 1) != 0 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16); }

template <int HD, int NT, int W>
struct Shared {
    static constexpr int kRows = 8 * NT, kState = HD + 2;
    // The warps' rings; at the end the same bytes hold [warp][row][values], then the block's own state.
    __host__ __device__ static constexpr int rings(int block) { return W * kStages * block; }
    static constexpr int kStates = (int)sizeof(float) * (W * kRows * kState + kRows * kState);
    __host__ __device__ static constexpr int bytes(int block) { return rings(block) > kStates ? rings(block) : kStates; }
};

// NG groups of scales a head, NT tiles of 8 query rows, W warps.  PLAIN: no soft cap, no penalty by distance, no scores written.
template <int HD, int NG, int NT, int W, bool PLAIN>
__global__ void __launch_bounds__(W * 32, NT == 1 ? 16 / W : 8 / W)
attention4_rows_kernel(const Call c, int n_splits, int cluster, int tiles, int* status) {
    using L = Layout<HD>;
    using S = Shared<HD, NT, W>;
    constexpr int kRows = S::kRows, kState = S::kState, kThreads = W * 32;
    constexpr int JK = HD / 32, JV = HD / 64;             // words of a lane: of a key, of a value row
    constexpr int kBlock = block_bytes(HD, NG);
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t bars[W][kStages];
    __shared__ float factor[W][kRows];
    __shared__ float block_m[kRows], block_l[kRows];

    const int split = blockIdx.x, seq = blockIdx.z, kvh = blockIdx.y / tiles, row_tile = blockIdx.y - kvh * tiles;
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    if (lane < kStages) lb_tc::mbar_init(&bars[warp][lane], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncwarp();
    lb_wait_for_predecessor();
    lb_dependents_may_launch();

    const Portion part = portion_of(c, seq);
    const int n_rows = part.count * c.per, row0 = row_tile * kRows;
    if (row0 >= n_rows) return;                            // the same for all blocks of a cluster
    const int rows_here = min(kRows, n_rows - row0);
    const int limit = min(c.max_keys, c.table_stride << c.pages.page_shift) - 1;          // no key past this place is read
    auto place_of = [&](int row) { return min(part.place + min(row, n_rows - 1) / c.per, limit); };
    const int p_lo = place_of(row0), p_hi = place_of(row0 + rows_here - 1);
    const int first_lo = p_lo < 0 ? 0 : lb_first_visible(p_lo, c.window), first_hi = p_hi < 0 ? 0 : lb_first_visible(p_hi, c.window);
    // The range's blocks of keys: all that any row sees, in equal parts.
    const int tile_lo = first_lo / kBlockKeys, all_tiles = p_hi >= 0 ? p_hi / kBlockKeys + 1 - tile_lo : 0;
    const int share = (all_tiles + n_splits - 1) / n_splits;
    const int tile0 = tile_lo + split * share, n_tiles = max(0, min(share, all_tiles - split * share));
    const int my_tiles = n_tiles > warp ? (n_tiles - warp + W - 1) / W : 0;
    const int32_t* table = c.table + (int64_t)seq * c.table_stride;

    uint8_t* ring = smem + warp * kStages * kBlock;
    int page_reg = 0;
    uint32_t missing = 0;                                  // a bit a stage: its keys are on no page
    auto tile_at = [&](int i) { return tile0 + warp + W * i; };
    auto fetch = [&](int i) {
        if ((i & 31) == 0) page_reg = i + lane < my_tiles ? table[tile_at(i + lane) * kBlockKeys >> c.pages.page_shift] : 0;
        const int64_t at = c.pages.at(__shfl_sync(0xffffffffu, page_reg, i & 31), kvh, tile_at(i) * kBlockKeys);
        const int stage = i % kStages;
        missing = (missing & ~(1u << stage)) | (at < 0 ? 1u << stage : 0u);
        if (at >= 0 && lane == 0) {
            lb_tc::mbar_expect_tx(&bars[warp][stage], kBlock);
            copy_block(ring + stage * kBlock, c.pages.memory + at, kBlock, &bars[warp][stage]);
        } else if (lane == 0) {
            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(lb_tc::smem_u32(&bars[warp][stage])) : "memory");
        }
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i)
        if (i < my_tiles) fetch(i);

    // The queries as the second operand: lane (g, t) has the dims 32 j + 8 t .. + 7 of row g, times a power of two that puts the row's largest at 2^14.
    uint32_t qf[NT][JK][4];
    float row_scale[NT][2];                                // of the rows 2 t and 2 t + 1, the accumulators' columns
    const bool q_wide = reinterpret_cast<uintptr_t>(c.q) % 16 == 0 && c.q_stride % 8 == 0;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        const int row = row0 + 8 * n + g;
        const bool there = row < n_rows;
        const __nv_bfloat16* from = c.q + (int64_t)(part.first + (there ? row / c.per : 0)) * c.q_stride + (int64_t)(kvh * c.per + (there ? row % c.per : 0)) * HD + 8 * t;
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < JK; ++j) {
            uint32_t u[4] = {0, 0, 0, 0};
            if (there && q_wide) {
                load_words<16>(reinterpret_cast<const uint8_t*>(from + 32 * j), u);
            } else if (there) {
#pragma unroll
                for (int e = 0; e < 4; ++e) u[e] = __bfloat16_as_ushort(from[32 * j + 2 * e]) | (uint32_t)__bfloat16_as_ushort(from[32 * j + 2 * e + 1]) << 16;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                qf[n][j][e] = u[e];
                top = max(top, max(u[e] & 0x7fffu, u[e] >> 16 & 0x7fffu));
            }
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^shift times the row; a row of zeros, or with values that are not finite, stays as it is.
        const int shift = top == 0 || top >= 0x7f80u ? 0 : 14 - (max((int)(top >> 7), 1) - 127);
        const float up = pow2(shift / 2), up2 = pow2(shift - shift / 2);
#pragma unroll
        for (int j = 0; j < JK; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                qf[n][j][e] = h2(__floats2half2_rn(__uint_as_float(qf[n][j][e] << 16) * up * up2, __uint_as_float(qf[n][j][e] & 0xffff0000u) * up * up2));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int s = __shfl_sync(0xffffffffu, shift, (2 * t + e) * 4);
            row_scale[n][e] = c.scale * kLbLog2e * pow2(-s / 2) * pow2(-s - -s / 2);
        }
    }
    float m[NT][2], l[NT][2], o[NT][JV * 4][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) m[n][e] = kLowest, l[n][e] = 0.0f;
#pragma unroll
        for (int i = 0; i < JV * 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][i][e] = 0.0f;
    }
    float f = kLeastScale - kRoom;
    uint32_t f_bits = (uint32_t)(127 + (int)kLeastScale) << 7;              // 2^(f + kRoom) as bfloat16: no scale seen is larger
    const lb_soft_cap capped(PLAIN ? 0.0f : c.soft_cap, 0.0f);
    const bool biased = !PLAIN && c.distance != nullptr;
    float r1[NT][2], r2[NT][2];
    int place[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int row = row0 + 8 * n + 2 * t + e;
            place[n][e] = place_of(row);
            r1[n][e] = r2[n][e] = 0.0f;
            if (biased && row < n_rows) {
                r1[n][e] = c.distance[kvh * c.per + row % c.per];
                r2[n][e] = c.distance[c.n_head + kvh * c.per + row % c.per];
            }
        }
    float* scores = PLAIN || c.scores == nullptr ? nullptr : c.scores + (((int64_t)seq * c.pages.n_kv_head + kvh) * c.max_rows + row0) * c.score_keys;

    bool gave_up = false;
    int done = 0;
    for (int i = 0; i < my_tiles; ++i) {
        const int stage = i % kStages;
        if (i + kStages - 1 < my_tiles) fetch(i + kStages - 1);
        // Bounded; one answer for the warp.
        if (!__all_sync(0xffffffffu, lb_tc::mbar_wait(&bars[warp][stage], (uint32_t)(i / kStages) & 1u, nullptr))) {
            gave_up = true;
            done = i;
            break;
        }
        const uint8_t* block = ring + stage * kBlock;
        const int key0 = tile_at(i) * kBlockKeys;
        // S^T of sixteen keys: a[0], a[1] key g and the columns 2 t and 2 t + 1, a[2], a[3] key g + 8.
        float z[NT][4];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) z[n][e] = 0.0f;
        {
            uint32_t lo[JK], hi[JK], sc[NG];                    // scales: NG of key g, then NG of key g + 8
            load_words<L::kPiece>(block + lane * L::kPiece, lo);
            load_words<L::kPiece>(block + 32 * L::kPiece + lane * L::kPiece, hi);
            load_words<4 * NG>(block + L::kScales + g * 4 * NG, sc);
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
                float a[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) a[n][e] = 0.0f;
#pragma unroll
                for (int j = gr * JK / NG; j < (gr + 1) * JK / NG; ++j) {
                    uint32_t x[4], y[4];
                    pairs_of(lo[j], x);
                    pairs_of(hi[j], y);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma_f16(a[n], x[0], y[0], x[1], y[1], qf[n][j][0], qf[n][j][1]);
                        mma_f16(a[n], x[2], y[2], x[3], y[3], qf[n][j][2], qf[n][j][3]);
                    }
                }
                const float s0 = number(sc, gr), s1 = number(sc, NG + gr);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    z[n][0] = fmaf(a[n][0], s0, z[n][0]);
                    z[n][1] = fmaf(a[n][1], s0, z[n][1]);
                    z[n][2] = fmaf(a[n][2], s1, z[n][2]);
                    z[n][3] = fmaf(a[n][3], s1, z[n][3]);
                }
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) z[n][e] *= row_scale[n][e & 1];
        if constexpr (!PLAIN) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int key = key0 + g + 8 * (e >> 1);
                    if (capped.on) z[n][e] = capped(z[n][e]);
                    if (biased) z[n][e] -= lb_distance_penalty_log2(r1[n][e & 1], r2[n][e & 1], max(place[n][e & 1] - key, 0));
                }
        }
        uint32_t vs[NG];
        load_words<4 * NG>(block + L::kScales + 32 * NG + g * 4 * NG, vs);
        const bool absent = (missing >> stage & 1u) != 0;
        if (key0 + kBlockKeys - 1 > p_lo || key0 < first_hi || absent) {
            // Keys that some row does not see: their scores are -inf, and the scales of those past every row (whatever the memory holds) 0.
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int key = key0 + g + 8 * (e >> 1), p = place[n][e & 1];
                    if (absent || key > p || key < lb_first_visible(max(p, 0), c.window)) z[n][e] = -CUDART_INF_F;
                }
#pragma unroll
            for (int i2 = 0; i2 < 2; ++i2) {
                const int key = key0 + g + 8 * i2;
                if (absent || key > p_hi || key < first_lo) {
                    if constexpr (NG == 1) {
                        vs[0] &= i2 == 0 ? 0xffff0000u : 0x0000ffffu;
                    } else {
#pragma unroll
                        for (int e = 0; e < NG / 2; ++e) vs[i2 * NG / 2 + e] = 0;
                    }
                }
            }
        }
        if constexpr (!PLAIN) {
            if (scores != nullptr) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int row = 8 * n + 2 * t + (e & 1), key = key0 + g + 8 * (e >> 1);
                        if (row < rows_here && key < c.score_keys) scores[(int64_t)row * c.score_keys + key] = z[n][e];
                    }
            }
        }
        // Does a score pass its row's reference, or a scale f?
        uint32_t top = vs[0];
#pragma unroll
        for (int e = 1; e < NG; ++e) top = __vmaxu2(top, vs[e]);
        top = max(top & 0xffffu, top >> 16);
        bool moved = top > f_bits;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) moved = moved || z[n][e] > m[n][e & 1] + kSlack;
        if (__any_sync(0xffffffffu, moved)) {
            top = __reduce_max_sync(0xffffffffu, top);
            float f_new = f;
            if (top > f_bits) {
                f_bits = (min(top, 0x7f00u) + 0x7fu) & 0x7f80u;         // the next power of two (2^127 at most; a NaN stays one whatever it is divided by)
                f_new = (float)((int)(f_bits >> 7) - 127) - kRoom;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float high = fmaxf(z[n][e], z[n][e + 2]);
#pragma unroll
                    for (int d = 4; d < 32; d *= 2) high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, d));
                    high = fmaxf(high, m[n][e]);
                    const float corr = ex2((m[n][e] - high) + (f - f_new));
                    m[n][e] = high;
                    l[n][e] *= corr;
#pragma unroll
                    for (int k = 0; k < JV * 4; ++k) {
                        o[n][k][e] *= corr;
                        o[n][k][e + 2] *= corr;
                    }
                }
            f = f_new;
        }
        uint32_t pf[NT][NG][2];                                          // p s of the groups, as the second operand
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float ref0 = m[n][0] + f, ref1 = m[n][1] + f;
            float p[4];
            p[0] = ex2(z[n][0] - ref0);
            p[1] = ex2(z[n][1] - ref1);
            p[2] = ex2(z[n][2] - ref0);
            p[3] = ex2(z[n][3] - ref1);
            l[n][0] += p[0] + p[2];
            l[n][1] += p[1] + p[3];
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
                const float s0 = number(vs, gr), s1 = number(vs, NG + gr);
                pf[n][gr][0] = turned(h2(__floats2half2_rn(p[0] * s0, p[1] * s0)));
                pf[n][gr][1] = turned(h2(__floats2half2_rn(p[2] * s1, p[3] * s1)));
            }
        }
        // O^T: lane (g, t) has the words of the keys 2 t, 2 t + 1 (x) and of those plus 8 (y).
        {
            uint32_t x[2 * JV], y[2 * JV];
            const int at = (t * 8 + L::v_turn(g, t)) * L::kPiece;
            load_words<L::kPiece>(block + L::kV + at, x);
            load_words<L::kPiece>(block + L::kV + 32 * L::kPiece + at, y);
#pragma unroll
            for (int j = 0; j < JV; ++j) {
                uint32_t a0[4], a1[4], a2[4], a3[4];
                pairs_of(__byte_perm(x[j], x[JV + j], 0x5410), a0);
                pairs_of(__byte_perm(x[j], x[JV + j], 0x7632), a1);
                pairs_of(__byte_perm(y[j], y[JV + j], 0x5410), a2);
                pairs_of(__byte_perm(y[j], y[JV + j], 0x7632), a3);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int gr = (64 * j + 32 * (k >> 1)) / (HD / NG);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_f16(o[n][j * 4 + k], a0[k], a1[k], a2[k], a3[k], pf[n][gr][0], pf[n][gr][1]);
                }
            }
        }
        __syncwarp();                                   // the stage is overwritten by the copy issued in the next trip
    }
    if (gave_up) {
        // The copies still in flight land before the block may leave (bounded as well); the result is wrong and the status word says so.
        if (lane == 0) atomicCAS(status, 0, (0xC << 12) | 1);
        for (int i = done; i < my_tiles && i < done + kStages; ++i) lb_tc::mbar_wait(&bars[warp][i % kStages], (uint32_t)(i / kStages) & 1u, nullptr);
    }

    // The warps' states: m + f, the sum and the values of a row.
    float* states = reinterpret_cast<float*>(smem);                 // [warp][row][kState]
    float* own = states + W * kRows * kState;                       // [row][kState]: the block's
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int d = 4; d < 32; d *= 2) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
    __syncthreads();                                                // the rings have been read
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            float* st = states + (warp * kRows + 8 * n + 2 * t + e) * kState;
            if (g == 0) {
                st[0] = m[n][e] + f;
                st[1] = l[n][e];
            }
#pragma unroll
            for (int j = 0; j < JV; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    *reinterpret_cast<float2*>(st + 2 + 64 * j + 32 * (k >> 1) + 4 * g + 2 * (k & 1)) = make_float2(o[n][j * 4 + k][e], o[n][j * 4 + k][e + 2]);
        }
    __syncthreads();
    if (threadIdx.x < kRows) {
        const int row = threadIdx.x;
        float mm = kLowest, ll = 0.0f;
        for (int w = 0; w < W; ++w) mm = fmaxf(mm, states[(w * kRows + row) * kState]);
        for (int w = 0; w < W; ++w) {
            const float* st = states + (w * kRows + row) * kState;
            factor[w][row] = st[1] == 0.0f ? 0.0f : exp2f(st[0] - mm);
            ll += st[1] * factor[w][row];
        }
        block_m[row] = mm;
        block_l[row] = ll;
        own[row * kState] = mm;
        own[row * kState + 1] = ll;
    }
    __syncthreads();
    const bool alone = n_splits == 1;
    const int64_t unit = ((int64_t)seq * c.pages.n_kv_head + kvh) * tiles + row_tile;
    // A row's result from its divisor's reference and sum (the sink joined) and a sum of values.
    auto finish = [&](int row, int d, float mm, float ll, float v) {
        const int r = row0 + row, head = kvh * c.per + r % c.per;
        if (c.sink != nullptr) v *= lb_sink_join_exp2(c.sink[head] * kLbLog2e, mm, ll);
        c.out[(int64_t)(part.first + r / c.per) * c.out_stride + head * HD + d] = __float2bfloat16_rn(ll == 0.0f ? 0.0f : v / ll);
        if (d == 0 && c.log_sums != nullptr) {
            const float top = c.sink != nullptr ? fmaxf(mm, c.sink[head] * kLbLog2e) : mm;
            c.log_sums[((int64_t)seq * c.pages.n_kv_head + kvh) * c.max_rows + r] = ll == 0.0f ? CUDART_INF_F : top + log2f(ll);
        }
    };
    for (int i = threadIdx.x; i < rows_here * HD; i += kThreads) {
        const int row = i / HD, d = i - row * HD;
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) v = fmaf(factor[w][row], states[(w * kRows + row) * kState + 2 + d], v);
        if (alone) finish(row, d, block_m[row], block_l[row], v);
        else if (cluster) own[row * kState + 2 + d] = v;
        else c.partial[((unit * n_splits + split) * kRows + row) * kState + 2 + d] = v;
    }
    if (alone) return;
    if (!cluster) {
        if (threadIdx.x < rows_here) {
            float* to = c.partial + ((unit * n_splits + split) * kRows + threadIdx.x) * kState;
            to[0] = block_m[threadIdx.x];
            to[1] = block_l[threadIdx.x];
        }
        return;
    }
    // The ranges' states meet: every block makes its share of the values from all blocks' shared memory.
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    const uint32_t own_at = lb_tc::smem_u32(own);
    auto remote = [&](int rank, int index) {
        uint32_t at;
        float v;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(own_at + 4u * (uint32_t)index), "r"(rank));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
        return v;
    };
    const int share_of = (rows_here * HD + n_splits - 1) / n_splits;
    for (int i = split * share_of + threadIdx.x; i < min((split + 1) * share_of, rows_here * HD); i += kThreads) {
        const int row = i / HD, d = i - row * HD;
        float mm = kLowest, ll = 0.0f, v = 0.0f;
        for (int s = 0; s < n_splits; ++s) mm = fmaxf(mm, remote(s, row * kState));
        for (int s = 0; s < n_splits; ++s) {
            const float sum = remote(s, row * kState + 1), w = sum == 0.0f ? 0.0f : exp2f(remote(s, row * kState) - mm);
            ll = fmaf(sum, w, ll);
            v = fmaf(remote(s, row * kState + 2 + d), w, v);
        }
        finish(row, d, mm, ll, v);
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The ranges' states of a row tile, where more blocks share a request's keys than a cluster has.
template <int HD>
__global__ void __launch_bounds__(256)
attention4_meet_kernel(const Call c, int n_splits, int tiles, int tile_rows) {
    constexpr int kState = HD + 2;
    lb_wait_for_predecessor();
    lb_dependents_may_launch();
    const int seq = blockIdx.z, kvh = blockIdx.y / tiles, row_tile = blockIdx.y - kvh * tiles;
    const Portion part = portion_of(c, seq);
    const int n_rows = part.count * c.per, r = row_tile * tile_rows + blockIdx.x, d = threadIdx.x;
    if (r >= n_rows || (int)blockIdx.x >= tile_rows || d >= HD) return;
    const int64_t unit = ((int64_t)seq * c.pages.n_kv_head + kvh) * tiles + row_tile;
    const float* from = c.partial + (unit * n_splits * tile_rows + blockIdx.x) * kState;
    const int64_t step = (int64_t)tile_rows * kState;
    float mm = kLowest, ll = 0.0f, v = 0.0f;
    for (int s = 0; s < n_splits; ++s) mm = fmaxf(mm, from[s * step]);
    for (int s = 0; s < n_splits; ++s) {
        const float sum = from[s * step + 1], w = sum == 0.0f ? 0.0f : exp2f(from[s * step] - mm);
        ll = fmaf(sum, w, ll);
        v = fmaf(from[s * step + 2 + d], w, v);
    }
    const int head = kvh * c.per + r % c.per;
    float top = mm;
    if (c.sink != nullptr) {
        top = fmaxf(mm, c.sink[head] * kLbLog2e);
        v *= lb_sink_join_exp2(c.sink[head] * kLbLog2e, mm, ll);
    }
    c.out[(int64_t)(part.first + r / c.per) * c.out_stride + head * HD + d] = __float2bfloat16_rn(ll == 0.0f ? 0.0f : v / ll);
    if (d == 0 && c.log_sums != nullptr) c.log_sums[((int64_t)seq * c.pages.n_kv_head + kvh) * c.max_rows + r] = ll == 0.0f ? CUDART_INF_F : top + log2f(ll);
}

template <int HD, int NG, int NT, int W, bool PLAIN>
int launch(const Call& c, const RowsPlan& p, cudaStream_t s) {
    using S = Shared<HD, NT, W>;
    int* status = nullptr;
    if (int rc = lb_tc_status_word(&status)) return rc;
    auto kernel = attention4_rows_kernel<HD, NG, NT, W, PLAIN>;
    const int smem = S::bytes(block_bytes(HD, NG));
    LB_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (p.cluster && p.splits > 8) LB_CHECK_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    const dim3 grid(p.splits, c.pages.n_kv_head * p.tiles, c.n_seq);
    LB_CHECK_CUDA(lb_launch_overlapped_cluster(0, p.cluster ? p.splits : 1, kernel, grid, dim3(W * 32), smem, s, c, p.splits, p.cluster, p.tiles, status));
    if (p.splits > 1 && !p.cluster) {
        const dim3 rows(p.rows, c.pages.n_kv_head * p.tiles, c.n_seq);
        LB_CHECK_CUDA(lb_launch_overlapped(attention4_meet_kernel<HD>, rows, dim3(HD), 0, s, c, p.splits, p.tiles, p.rows));
    }
    return LB_OK;
}

template <int HD, int NG>
int launch_for(const Call& c, const RowsPlan& p, cudaStream_t s) {
    const bool plain = c.distance == nullptr && c.soft_cap <= 0.0f && c.scores == nullptr;
    if (p.rows == 8) return plain ? launch<HD, NG, 1, 8, true>(c, p, s) : launch<HD, NG, 1, 8, false>(c, p, s);
    return plain ? launch<HD, NG, 2, 8, true>(c, p, s) : launch<HD, NG, 2, 8, false>(c, p, s);
}

}  // namespace

RowsPlan rows_plan(int n_seq, int n_kv_head, int max_rows, int max_keys, int head_dim, int n_sm) {
    (void)head_dim;
    RowsPlan p;
    p.rows = max_rows > 8 ? 16 : 8;
    p.tiles = (max_rows + p.rows - 1) / p.rows;
    p.warps = 8;
    // Two blocks an SM; a range of fewer than 128 keys has no work for eight warps.
    const int64_t work = std::max<int64_t>(1, (int64_t)n_seq * n_kv_head * p.tiles);
    const int64_t want = std::min<int64_t>((2 * n_sm + work - 1) / work, std::max(1, max_keys / 128));
    p.splits = want > 16 ? (int)std::min<int64_t>(want, 64) : want > 8 ? 16 : (int)std::max<int64_t>(1, want);
    p.cluster = p.splits > 1 && p.splits <= 16;
    return p;
}

int few_rows(const Call& c, int head_dim, const RowsPlan& p, cudaStream_t s) {
    if (head_dim == 64) return c.pages.groups == 1 ? launch_for<64, 1>(c, p, s) : launch_for<64, 2>(c, p, s);
    return c.pages.groups == 1 ? launch_for<128, 1>(c, p, s) : c.pages.groups == 2 ? launch_for<128, 2>(c, p, s) : launch_for<128, 4>(c, p, s);
}

}  // namespace lb_a4

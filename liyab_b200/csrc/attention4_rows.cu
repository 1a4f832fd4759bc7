// Attention over a 4-bit cache for few query rows: single tokens, drafts of a few, the last tokens of a prompt.
//
// The query rows of a request that share a key/value head (its tokens' heads, in the order of the tokens) are cut into tiles of 4 or 8.  A warp takes blocks of sixteen keys in pairs, each
// block fetched by one bulk copy into a ring of the warp's own.  A lane finds its values there in the order of the operands (cache4.cuh).  Then
//   S^T = K q^T      mma.sync m16n8k32 on bytes: the first operand is n + 8 as it lies (a mask, a shift), the second a row of queries as whole numbers of 16 bits in two digits, so a
//                    column is a row's digit.  The sums start at -8 times the digits' sum and at the bits of a float, so that two subtractions and a multiply-add make the number; each group's
//                    meets its key's scale in 32 bits;
//   p = 2^(S - m)    m a row's reference in 32 bits;
//   O^T += V^T p^T   mma.sync m16n8k16 on float16: rows are dims, n - 8 made of the nibbles exactly (w & 0x000f000f | 0x64006400 is 1024 + n of two values, less 1032); p times the value's
//                    scale, rounded to float16, turned by movmatrix into the second operand.
// What is rounded: p s to float16 (2^-12, or 2^-31 of the warp's largest value scale), and queries more than 2^6 below their row's largest (to 2^-15 of it); a row's 16 bits hold bfloat16's
// eight of all others.  A power of two a row puts its largest at 2^14.  The values' scales have any size that bfloat16 has, so they are taken in units of 2^f, f the exponent of the warp's largest
// (2^-120 at least), less 6: 2^(S - m) s is at most 2^14.  p takes 2^-f along as far as that leaves it and its sum well within float32's range, f in -40 .. 40; what is beyond, the scales are multiplied
// by.  A state's sum is relative to m alone, and it carries f, which is O's.  m moves when a score passes it by more than 2^8, or a scale f: the warp votes, which costs a few instructions a pair where
// searching the maximum cost thirty a tile.  A scale that is NaN (of a group that was not finite) is no f and no factor: it would meet p = 0 of rows that do not see its key.  It passes every f, so it
// is met where the warp has voted: its products are 0, and the sums of the rows that see it are NaN from there on.
//
// Two ways to share the keys out (rows_plan chooses by an estimate of both).  WHOLE: a block has a request's row tile and key/value head, its eight warps a stretch of the keys each, whose states meet
// in shared memory and become the result: no scratch memory, one launch.  Else all warps of the launch take equal shares of all tiles of all requests (256 at most to a launch row), wherever they
// begin and end, and another launch joins the states of a row's runs in their order.
//
// What bounds it.  A block of sixteen keys takes some 257 instructions for heads of 128 with four rows, most of them on the pipe for integers and halves at two cycles each, so the GPU gets through
// 5.1 TB/s of cache (heads of 64: 4.3), 0.78 of the copy bandwidth, after a start of 8 us (requests, block tables, first keys, queries: four trips to memory, and the launch)
// and before a join of 3 to 6.  8 requests on 16,384 keys, 32 heads over 8 of 128: 38 us, 3.8 TB/s; 64 on 1,024, 25 heads of 64: 31.5 us; 1 on 131,072: 38; 1 on 512, 25 heads of 64: 5.5.
// Float16 products for K as well, a tile at a time, took 67 us for the first, with a block to a range of one request's keys.  Five blocks of four warps an SM for heads of 64, not four: 34.8 us for the
// second against 32.0; twice the blocks for the third 47 against 38.7; tiles of sixteen rows lose to two of eight, as their registers leave half the warps; a third pair in the ring changes nothing.
#include "attention4.h"
#include "attention4_join.cuh"
#include "attention4_parts.cuh"

#include <float.h>
#include <math_constants.h>

#include <algorithm>
#include <cmath>
#include <limits>

namespace lb_a4 {
namespace {

using namespace lb_c4;

constexpr int kStages = 2;                     // pairs of tiles in a warp's ring
constexpr float kSlack = 8.0f;                 // how far a score may pass its row's reference (base 2)
constexpr int kLeastScale = -120;              // the exponent of the largest value scale, before any
constexpr int kEven = 40;                      // of f, p has -kEven .. kEven
constexpr int kRoom = 6;                       // p s reaches 2^(kRoom + kSlack) = 2^14 of float16's 2^16; what lies 2^-30 below the largest scale loses bits

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
constexpr float kMagic = 12582912.0f;          // 1.5 2^23
// Sums of products of bytes, n + 8 by a query's digit.  kSumBits: the bits of 1.5 2^11, after which integers up to 2^22 either way are the bits of that number plus themselves in units of 2^-12: a sum,
// 2^25 at most, times a key's scale stays within float32's range for scales up to 2^114 (in units of 1 up to 2^102).
constexpr int kSumBits = 0x45400000, kSumUnit = 12;
constexpr float kSum = 3072.0f;
__device__ __forceinline__ void mma_u8s8_first(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, int c0, int c1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %10, %11};"
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c0), "r"(c1));
}
__device__ __forceinline__ void mma_u8s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
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
// Two bfloat16 numbers times a power of two, exact but below the smallest normal number.
__device__ __forceinline__ uint32_t scaled(uint32_t v, uint32_t by) {
    const __nv_bfloat162 y = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&by));
    return *reinterpret_cast<const uint32_t*>(&y);
}
// A block's warps.
__host__ __device__ constexpr int warps_of(int nt, bool whole) { return whole || nt == 1 ? 8 : 4; }
constexpr int kMostRequests = 256;             // of a launch row (grid.y)
constexpr int kLeastTiles = 4;                 // of a warp

// Blocks an SM.  (Heads of 64 have registers for three with one tile of rows: 64 x 1024 keys 34.8 us against 32.0.)
__host__ __device__ constexpr int blocks_per_sm(int hd, int nt, bool whole) { return nt == 1 ? 2 : whole ? 1 : hd == 64 ? 4 : 3; }

// The blocks of keys of a request that any of its rows sees: the first and how many.
__device__ __forceinline__ void tiles_of(const Call& c, const Portion& p, int* first, int* count) {
    const int limit = min(c.max_keys, c.table_stride << c.pages.page_shift) - 1;
    const int lo = min(p.place, limit), hi = p.count > 0 ? min(p.place + p.count - 1, limit) : -1;
    *first = lo < 0 ? 0 : lb_first_visible(lo, c.window) / kBlockKeys;
    *count = hi < 0 ? 0 : hi / kBlockKeys + 1 - *first;
}

// A request of a launch row: its tokens, its first tile of keys and how many, its row tiles for each key/value head.
struct Request {
    Portion part;
    int first, count, in_row;
};

// How many tiles a warp takes, of `total` in its launch row.
__host__ __device__ __forceinline__ int share_of(int total, int n_warps) {
    const int even = (total + n_warps - 1) / n_warps;
    return even > kLeastTiles ? even : kLeastTiles;
}

// NG groups of scales a head, NT tiles of 4 query rows (two digits each).  PLAIN: no soft cap, no penalty by distance, no scores written.  WHOLE: a block has one request's (blockIdx.y) row tile
// and key/value head (blockIdx.x), whose keys its warps share out and whose result it makes itself; else the states of the warps' runs meet in another launch.
template <int HD, int NG, int NT, bool PLAIN, bool WHOLE>
__global__ void __launch_bounds__(warps_of(NT, WHOLE) * 32, blocks_per_sm(HD, NT, WHOLE))
attention4_rows_kernel(const Call c, int per_row, int tiles, int* status) {
    using L = Layout<HD>;
    constexpr int kRows = 4 * NT, kState = HD + 4;         // a state is a reference, a sum, the values' unit, a place, the values
    constexpr int JK = HD / 32, JV = HD / 64;             // words of a lane: of a key, of a value row
    constexpr int kBlock = block_bytes(HD, NG), kWarps = warps_of(NT, WHOLE);
    // The columns of V^T p^T: with four rows a pair of columns is a row times the scales of two groups, else two rows, an operand for each group.
    constexpr int VT = NT == 1 ? 1 : NT / 2, VG = NT == 1 ? (NG + 1) / 2 : NG;
    // The warps' rings, (WHOLE) their states, then the list of requests, behind where their tiles start in the row's order.
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t bars[kWarps][kStages];
    __shared__ int found[kWarps][64];                      // the cache's blocks of the tiles to come; -1: on no page
    float* states = reinterpret_cast<float*>(smem + kWarps * kStages * 2 * kBlock);
    int* starts = reinterpret_cast<int*>(states + (WHOLE ? kWarps * kRows * kState : 0));
    Request* requests = reinterpret_cast<Request*>(starts + per_row + 1);

    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int seq0 = blockIdx.y * per_row, n_seq = min(per_row, c.n_seq - seq0), kv = c.pages.n_kv_head;
    if (lane < kStages) lb_tc::mbar_init(&bars[warp][lane], 2);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    lb_wait_for_predecessor();
    lb_dependents_may_launch();
    if (warp == 0) {
        int sum = 0;
        for (int s0 = 0; s0 < n_seq; s0 += 32) {
            const int s = s0 + lane;
            int mine = 0;
            if (s < n_seq) {
                Request r;
                r.part = portion_of(c, seq0 + s);
                tiles_of(c, r.part, &r.first, &r.count);
                r.in_row = c.q_start == nullptr ? tiles : r.part.count > 0 ? (r.part.count * c.per + kRows - 1) / kRows : 0;
                requests[s] = r;
                mine = kv * r.in_row * r.count;
            }
            int before = mine;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const int v = __shfl_up_sync(0xffffffffu, before, o);
                if (lane >= o) before += v;
            }
            if (s < n_seq) starts[s] = sum + before - mine;
            sum += __shfl_sync(0xffffffffu, before, 31);
        }
        if (lane == 0) starts[n_seq] = sum;
    }
    __syncthreads();
    const int total = starts[n_seq], n_warps = gridDim.x * kWarps, me = blockIdx.x * kWarps + warp;
    int begin, end;
    if constexpr (WHOLE) {
        if ((int)blockIdx.x >= kv * requests[0].in_row) return;
        const int count = requests[0].count, share = (count + kWarps - 1) / kWarps;
        begin = blockIdx.x * count + min(warp * share, count);
        end = blockIdx.x * count + min((warp + 1) * share, count);
    } else {
        const int share = share_of(total, n_warps);
        if (blockIdx.x == 0)                                // for the launch that joins the states
            for (int s = threadIdx.x; s <= n_seq; s += kWarps * 32) c.starts[(int64_t)blockIdx.y * (per_row + 1) + s] = starts[s];
        begin = min((int64_t)me * share, (int64_t)total);
        end = min((int64_t)(me + 1) * share, (int64_t)total);
        if (begin >= end) return;
    }
    // The request that tile x of the row belongs to.
    auto request_of = [&](int x) {
        int lo = 0, hi = n_seq - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (starts[mid] <= x) lo = mid;
            else hi = mid - 1;
        }
        return lo;
    };
    uint8_t* ring = smem + warp * kStages * 2 * kBlock;
    const int n_tiles = end - begin;
    // Tiles come in pairs, counted from the warp's first: a barrier a pair, on which two lanes arrive with a tile each.
    const int n_pairs = (n_tiles + 1) >> 1;
    int listed = 0, asked = 0;                             // tiles whose blocks are found, pairs asked for
    bool all_there = true;                                 // no tile listed so far is on no page
    auto fetch = [&]() {
        if (asked >= n_pairs) return;
        if (2 * asked + 2 > listed) {
            const int x = begin + listed + lane;
            int at = -1;
            if (x < end) {
                const int s = request_of(x), count = requests[s].count, in_row = requests[s].in_row;
                const int unit = (x - starts[s]) / count, tile = requests[s].first + x - starts[s] - unit * count, kvh = in_row == 1 ? unit : unit / in_row;
                const int page = c.table[(int64_t)(seq0 + s) * c.table_stride + (tile * kBlockKeys >> c.pages.page_shift)];
                if ((unsigned)page < (unsigned)c.pages.n_pages) at = ((page * kv + kvh) << (c.pages.page_shift - 4)) + (tile & ((1 << (c.pages.page_shift - 4)) - 1));
            }
            found[warp][(listed + lane) & 63] = at;
            all_there = all_there && __all_sync(0xffffffffu, at >= 0 || x >= end);
            listed += 32;
            __syncwarp();
        }
        if (lane < 2 - c.withhold) {
            const int stage = asked % kStages, at = found[warp][(2 * asked + lane) & 63];
            if (at >= 0) {
                lb_tc::mbar_expect_tx(&bars[warp][stage], kBlock);
                copy_block(ring + (2 * stage + lane) * kBlock, c.pages.memory + (int64_t)at * kBlock, kBlock, &bars[warp][stage]);
            } else {
                asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(lb_tc::smem_u32(&bars[warp][stage])) : "memory");
            }
        }
        ++asked;
        __syncwarp();
    };
#pragma unroll 1
    for (int i = 0; i < kStages; ++i) fetch();

    const lb_soft_cap capped(PLAIN ? 0.0f : c.soft_cap, 0.0f);
    const bool biased = !PLAIN && c.distance != nullptr;
    const int limit = min(c.max_keys, c.table_stride << c.pages.page_shift) - 1;          // no key past this place is read
    const bool q_wide = reinterpret_cast<uintptr_t>(c.q) % 16 == 0 && c.q_stride % 8 == 0;
    bool gave_up = false;
    int done = 0;
    // A run: the tiles of one request, key/value head and row tile.
    while (done < n_tiles && !gave_up) {
        const int s = request_of(begin + done), seq = seq0 + s;
        const Portion part = requests[s].part;
        const int in_row = requests[s].in_row, count = requests[s].count;
        const int unit = (begin + done - starts[s]) / count, kvh = in_row == 1 ? unit : unit / in_row, row_tile = unit - kvh * in_row;
        const int tile0 = requests[s].first + begin + done - starts[s] - unit * count;
        const int run_end = min(n_tiles, starts[s] + (unit + 1) * count - begin), run_begin = done;
        const int n_rows = part.count * c.per, row0 = row_tile * kRows, rows_here = min(kRows, n_rows - row0);
        auto token_of = [&](int row) { return part.count == 1 ? 0 : row / c.per; };
        auto place_of = [&](int row) { return min(part.place + token_of(min(row, n_rows - 1)), limit); };
        const int p_lo = place_of(row0), p_hi = place_of(row0 + rows_here - 1);
        const int first_lo = p_lo < 0 ? 0 : lb_first_visible(p_lo, c.window), first_hi = p_hi < 0 ? 0 : lb_first_visible(p_hi, c.window);

        // The queries as the second operand: columns are (row, digit).  A row times a power of two, so that its largest is in 2^14 .. 2^15, is rounded to 16 bits, 256 high + low, both
        // -128 .. 127; lane (g, t) has digit g % 2 of the dims 32 j + 8 t .. + 7 of row g / 2, in the order of the nibbles of a key's word.  An operand's keys are n + 8, so the sums start
        // at -8 times the digits' sum, and at the bits of 1.5 2^11: what they come to is a float's bits.
        uint32_t qd[NT][JK][2];
        int base[NT][NG][2];                                   // of columns 2 t and 2 t + 1: high and low digit of row t
        float row_scale[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int row = row0 + 4 * n + (g >> 1);
            const bool there = row < n_rows;
            const int token = there ? token_of(row) : 0, head = there ? row - token * c.per : 0;
            const __nv_bfloat16* from = c.q + (int64_t)(part.first + token) * c.q_stride + (int64_t)(kvh * c.per + head) * HD + 8 * t;
            uint32_t top = 0, u[JK][4];
#pragma unroll
            for (int j = 0; j < JK; ++j) {
#pragma unroll
                for (int e = 0; e < 4; ++e) u[j][e] = 0;
                if (there && q_wide) {
                    load_words<16>(reinterpret_cast<const uint8_t*>(from + 32 * j), u[j]);
                } else if (there) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) u[j][e] = __bfloat16_as_ushort(from[32 * j + 2 * e]) | (uint32_t)__bfloat16_as_ushort(from[32 * j + 2 * e + 1]) << 16;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) top = max(top, max(u[j][e] & 0x7fffu, u[j][e] >> 16 & 0x7fffu));
            }
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // (A largest value of eight ones, 32,640 of 2^15, would have a high digit of 128: it goes a bit lower.)  A row that is not finite has NaN for a factor.
            const int shift = top == 0 || top >= 0x7f80u ? 0 : 14 - (max((int)(top >> 7), 1) - 127) - ((top & 0x7fu) == 0x7fu);
            const float up = pow2(shift / 2), up2 = pow2(shift - shift / 2);
            // x 2^shift + 1.5 2^23 has the 16 bits below: byte 0 is the low digit, byte 1, with the carry of a negative low one, the high digit.
            const uint32_t carry = (g & 1) != 0 ? 0u : 0x80u, pick = (g & 1) != 0 ? 0x40u : 0x51u;
            int sums[JK];
#pragma unroll
            for (int j = 0; j < JK; ++j) {
                uint32_t v[8];
#pragma unroll
                for (int d = 0; d < 8; ++d) {
                    const float x = __uint_as_float((d & 1) != 0 ? u[j][d / 2] & 0xffff0000u : u[j][d / 2] << 16);
                    v[d] = __float_as_uint(fmaf(top >= 0x7f80u ? 0.0f : x * up, up2, kMagic)) + carry;
                }
                auto four = [&](int a, int b, int cc, int dd) { return __byte_perm(__byte_perm(v[a], v[b], pick), __byte_perm(v[cc], v[dd], pick), 0x5410u); };
                qd[n][j][0] = four(0, 4, 1, 5);                 // nibbles 0, 2, 4, 6
                qd[n][j][1] = four(2, 6, 3, 7);                 // nibbles 1, 3, 5, 7
                sums[j] = __dp4a((int)qd[n][j][0], 0x01010101, __dp4a((int)qd[n][j][1], 0x01010101, 0));
                sums[j] += __shfl_xor_sync(0xffffffffu, sums[j], 1);
                sums[j] += __shfl_xor_sync(0xffffffffu, sums[j], 2);
            }
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
                int sum = 0;
#pragma unroll
                for (int j = gr * JK / NG; j < (gr + 1) * JK / NG; ++j) sum += sums[j];
#pragma unroll
                for (int e = 0; e < 2; ++e) base[n][gr][e] = kSumBits - 8 * __shfl_sync(0xffffffffu, sum, (2 * t + e) * 4);
            }
            const int sh = __shfl_sync(0xffffffffu, shift, 8 * t) - kSumUnit;
            const uint32_t row_top = __shfl_sync(0xffffffffu, top, 8 * t);
            row_scale[n] = row_top >= 0x7f80u ? CUDART_NAN_F : c.scale * kLbLog2e * pow2(-sh / 2) * pow2(-sh - -sh / 2);
        }
        // m: a row's largest score, or near it; ref: m and p's share of f, what scores are taken relative to; passes: m and the slack.
        float m[NT], l[NT], ref[NT], passes[NT], o[VT][JV * 4][4];
#pragma unroll
        for (int n = 0; n < NT; ++n) m[n] = ref[n] = passes[n] = kLowest, l[n] = 0.0f;
#pragma unroll
        for (int n = 0; n < VT; ++n)
#pragma unroll
            for (int i = 0; i < JV * 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][i][e] = 0.0f;
        int f = kLeastScale - kRoom;
        uint32_t most_bits = 0;                                                 // 2^(f + kRoom) as bfloat16: a scale that is larger moves f; 0 where every pair's scales are to be multiplied
        auto share_of_p = [](int units) { return min(max(units, -kEven), kEven); };
        float r1[NT], r2[NT];
        int place[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int row = row0 + 4 * n + t;
            place[n] = place_of(row);
            r1[n] = r2[n] = 0.0f;
            if (biased && row < n_rows) {
                const int head = kvh * c.per + row - token_of(row) * c.per;
                r1[n] = c.distance[head];
                r2[n] = c.distance[c.n_head + head];
            }
        }
        float* scores = PLAIN || c.scores == nullptr ? nullptr : c.scores + (((int64_t)seq * kv + kvh) * c.max_rows + row0) * c.score_keys;

        int stage = (done >> 1) % kStages;
        uint32_t parity = (uint32_t)((done >> 1) / kStages) & 1u;
        while (done < run_end) {
            // A pair of tiles; where the run begins or ends within one, the other of its two is masked.
            const int pair = done >> 1;
            if (!wait(&bars[warp][stage], parity, nullptr)) {               // bounded; one answer for the warp
                gave_up = true;
                break;
            }
            const int key0 = (tile0 + 2 * pair - run_begin) * kBlockKeys;
            const uint8_t* block = ring + 2 * stage * kBlock;
            const bool half = 2 * pair < run_begin || 2 * pair + 2 > run_end;
            float z[NT][2][2];                                     // [tile][key g, key g + 8] of row t
            uint32_t vs[2][NG];                                    // the values' scales: NG of key g, then NG of key g + 8
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                uint32_t lo[JK], hi[JK], sc[NG];
                load_words<L::kPiece>(block + u * kBlock + lane * L::kPiece, lo);
                load_words<L::kPiece>(block + u * kBlock + 32 * L::kPiece + lane * L::kPiece, hi);
                load_words<4 * NG>(block + u * kBlock + L::kScales + g * 4 * NG, sc);
                load_words<4 * NG>(block + u * kBlock + L::kScales + 32 * NG + g * 4 * NG, vs[u]);
#pragma unroll
                for (int gr = 0; gr < NG; ++gr) {
                    int a[NT][4];
#pragma unroll
                    for (int j = gr * JK / NG; j < (gr + 1) * JK / NG; ++j) {
                        const uint32_t a0 = lo[j] & 0x0f0f0f0fu, a1 = hi[j] & 0x0f0f0f0fu, a2 = lo[j] >> 4 & 0x0f0f0f0fu, a3 = hi[j] >> 4 & 0x0f0f0f0fu;
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            if (j == gr * JK / NG) mma_u8s8_first(a[n], a0, a1, a2, a3, qd[n][j][0], qd[n][j][1], base[n][gr][0], base[n][gr][1]);
                            else mma_u8s8(a[n], a0, a1, a2, a3, qd[n][j][0], qd[n][j][1]);
                        }
                    }
                    const float s0 = number(sc, gr), s1 = number(sc, NG + gr);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float k0 = fmaf(__int_as_float(a[n][0]) - kSum, 256.0f, __int_as_float(a[n][1]) - kSum);
                        const float k1 = fmaf(__int_as_float(a[n][2]) - kSum, 256.0f, __int_as_float(a[n][3]) - kSum);
                        z[n][u][0] = gr == 0 ? k0 * s0 : fmaf(k0, s0, z[n][u][0]);
                        z[n][u][1] = gr == 0 ? k1 * s1 : fmaf(k1, s1, z[n][u][1]);
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        z[n][u][e] *= row_scale[n];
                        if constexpr (!PLAIN) {
                            if (capped.on) z[n][u][e] = capped(z[n][u][e]);
                            if (biased) z[n][u][e] -= lb_distance_penalty_log2(r1[n], r2[n], max(place[n] - (key0 + 16 * u + g + 8 * e), 0));
                        }
                    }
            }
            if (key0 + 2 * kBlockKeys - 1 > p_lo || key0 < first_hi || half || !all_there) {
                // Keys that some row does not see: their scores are -inf, and the scales of those past every row (whatever the memory holds) 0.
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int key = key0 + 16 * u + g + 8 * e;
                        const bool absent = 2 * pair + u < run_begin || 2 * pair + u >= run_end || found[warp][(2 * pair + u) & 63] < 0;
#pragma unroll
                        for (int n = 0; n < NT; ++n)
                            if (absent || key > place[n] || key < lb_first_visible(max(place[n], 0), c.window)) z[n][u][e] = -CUDART_INF_F;
                        if (absent || key > p_hi || key < first_lo) {
                            if constexpr (NG == 1) {
                                vs[u][0] &= e == 0 ? 0xffff0000u : 0x0000ffffu;
                            } else {
#pragma unroll
                                for (int i = 0; i < NG / 2; ++i) vs[u][e * NG / 2 + i] = 0;
                            }
                        }
                    }
            }
            if constexpr (!PLAIN) {
                if (scores != nullptr) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int u = 0; u < 2; ++u)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const int row = 4 * n + t, key = key0 + 16 * u + g + 8 * e;
                                if (row < rows_here && 2 * pair + u >= run_begin && 2 * pair + u < run_end && key < c.score_keys) scores[(int64_t)row * c.score_keys + key] = z[n][u][e];
                            }
                }
            }
            // Does a score pass its row's reference, or a scale f?
            uint32_t top = __vmaxu2(vs[0][0], vs[1][0]);
#pragma unroll
            for (int i = 1; i < NG; ++i) top = __vmaxu2(top, __vmaxu2(vs[0][i], vs[1][i]));
            bool moved = (top >> 16) > most_bits || (top & 0xffffu) > most_bits;
#pragma unroll
            for (int n = 0; n < NT; ++n) moved = moved || fmaxf(fmaxf(z[n][0][0], z[n][0][1]), fmaxf(z[n][1][0], z[n][1][1])) > passes[n];
            if (__any_sync(0xffffffffu, moved)) {
                top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
                if (top >= 0x7f80u) {
                    // A scale that is NaN is 0 in the products, and what the rows that see its key have of the group's dims becomes NaN, which no later factor or sum changes.
                    uint32_t nans = 0;                          // a bit a row and group
                    top = 0;
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int i = 0; i < 2 * NG; ++i) {
                            const uint32_t half_word = i % 2 != 0 ? 0xffff0000u : 0x0000ffffu;
                            if ((vs[u][i / 2] & half_word & 0x7fff7fffu) >= (0x7f807f80u & half_word)) {
                                vs[u][i / 2] &= ~half_word;
#pragma unroll
                                for (int n = 0; n < NT; ++n) nans |= z[n][u][i / NG] != -CUDART_INF_F ? 1u << (n * NG + i % NG) : 0u;
                            }
                            if (i % 2 != 0) top = __vmaxu2(top, vs[u][i / 2]);
                        }
                    top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
#pragma unroll
                    for (int d = 4; d < 32; d *= 2) nans |= __shfl_xor_sync(0xffffffffu, nans, d);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int k = 0; k < JV * 4; ++k) {
                            const int gr = (64 * (k / 4) + 32 * (k % 4 >> 1)) / (HD / NG), e = NT == 1 ? gr & 1 : n & 1;
                            if ((nans >> (n * NG + gr) & 1u) != 0) o[n / 2][k][e] = o[n / 2][k][e + 2] = CUDART_NAN_F;
                        }
                }
                const int f_old = f;
                f = max(f, (int)((min(top, 0x7f00u) + 0x7fu) >> 7) - 127 - kRoom);             // the next power of two (2^127 at most)
                const int of_p = share_of_p(f);
                most_bits = f == of_p ? (uint32_t)(127 + kRoom + f) << 7 : 0;
                if (f != of_p) {
                    const uint32_t by = (uint32_t)(127 - (f - of_p)) * 0x00800080u;            // a power of two, twice
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int i = 0; i < NG; ++i) vs[u][i] = scaled(vs[u][i], by);
                }
                float corr[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float high = fmaxf(fmaxf(z[n][0][0], z[n][0][1]), fmaxf(z[n][1][0], z[n][1][1]));
#pragma unroll
                    for (int d = 4; d < 32; d *= 2) high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, d));
                    high = fmaxf(high, m[n]);
                    corr[n] = ex2((m[n] - high) + (float)(f_old - f));
                    l[n] *= ex2((m[n] - high) + (float)(share_of_p(f_old) - of_p));
                    m[n] = high;
                    ref[n] = high + (float)of_p;
                    passes[n] = high + kSlack;
                }
#pragma unroll
                for (int v = 0; v < VT; ++v)
#pragma unroll
                    for (int k = 0; k < JV * 4; ++k)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[v][k][e] *= NT == 1 ? corr[0] : corr[(2 * v + (e & 1)) % NT];
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                uint32_t pf[VT][VG][2];                                          // p s, as the second operand
                float p[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    p[n][0] = ex2(z[n][u][0] - ref[n]);
                    p[n][1] = ex2(z[n][u][1] - ref[n]);
                    l[n] += p[n][0] + p[n][1];
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float sv[NG];
#pragma unroll
                    for (int gr = 0; gr < NG; ++gr) sv[gr] = number(vs[u], e * NG + gr);
#pragma unroll
                    for (int v = 0; v < VT; ++v)
#pragma unroll
                        for (int x = 0; x < VG; ++x)
                            pf[v][x][e] = turned(h2(NT == 1 ? __floats2half2_rn(p[0][e] * sv[2 * x], p[0][e] * sv[(2 * x + 1) % NG])
                                                            : __floats2half2_rn(p[2 * v][e] * sv[x % NG], p[(2 * v + 1) % NT][e] * sv[x % NG])));
                }
                // V^T p^T: lane (g, t) has the words of the keys 2 t, 2 t + 1 (x) and of those plus 8 (y).
                uint32_t x[2 * JV], y[2 * JV];
                const int at = (t * 8 + L::v_turn(g, t)) * L::kPiece;
                load_words<L::kPiece>(block + u * kBlock + L::kV + at, x);
                load_words<L::kPiece>(block + u * kBlock + L::kV + 32 * L::kPiece + at, y);
#pragma unroll
                for (int j = 0; j < JV; ++j) {
                    __half2 a0[4], a1[4], a2[4], a3[4];
                    pairs_of(__byte_perm(x[j], x[JV + j], 0x5410), a0);
                    pairs_of(__byte_perm(x[j], x[JV + j], 0x7632), a1);
                    pairs_of(__byte_perm(y[j], y[JV + j], 0x5410), a2);
                    pairs_of(__byte_perm(y[j], y[JV + j], 0x7632), a3);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int gr = (64 * j + 32 * (k >> 1)) / (HD / NG), x2 = NT == 1 ? gr / 2 : gr;
#pragma unroll
                        for (int v = 0; v < VT; ++v) mma_f16(o[v][j * 4 + k], h2(a0[k]), h2(a1[k]), h2(a2[k]), h2(a3[k]), pf[v][x2][0], pf[v][x2][1]);
                    }
                }
            }
            __syncwarp();                                   // the pair is overwritten by the copies asked for next
            done = min(2 * pair + 2, run_end);
            if ((done & 1) == 0) {                          // (else the next run has the rest of it)
                fetch();
                parity ^= stage == kStages - 1;
                stage = stage == kStages - 1 ? 0 : stage + 1;
            }
        }
        if (gave_up) break;

        // The run's state: m, the sum, f and the values of its rows.
        float* state = WHOLE ? states + warp * (kRows * kState) : c.partial + ((int64_t)blockIdx.y * (n_warps + (int64_t)per_row * kv * tiles) + me + ((int64_t)s * kv + kvh) * tiles + row_tile) * (kRows * kState);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int d = 4; d < 32; d *= 2) l[n] += __shfl_xor_sync(0xffffffffu, l[n], d);
            const int row = 4 * n + t;
            if (row >= rows_here) continue;
            float* to = state + row * kState;
            if (g == 0) *reinterpret_cast<float4*>(to) = make_float4(m[n], l[n] * pow2(share_of_p(f)), (float)f, 0.0f);
#pragma unroll
            for (int j = 0; j < JV; ++j)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int gr = (64 * j + 32 * (k >> 1)) / (HD / NG), e = NT == 1 ? gr & 1 : n & 1;
                    *reinterpret_cast<float2*>(to + 4 + 64 * j + 32 * (k >> 1) + 4 * g + 2 * (k & 1)) = make_float2(o[n / 2][j * 4 + k][e], o[n / 2][j * 4 + k][e + 2]);
                }
        }
    }
    if (gave_up) {
        // The copies still in flight land before the block may leave (bounded as well); the result is wrong and the status word says so.
        if (lane == 0) atomicCAS(status, 0, (0xC << 12) | 1);
        for (int i = done >> 1; i < asked; ++i) lb_tc::mbar_wait(&bars[warp][i % kStages], (uint32_t)(i / kStages) & 1u, nullptr);
    }
    if constexpr (WHOLE) {
        // Every warp's state, also of those without keys (and of one that gave up), then a warp a row.
        static_assert(kRows <= kWarps, "a warp a row");
        if (n_tiles <= 0 || gave_up)
            for (int i = lane; i < kRows * kState; i += 32) states[warp * (kRows * kState) + i] = 0.0f;
        __syncthreads();
        const Portion part = requests[0].part;
        const int in_row = requests[0].in_row, kvh = blockIdx.x / in_row, r = ((int)blockIdx.x - kvh * in_row) * kRows + warp;
        if (warp < kRows && r < part.count * c.per) join_row<HD>(c, part, seq0, kvh, r, states + warp * kState, kRows * kState, kWarps, 0, nullptr);
    }
}

// Joins the states of the rows' runs, a team of warps a row: bound by its chain of trips to memory (requests, starts, the states' sums and eight of their values at once), which costs 3.5 us, and by the
// states where a row has many (1 request of 131,072 keys: 296 a row, 6 us).
template <int HD>
__global__ void __launch_bounds__(1024)
attention4_join_kernel(const Call c, int per_row, int n_warps, int tiles, int rows_shift, int team_shift) {
    constexpr int kState = HD + 4;
    __shared__ float joined[32][HD + 3];
    const int kv = c.pages.n_kv_head, seq = blockIdx.z, kvh = blockIdx.y, row_of = seq < per_row ? 0 : seq / per_row, s = seq - row_of * per_row;
    const int r = blockIdx.x * (blockDim.x >> 5 >> team_shift) + (threadIdx.x >> 5 >> team_shift);
    lb_wait_for_predecessor();
    lb_dependents_may_launch();
    const Portion part = portion_of(c, seq);
    const float* state = nullptr;
    int runs = 0;
    if (r < part.count * c.per) {
        const int row_tile = r >> rows_shift, in_row = c.q_start == nullptr ? tiles : ((part.count * c.per - 1) >> rows_shift) + 1;
        const int* starts = c.starts + (int64_t)row_of * (per_row + 1);
        const int start = starts[s], units = kv * in_row, n_seq = min(per_row, c.n_seq - row_of * per_row), share = share_of(starts[n_seq], n_warps);
        const int count = units == 1 ? starts[s + 1] - start : (starts[s + 1] - start) / units;
        const int from = start + (kvh * in_row + row_tile) * count, first = from / share;
        runs = count > 0 ? (from + count - 1) / share - first + 1 : 0;
        state = c.partial + (((((int64_t)row_of * (n_warps + (int64_t)per_row * kv * tiles) + first + ((int64_t)s * kv + kvh) * tiles + row_tile) << rows_shift) + r - (row_tile << rows_shift)) *
                             kState);
    }
    join_row<HD>(c, part, seq, kvh, r, state, kState << rows_shift, runs, team_shift, joined);
}

template <int HD, int NG, int NT, bool PLAIN>
int launch(const Call& c, const RowsPlan& p, cudaStream_t s) {
    int* status = nullptr;
    if (int rc = lb_tc_status_word(&status)) return rc;
    if (p.whole) {
        auto kernel = attention4_rows_kernel<HD, NG, NT, PLAIN, true>;
        constexpr int kWarps = warps_of(NT, true), smem = kWarps * (kStages * 2 * block_bytes(HD, NG) + 4 * NT * (HD + 4) * 4) + 8 + (int)sizeof(Request);
        static std::atomic<uint64_t> asked{0};
        if (int rc = allow_shared(kernel, smem, asked)) return rc;
        LB_CHECK_CUDA(lb_launch_overlapped(kernel, dim3(c.pages.n_kv_head * p.tiles, c.n_seq), dim3(kWarps * 32), smem, s, c, 1, p.tiles, status));
        return LB_OK;
    }
    constexpr int kWarps = warps_of(NT, false);
    auto kernel = attention4_rows_kernel<HD, NG, NT, PLAIN, false>;
    const int smem = kWarps * kStages * 2 * block_bytes(HD, NG) + 4 * (p.per_row + 1) + (int)sizeof(Request) * p.per_row;
    static std::atomic<uint64_t> asked{0};
    if (int rc = allow_shared(kernel, kWarps * kStages * 2 * block_bytes(HD, NG) + 4 * (kMostRequests + 1) + (int)sizeof(Request) * kMostRequests, asked)) return rc;
    LB_CHECK_CUDA(lb_launch_overlapped(kernel, dim3(p.blocks, (c.n_seq + p.per_row - 1) / p.per_row), dim3(kWarps * 32), smem, s, c, p.per_row, p.tiles, status));
    // Blocks of four warps or more, but no warps past the rows.
    int join_warps = p.join_team;
    while (join_warps < 4 && join_warps < c.max_rows * p.join_team) join_warps *= 2;
    const int teams = join_warps / p.join_team;
    LB_CHECK_CUDA(lb_launch_overlapped(attention4_join_kernel<HD>, dim3((c.max_rows + teams - 1) / teams, c.pages.n_kv_head, c.n_seq), dim3(32 * join_warps), 0, s, c, p.per_row,
                                       p.blocks * kWarps, p.tiles, __builtin_ctz((unsigned)p.rows), __builtin_ctz((unsigned)p.join_team)));
    return LB_OK;
}

template <int HD, int NG>
int launch_for(const Call& c, const RowsPlan& p, cudaStream_t s) {
    const bool plain = c.distance == nullptr && c.soft_cap <= 0.0f && c.scores == nullptr;
    if (p.rows == 4) return plain ? launch<HD, NG, 1, true>(c, p, s) : launch<HD, NG, 1, false>(c, p, s);
    return plain ? launch<HD, NG, 2, true>(c, p, s) : launch<HD, NG, 2, false>(c, p, s);
}

}  // namespace

RowsPlan rows_plan(int n_seq, int n_kv_head, int max_rows, int max_keys, int head_dim, int n_sm) {
    RowsPlan p = {};
    p.rows = max_rows > 4 ? 8 : 4;
    p.tiles = (max_rows + p.rows - 1) / p.rows;
    // A launch row numbers its tiles in 32 bits: a request of more is not this kernel's.
    const int64_t units = (int64_t)n_kv_head * p.tiles, most = units * ((max_keys + kBlockKeys - 1) / kBlockKeys);
    p.fits = most <= 1 << 30;
    if (!p.fits) {
        p.us = std::numeric_limits<double>::infinity();
        return p;
    }
    p.per_row = (int)std::max<int64_t>(1, std::min<int64_t>({(int64_t)std::max(1, n_seq), (int64_t)kMostRequests, ((int64_t)1 << 30) / std::max<int64_t>(1, most)}));
    const int kWarps = warps_of(p.rows / 4, false);
    const int64_t warps = std::min<int64_t>((int64_t)n_sm * blocks_per_sm(head_dim, p.rows / 4, false) * kWarps, (most * p.per_row + kLeastTiles - 1) / kLeastTiles);
    p.blocks = (int)std::max<int64_t>(1, (warps + kWarps - 1) / kWarps);
    // Runs that a row has, about; a warp takes eight of them or fewer, whose values are on their way at once.
    const int64_t runs = p.blocks * kWarps / (units * p.per_row) + 2;
    p.join_team = 1;
    while (p.join_team < 32 && p.join_team * 8 < runs) p.join_team *= 2;
    const int64_t rows = (std::max(1, n_seq) + p.per_row - 1) / p.per_row;
    p.states = rows * (p.blocks * kWarps + p.per_row * units) * p.rows * (head_dim + 4) * 4;
    p.starts = rows * (p.per_row + 1) * 4;
    // Which way: by an estimate of both in microseconds, from 150 calls of 1 to 64 requests on 64 to 8,192 keys (25 heads of 64; 32 over 8, and over 4, of 128).  Blocks that have a row tile's keys to
    // themselves: a start and an end for each wave of them, and the keys, which all SMs' blocks read side by side (1 request, 25 heads of 64, 512 keys 5.9 us, the other way 8.6; 16 requests, 8 heads,
    // 2,048 keys 13.5 / 20).  Warps that share all tiles: a start, a join, and the tiles of a warp (1 request, 8 heads, 8,192 keys 39 / 13; 16 requests 42 / 40).
    const bool wide = head_dim == 128, two = p.rows == 8;
    const double all = (double)units * n_seq, thousands = max_keys / 1024.0;
    const double waves = std::ceil(all / (n_sm * blocks_per_sm(head_dim, p.rows / 4, true)));
    const double one = two ? (wide ? 4.55 : 3.3) : wide ? 4.25 : 2.9, shared = two ? (wide ? 0.0375 : 0.022) : wide ? 0.0286 : 0.0165;
    const double whole_us = 1.3 + (two ? 5.0 : 4.2) * waves + thousands * std::max(one, shared * all);
    const double tiles_of_warp = std::max<double>(kLeastTiles, (double)most * n_seq / (n_sm * blocks_per_sm(head_dim, p.rows / 4, false) * kWarps));
    const double shared_us = 9.0 + tiles_of_warp * (two ? (wide ? 0.85 : 0.6) : wide ? 1.2 : 0.62) + std::min(tiles_of_warp, 10.0) * (wide && !two ? 0.0 : 0.25) + (tiles_of_warp > kLeastTiles ? 2.0 : 0.0);
    // (The estimates take every request to be as long as the longest.  Where they are not, sharing gains and a block's own keys do not: 16 requests of 2,048 keys on average and 4,096 at most 38 us and
    // 30.  So a block has its own keys only where that is clearly the shorter.)
    p.whole = whole_us < 0.8 * shared_us;
    p.us = p.whole ? whole_us : shared_us;
    if (p.whole) p.states = p.starts = 0;
    return p;
}

int few_rows(const Call& c, int head_dim, const RowsPlan& p, cudaStream_t s) {
    if (head_dim == 64) return c.pages.groups == 1 ? launch_for<64, 1>(c, p, s) : launch_for<64, 2>(c, p, s);
    return c.pages.groups == 1 ? launch_for<128, 1>(c, p, s) : c.pages.groups == 2 ? launch_for<128, 2>(c, p, s) : launch_for<128, 4>(c, p, s);
}

}  // namespace lb_a4

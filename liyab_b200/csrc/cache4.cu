// The 4-bit cache's own work: rows in, values out, and eviction.
//
// append4 and cache4_values move each value once; eight threads have a row of keys or of values, in the order of cache4.cuh.  They are bound by instructions, 281 a warp of 512 values in and 123 out:
// 4,096 tokens of 8 heads of 128 go in in 11.2 us by themselves from cold memory (477 instructions a warp, with keys and values in each and a corrected division a value: 16), 16,384 rows of 8 heads come
// out in 16 us (85 MB, 5.3 TB/s).
// evict4 is two launches.  The first chooses: a block (a cluster of up to eight for more than 8,192 keys) a request and key/value head finds the weight of the last key that stays by a radix selection over the
// weights as ordered integers (three passes over 11, 11 and 10 bits), then every warp counts its stretch of the keys and writes those that stay in their order.  It is bound by the passes' chains of
// barriers and, for long requests, by their instructions on the SMs that have a request and head (from cold memory 12 x 2,048 keys 11.0 us, 64 x 8,192 keys 16;
// without a look at the pages 9.3 and 14; with zeros counted by votes and one key a step 17 then).  The second copies: a warp a block of sixteen keys of the
// destination, whose pieces it gathers, all asked for before the first is stored (64 x 2,048 keys of 128 dims, 36 MB read and written, 11 us; a piece at a time 12.2).  The destination is never
// a source, so nothing waits for anything.
#include "attention4.h"
#include "cache4.cuh"
#include "linear4.h"

#include <math_constants.h>

#include <algorithm>

namespace lb_c4 {

int pages_of(const lb_cache4* c, const char* what, Pages* p) {
    LB_CHECK_ARG(c != nullptr, "%s: no cache", what);
    LB_CHECK_ARG(c->head_dim == 64 || c->head_dim == 128, "%s: heads of %d values (64 or 128)", what, c->head_dim);
    LB_CHECK_ARG((c->group == 32 || c->group == 64 || c->group == 128) && c->group <= c->head_dim, "%s: groups of %d values (32, 64 or 128, up to a head)", what, c->group);
    LB_CHECK_ARG(c->page_size >= 16 && c->page_size <= (1 << 20) && (c->page_size & (c->page_size - 1)) == 0, "%s: pages of %d keys (a power of two, 16 or more)", what, c->page_size);
    LB_CHECK_ARG(c->n_pages >= 0 && c->n_kv_head > 0 && c->n_kv_head <= 65535, "%s: %d pages of %d heads", what, c->n_pages, c->n_kv_head);
    LB_CHECK_ARG((int64_t)c->n_pages * c->page_size <= INT32_MAX, "%s: %d pages of %d keys have slots past 32 bits", what, c->n_pages, c->page_size);
    LB_CHECK_ARG((int64_t)c->n_pages * c->n_kv_head * (c->page_size / 16) <= INT32_MAX, "%s: %d pages of %d heads are more than 2^31 blocks of keys", what, c->n_pages, c->n_kv_head);
    LB_CHECK_ARG((c->memory != nullptr || c->n_pages == 0) && reinterpret_cast<uintptr_t>(c->memory) % 16 == 0, "%s: the cache's memory is missing or not 16-byte aligned", what);
    p->memory = static_cast<uint8_t*>(c->memory);
    p->n_pages = c->n_pages;
    p->n_kv_head = c->n_kv_head;
    p->page_shift = __builtin_ctz((unsigned)c->page_size);
    p->groups = c->head_dim / c->group;
    p->block = block_bytes(c->head_dim, p->groups);
    return LB_OK;
}

}  // namespace lb_c4

namespace {

using namespace lb_c4;

// N (4 or 8) neighbouring values of a row as 32-bit numbers, and the bits of the largest |x|.  (Compared as integers, where a NaN is the largest of all: fmaxf would drop it.)
template <typename T, int N>
__device__ __forceinline__ uint32_t load_values(const T* p, bool wide, float* v) {
    if constexpr (sizeof(T) == 4) {
        if (wide) {
#pragma unroll
            for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(v + i) = *reinterpret_cast<const float4*>(p + i);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = p[i];
        }
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) top = max(top, __float_as_uint(v[i]) << 1);
        return top >> 1;
    } else {
        uint32_t u[N / 2], top = 0;
        if (wide) {
            if constexpr (N == 8) *reinterpret_cast<uint4*>(u) = *reinterpret_cast<const uint4*>(p);
            else *reinterpret_cast<uint2*>(u) = *reinterpret_cast<const uint2*>(p);
        } else {
#pragma unroll
            for (int i = 0; i < N / 2; ++i) u[i] = __bfloat16_as_ushort(p[2 * i]) | (uint32_t)__bfloat16_as_ushort(p[2 * i + 1]) << 16;
        }
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            v[2 * i] = __uint_as_float(u[i] << 16);
            v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
            top = __vmaxu2(top, u[i] & 0x7fff7fffu);
        }
        return max(top << 16, top & 0xffff0000u);
    }
}

// The scale of a group whose largest |x| this is, bfloat16(x / 7); the rounding that follows divides by what was stored.
template <typename T>
__device__ __forceinline__ __nv_bfloat16 group_scale(uint32_t top) {
    const float a = __uint_as_float(top);
    if (top >= 0x7f800000u) return __float2bfloat16_rn(CUDART_NAN_F);
    // A bfloat16 number over seven is never within 2^-12 of the middle of two bfloat16 numbers (seven times a middle has nine bits or more and is odd), so the product with 1 / 7 rounds alike.
    if (sizeof(T) == 2 && top >= 0x04000000u) return __float2bfloat16_rn(a * 0.14285715f);
    return __float2bfloat16_rn(__fdiv_rn(a, 7.0f));
}

// A scale and its rounded reciprocal, and whether that is within float32's range.
struct Divisor {
    float s, r;
    __device__ __forceinline__ bool plain() const { return s >= 0x1p-90f; }
};
__device__ __forceinline__ Divisor divisor(__nv_bfloat16 scale) {
    const float s = __bfloat162float(scale);
    return Divisor{s, __frcp_rn(s)};
}

// Eight values over their scales (the first four over a), the quotients rounded to 32 bits and then to the nearest even integer, as nibbles n + 8: nibble n is value 2 (n % 4) + n / 4, of keys and of
// values.  |x| is at most 7.03 s as long as s is a normal number, so the integers are -7 .. 7.  They come out of an addition of 1.5 2^23, whose bits are a number in base 16 as they are: what the
// eight times 0x4b400000 come to is taken off at the end, modulo 2^32.
// The quotient of float32 numbers is x r corrected by its rest times r, r the scale's rounded reciprocal (Markstein's division, correctly rounded).  That of bfloat16 numbers (eight bits each) lies on
// the middle of two integers or 2^-10 away from it at least: (2 a 2^d - (2 k + 1) b) / 2 b for whole a, b < 256, where d >= -2 as a quotient below 1 / 4 rounds to 0.  So x r, off by 2^-21 at
// most, rounded to a multiple of 2^-11 by adding 6144 lies on the same side of the middle, or on it.
template <typename T>
__device__ __forceinline__ uint32_t eight_nibbles(const float* x, const Divisor& a, const Divisor& b) {
    constexpr float kMagic = 12582912.0f, kCoarse = 6144.0f;
    if (a.plain() && b.plain()) {
        uint32_t word = 0;
#pragma unroll
        for (int n = 7; n >= 0; --n) {
            const int d = 2 * (n & 3) + (n >> 2);
            const float s = d < 4 ? a.s : b.s, r = d < 4 ? a.r : b.r;
            float whole;
            if constexpr (sizeof(T) == 2) {
                whole = fmaf(x[d], r, kCoarse) + (kMagic - kCoarse);
            } else {
                const float q = x[d] * r;
                whole = fmaf(fmaf(-q, s, x[d]), r, q) + kMagic;
            }
            word = (word << 4) + __float_as_uint(whole);
        }
        return word + (8u - 0x4b400000u) * 0x11111111u;
    }
    uint32_t word = 0;                                     // scales of 0, NaN, or with a reciprocal past float32's range
#pragma unroll 1
    for (int n = 0; n < 8; ++n) {
        const int d = 2 * (n & 3) + (n >> 2);
        float v = x[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) v = i == d ? x[i] : v;
        const float s = d < 4 ? a.s : b.s, q = s > 0.0f ? rintf(__fdiv_rn(v, s)) : 0.0f;
        word |= (uint32_t)((int)fminf(fmaxf(q, -8.0f), 7.0f) + 8) << (4 * n);
    }
    return word;
}

// Eight threads have a row of keys (OF 0) or values (1), HD / 64 words each; they are neighbours in a warp, which has four rows of the same kind.  A block has sixteen tokens' rows of one head, keys
// and values.
template <int HD, int NG, int OF>
struct Share {
    static constexpr int kWords = HD / 64, kGroup = HD / NG;
    // A thread's groups, and that of word i's first (second) four values.  Keys: a word lies in one group of 32, which four threads share.  Values: a word's halves lie in two groups of 32, which
    // eight threads share.
    static constexpr int kGroups = OF == 0 ? (kGroup == 32 ? kWords : 1) : kGroup == 32 ? 2 * kWords : kGroup == 64 ? kWords : 1;
    static constexpr bool kAll = OF == 1 || kGroup == HD;               // whether eight threads share a group
    __device__ static constexpr int group(int i, int second) { return OF == 0 ? (kGroup == 32 ? i : 0) : kGroup == 32 ? 2 * i + second : kGroup == 64 ? i : 0; }
    // The first dim of a word's first, and of its second four values; r: the thread of the eight.
    __device__ static int dim(int r, int i, int second) { return OF == 0 ? 32 * ((r >> 2) * kWords + i) + 8 * (r & 3) + 4 * second : 64 * i + 32 * second + 4 * r; }
    // Which of the row's scales a thread's is.
    __device__ static int scale(int r, int gr) { return kGroups == NG ? gr : OF == 0 ? (r >> 2) * kGroups + gr : 0; }
    __device__ static int place(int key, int r) { return OF == 0 ? Layout<HD>::k_word(key, 4 * (r >> 2) * kWords + (r & 3)) : Layout<HD>::v_word(key, r, 0); }
};
constexpr int kBlockRows = 16;

template <typename T, int HD, int NG, int OF>
__device__ __forceinline__ void append_row(const T* __restrict__ rows, int64_t ld, const int32_t* __restrict__ slot_mapping, const Pages& pages, int n_tokens, bool wide) {
    using S = Share<HD, NG, OF>;
    constexpr int W = S::kWords;
    const int token = blockIdx.x * kBlockRows + ((threadIdx.x & 127) >> 3), head = blockIdx.y, r = threadIdx.x & 7;
    // Threads past the end and those of skipped rows go along with the shuffles.
    const int slot = token < n_tokens ? slot_mapping[token] : -1;
    const bool there = slot >= 0 && slot >> pages.page_shift < pages.n_pages;
    float x[W][8] = {};
    uint32_t top[S::kGroups] = {};
    const T* from = rows + (int64_t)token * ld + head * HD;
    if (there) {
#pragma unroll
        for (int i = 0; i < W; ++i) {
            if constexpr (OF == 0) {
                top[S::group(i, 0)] = max(top[S::group(i, 0)], load_values<T, 8>(from + S::dim(r, i, 0), wide, x[i]));
            } else {
#pragma unroll
                for (int e = 0; e < 2; ++e) top[S::group(i, e)] = max(top[S::group(i, e)], load_values<T, 4>(from + S::dim(r, i, e), wide, x[i] + 4 * e));
            }
        }
    }
#pragma unroll
    for (int gr = 0; gr < S::kGroups; ++gr) {
        top[gr] = max(top[gr], __shfl_xor_sync(0xffffffffu, top[gr], 1));
        top[gr] = max(top[gr], __shfl_xor_sync(0xffffffffu, top[gr], 2));
        if (S::kAll) top[gr] = max(top[gr], __shfl_xor_sync(0xffffffffu, top[gr], 4));
    }
    if (!there) return;
    uint8_t* block = pages.memory + pages.at(slot >> pages.page_shift, head, slot);
    const int key = slot & 15;
    __nv_bfloat16* scales = reinterpret_cast<__nv_bfloat16*>(block + Layout<HD>::scale(key, NG, OF));
    Divisor by[S::kGroups];
#pragma unroll
    for (int gr = 0; gr < S::kGroups; ++gr) {
        const __nv_bfloat16 scale = group_scale<T>(top[gr]);
        by[gr] = divisor(scale);
        if ((S::kAll ? r : r & 3) == 0) scales[S::scale(r, gr)] = scale;
    }
    uint32_t word[W];
#pragma unroll
    for (int i = 0; i < W; ++i) word[i] = eight_nibbles<T>(x[i], by[S::group(i, 0)], by[S::group(i, 1)]);
    // A thread's words are neighbours.
    if constexpr (W == 2) *reinterpret_cast<uint2*>(block + S::place(key, r)) = make_uint2(word[0], word[W - 1]);
    else *reinterpret_cast<uint32_t*>(block + S::place(key, r)) = word[0];
}

template <typename T, int HD, int NG>
__global__ void __launch_bounds__(256)
append4_kernel(const T* __restrict__ k, int64_t ldk, const T* __restrict__ v, int64_t ldv, const int32_t* __restrict__ slot_mapping, const Pages pages, int n_tokens, int wide) {
    lb_wait_for_predecessor();
    lb_dependents_may_launch();
    if (threadIdx.x < 128) append_row<T, HD, NG, 0>(k, ldk, slot_mapping, pages, n_tokens, wide != 0);
    else append_row<T, HD, NG, 1>(v, ldv, slot_mapping, pages, n_tokens, wide != 0);
}

__device__ __forceinline__ void store4(float* p, bool wide, const float* v) {
    if (wide) {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = v[i];
    }
}

template <typename T, int HD, int NG, int OF>
__device__ __forceinline__ void row_values(const Pages& pages, const int32_t* __restrict__ slots, int n, T* __restrict__ rows, int64_t ld, bool wide) {
    using S = Share<HD, NG, OF>;
    constexpr int W = S::kWords;
    const int i = blockIdx.x * kBlockRows + ((threadIdx.x & 127) >> 3), head = blockIdx.y, r = threadIdx.x & 7;
    if (i >= n) return;
    const int slot = slots[i];
    if (slot < 0 || slot >> pages.page_shift >= pages.n_pages) return;
    const uint8_t* block = pages.memory + pages.at(slot >> pages.page_shift, head, slot);
    const int key = slot & 15;
    const __nv_bfloat16* scales = reinterpret_cast<const __nv_bfloat16*>(block + Layout<HD>::scale(key, NG, OF));
    T* to = rows + (int64_t)i * ld + head * HD;
    uint32_t word[W];
    if constexpr (W == 2) {
        const uint2 u = *reinterpret_cast<const uint2*>(block + S::place(key, r));
        word[0] = u.x;
        word[W - 1] = u.y;
    } else {
        word[0] = *reinterpret_cast<const uint32_t*>(block + S::place(key, r));
    }
    __nv_bfloat16 by[S::kGroups];
#pragma unroll
    for (int gr = 0; gr < S::kGroups; ++gr) by[gr] = scales[S::scale(r, gr)];
#pragma unroll
    for (int j = 0; j < W; ++j) {
        const int da = S::dim(r, j, 0), db = S::dim(r, j, 1);
        const __nv_bfloat16 sa = by[S::group(j, 0)], sb = by[S::group(j, 1)];
        if constexpr (sizeof(T) == 2) {
            // 128 + n as bfloat16 less 136, times the scale: one rounding.  Value d of a word is nibble d / 2 + 4 (d % 2).
            const __nv_bfloat162 offset = __float2bfloat162_rn(-136.0f);
            uint32_t x[4];
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const uint32_t u = (word[j] >> (4 * d) & 0x000f000fu) | 0x43004300u;
                const __nv_bfloat162 y = __hmul2(__hadd2(*reinterpret_cast<const __nv_bfloat162*>(&u), offset), __bfloat162bfloat162(d < 2 ? sa : sb));
                x[d] = *reinterpret_cast<const uint32_t*>(&y);
            }
            if (!wide) {
#pragma unroll
                for (int d = 0; d < 8; ++d) to[(d < 4 ? da : db) + d % 4] = __ushort_as_bfloat16((uint16_t)(x[d / 2] >> (16 * (d % 2))));
            } else if constexpr (OF == 0) {
                *reinterpret_cast<uint4*>(to + da) = make_uint4(x[0], x[1], x[2], x[3]);
            } else {
                *reinterpret_cast<uint2*>(to + da) = make_uint2(x[0], x[1]);
                *reinterpret_cast<uint2*>(to + db) = make_uint2(x[2], x[3]);
            }
        } else {
            // 1.5 2^23 + n + 8, less that and 8, times the scale: exact.
            const float fa = __bfloat162float(sa), fb = __bfloat162float(sb);
            float x[8];
#pragma unroll
            for (int d = 0; d < 8; ++d) x[d] = (__uint_as_float((word[j] >> (4 * (d / 2 + 4 * (d % 2))) & 15u) | 0x4b400000u) - 12582920.0f) * (d < 4 ? fa : fb);
            store4(to + da, wide, x);
            store4(to + db, wide, x + 4);
        }
    }
}

template <typename T, int HD, int NG>
__global__ void __launch_bounds__(256)
cache4_values_kernel(const Pages pages, const int32_t* __restrict__ slots, int n, T* __restrict__ k, int64_t ldk, T* __restrict__ v, int64_t ldv, int wide) {
    lb_wait_for_predecessor();
    lb_dependents_may_launch();
    if (threadIdx.x < 128) row_values<T, HD, NG, 0>(pages, slots, n, k, ldk, wide != 0);
    else row_values<T, HD, NG, 1>(pages, slots, n, v, ldv, wide != 0);
}

// ---- eviction ----

constexpr int kChoiceThreads = 1024, kBins = 2048, kMostHeld = 49152;

// Floats as integers of the same order; -0 is 0, a NaN the largest.
__device__ __forceinline__ uint32_t ordered(float v) {
    if (isnan(v)) return 0xffffffffu;
    const uint32_t b = __float_as_uint(v + 0.0f);
    return (b & 0x80000000u) != 0 ? ~b : b | 0x80000000u;
}

struct Choice {
    const float* mass;
    const int32_t* mass_rows;
    const int32_t* n_keys;
    int32_t* kept;
    float* dest_mass;
    const int32_t* table;
    int64_t mass_stride, mass_head_stride, dest_stride, dest_head_stride;
    int keep, recent, max_keys, n_mass, n_dest_mass, table_stride, page_shift, n_pages;
};

// A barrier of the cluster's threads (`blocks` 1: of the block's), and a pair of numbers in block r's shared memory.
__device__ __forceinline__ void meet(int blocks) {
    if (blocks == 1) {
        __syncthreads();
    } else {
        asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
    }
}
__device__ __forceinline__ uint2 of_block(const uint32_t* here, int r) {
    uint2 v;
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(here)), "r"(r));
    asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
    return v;
}

// `blocks` blocks, a cluster, share a request's and head's keys: their counts meet in each other's shared memory.
// Keys on pages that are not there do not stay: of the old keys their place in the order is 0, below every number's, and no more stay than are there; of the newest they are left out, and as many more
// of the old ones stay.
// (1,024 threads also for few keys: 1 request of 2,048, 12 heads, 14.9 us in all; with 512 16.6, with 256 23.2, as the passes wait for shared memory.)
template <bool SHARED>
__global__ void __launch_bounds__(kChoiceThreads)
evict4_choose_kernel(const Choice c, int held, int n_blocks) {
    const int blocks = SHARED ? n_blocks : 1;
    constexpr int THREADS = kChoiceThreads, kOwn = kBins / THREADS;
    static_assert(kOwn == 2, "a thread's bins are read as a pair");
    extern __shared__ uint32_t keys_s[];       // the first `held` of the block's keys' weights as ordered integers
    __shared__ __align__(16) uint32_t both[2][kBins];         // a pass's counts, in turns: the others of the cluster may be at the last pass's still
    __shared__ __align__(8) uint32_t kept_here[2];          // keys of this block above the threshold, and at it
    __shared__ uint32_t sums[THREADS / 32];
    __shared__ uint32_t found[2];              // the bin that holds the last key to stay, and how many of it stay
    __shared__ int gone[2];                    // how many of the old keys, and of the newest, are not there
    if (threadIdx.x < 2) gone[threadIdx.x] = 0;
    lb_wait_for_predecessor();
    lb_dependents_may_launch();
    const int head = blockIdx.x / blocks, rank = blockIdx.x - head * blocks, n_head = gridDim.x / blocks, seq = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n = min(max(c.n_keys[seq], 0), c.max_keys);
    const int r = c.mass_rows != nullptr ? c.mass_rows[seq] : seq;
    const bool weighed = (unsigned)r < (unsigned)c.n_mass;
    const float* mass = c.mass + (weighed ? (int64_t)r * c.mass_stride + (int64_t)head * c.mass_head_stride : 0);
    int32_t* kept = c.kept + ((int64_t)seq * n_head + head) * c.keep;
    float* dest = c.dest_mass != nullptr && (unsigned)r < (unsigned)c.n_dest_mass ? c.dest_mass + (int64_t)r * c.dest_stride + (int64_t)head * c.dest_head_stride : nullptr;
    const int old = n - min(c.recent, n);
    const int32_t* table = c.table + (int64_t)seq * c.table_stride;
    auto absent = [&](int key) { return (unsigned)table[key >> c.page_shift] >= (unsigned)c.n_pages; };
    const int n_table = (n + (1 << c.page_shift) - 1) >> c.page_shift;
    int page = (int)threadIdx.x < n_table ? table[threadIdx.x] : 0;               // (asked for ahead of the weights, and looked at behind them)
    // The block's stretch of the old keys.
    const int share = ((old + blocks - 1) / blocks + 31) / 32 * 32, lo = min(old, rank * share), mine = min(old, lo + share) - lo, in_shared = min(mine, held);
    for (int i0 = threadIdx.x; i0 < in_shared; i0 += 4 * THREADS) {
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = weighed && i0 + j * THREADS < mine ? mass[lo + i0 + j * THREADS] : 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i0 + j * THREADS < in_shared) keys_s[i0 + j * THREADS] = ordered(v[j]);
    }
    for (int i = 4 * threadIdx.x; i < kBins; i += 4 * THREADS) *reinterpret_cast<uint4*>(both[0] + i) = make_uint4(0, 0, 0, 0);
    asm volatile("" : "+r"(page) : : "memory");
    __syncthreads();
#pragma unroll 1
    for (int p = threadIdx.x; p < n_table; p += THREADS) {
        if (p >= THREADS) page = table[p];
        if ((unsigned)page >= (unsigned)c.n_pages) {
            const int first = p << c.page_shift, end = min(first + (1 << c.page_shift), n);
            for (int i = max(first - lo, 0); i < min(end - lo, in_shared); ++i) keys_s[i] = 0;
            if (first < old) atomicAdd(&gone[0], min(end, old) - first);
            if (end > old) atomicAdd(&gone[1], end - max(first, old));
        }
    }
    __syncthreads();
    const int new_there = n - old - gone[1], by_weight = min(old - gone[0], c.keep - new_there), stay = by_weight + new_there;         // recent <= keep, so by_weight is never negative
    auto key_at = [&](int i) { return i < held ? keys_s[i] : absent(lo + i) ? 0u : weighed ? ordered(mass[lo + i]) : 0x80000000u; };
    // The sum of what the warps before this one left.
    auto before = [&](const uint32_t* of_warps) { return __reduce_add_sync(0xffffffffu, lane < warp ? of_warps[lane] : 0u); };
    // The by_weight-th largest key among the first `old`: `threshold` its prefix so far, `left` how many keys with that prefix stay.
    uint32_t threshold = 0, left = (uint32_t)by_weight;
    if (by_weight < old && by_weight > 0) {
        int low = 32;
#pragma unroll 1
        for (int pass = 0; pass < 3; ++pass) {
            const int bits = pass < 2 ? 11 : 10, high = low;
            low -= bits;
            const uint32_t mask = (1u << bits) - 1u, prefix = pass == 0 ? 0u : threshold >> high;
            uint32_t* bins = both[pass & 1];
            if (pass > 0) {
                for (int i = 4 * threadIdx.x; i < kBins; i += 4 * THREADS) *reinterpret_cast<uint4*>(bins + i) = make_uint4(0, 0, 0, 0);
                __syncthreads();
            }
            // Many weights are 0: they are counted in a register and enter with one addition a warp.
            uint32_t zeros = 0;
            auto enter = [&](uint32_t key) {
                if (pass != 0 && key >> high != prefix) return;
                if (key == 0x80000000u) ++zeros;
                else atomicAdd(&bins[key >> low & mask], 1u);
            };
            int i = threadIdx.x;
            for (; i + 3 * THREADS < in_shared; i += 4 * THREADS) {
                uint32_t key[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) key[j] = keys_s[i + j * THREADS];
#pragma unroll
                for (int j = 0; j < 4; ++j) enter(key[j]);
            }
            for (; i < in_shared; i += THREADS) enter(keys_s[i]);
#pragma unroll 1
            for (; i < mine; i += THREADS) enter(key_at(i));
            zeros = __reduce_add_sync(0xffffffffu, zeros);
            if (zeros != 0 && lane == 0) atomicAdd(&bins[0x80000000u >> low & mask], zeros);
            meet(blocks);
            // Two neighbouring bins a thread, from the largest down, of all the cluster's blocks: how many keys lie in larger bins.  Every block does the same sums.
            const int top = kBins - 1 - kOwn * threadIdx.x;
            uint32_t own[kOwn] = {};
            for (int r = 0; r < blocks; ++r) {
                const uint2 two = blocks == 1 ? *reinterpret_cast<const uint2*>(bins + top - 1) : of_block(bins + top - 1, r);
                own[0] += two.y;
                own[1] += two.x;
            }
            const uint32_t sum = own[0] + own[1];
            uint32_t larger = sum;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const uint32_t v = __shfl_up_sync(0xffffffffu, larger, o);
                if (lane >= o) larger += v;
            }
            if (lane == 31) sums[warp] = larger;
            __syncthreads();
            larger += before(sums) - sum;
            if (larger < left && left <= larger + sum) {
#pragma unroll
                for (int j = 0; j < kOwn; ++j) {
                    if (larger < left && left <= larger + own[j]) {
                        found[0] = (uint32_t)(top - j);
                        found[1] = left - larger;
                    }
                    larger += own[j];
                }
            }
            __syncthreads();
            threshold |= found[0] << low;
            left = found[1];
        }
    } else if (by_weight == 0) {
        threshold = 0xffffffffu;       // none stays by its weight
        left = 0;
    } else {
        left = 0xffffffffu;            // all do
    }
    // A warp has a stretch of the keys: it counts those above the threshold and those at it, the warps' counts meet, and it writes its own.
    const int stretch = (mine + THREADS - 1) / THREADS * 32, from = min(mine, warp * stretch), to = min(mine, from + stretch);
    const int to_shared = min(to, held);
    uint32_t above = 0, at = 0;
    auto count = [&](uint32_t key) {
        above += key > threshold;
        at += key == threshold;
    };
    for (int i = from + lane; i < to_shared; i += 32) count(keys_s[i]);
#pragma unroll 1
    for (int i = max(from, held) + lane; i < to; i += 32) count(key_at(i));
    above = __reduce_add_sync(0xffffffffu, above);
    at = __reduce_add_sync(0xffffffffu, at);
    uint32_t* counts = both[1];                // (the last pass's are the other; no block reads these any more)
    if (lane == 0) {
        counts[warp] = above;
        counts[32 + warp] = at;
    }
    __syncthreads();
    uint32_t place = before(counts), ties = before(counts + 32);
    if (blocks > 1) {
        if (threadIdx.x == THREADS - 1) {
            kept_here[0] = place + above;
            kept_here[1] = ties + at;
        }
        meet(blocks);
        for (int r = 0; r < rank; ++r) {
            const uint2 two = of_block(kept_here, r);
            place += two.x;
            ties += two.y;
        }
    }
    place += min(ties, left);
    auto write = [&](int i, uint32_t key) {
        const bool tie = i < to && key == threshold;
        const uint32_t tie_mask = __ballot_sync(0xffffffffu, tie);
        const uint32_t below = (1u << lane) - 1u;
        const bool stays = i < to && (key > threshold || (tie && ties + __popc(tie_mask & below) < left));
        const uint32_t mask = __ballot_sync(0xffffffffu, stays);
        const uint32_t p = place + __popc(mask & below);
        if (stays && p < (uint32_t)c.keep) {
            kept[p] = lo + i;
            if (dest != nullptr) dest[p] = weighed ? mass[lo + i] : 0.0f;
        }
        place += __popc(mask);
        ties += __popc(tie_mask);
    };
    for (int i0 = from; i0 < to_shared; i0 += 32) write(i0 + lane, i0 + lane < to ? keys_s[i0 + lane] : 0);
#pragma unroll 1
    for (int i0 = max(from, held); i0 < to; i0 += 32) write(i0 + lane, i0 + lane < to ? key_at(i0 + lane) : 0);
    // The newest, in their order; where some are not there a warp goes through them.
    if (gone[1] != 0 && rank == 0 && warp == 0) {
        int p = by_weight;
        for (int k0 = old; k0 < n; k0 += 32) {
            const int key = k0 + lane;
            const bool there = key < n && !absent(key);
            const uint32_t mask = __ballot_sync(0xffffffffu, there);
            if (there) {
                const int i = p + __popc(mask & ((1u << lane) - 1u));
                kept[i] = key;
                if (dest != nullptr) dest[i] = weighed ? mass[key] : 0.0f;
            }
            p += __popc(mask);
        }
    }
    for (int i = (gone[1] != 0 ? stay : by_weight) + rank * THREADS + threadIdx.x; i < c.keep; i += blocks * THREADS) {
        const int key = old + i - by_weight;
        const bool there = i < stay;
        kept[i] = there ? key : -1;
        if (dest != nullptr) dest[i] = there && weighed ? mass[key] : 0.0f;
    }
    if (blocks > 1) meet(blocks);              // no block leaves while another reads its counts
}

template <int HD>
__global__ void __launch_bounds__(128)
evict4_copy_kernel(const Pages pages, const int32_t* __restrict__ table, int table_stride, const int32_t* __restrict__ dest_table, int dest_stride,
                   const int32_t* __restrict__ kept, int keep, int max_keys) {
    using L = Layout<HD>;
    constexpr int P = L::kPiece;
    using Piece = typename std::conditional<P == 16, uint4, uint2>::type;         // of a key's K bytes
    using Half = typename std::conditional<P == 16, uint2, uint32_t>::type;       // of a key's V bytes
    lb_wait_for_predecessor();
    lb_dependents_may_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tile = blockIdx.x * 4 + warp, head = blockIdx.y, seq = blockIdx.z;
    if (tile * 16 >= keep) return;
    const int32_t* my_kept = kept + ((int64_t)seq * pages.n_kv_head + head) * keep;
    // Lane i < 16 knows where key i of the tile comes from.
    int64_t source = -1;
    int from = 0;
    if (lane < 16 && tile * 16 + lane < keep) {
        from = my_kept[tile * 16 + lane];
        if (from >= 0 && from < max_keys) source = pages.at(table[(int64_t)seq * table_stride + (from >> pages.page_shift)], head, from);
    }
    if (__ballot_sync(0xffffffffu, source >= 0) == 0) return;
    const int64_t dest_at = pages.at(dest_table[(int64_t)seq * dest_stride + (tile * 16 >> pages.page_shift)], head, tile * 16);
    if (dest_at < 0) return;
    uint8_t* dest = pages.memory + dest_at;
    const int key_from = from & 15;
    auto source_of = [&](int key, int* place) -> const uint8_t* {
        const int64_t at = __shfl_sync(0xffffffffu, source, key);
        *place = __shfl_sync(0xffffffffu, key_from, key);
        return at < 0 ? nullptr : pages.memory + at;
    };
    // A lane's pieces: K of the keys g and g + 8, V of every fourth key (eight lanes each), the scales of a key's K or V.  All are on their way before the first is stored.
    Piece k[2];
    Half v[4];
    uint16_t scale[4];
    bool there[6], scaled;
    const int of = lane >> 4;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        int place;
        const uint8_t* block = source_of(8 * i + (lane >> 2), &place);
        there[i] = block != nullptr;
        if (there[i]) k[i] = *reinterpret_cast<const Piece*>(block + L::k_word(place, lane & 3));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        int place;
        const uint8_t* block = source_of(4 * i + (lane >> 3), &place);
        there[2 + i] = block != nullptr;
        if (there[2 + i]) v[i] = *reinterpret_cast<const Half*>(block + L::v_word(place, lane & 7, 0));
    }
    {
        int place;
        const uint8_t* block = source_of(lane & 15, &place);
        scaled = block != nullptr;
#pragma unroll
        for (int s = 0; s < HD / 32; ++s)
            if (scaled && s < pages.groups) scale[s] = reinterpret_cast<const uint16_t*>(block + L::scale(place, pages.groups, of))[s];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (there[i]) *reinterpret_cast<Piece*>(dest + L::k_word(8 * i + (lane >> 2), lane & 3)) = k[i];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (there[2 + i]) *reinterpret_cast<Half*>(dest + L::v_word(4 * i + (lane >> 3), lane & 7, 0)) = v[i];
#pragma unroll
    for (int s = 0; s < HD / 32; ++s)
        if (scaled && s < pages.groups) reinterpret_cast<uint16_t*>(dest + L::scale(lane & 15, pages.groups, of))[s] = scale[s];
}

bool wide_rows(const void* p, int64_t ld, int bytes) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * bytes % 16 == 0; }

template <typename T>
int append_rows(const T* k, int64_t ldk, const T* v, int64_t ldv, const int32_t* slots, const Pages& pages, int hd, int n, cudaStream_t s) {
    const int wide = wide_rows(k, ldk, sizeof(T)) && wide_rows(v, ldv, sizeof(T));
    const dim3 blocks((unsigned)((n + (int64_t)kBlockRows - 1) / kBlockRows), (unsigned)pages.n_kv_head);
    LB_CHECK_CUDA(lb_launch_overlapped(hd == 64 ? (pages.groups == 1 ? append4_kernel<T, 64, 1> : append4_kernel<T, 64, 2>)
                                       : pages.groups == 1 ? append4_kernel<T, 128, 1> : pages.groups == 2 ? append4_kernel<T, 128, 2> : append4_kernel<T, 128, 4>, blocks, dim3(256), 0, s, k, ldk, v, ldv, slots, pages, n, wide));
    return LB_OK;
}

template <typename T>
int value_rows(const Pages& pages, const int32_t* slots, int n, T* k, int64_t ldk, T* v, int64_t ldv, int hd, cudaStream_t s) {
    const int wide = wide_rows(k, ldk, sizeof(T)) && wide_rows(v, ldv, sizeof(T));
    const dim3 blocks((unsigned)((n + (int64_t)kBlockRows - 1) / kBlockRows), (unsigned)pages.n_kv_head);
    LB_CHECK_CUDA(lb_launch_overlapped(hd == 64 ? (pages.groups == 1 ? cache4_values_kernel<T, 64, 1> : cache4_values_kernel<T, 64, 2>)
                                       : pages.groups == 1 ? cache4_values_kernel<T, 128, 1> : pages.groups == 2 ? cache4_values_kernel<T, 128, 2> : cache4_values_kernel<T, 128, 4>, blocks, dim3(256), 0, s, pages, slots, n, k, ldk, v, ldv,
                                       wide));
    return LB_OK;
}

int rows_check(const char* what, int dtype, const void* k, int64_t ldk, const void* v, int64_t ldv, const int32_t* slots, const lb_cache4* cache, int n, Pages* pages) {
    if (int rc = pages_of(cache, what, pages)) return rc;
    LB_CHECK_ARG(dtype == LB_F32 || dtype == LB_BF16, "%s: rows are float32 or bfloat16", what);
    LB_CHECK_ARG(n >= 0 && (n == 0 || (k != nullptr && v != nullptr && slots != nullptr)), "%s: %d rows, or no memory for them", what, n);
    const int width = cache->n_kv_head * cache->head_dim, bytes = dtype == LB_F32 ? 4 : 2;
    LB_CHECK_ARG(n < 2 || (ldk >= width && ldv >= width), "%s: rows overlap", what);
    LB_CHECK_ARG(reinterpret_cast<uintptr_t>(k) % bytes == 0 && reinterpret_cast<uintptr_t>(v) % bytes == 0 && reinterpret_cast<uintptr_t>(slots) % 4 == 0,
                 "%s: pointers off their type's alignment", what);
    return n > 0 ? device_check(what, cache->device) : LB_OK;
}

}  // namespace

extern "C" int lb_cache4_bytes(int n_pages, int n_kv_head, int head_dim, int page_size, int group, int64_t* bytes) {
    LB_CHECK_ARG(bytes != nullptr, "cache4: no place for the size");
    const lb_cache4 c = {reinterpret_cast<void*>(16), n_pages, n_kv_head, head_dim, page_size, group, 0};
    Pages p;
    if (int rc = pages_of(&c, "cache4", &p)) return rc;
    *bytes = (int64_t)n_pages * n_kv_head * (page_size / 16) * p.block;
    return LB_OK;
}

extern "C" int lb_append4(int dtype, const void* k, int64_t ldk, const void* v, int64_t ldv, const int32_t* slot_mapping, const lb_cache4* cache, int n_tokens, void* stream) {
    Pages pages;
    if (int rc = rows_check("append4", dtype, k, ldk, v, ldv, slot_mapping, cache, n_tokens, &pages)) return rc;
    if (n_tokens == 0 || pages.n_pages == 0) return LB_OK;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == LB_F32) return append_rows<float>((const float*)k, ldk, (const float*)v, ldv, slot_mapping, pages, cache->head_dim, n_tokens, s);
    return append_rows<__nv_bfloat16>((const __nv_bfloat16*)k, ldk, (const __nv_bfloat16*)v, ldv, slot_mapping, pages, cache->head_dim, n_tokens, s);
}

extern "C" int lb_cache4_values(int dtype, const lb_cache4* cache, const int32_t* slots, int n, void* k, int64_t ldk, void* v, int64_t ldv, void* stream) {
    Pages pages;
    if (int rc = rows_check("cache4_values", dtype, k, ldk, v, ldv, slots, cache, n, &pages)) return rc;
    if (n == 0 || pages.n_pages == 0) return LB_OK;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == LB_F32) return value_rows<float>(pages, slots, n, (float*)k, ldk, (float*)v, ldv, cache->head_dim, s);
    return value_rows<__nv_bfloat16>(pages, slots, n, (__nv_bfloat16*)k, ldk, (__nv_bfloat16*)v, ldv, cache->head_dim, s);
}

extern "C" int lb_evict4(const lb_evict4_args* args) {
    LB_CHECK_ARG(args != nullptr, "evict4: no arguments");
    const lb_evict4_args& a = *args;
    Pages pages;
    if (int rc = pages_of(a.cache, "evict4", &pages)) return rc;
    LB_CHECK_ARG(a.n_seq >= 0 && a.n_seq <= 65535, "evict4: %d requests (up to 65535)", a.n_seq);
    LB_CHECK_ARG(a.keep > 0 && a.recent >= 0 && a.recent <= a.keep, "evict4: keep %d keys, %d of them the newest", a.keep, a.recent);
    LB_CHECK_ARG(a.max_keys <= 1 << 30 && a.keep <= 1 << 30, "evict4: %d keys, of which %d stay, are more than one launch takes", a.max_keys, a.keep);
    LB_CHECK_ARG(a.max_keys >= 0 && (int64_t)a.table_stride * a.cache->page_size >= a.max_keys, "evict4: %d keys, block tables of %d pages", a.max_keys, a.table_stride);
    LB_CHECK_ARG((int64_t)a.dest_table_stride * a.cache->page_size >= a.keep, "evict4: %d keys stay, destination tables of %d pages", a.keep, a.dest_table_stride);
    LB_CHECK_ARG(a.n_mass >= 0 && a.n_dest_mass >= 0 && a.mass_head_stride >= 0 && a.mass_stride >= 0 && a.dest_stride >= 0 && a.dest_head_stride >= 0,
                 "evict4: weights of no size");
    if (a.n_seq == 0) return LB_OK;
    LB_CHECK_ARG(a.mass != nullptr && a.block_table != nullptr && a.n_keys != nullptr && a.dest_table != nullptr && a.kept != nullptr, "evict4: a pointer is missing");
    const lb_a4::WeightRows mass = {a.mass, a.mass_stride, a.mass_head_stride, a.n_mass, pages.n_kv_head, a.max_keys};
    const lb_a4::WeightRows dest_mass = {a.dest_mass, a.dest_stride, a.dest_head_stride, a.n_dest_mass, pages.n_kv_head, a.keep};
    LB_CHECK_ARG(a.dest_mass == nullptr || (a.dest_mass != a.mass && lb_a4::rows_disjoint(mass, dest_mass)), "evict4: the kept keys' weights go to memory of their own");
    LB_CHECK_ARG(a.dest_mass == nullptr || lb_a4::rows_apart(dest_mass), "evict4: the kept keys' weights go to rows that overlap (%lld and %lld numbers apart, of %d keys)", (long long)a.dest_stride,
                 (long long)a.dest_head_stride, a.keep);
    if (int rc = device_check("evict4", a.cache->device)) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(a.stream);
    const Choice c = {a.mass, a.mass_rows, a.n_keys, a.kept, a.dest_mass, a.block_table, a.mass_stride, a.mass_head_stride, a.dest_stride, a.dest_head_stride, a.keep, a.recent, a.max_keys,
                      a.n_mass, a.n_dest_mass, a.table_stride, pages.page_shift, pages.n_pages};
    // A block a request and head up to 8,192 keys (8 x 8,192 keys, 8 heads: 38.9 us, by two blocks each 39.8, whose barriers cost what they save); for more as many as there are SMs for (1 x 131,072
    // keys, 8 heads: 56 us by eight blocks each, 230 by one).
    int blocks = 1;
    while (blocks < 8 && (int64_t)pages.n_kv_head * a.n_seq * blocks * 2 <= linear4_sm_count() && a.max_keys > 8192 * blocks) blocks *= 2;
    const int held = std::min(((a.max_keys + blocks - 1) / blocks + 31) / 32 * 32, kMostHeld);
    auto choose = blocks > 1 ? evict4_choose_kernel<true> : evict4_choose_kernel<false>;
    static std::atomic<uint64_t> asked[2];
    if (int rc = lb_a4::allow_shared(choose, 4 * kMostHeld, asked[blocks > 1])) return rc;
    LB_CHECK_CUDA(lb_launch_overlapped_cluster(0, blocks, choose, dim3(pages.n_kv_head * blocks, a.n_seq), dim3(kChoiceThreads), 4 * held, s, c, held, blocks));
    const dim3 grid((a.keep - 1) / 64 + 1, pages.n_kv_head, a.n_seq);
    LB_CHECK_CUDA(lb_launch_overlapped(a.cache->head_dim == 128 ? evict4_copy_kernel<128> : evict4_copy_kernel<64>, grid, dim3(128), 0, s, pages, a.block_table, a.table_stride,
                                       a.dest_table, a.dest_table_stride, a.kept, a.keep, a.max_keys));
    return LB_OK;
}

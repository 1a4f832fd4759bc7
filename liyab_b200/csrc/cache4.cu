// The 4-bit cache's own work: rows in, values out, and eviction.
//
// append4 and cache4_values move each value once and are bound by memory; a thread has a word (eight values) of a row, in the order of cache4.cuh.
// evict4 is two launches.  The first chooses: a block a request and key/value head finds the weight of the last key that stays by a radix selection over the
// weights as ordered integers (three passes over 11, 11 and 10 bits), then every warp counts its stretch of the keys and writes those that stay in their order.  The
// second copies: a warp a block of sixteen keys of the destination, whose pieces it gathers.  The destination is never a source, so nothing waits for anything.
#include "cache4.cuh"
#include "linear4.h"

#include <math_constants.h>

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

// `count` (4 or 8) neighbouring values of a row.
template <typename T, int N>
__device__ __forceinline__ void load_values(const T* p, bool wide, float* v) {
    if (wide) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(v + i) = *reinterpret_cast<const float4*>(p + i);
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                const uint2 u = *reinterpret_cast<const uint2*>(p + i);
                v[i] = __uint_as_float(u.x << 16);
                v[i + 1] = __uint_as_float(u.x & 0xffff0000u);
                v[i + 2] = __uint_as_float(u.y << 16);
                v[i + 3] = __uint_as_float(u.y & 0xffff0000u);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = lb_to_float(p[i]);
    }
}

// max |v| as an integer that orders like it, a NaN above all.
__device__ __forceinline__ uint32_t size_of(const float* v, int n) {
    uint32_t top = 0;
    for (int i = 0; i < n; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    return top;
}

// The scale of a group whose largest |x| this is, bfloat16(x / 7); the rounding that follows divides by what was stored.
__device__ __forceinline__ __nv_bfloat16 group_scale(uint32_t top) {
    return __float2bfloat16_rn(top < 0x7f800000u ? __fdiv_rn(__uint_as_float(top), 7.0f) : CUDART_NAN_F);
}
__device__ __forceinline__ uint32_t nibble(float x, float s) {
    const float r = s > 0.0f ? rintf(__fdiv_rn(x, s)) : 0.0f;            // a scale of 0 or NaN: 0
    return (uint32_t)((int)fminf(fmaxf(r, -8.0f), 7.0f) + 8);
}

// A thread a word: threads are [token][head][K words, V words].
template <typename T, int HD>
__global__ void __launch_bounds__(256)
append4_kernel(const T* __restrict__ k, int64_t ldk, const T* __restrict__ v, int64_t ldv, const int32_t* __restrict__ slot_mapping, const Pages pages, int n_tokens, int wide) {
    using L = Layout<HD>;
    constexpr int W = L::kWords;
    lb_wait_for_predecessor();
    lb_dependents_may_launch();
    const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, row = id / (2 * W);
    const int w = (int)(id % W), of = (int)(id / W & 1);
    const int head = (int)(row % pages.n_kv_head);
    const int64_t token = row / pages.n_kv_head;
    // The threads of a row are neighbours in one warp; those past the end and those of skipped rows go along with the shuffles.
    const int slot = token < n_tokens ? slot_mapping[token] : -1;
    const bool there = slot >= 0 && slot >> pages.page_shift < pages.n_pages;
    float x[8] = {};
    uint32_t a, b;                                     // the largest of its values in the first, and in the second group that it touches
    const int g = w & 7, j = w >> 3;
    if (of == 0) {
        if (there) load_values<T, 8>(k + token * ldk + head * HD + 8 * w, wide, x);
        a = b = size_of(x, 8);
    } else {
        if (there) {
            load_values<T, 4>(v + token * ldv + head * HD + 64 * j + 4 * g, wide, x);
            load_values<T, 4>(v + token * ldv + head * HD + 64 * j + 32 + 4 * g, wide, x + 4);
        }
        a = size_of(x, 4);
        b = size_of(x + 4, 4);
    }
    auto meet = [&](int distance) {
        a = max(a, __shfl_xor_sync(0xffffffffu, a, distance));
        b = max(b, __shfl_xor_sync(0xffffffffu, b, distance));
    };
    const int group = HD / pages.groups;
    meet(1);
    meet(2);
    // Eight threads of values have two groups of 32 between them, of keys one of 64.
    const uint32_t a4 = a, b4 = b;
    meet(4);
    if (of == 0) {
        if (group == 32) a = b = a4;
        (void)b4;
    } else if (group != 32) {
        a = b = max(a, b);
    }
    if constexpr (HD == 128) {
        const uint32_t far = __shfl_xor_sync(0xffffffffu, a, 8);
        if (group == 128) a = b = max(a, far);
    }
    if (!there) return;
    const __nv_bfloat16 sa = group_scale(a), sb = group_scale(b);
    const float fa = __bfloat162float(sa), fb = __bfloat162float(sb);
    uint8_t* block = pages.memory + pages.at(slot >> pages.page_shift, head, slot);
    const int key = slot & 15;
    uint32_t word = 0;
    __nv_bfloat16* scales = reinterpret_cast<__nv_bfloat16*>(block + L::scale(key, pages.groups, of));
    if (of == 0) {
#pragma unroll
        for (int d = 0; d < 8; ++d) word |= nibble(x[d], fa) << (4 * (d / 2 + 4 * (d % 2)));
        *reinterpret_cast<uint32_t*>(block + L::k_word(key, w)) = word;
        if (8 * w % group == 0) scales[8 * w / group] = sa;
    } else {
        // Nibble n is value 2 (n % 2) + n / 4 of the four in the first (n % 4 < 2) or the second group.
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            const int second = (n & 3) >> 1;
            word |= nibble(x[4 * second + 2 * (n & 1) + (n >> 2)], second != 0 ? fb : fa) << (4 * n);
        }
        *reinterpret_cast<uint32_t*>(block + L::v_word(key, g, j)) = word;
        if (g == 0 && 64 * j % group == 0) scales[64 * j / group] = sa;
        if (g == 0 && group == 32) scales[2 * j + 1] = sb;
    }
}

template <typename T>
__device__ __forceinline__ void store4(T* p, bool wide, const float* v) {
    if (wide) {
        if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            const __nv_bfloat162 lo = __floats2bfloat162_rn(v[0], v[1]), hi = __floats2bfloat162_rn(v[2], v[3]);
            *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i] = lb_from_float<T>(v[i]);
    }
}

template <typename T, int HD>
__global__ void __launch_bounds__(256)
cache4_values_kernel(const Pages pages, const int32_t* __restrict__ slots, int n, T* __restrict__ k, int64_t ldk, T* __restrict__ v, int64_t ldv, int wide) {
    using L = Layout<HD>;
    constexpr int W = L::kWords;
    lb_wait_for_predecessor();
    lb_dependents_may_launch();
    const int64_t id = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, row = id / (2 * W);
    const int w = (int)(id % W), of = (int)(id / W & 1), head = (int)(row % pages.n_kv_head);
    const int64_t i = row / pages.n_kv_head;
    if (i >= n) return;
    const int slot = slots[i];
    if (slot < 0 || slot >> pages.page_shift >= pages.n_pages) return;
    const uint8_t* block = pages.memory + pages.at(slot >> pages.page_shift, head, slot);
    const int key = slot & 15, group = HD / pages.groups, g = w & 7, j = w >> 3;
    const __nv_bfloat16* scales = reinterpret_cast<const __nv_bfloat16*>(block + L::scale(key, pages.groups, of));
    const uint32_t word = *reinterpret_cast<const uint32_t*>(block + (of == 0 ? L::k_word(key, w) : L::v_word(key, g, j)));
    float x[8];
    if (of == 0) {
        const float s = __bfloat162float(scales[8 * w / group]);
#pragma unroll
        for (int d = 0; d < 8; ++d) x[d] = (float)((int)(word >> (4 * (d / 2 + 4 * (d % 2))) & 15u) - 8) * s;
        T* to = k + i * ldk + head * HD + 8 * w;
        store4(to, wide, x);
        store4(to + 4, wide, x + 4);
    } else {
        const float sa = __bfloat162float(scales[64 * j / group]), sb = __bfloat162float(scales[(64 * j + 32) / group]);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int second = e >> 2, d = e & 3, nib = 2 * second + (d >> 1) + 4 * (d & 1);
            x[e] = (float)((int)(word >> (4 * nib) & 15u) - 8) * (second != 0 ? sb : sa);
        }
        T* to = v + i * ldv + head * HD + 64 * j + 4 * g;
        store4(to, wide, x);
        store4(to + 32, wide, x + 4);
    }
}

// ---- eviction ----

constexpr int kChoiceThreads = 1024, kBins = 2048;

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
    int64_t mass_stride, mass_head_stride, dest_stride, dest_head_stride;
    int keep, recent, max_keys, n_mass, n_dest_mass;
};

__global__ void __launch_bounds__(kChoiceThreads)
evict4_choose_kernel(const Choice c) {
    __shared__ uint32_t bins[kBins];
    __shared__ uint32_t sums[32];
    __shared__ uint32_t found[2];              // the bin that holds the last key to stay, and how many of it stay
    lb_wait_for_predecessor();
    lb_dependents_may_launch();
    const int head = blockIdx.x, seq = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n = min(max(c.n_keys[seq], 0), c.max_keys);
    const int r = c.mass_rows != nullptr ? c.mass_rows[seq] : seq;
    const bool weighed = (unsigned)r < (unsigned)c.n_mass;
    const float* mass = c.mass + (weighed ? (int64_t)r * c.mass_stride + (int64_t)head * c.mass_head_stride : 0);
    int32_t* kept = c.kept + ((int64_t)seq * gridDim.x + head) * c.keep;
    float* dest = c.dest_mass != nullptr && (unsigned)r < (unsigned)c.n_dest_mass ? c.dest_mass + (int64_t)r * c.dest_stride + (int64_t)head * c.dest_head_stride : nullptr;
    const int stay = min(n, c.keep), old = n - min(c.recent, n);
    const int by_weight = stay - (n - old);           // of the `old` first keys; recent <= keep, so never negative
    auto key_at = [&](int i) { return weighed ? ordered(mass[i]) : 0u; };
    // The by_weight-th largest key among the first `old`: `above` its prefix so far, `left` how many keys with that prefix stay.
    uint32_t threshold = 0, left = (uint32_t)by_weight;
    if (by_weight < old && by_weight > 0) {
        int low = 32;
        for (int pass = 0; pass < 3; ++pass) {
            const int bits = pass < 2 ? 11 : 10, high = low;
            low -= bits;
            for (int i = threadIdx.x; i < kBins; i += kChoiceThreads) bins[i] = 0;
            __syncthreads();
            for (int i = threadIdx.x; i < old; i += kChoiceThreads) {
                const uint32_t key = key_at(i);
                if (pass == 0 || key >> high == threshold >> high) atomicAdd(&bins[key >> low & ((1u << bits) - 1u)], 1u);
            }
            __syncthreads();
            // Two bins a thread, from the largest down: how many keys lie in larger bins.
            const int top = kBins - 1 - 2 * threadIdx.x;
            const uint32_t b0 = bins[top], b1 = bins[top - 1];
            uint32_t sum = b0 + b1;
            for (int o = 1; o < 32; o *= 2) {
                const uint32_t before = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += before;
            }
            if (lane == 31) sums[warp] = sum;
            __syncthreads();
            uint32_t larger = sum - b0 - b1;
            for (int i = 0; i < warp; ++i) larger += sums[i];
            if (larger < left && left <= larger + b0) {
                found[0] = (uint32_t)top;
                found[1] = left - larger;
            } else if (larger + b0 < left && left <= larger + b0 + b1) {
                found[0] = (uint32_t)(top - 1);
                found[1] = left - larger - b0;
            }
            __syncthreads();
            threshold |= found[0] << low;
            left = found[1];
        }
    } else if (by_weight <= 0) {
        threshold = 0xffffffffu;       // none stays by its weight
        left = 0;
    } else {
        left = 0xffffffffu;            // all do
    }
    // A warp has a stretch of the keys: it counts those above the threshold and those at it, the warps' counts meet, and it writes its own.
    const int stretch = (old + 32 * 32 - 1) / (32 * 32) * 32, from = min(old, warp * stretch), to = min(old, from + stretch);
    uint32_t above = 0, at = 0;
    for (int i = from + lane; i < to; i += 32) {
        const uint32_t key = key_at(i);
        above += key > threshold;
        at += key == threshold;
    }
    above = __reduce_add_sync(0xffffffffu, above);
    at = __reduce_add_sync(0xffffffffu, at);
    __syncthreads();
    if (lane == 0) {
        bins[warp] = above;
        bins[32 + warp] = at;
    }
    __syncthreads();
    uint32_t place = 0, ties = 0;
    for (int i = 0; i < warp; ++i) {
        place += bins[i];
        ties += bins[32 + i];
    }
    place += min(ties, left);
    for (int i0 = from; i0 < to; i0 += 32) {
        const int i = i0 + lane;
        const uint32_t key = i < to ? key_at(i) : 0;
        const bool tie = i < to && key == threshold;
        const uint32_t tie_mask = __ballot_sync(0xffffffffu, tie);
        const uint32_t below = (1u << lane) - 1u;
        const bool stays = i < to && (key > threshold || (tie && ties + __popc(tie_mask & below) < left));
        const uint32_t mask = __ballot_sync(0xffffffffu, stays);
        const uint32_t p = place + __popc(mask & below);
        if (stays && p < (uint32_t)c.keep) {
            kept[p] = i;
            if (dest != nullptr) dest[p] = weighed ? mass[i] : 0.0f;
        }
        place += __popc(mask);
        ties += __popc(tie_mask);
    }
    for (int i = max(by_weight, 0) + threadIdx.x; i < c.keep; i += kChoiceThreads) {
        const int key = old + i - max(by_weight, 0);
        const bool there = i < stay;
        kept[i] = there ? key : -1;
        if (dest != nullptr) dest[i] = there && weighed ? mass[key] : 0.0f;
    }
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
#pragma unroll
    for (int i = 0; i < 2; ++i) {                     // K: a lane's pieces of keys g and g + 8
        const int key = 8 * i + (lane >> 2);
        int place;
        const uint8_t* block = source_of(key, &place);
        if (block != nullptr) *reinterpret_cast<Piece*>(dest + L::k_word(key, lane & 3)) = *reinterpret_cast<const Piece*>(block + L::k_word(place, lane & 3));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {                     // V: four keys, eight pieces each
        const int key = 4 * i + (lane >> 3), g = lane & 7;
        int place;
        const uint8_t* block = source_of(key, &place);
        if (block != nullptr) *reinterpret_cast<Half*>(dest + L::v_word(key, g, 0)) = *reinterpret_cast<const Half*>(block + L::v_word(place, g, 0));
    }
    {
        const int key = lane & 15, of = lane >> 4;
        int place;
        const uint8_t* block = source_of(key, &place);
        if (block != nullptr)
            for (int s = 0; s < pages.groups; ++s)
                reinterpret_cast<uint16_t*>(dest + L::scale(key, pages.groups, of))[s] = reinterpret_cast<const uint16_t*>(block + L::scale(place, pages.groups, of))[s];
    }
}

bool wide_rows(const void* p, int64_t ld, int bytes) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * bytes % 16 == 0; }

template <typename T>
int append_rows(const T* k, int64_t ldk, const T* v, int64_t ldv, const int32_t* slots, const Pages& pages, int hd, int n, cudaStream_t s) {
    const int wide = wide_rows(k, ldk, sizeof(T)) && wide_rows(v, ldv, sizeof(T));
    const int64_t threads = (int64_t)n * pages.n_kv_head * 2 * (hd / 8), blocks = (threads + 255) / 256;
    LB_CHECK_ARG(blocks <= INT32_MAX, "append4: %d tokens are more than one launch takes", n);
    LB_CHECK_CUDA(lb_launch_overlapped(hd == 128 ? append4_kernel<T, 128> : append4_kernel<T, 64>, dim3((unsigned)blocks), dim3(256), 0, s, k, ldk, v, ldv, slots, pages, n, wide));
    return LB_OK;
}

template <typename T>
int value_rows(const Pages& pages, const int32_t* slots, int n, T* k, int64_t ldk, T* v, int64_t ldv, int hd, cudaStream_t s) {
    const int wide = wide_rows(k, ldk, sizeof(T)) && wide_rows(v, ldv, sizeof(T));
    const int64_t threads = (int64_t)n * pages.n_kv_head * 2 * (hd / 8), blocks = (threads + 255) / 256;
    LB_CHECK_ARG(blocks <= INT32_MAX, "cache4_values: %d rows are more than one launch takes", n);
    LB_CHECK_CUDA(lb_launch_overlapped(hd == 128 ? cache4_values_kernel<T, 128> : cache4_values_kernel<T, 64>, dim3((unsigned)blocks), dim3(256), 0, s, pages, slots, n, k, ldk, v, ldv,
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
    LB_CHECK_ARG(a.max_keys >= 0 && (int64_t)a.table_stride * a.cache->page_size >= a.max_keys, "evict4: %d keys, block tables of %d pages", a.max_keys, a.table_stride);
    LB_CHECK_ARG((int64_t)a.dest_table_stride * a.cache->page_size >= a.keep, "evict4: %d keys stay, destination tables of %d pages", a.keep, a.dest_table_stride);
    LB_CHECK_ARG(a.n_mass >= 0 && a.n_dest_mass >= 0 && a.mass_head_stride >= 0 && a.mass_stride >= 0 && a.dest_stride >= 0 && a.dest_head_stride >= 0,
                 "evict4: weights of no size");
    if (a.n_seq == 0) return LB_OK;
    LB_CHECK_ARG(a.mass != nullptr && a.block_table != nullptr && a.n_keys != nullptr && a.dest_table != nullptr && a.kept != nullptr, "evict4: a pointer is missing");
    LB_CHECK_ARG(a.dest_mass == nullptr || a.dest_mass != a.mass, "evict4: the kept keys' weights go to memory of their own");
    if (int rc = device_check("evict4", a.cache->device)) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(a.stream);
    const Choice c = {a.mass, a.mass_rows, a.n_keys, a.kept, a.dest_mass, a.mass_stride, a.mass_head_stride, a.dest_stride, a.dest_head_stride, a.keep, a.recent, a.max_keys,
                      a.n_mass, a.n_dest_mass};
    LB_CHECK_CUDA(lb_launch_overlapped(evict4_choose_kernel, dim3(pages.n_kv_head, a.n_seq), dim3(kChoiceThreads), 0, s, c));
    const dim3 grid((a.keep + 63) / 64, pages.n_kv_head, a.n_seq);
    LB_CHECK_CUDA(lb_launch_overlapped(a.cache->head_dim == 128 ? evict4_copy_kernel<128> : evict4_copy_kernel<64>, grid, dim3(128), 0, s, pages, a.block_table, a.table_stride,
                                       a.dest_table, a.dest_table_stride, a.kept, a.keep, a.max_keys));
    return LB_OK;
}

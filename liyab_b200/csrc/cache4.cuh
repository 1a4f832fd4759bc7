// Where the values of a 4-bit cache lie, for the kernels that fill it and those that read it (see api.h, "4-bit cache").
//
// A page is, for each key/value head, page_size / 16 blocks of sixteen neighbouring keys.  A block is one run of memory, so that one bulk copy fetches a tile of keys
// with their values and scales: [K nibbles 8 hd bytes][V nibbles 8 hd][K scales][V scales], scales bfloat16, hd / group a row.  The order inside a block is that of the
// operands of mma.sync (m16n8k32 on bytes for the keys, m16n8k16 on halves for the values), so that a lane (g = lane / 4, t = lane % 4) finds its values of a tile in 16-byte pieces (8 for heads of 64) without bank conflicts:
//   K, the first operand of K q^T (rows are keys): lane (g, t) has of the keys g and g + 8 the words t, 4 + t, ..: dims 8 w .. 8 w + 7, so that the dims of one product
//      are the same 32, one group of the scales.  Dim 8 w + d is nibble d / 2 + 4 (d % 2) of its word: a mask gives four of them in the bytes of a register, a shift and a mask two neighbours in
//      its halves.
//   V, the first operand of V^T p^T (rows are dims): lane (g, t) has of the keys 2 t, 2 t + 1 (and of those plus 8) the words (g, j): nibble n is dim
//      64 j + 32 (n % 4 / 2) + 4 g + 2 (n % 2) + n / 4, so that the sixteen dims of one product lie in the same 32 as well; the low (high) halves of two keys' words, put beside each
//      other, are the operand's row g (g + 8).
// A key's K bytes are one run of hd / 2, its V bytes lie in one run of hd.
#pragma once

#include "api.h"
#include "common.cuh"

namespace lb_c4 {

constexpr int kBlockKeys = 16;

// Bytes of a block of sixteen keys.
__host__ __device__ constexpr int block_bytes(int hd, int groups) { return 16 * hd + 64 * groups; }

template <int HD>
struct Layout {
    static constexpr int kPiece = HD / 8;              // bytes of a lane's share of eight keys (K), of a pair of keys (V)
    static constexpr int kWords = HD / 8;              // words of a row
    static constexpr int kV = 8 * HD, kScales = 16 * HD;
    // The order of the lanes' pieces of V: by pairs of keys, turned so that the lanes that are served together meet all banks.
    __device__ static constexpr int v_turn(int g, int t) { return HD == 128 ? (g + 2 * t) & 7 : (g + 4 * (t >> 1)) & 7; }
    __device__ static constexpr int k_word(int key, int w) { return (key >> 3) * 32 * kPiece + ((key & 7) * 4 + (w & 3)) * kPiece + (w >> 2) * 4; }
    __device__ static constexpr int v_word(int key, int g, int j) {
        const int t = (key & 7) >> 1;
        return kV + (key >> 3) * 32 * kPiece + (t * 8 + v_turn(g, t)) * kPiece + (key & 1) * (kPiece / 2) + j * 4;
    }
    // of: 0 keys, 1 values
    __device__ static constexpr int scale(int key, int groups, int of) { return kScales + of * 32 * groups + ((key & 7) * 2 + (key >> 3)) * groups * 2; }
};

// What the kernels know of a cache.
struct Pages {
    uint8_t* memory;
    int n_pages, n_kv_head, page_shift, groups, block;
    // The block that holds `key` of a request whose pages the table names; -1: no such page.
    __device__ __forceinline__ int64_t at(int page, int head, int key) const {
        if ((unsigned)page >= (unsigned)n_pages) return -1;
        const int in_page = key & ((1 << page_shift) - 1);
        return (int64_t)(((page * n_kv_head + head) << (page_shift - 4)) + (in_page >> 4)) * block;          // (a cache has fewer than 2^31 blocks)
    }
};

// Checks a cache and turns it into what the kernels know of it (host).
int pages_of(const lb_cache4* cache, const char* what, Pages* pages);

}  // namespace lb_c4

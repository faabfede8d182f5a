// cache_parts.h - the paged key-value cache as its kernels see it: where a token's keys and values lie, and where a
// sequence's rows are.
//
// A page holds `page` tokens (32 << page_shift) of every kv head of one layer, head after head, a head in blocks of 32
// tokens.  A block is its keys, then its values, each in the order in which 16 x 16 x 32 matrix instructions take operands:
// the attention of few rows reads whole 1 KiB runs straight into registers.
//   Token t = b4 b3 b2 b1 b0 of a block is row m = b4 b2 b1 b0 of tile t16 = b3 of 16 tokens, so that after S^T the lanes of
//   quarter q4 = b4 b2 have the scores of eight tokens in slots s = b3 b1 b0; in the order of 32 x 32 x 16 instructions these are the eight
//   that half b2 of the lanes has for 16 tokens b4: values serve both shapes as they lie, and P never moves.
//   keys: operand A of S^T = K Q^T.  Tile t16, group g of 32 dimensions; lane l = m | q4 << 4 holds dimensions 32 g + 8 q4 + 0..7.
//         16 bits  16 B per (t16, g, lane): ((t16 G + g) 64 + l) 16
//         Q8       8 B, both tiles in 16 B: (g 64 + l) 16 + 8 t16, byte = q + 128
//         Q4       one word, both tiles of two groups in 16 B (of the last, odd group in 8 B); nibble of dimension slot s at bit
//                  16 (s & 1) + 4 (s >> 1 & 1) + 8 (s >> 2), value q + 8
//   values: operand A of Y^T = V^T P^T.  Tile dt of 16 dimensions; lane l = dimension & 15 | q4 << 4 holds the eight tokens of
//       quarter q4, slot after slot.
//         16 bits  16 B per (dt, lane), 2 B per token
//         Q8       8 B, tiles 2 g and 2 g + 1 in 16 B; byte = q + 128.  A byte belongs to one token.
//         Q4       8 B per (g, lane), tile 2 g in the low nibbles and 2 g + 1 in the high ones: here too a byte belongs to one
//                  token; bytes of slots 0..3 in the order 0 2 1 3 (so of 4..7); two groups in 16 B as for the keys
//   Q4, Q8: f16 scales [G][q4][s] behind the data, keys' and values' alike.
// No byte is shared by two tokens, so rows of different sequences may be written in any order.
#pragma once

#include "cybq_device.h"

namespace cybq {

// codes of enum cybq_cache_kind
constexpr int kCacheF16 = 1, kCacheBF16 = 2, kCacheQ4 = 4, kCacheQ8 = 8;
constexpr int kBlockTokens = 32;

__host__ __device__ constexpr bool cache_quantised(int kind) { return kind == kCacheQ4 || kind == kCacheQ8; }
// bytes of 32 tokens' keys (or values), without and with their scales
__host__ __device__ constexpr int cache_data_bytes(int kind, int dim) { return kBlockTokens * dim * (cache_quantised(kind) ? kind : 16) / 8; }
__host__ __device__ constexpr int cache_half_bytes(int kind, int dim) { return cache_data_bytes(kind, dim) + (cache_quantised(kind) ? 2 * dim : 0); }
__host__ __device__ constexpr int cache_block_bytes(int kind, int dim) { return 2 * cache_half_bytes(kind, dim); }

struct CacheView {               // one layer
    uint8_t* base;
    int64_t page_bytes;
    int pages;
    int page_shift;              // blocks of a page: 1 << page_shift
    int kv_heads, dim, kind;
};

struct BatchView {
    const int32_t* starts;       // [seqs + 1]
    const int32_t* lengths;      // [seqs]
    const int32_t* tables;       // [seqs][table_pages]
    int seqs, rows, max_new, table_pages;
};

// Q4: byte offset of the 4 (keys) or 8 (values) bytes of group g and lane l; `step` = 4 t16 for keys
template <int G>
__host__ __device__ constexpr int q4_place(int g, int l, int step)
{
    return (g | 1) < G ? ((g >> 1) * 64 + l) * 16 + (g & 1) * 8 + step : (G >> 1) * 1024 + l * 8 + step;
}

// byte offset, within the keys of a block, of dimensions 32 g + 8 q4 + 0..7 of token t
template <int KIND, int G>
__host__ __device__ constexpr int key_place(int t, int g, int q4)
{
    const int t16 = t >> 3 & 1, l = (t >> 4) << 3 | (t & 7) | q4 << 4;
    return KIND == kCacheQ8 ? (g * 64 + l) * 16 + 8 * t16 : KIND == kCacheQ4 ? q4_place<G>(g, l, 4 * t16) : ((t16 * G + g) * 64 + l) * 16;
}

// slot and lane group of token t of a block
__host__ __device__ constexpr int token_slot(int t) { return (t & 3) | (t >> 3 & 1) << 2; }
__host__ __device__ constexpr int token_q4(int t) { return (t >> 4) << 1 | (t >> 2 & 1); }

// byte offset, within the values of a block, of dimension d of token t (Q4: of the byte of dimensions d and d + 16, d & 16 == 0)
template <int KIND, int G>
__host__ __device__ constexpr int value_place(int t, int d)
{
    const int l = (d & 15) | token_q4(t) << 4, s = token_slot(t);
    if (KIND == kCacheQ8) return ((d >> 5) * 64 + l) * 16 + (d >> 4 & 1) * 8 + s;
    if (KIND == kCacheQ4) return q4_place<G>(d >> 5, l, 0) + (s & 4) + ((s & 1) << 1 | (s >> 1 & 1));
    return ((d >> 4) * 64 + l) * 16 + 2 * s;
}

// byte offset of a scale behind the data
__host__ __device__ constexpr int scale_place(int t, int g) { return ((g * 4 + token_q4(t)) * 8 + token_slot(t)) * 2; }

// One sequence's rows: row0 .. row0 + n are its last n tokens, of len; positions at and behind the table's end have no page.
// Starts that fall, or leave 0 .. rows, make a sequence without rows, or one that ends with the rows.
struct Seq {
    int row0, n, len;
};
// the table ends at 2^30 tokens: rows of a longer sequence lie behind it, whatever its length
constexpr int kMaxLength = (1 << 30) + (1 << 25);
__device__ __forceinline__ Seq seq_of(const BatchView& t, int b)
{
    Seq s;
    const int first = t.starts[b], last = t.starts[b + 1];
    s.row0 = first;
    s.n = first < 0 || first >= t.rows || last <= first ? 0 : min(min(last, t.rows) - first, t.max_new);
    s.len = min(max(t.lengths[b], 0), kMaxLength);
    return s;
}

// inclusive sum over the wave's lanes
__device__ __forceinline__ int wave_prefix(int v)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);       // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);      // row_bcast 15, 31
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return v;
}

// The blocks of 32 positions that a sequence's rows touch (positions below zero count too: their rows have no token)
__device__ __forceinline__ int row_blocks(const Seq& s)
{
    const int p0 = s.len - s.n;
    return s.n ? ((s.len - 1) >> 5) - (p0 >> 5) + 1 : 0;
}

}  // namespace cybq

// 8-bit paged KV cache: layout, row lookup and scale arithmetic shared by the
// append, read and attention kernels, gfx950.
//
// A block is 16 consecutive tokens of one KV head and shares one scale 2^e, K
// and V apart: value = (byte - 128) * 2^e.  A page holds page_tokens tokens of
// every KV head:
//   K       [n_pages][n_kv][page_tokens][hd]          a token's dims together
//   V       [n_pages][n_kv][page_tokens / 16][hd][16] a dim's 16 tokens together
//   k_exp,
//   v_exp   [n_pages][n_kv][page_tokens / 16]         int8
// Scales are powers of two, so raising one is a rounded shift of the block's
// bytes (all raises of a block together cost less than one step: 1/2 + 1/4 +
// ...), and scores and sums are scaled without rounding.  V lies transposed
// because 16 bytes of one dim are then a lane's operand of P.V as they stand;
// 16 is the tokens a lane of the 64-token attention step holds.
#pragma once
#include "vte_common.h"

#define KVP_BLOCK 16
#define KVP_E_MIN (-126)
#define KVP_E_NAN (-128)  // a block that received an Inf or a NaN reads as NaN
#define KVP_ZERO 128      // the byte of 0

struct KvPages {
    uint8_t *k, *v;
    int8_t *k_exp, *v_exp;
    int n_pages, page_log2, n_kv;
};
struct KvRows {
    const int *row_start, *kv_offset, *page_table;
    int batch, rows, max_rows, max_pages;
};

__device__ __forceinline__ int kvp_capacity(const KvPages& c, const KvRows& r) { return r.max_pages << c.page_log2; }

// Sequence b's new rows [first, first + n), and the position of the first; n = 0
// for a sequence that is not running (kv_offset < 0).
struct KvSeq {
    int first, n, pos;
};
__device__ __forceinline__ KvSeq kvp_place(const KvRows& r, int b) {  // its rows, whether it runs or not
    KvSeq s;
    s.pos = min(r.kv_offset[b], 1 << 30);  // (no table reaches further; pos + row stays an int)
    if (r.row_start == nullptr) {
        s.first = b;
        s.n = r.max_rows;
    } else {
        s.first = min(max(r.row_start[b], 0), r.rows);
        s.n = max(min(min(max(r.row_start[b + 1], 0), r.rows) - s.first, r.max_rows), 0);
    }
    return s;
}
__device__ __forceinline__ KvSeq kvp_seq(const KvRows& r, int b) {
    KvSeq s = kvp_place(r, b);
    if (s.pos < 0) s.n = 0;
    return s;
}
// The sequence of a row: the last one that starts at or before it, -1 behind the last sequence.
__device__ __forceinline__ int kvp_row_seq(const KvRows& r, int row) {
    if (r.row_start == nullptr) return row < r.batch ? row : -1;
    if (row < r.row_start[0] || row >= r.row_start[r.batch]) return -1;
    int lo = 0, hi = r.batch - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (r.row_start[mid] <= row) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
// Tokens of a sequence that a row at position `pos` sees (itself the last).
__device__ __forceinline__ int kvp_len(int pos, int cap) { return pos < cap ? pos + 1 : cap; }
// Page of table entry j of sequence b; -1 where the entry is no page of the cache.
__device__ __forceinline__ int kvp_page(const KvPages& c, const KvRows& r, int b, int j) {
    const int p = r.page_table[(size_t)b * r.max_pages + j];
    return (unsigned)p < (unsigned)c.n_pages ? p : -1;
}

// 2^e of a stored exponent (NaN for KVP_E_NAN).
__device__ __forceinline__ float kvp_scale(int e) {
    return __uint_as_float(e == KVP_E_NAN ? 0x7FC00000u : (uint32_t)(e + 127) << 23);
}
// The smallest e >= KVP_E_MIN with amax <= 127 * 2^e, amax finite and >= 0:
// amax = m 2^x with m in [1/2, 1) gives x - 7, or x - 6 where m > 127/128.
__device__ __forceinline__ int kvp_exponent(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = (int)(u >> 23) - 126 - 7 + ((u & 0x7FFFFFu) > 0x7E0000u ? 1 : 0);
    return max(e, KVP_E_MIN);
}
__device__ __forceinline__ uint32_t kvp_code(float x, float inv) { return (uint32_t)(__float2int_rn(x * inv) + KVP_ZERO); }

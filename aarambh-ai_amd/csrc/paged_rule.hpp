// Pages of the paged key / value cache: where an element lies in a page, which rows and
// positions a sequence has, and which pages its tokens are in.
// Plain C++ once __host__, __device__ and __forceinline__ are defined: the host test includes it.
#pragma once
#include <stdint.h>

namespace aarh {

// Bits of a sequence's status word.
enum { PAGE_SEQ_BAD_PAGE = 1, PAGE_SEQ_BAD_LENGTH = 2 };

// Tokens of a page come in blocks of PAGE_BLK, each stored in the order in which the matrix
// instructions take it.
constexpr int PAGE_BLK = 32;

// Element (token t < 32, dimension d) of a block of keys.  A 16-byte piece is one lane's operand
// of the product K Q^T: 16-bit keys [t / 4 % 2][d / 64][d / 8 % 2][lane][8], INT8 keys
// [t / 4 % 2][d / 64][lane][16] (both halves of d / 8 % 2), lane = d / 16 % 4 * 16 + t / 8 * 4 + t % 4.
// Rows of the product are then tokens in the order that makes a lane's eight scores the
// eight consecutive tokens which its piece of V^T holds.
__host__ __device__ __forceinline__ int page_k_at(int t, int d, int hd, bool i8) {
    const int ts = (t >> 2) & 1, lane = ((d >> 4) & 3) * 16 + (t >> 3) * 4 + (t & 3);
    const int c = ts * (hd >> 6) + (d >> 6);
    return i8 ? (c * 64 + lane) * 16 + (d & 15) : ((c * 2 + ((d >> 3) & 1)) * 64 + lane) * 8 + (d & 7);
}

// Element (t, d) of a block of values, kept as V^T: 16 bits [d][t]; INT8 [d / 32][t / 8][d % 16][d / 16 % 2][8].
__host__ __device__ __forceinline__ int page_v_at(int t, int d, int hd, bool i8) {
    (void)hd;
    return i8 ? (((d >> 5) * 4 + (t >> 3)) * 16 + (d & 15)) * 16 + ((d >> 4) & 1) * 8 + (t & 7) : d * 32 + t;
}

// A sequence of a call: its new rows row0 .. row0 + rows - 1 of the activation buffers are the
// last `rows` of its kv_len cached tokens.
struct PageSeq {
    int row0, rows, kv_len;
};

// Reads sequence b from the call's arrays.  false: the arrays contradict each other or the
// bounds the call was made with, and the sequence is left out (PAGE_SEQ_BAD_LENGTH).
__host__ __device__ __forceinline__ bool page_seq(const int32_t* row_off, const int32_t* kv_len, int b, int rows_total,
                                                  int max_rows, int max_kv, PageSeq* s) {
    const int64_t r0 = row_off[b], r1 = row_off[b + 1];
    const int n = kv_len[b];
    s->row0 = 0;
    s->rows = 0;
    s->kv_len = 0;
    if (r0 < 0 || r1 < r0 || r1 > rows_total || r1 - r0 > max_rows || n < r1 - r0 || n > max_kv) return false;
    s->row0 = (int)r0;
    s->rows = (int)(r1 - r0);
    s->kv_len = n;
    return true;
}

// Page of token t in a sequence's table, or -1 where the table holds none of the pool's pages.
__host__ __device__ __forceinline__ int page_of(const int32_t* table, int t, int page_shift, int n_pages) {
    const int p = table[t >> page_shift];
    return p >= 0 && p < n_pages ? p : -1;
}

}  // namespace aarh

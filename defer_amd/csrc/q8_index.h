// q8_index.h -- where the rows, positions and pages of the 8-bit operators
// are: plain arithmetic, the same on the host and in the kernels.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define Q8_HD __host__ __device__ __forceinline__
#else
#define Q8_HD inline
#endif

namespace q8 {

constexpr int PAGE = 64;               // positions of a page
constexpr int UNIT = 128;              // attention positions of a unit (short sequences)
constexpr int UNIT_GROWS = 8192;       // ... which grows by as much every so many positions
constexpr int MAX_UNITS = UNIT_GROWS / UNIT;  // so a row has at most so many units
constexpr uint32_t MAX_HEAD_DIM = 256;
constexpr uint32_t MAX_K = 131072;     // sums of fewer code products than this fit 32 bits
constexpr uint32_t MAX_TREE = 64;      // drafted rows of a sequence: a wave's lanes
constexpr uint32_t MAX_SCORE = 1u << 20;   // logits of a row
constexpr uint32_t MAX_TOP = 32;           // alternatives of a row

// The head size as a page holds it.
Q8_HD uint32_t padded(uint32_t head_dim) { return (head_dim + 63) / 64 * 64; }

// The rows of a call that belong to one sequence: rows [start, start + n),
// the last n of its len positions. What the arrays hold is clamped to the
// call's rows, so no row outside them is ever touched.
struct Span {
  int start, n, len;
  // Position of the sequence's j-th row (negative: the row has none).
  Q8_HD int64_t pos(int j) const { return (int64_t)len - n + j; }
};
Q8_HD Span span_of(const int32_t* row_start, const int32_t* kv_len, uint32_t i, uint32_t rows) {
  Span s;
  const int64_t lo = row_start ? row_start[i] : (int64_t)i;
  const int64_t hi = row_start ? row_start[i + 1] : (int64_t)i + 1;
  const int64_t a = lo < 0 ? 0 : lo > (int64_t)rows ? (int64_t)rows : lo;
  const int64_t b = hi < a ? a : hi > (int64_t)rows ? (int64_t)rows : hi;
  s.start = (int)a;
  s.n = (int)(b - a);
  s.len = kv_len[i];
  return s;
}

// The page of a sequence's block of 64 positions, or -1: the block is behind
// the table's end or its entry names no page. (No table: page = block.)
Q8_HD int page_of(const int32_t* table, uint32_t width, uint32_t pages, int64_t block) {
  if (block < 0 || block >= (int64_t)width) return -1;
  const int p = table ? table[block] : (int)block;
  return p >= 0 && (uint32_t)p < pages ? p : -1;
}

// Attention sums a row's positions in units that depend on its own position
// only, so the row's bits do not depend on the other rows of the call.
Q8_HD int unit_len(int64_t pos) { return (int)(UNIT * (1 + pos / UNIT_GROWS)); }
Q8_HD int unit_count(int64_t pos) { return pos < 0 ? 0 : (int)(pos / unit_len(pos)) + 1; }
// The most units any row of a call has whose sequences are at most `len` long.
Q8_HD int most_units(int64_t len) {
  const int64_t n = (len + UNIT - 1) / UNIT;
  return n < 1 ? 1 : n > MAX_UNITS ? MAX_UNITS : (int)n;
}

// Whether two sets of rows share a byte: rows of ar and br bytes from a and b on,
// as and bs bytes apart (at least their length; any number where there is one row).
inline bool share(const void* a, int64_t as, uint32_t a_rows, int64_t ar, const void* b, int64_t bs, uint32_t b_rows, int64_t br) {
  const int64_t x = (int64_t)(uintptr_t)a, y = (int64_t)(uintptr_t)b;
  const int64_t na = a_rows, nb = b_rows;
  if (!na || !nb) return false;
  if (na == 1) as = ar;
  if (nb == 1) bs = br;
  if (x + (na - 1) * as + ar <= y || y + (nb - 1) * bs + br <= x) return false;
  if (as == bs) {  // columns of one matrix: the later one's first row lies between two of the other's
    const int64_t d = x < y ? y - x : x - y, n = x < y ? na : nb, k = d / as, left = d % as;
    const int64_t first = x < y ? ar : br, later = x < y ? br : ar;
    return (k < n && left < first) || (k + 1 < n && as - left < later);
  }
  for (int64_t i = 0, j = 0; i < na && j < nb;) {
    const int64_t p = x + i * as, q = y + j * bs;
    if (p + ar <= q)
      ++i;
    else if (q + br <= p)
      ++j;
    else
      return true;
  }
  return false;
}
// ... other than row by row, each row the same in both.
inline bool overlap(const void* a, int64_t as, uint32_t a_rows, int64_t ar, const void* b, int64_t bs, uint32_t b_rows, int64_t br) {
  const bool same = a == b && a_rows == b_rows && ar == br && (as == bs || a_rows == 1);
  return !same && share(a, as, a_rows, ar, b, bs, b_rows, br);
}
inline bool overlap(const void* a, int64_t as, uint32_t a_rows, const void* b, int64_t bs, uint32_t b_rows, int64_t row) {
  return overlap(a, as, a_rows, row, b, bs, b_rows, row);
}

}  // namespace q8

// kx_paged_place.h -- where the rows of a ragged batch and the places of a paged cache lie: arithmetic on what the caller's tables say, in
// plain C++ for host and device.  Nothing here trusts a table: whatever it holds, rows stay in [0, tokens) and pages in [0, pages).
#pragma once
#include <stdint.h>

#if defined(__HIPCC__)
#define KXP_FN __host__ __device__ __forceinline__
#else
#define KXP_FN inline
#endif

namespace kxpage {

constexpr int UNIT = 64;                        // tokens that are read and written together; a page is a whole number of them
constexpr int LEAST = -100;                     // smallest exponent of a scale
constexpr int BAD_PAGE = 1, BAD_POSITION = 2, BAD_ROWS = 4;  // what kx_paged_faults reports

// Rows [first, first + n) of a sequence, its first one at position pos.
struct Rows {
  int first, n, pos, fault;
};
// from: start[b], to: start[b + 1]; cap: positions that the table has pages for
KXP_FN Rows rows_of(int from, int to, int pos, int tokens, int cap) {
  Rows r = {from, to - from, pos, 0};
  if (from < 0 || to < from || to > tokens) return {0, 0, 0, BAD_ROWS};
  if (r.n && (pos < 0 || pos > cap - r.n)) return {from, 0, 0, BAD_POSITION};
  return r;
}
// units that n positions from pos on touch
KXP_FN int units_of(int pos, int n) { return n > 0 ? (pos + n - 1) / UNIT - pos / UNIT + 1 : 0; }
KXP_FN bool page_ok(int id, int pages) { return id >= 0 && id < pages; }

// Place of token t of 64 in a row of cached values.  The matrix cores' sums of scores leave tokens 4 q .. 4 q + 3 of a block of 16 in quarter q of the
// wave, and the product with the values takes 8 tokens a quarter, which may be any as long as both operands agree: blocks 2 h and 2 h + 1 one
// after the other.  A quarter's 16 tokens of both halves then are 16 bytes in a row.
KXP_FN int place_of(int t) { return (t >> 2 & 3) << 4 | (t >> 5) << 3 | (t >> 4 & 1) << 2 | (t & 3); }
KXP_FN int token_of(int place) { return (place >> 3 & 1) << 5 | (place >> 2 & 1) << 4 | (place >> 4) << 2 | (place & 3); }

// The least e >= LEAST with x <= 448 * 2^e for the positive finite float of these bits: 1.75 * 2^8 is 448.
KXP_FN int exponent_of(uint32_t bits) {
  const int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < LEAST ? LEAST : e;
}
KXP_FN uint32_t scale_bits(int e) { return (uint32_t)(e + 127) << 23; }                 // 2^e
KXP_FN int scale_exponent(uint32_t bits) { return (int)(bits >> 23 & 0xffu) - 127; }    // of a scale

// Padded widths of cached rows: the tile of the attention kernels that holds both.
struct Widths {
  int k, v;
};
KXP_FN Widths widths_of(int dim, int vdim) {
  const Widths w[4] = {{64, 64}, {128, 128}, {192, 128}, {256, 256}};
  for (int i = 0; i < 4; ++i)
    if (dim <= w[i].k && vdim <= w[i].v) return w[i];
  return {0, 0};
}

}  // namespace kxpage

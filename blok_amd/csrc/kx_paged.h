// kx_paged.h -- a cache of keys and values in pages, in 8 bits with a scale for each block of tokens and head, and the attention over it
// (kx_paged_cache.hip, kx_paged_attend.hip).  No counterpart in the reference, whose cache is 32-bit tiles on a disk (src/kimi_exec.cu:192-238).
//
// An element is an e4m3 code times its block's scale 2^e, with e the least whole number from -100 on that keeps the block's largest magnitude within
// 448 * 2^e.  Scales are powers of two, so that a block whose scale grows when a token is appended keeps the elements it has: dividing a code by a power
// of two rounds only where the result is below the smallest normal number, 2^-6.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "kx_paged_place.h"

struct KxDivider {
  int d = 1;
  uint32_t m = 0;  // (2^32 - 1) / d
};
struct KxPagedSpec {
  int heads = 0, kv_heads = 0, dim = 0, vdim = 0, page = 0, block = 0, rot = 0, pairs = 0, size = 0;
  float scale = 1;
  int dp = 0, vp = 0;  // padded widths
};
struct KxPagedArgs {
  KxPagedSpec s;
  uint8_t *k = nullptr, *v = nullptr;    // [pages][kv_heads][page][dp]; [pages][kv_heads][page / 64][vp][64], a row's tokens by kxpage::place_of
  float *ks = nullptr, *vs = nullptr;    // [pages][kv_heads][page / block]
  const int *table = nullptr;            // [batch][table_ld]
  int pages = 0, table_ld = 0;
  const int *start = nullptr, *pos = nullptr;  // [batch + 1], [batch]
  int batch = 0, tokens = 0, longest = 0;
  const float *proj = nullptr;  // f32 [tokens][proj_ld]
  int proj_ld = 0, q_off = 0, k_off = 0, v_off = 0;
  const double *turn = nullptr;  // [rot / 2] turns per position
  void *out = nullptr;           // attention: [tokens][out_ld] of the number format; read: keys
  void *out_v = nullptr;         // read: values
  int out_ld = 0, out_v_ld = 0;
  bool wide_k = false, wide_v = false;  // rows of results are whole pieces: of 16 bytes read, of 4 elements of an attention
  int *fault = nullptr;          // KX_PAGED_* bits
  // attention: sums of parts of the positions, and who has handed his in
  float *part = nullptr;
  size_t part_floats = 0;
  int *arrived = nullptr;
  int arrivals = 0;
  KxDivider by_g, by_kv, per_page, by_splits;  // heads of a head of keys, heads of keys, groups of a page, parts
  int block_bits = 0;                          // of the size of a block
  int chunk = 0, splits = 0;     // units of a part (set by the launcher)
};
int kx_paged_append_launch(const KxPagedArgs &a, hipStream_t st);
int kx_paged_read_launch(const KxPagedArgs &a, hipStream_t st);
int kx_paged_attend_launch(bool f32, const KxPagedArgs &a, hipStream_t st);
// counters and floats of parts that steps of up to max_tokens rows of max_batch sequences can use
int kx_paged_arrivals(const KxPagedSpec &s, int max_batch, int max_tokens);
size_t kx_paged_part_floats(const KxPagedSpec &s, int max_batch, int max_tokens);

namespace kxpage {
inline KxDivider divider(int d) { return {d, 0xffffffffu / (uint32_t)d}; }
}

#if defined(__HIPCC__)
namespace kxpage {

// n / d for n >= 0: 2^32 / d - 1 <= m < 2^32 / d, so that n m / 2^32 lies above n / d - 1 and the whole number below it is the quotient or one less
__device__ __forceinline__ int quotient(int n, KxDivider v) {
  const int q = (int)__umulhi((uint32_t)n, v.m);
  return q + (n - q * v.d >= v.d ? 1 : 0);
}

// Which sequence a workgroup's task belongs to, where every sequence has count(rows) tasks in a row; n: rows.n is 0 past the last task.  All lanes
// of a wave call it and get the same.
struct Task {
  int seq, index;
  Rows r;
};
template <class Count>
__device__ __forceinline__ Task find_task(const KxPagedArgs &a, int task, Count count) {
  const int lane = threadIdx.x & 63, cap = a.table_ld * a.s.page;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const int b = min(b0 + lane, a.batch - 1);
    Rows r = rows_of(a.start[b], a.start[b + 1], a.pos[b], a.tokens, cap);
    if (b0 + lane >= a.batch) r.n = 0;
    if (r.fault && b0 + lane < a.batch) atomicOr(a.fault, r.fault);
    const int mine = count(r);
    int upto = mine;
    if (__builtin_amdgcn_ballot_w64(mine > 1)) {
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(upto, d);
        if (lane >= d) upto += o;
      }
    } else {  // a step of one row each
      const uint64_t some = __builtin_amdgcn_ballot_w64(mine > 0);
      upto += (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(some >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)some, 0));
    }
    const uint64_t past = __builtin_amdgcn_ballot_w64(upto > task);
    if (past) {
      const int l = __builtin_ctzll(past);
      auto of = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
      return {b0 + l, task - of(upto - mine), {of(r.first), of(r.n), of(r.pos), 0}};
    }
    task -= __builtin_amdgcn_readlane(upto, 63);
  }
  return {0, 0, {0, 0, 0, 0}};
}

// Sine and cosine of so many turns, by the series of both about 0 up to an eighth of a turn: the first omitted term is below 2^-60 for double,
// 2^-29 for float.
__device__ __forceinline__ void turned(double turns, double &c, double &s) {
  const double n = __builtin_rint(turns * 4.0), x = __builtin_fma(turns, 4.0, -n) * 1.5707963267948966, z = x * x;
  double a = 1.0 / 355687428096000.0, b = 1.0 / 20922789888000.0;
  a = __builtin_fma(a, z, -1.0 / 1307674368000.0);
  a = __builtin_fma(a, z, 1.0 / 6227020800.0);
  a = __builtin_fma(a, z, -1.0 / 39916800.0);
  a = __builtin_fma(a, z, 1.0 / 362880.0);
  a = __builtin_fma(a, z, -1.0 / 5040.0);
  a = __builtin_fma(a, z, 1.0 / 120.0);
  a = __builtin_fma(a, z, -1.0 / 6.0);
  a = __builtin_fma(a * z, x, x);
  b = __builtin_fma(b, z, -1.0 / 87178291200.0);
  b = __builtin_fma(b, z, 1.0 / 479001600.0);
  b = __builtin_fma(b, z, -1.0 / 3628800.0);
  b = __builtin_fma(b, z, 1.0 / 40320.0);
  b = __builtin_fma(b, z, -1.0 / 720.0);
  b = __builtin_fma(b, z, 1.0 / 24.0);
  b = __builtin_fma(b, z, -0.5);
  b = __builtin_fma(b, z, 1.0);
  const int q = (int)n & 3;
  const double u = q & 1 ? b : a, w = q & 1 ? a : b;
  s = q & 2 ? -u : u;
  c = (q + 1) & 2 ? -w : w;
}
__device__ __forceinline__ void turned(float quarters, int n, float &c, float &s) {  // n + quarters quarter turns, |quarters| <= 1 / 2
  const float x = quarters * 1.57079632679f, z = x * x;
  float a = 1.0f / 362880.0f, b = -1.0f / 3628800.0f;
  a = __builtin_fmaf(a, z, -1.0f / 5040.0f);
  a = __builtin_fmaf(a, z, 1.0f / 120.0f);
  a = __builtin_fmaf(a, z, -1.0f / 6.0f);
  a = __builtin_fmaf(a * z, x, x);
  b = __builtin_fmaf(b, z, 1.0f / 40320.0f);
  b = __builtin_fmaf(b, z, -1.0f / 720.0f);
  b = __builtin_fmaf(b, z, 1.0f / 24.0f);
  b = __builtin_fmaf(b, z, -0.5f);
  b = __builtin_fmaf(b, z, 1.0f);
  const float u = n & 1 ? b : a, w = n & 1 ? a : b;
  s = n & 2 ? -u : u;
  c = (n + 1) & 2 ? -w : w;
}
// turns per position times position, as whole quarter turns (mod 4) and a rest; exact to 2^-53 of the turns
__device__ __forceinline__ void quarters_of(double turn, int pos, float &rest, int &n) {
  double t = turn * (double)pos;
  t = (t - __builtin_rint(t)) * 4.0;
  const double r = __builtin_rint(t);
  n = (int)r & 3;
  rest = (float)(t - r);
}
// first and second dimension of pair p of a row whose first rot dimensions turn
__device__ __forceinline__ int2 pair_of(int p, int rot, int pairs) { return p >= rot / 2 || pairs ? make_int2(2 * p, 2 * p + 1) : make_int2(p, p + rot / 2); }

}  // namespace kxpage
#endif

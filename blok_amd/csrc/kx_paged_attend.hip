// kx_paged_attend.hip -- attention of the newest positions of a ragged batch over a paged cache of 8-bit keys and values (kx_paged.h).  No counterpart
// in the reference, whose attention goes over 32-bit tiles of one sequence (tiled_attention, src/kimi_exec.cu:692-716).
//
// With codes k, v and scales 2^a, 2^b of a token's blocks, and all in powers of two: x_t = (q . k_t) 2^a scale log2(e) + b,
//   out = sum_t 2^(x_t - M) v_t / sum_t 2^(x_t - b - M),  M at most 4 below the largest x so far.
// The values' scale is a part of the exponent, so that the products with the values are of codes and the largest of these weights lies between 1 and 2^4.
// A wave has 16 NQ columns -- a column is a query head of a row, all of them of one head of keys -- and goes through groups of 64 tokens on its own:
//   S^T = K Q^T (v_mfma_f32_16x16x32_f16) leaves each lane scores of one column and of 4 tokens of each block of 16, which is the operand that
//   O^T += V^T P^T wants, with the values' tokens in the order of kxpage::place_of.  Nothing passes through LDS or between lanes but the largest x.
// Codes become f16 in registers, exactly; a query is divided by a power of two and rounded to f16 (2^-11 of an element or 2^-39 of its largest, against the 2^-8 of the bf16
// result; in the 32-bit format it is the sum of two, 2^-22 of an element).  For bf16 results weights times 2^11, which is taken out of the values' codes, are rounded to f16, too: 2^-11 of each
// that is at least 2^-25 of the largest, and 2^-36 of the largest below that.  Many small weights beside a large one make a result as well: in the 32-bit format, a
// weight is the sum of three bf16, which hold any float, and costs two more products (4 sequences of 300 rows after 2700, 177 us with two f16, 203 with three bf16).
// Sums, M and denominators are 32-bit.
// Two forms: few columns a sequence (SHARE): the waves of a workgroup take groups of tokens in turn and are added up in LDS; many: every wave has columns
// of its own.  In both the positions may be split between workgroups, and the last one in adds the parts (kx_arrive.h), in order.
// What bounds it: few columns, HBM -- one position after 131072, 269 MB, 52 us, 11 of them the start and the parts; 64 sequences of up to 8192, 640 MB, 124 us, whose
// lengths differ -- and for short caches the chain from the tables to the pages and the hand-over, 11 us after 4096.  Many columns: vector instructions (128 conversions
// of codes and 32 exponentials for 64 products of a wave), which a SIMD issues in 55 % of the cycles, with its matrix core busy in 24 % and 1.6 waves on average: 580
// TFLOP/s of 1200.
#include <algorithm>
#include <type_traits>
#include "kx_arrive.h"
#include "kx_common.h"
#include "kx_math.h"
#include "kx_paged.h"
#include "kx_read_once.h"
#include "kx_wave.h"

namespace {

using namespace kxpage;

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));

template <class T>
using Constant = const __attribute__((address_space(4))) T *;  // loaded from by scalar loads, since no launch writes what it reads there
struct Scales {
  uint32_t k[4], v[4];
};

constexpr float NONE = -1e30f;  // M where nothing has been seen
constexpr float GROWTH = 4.0f;  // by so much x may be above M before the sums are divided by what M grows
constexpr int ROOM = 11;        // weights are times 2^ROOM beside the matrix cores: the largest at least that, and below 2^15.  7 beside a growth of 8, and 13 beside 2, are as fast
constexpr int FAR = 96;         // where a block's scale is so many powers of two below the largest so far (values of zero have the least), a weight times its scale may be no float
                                // any more and the weight still count: such weights go into the denominator without it.  The test costs 1 % where columns are many
constexpr int STATS = 4096;     // columns times parts of a task

__device__ __forceinline__ h8 unpacked(uint32_t lo, uint32_t hi) {
  const h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.0f, true);
  const h2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.0f, true);
  return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// codes divided by 2^ROOM, exactly: the smallest is 2^-9, and f16 has 2^-24
__device__ __forceinline__ h8 unpacked_down(uint32_t lo, uint32_t hi) {
  constexpr float down = 1.0f / (1 << ROOM);
  const h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, down, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, down, true);
  const h2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, down, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, down, true);
  return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ b8 unpacked_down_wide(uint32_t lo, uint32_t hi) {  // as bf16
  constexpr float down = 1.0f / (1 << ROOM);
  const b2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, down, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, down, true);
  const b2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, down, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, down, true);
  return b8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ f4 mfma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f4 mfma(b8 a, b8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
// over the four quarters of the wave
__device__ __forceinline__ float quarters_max(float v) {
  float o = v;
  kxw::swap_halves32(v, o);
  v = o = fmaxf(v, o);
  kxw::swap_rows16(v, o);
  return fmaxf(v, o);
}
__device__ __forceinline__ uint32_t quarters_max(uint32_t v) {
  float f = kx_bits_f32(v), o = f;
  kxw::swap_halves32(f, o);
  f = o = kx_bits_f32(max(kx_f32_bits(f), kx_f32_bits(o)));
  kxw::swap_rows16(f, o);
  return max(kx_f32_bits(f), kx_f32_bits(o));
}
__device__ __forceinline__ float quarters_sum(float v) {
  float o = v;
  kxw::swap_halves32(v, o);
  v = o = v + o;
  kxw::swap_rows16(v, o);
  return v + o;
}
__device__ __forceinline__ h2 halves_of(float a, float b) { return __builtin_convertvector((f2{a, b}), h2); }
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
// x without what a weight has of the values' scale 2^e and of ROOM
__device__ __forceinline__ float unscaled(float x, uint32_t scale) { return __builtin_amdgcn_ldexpf(x, -(scale_exponent(scale) + ROOM)); }
// x 2^d for a d that may lie below the exponents of floats
__device__ __forceinline__ float lowered(float x, float d) {
  const float f = exp2_(0.5f * d);
  return x * f * f;
}

template <bool ONCE>
__device__ __forceinline__ uint4 piece(const uint8_t *p) {
  if constexpr (ONCE) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    const u4 w = __builtin_nontemporal_load((const u4 *)p);
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  return *(const uint4 *)p;
}

template <int DP_, int VP_, int NQ_, bool SHARE_, bool F32_, bool ONCE_ = false>
struct Form {
  static constexpr int DP = DP_, VP = VP_, NQ = NQ_, NW = 4, THREADS = NW * 64, TILE = 16 * NQ;  // columns of a wave
  static constexpr bool SHARE = SHARE_, F32 = F32_, ONCE = ONCE_;
  static constexpr int COLS = SHARE ? TILE : NW * TILE;                         // of a workgroup
  static constexpr size_t PART = (size_t)COLS * (VP + 2);                       // floats of a part: sums, then M and denominator
  static constexpr int REGISTERS = NQ * (DP / 8 * (F32 ? 2 : 1) + VP / 4 + 16) + DP / 4 + VP / 4;
  static constexpr int WAVES = REGISTERS > 200 ? 1 : 2;                         // per SIMD
  static constexpr int SUB = NQ == 1 ? 4 : 2;                                   // blocks of 16 tokens that are multiplied at a time
  static constexpr int QLD = DP + 4, OLD = 68;                                  // floats of a row in LDS: a query; 64 sums of a column
  static constexpr int Q_FLOATS = (SHARE ? TILE : NW * 16) * QLD, O_FLOATS = NW * 16 * OLD + 2 * NW * TILE;
  static constexpr int LDS = Q_FLOATS > O_FLOATS ? Q_FLOATS : O_FLOATS;
};

template <class FM>
__global__ void __launch_bounds__(FM::THREADS, FM::WAVES) attend_k(KxPagedArgs a) {
  constexpr int DP = FM::DP, VP = FM::VP, NQ = FM::NQ, NW = FM::NW, TILE = FM::TILE, COLS = FM::COLS;
  constexpr bool SHARE = FM::SHARE, F32 = FM::F32;
  __shared__ __attribute__((aligned(16))) float lds[FM::LDS > 2 * STATS ? FM::LDS : 2 * STATS];
  __shared__ int last;
  const KxPagedSpec &s = a.s;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lc = lane & 15, lq = lane >> 4, g = a.by_g.d;
  const int rest = quotient(blockIdx.x, a.by_kv), head = blockIdx.x - rest * s.kv_heads, task = quotient(rest, a.by_splits), split = rest - task * a.splits;
  const Task t = find_task(a, task, [&](const Rows &r) { return (r.n * g + COLS - 1) / COLS; });
  if (!t.r.n) return;
  const int R = t.r.n * g, pos = t.r.pos;
  auto row_of = [&](int column) { return quotient(column, a.by_g); };
  auto low = [&](int hi) { return s.size ? max(hi - s.size + 1, 0) : 0; };
  // the workgroup's units and its part of them
  const int w0 = t.index * COLS, hi_all = pos + row_of(min(w0 + COLS, R) - 1), first = low(pos + row_of(w0)) / UNIT, units = hi_all / UNIT - first + 1;
  const int chunk = max(a.chunk, quotient(units + a.splits - 1, a.by_splits)), used = units <= a.chunk ? 1 : (units + chunk - 1) / chunk;
  if (split >= used) return;
  // the wave's columns
  const int c0 = w0 + (SHARE ? 0 : wave * TILE);
  const bool idle = c0 >= R;
  const int hi_min = pos + row_of(min(c0, R - 1)), hi_max = pos + row_of(min(c0 + TILE - 1, R - 1));
  int hi[NQ], lo[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    hi[n] = pos + row_of(min(c0 + n * 16 + lc, R - 1));
    lo[n] = low(hi[n]);
  }

  // queries: asked for first, a wave a column and a lane a pair of dimensions; turned by their positions into LDS, and from there to the lanes in the order of the
  // keys' loads.  All columns at once where the waves share them, 16 at a time where each has its own.
  constexpr int PP = (DP / 2 + 63) / 64, MINE = SHARE ? TILE / NW : 16, NTH = SHARE ? NW : 1;  // pairs of a lane; a wave's columns at a time, every NTH
  const int q_first = SHARE ? wave : 0;
  auto column = [&](int n, int k) { return min(c0 + n * 16 + k * NTH + q_first, R - 1); };
  float qx[MINE][PP][2];
  auto ask_queries = [&](int n) {
#pragma unroll
    for (int k = 0; k < MINE; ++k) {
      const int c = column(n, k), at = row_of(c);
      const float *const x = a.proj + (size_t)(t.r.first + at) * a.proj_ld + a.q_off + (size_t)(head * g + c - at * g) * s.dim;
#pragma unroll
      for (int p = 0; p < PP; ++p) {
        const int2 d = pair_of(lane + 64 * p, s.rot, s.pairs);
        qx[k][p][0] = d.x < s.dim ? x[d.x] : 0.0f;
        qx[k][p][1] = d.y < s.dim ? x[d.y] : 0.0f;
      }
    }
  };
  double turn[PP];
#pragma unroll
  for (int p = 0; p < PP; ++p) turn[p] = lane + 64 * p < s.rot / 2 ? a.turn[lane + 64 * p] : 0.0;
  ask_queries(0);

  const int u_to = idle ? 0 : min(first + min((split + 1) * chunk, units), hi_max / UNIT + 1);
  const int u_from = max(first + split * chunk, low(hi_min) / UNIT) + (SHARE ? wave : 0);
  constexpr int STEP = SHARE ? NW : 1;
  const Constant<int> table = (Constant<int>)(uintptr_t)(a.table + (size_t)t.seq * a.table_ld);
  const int lo_tile = low(hi_min), lo_most = low(hi_max), per_page = s.page / UNIT, scales_per_page = s.page / s.block;
  // keys and values of a group are asked for as soon as those of the one before have been used, its page two groups ahead; pages and scales by scalar loads
  uint4 kr[4][DP / 64], vr[VP / 16];
  auto page_at = [&](int u) { return table[quotient(min(u, u_to - 1), a.per_page)]; };
  auto in_page = [&](int u) { return (u - quotient(u, a.per_page) * per_page) * UNIT; };
  auto head_of = [&](int id) { return (size_t)(page_ok(id, a.pages) ? id : 0) * s.kv_heads + head; };
  auto load_k = [&](int u, int id) {
    const uint8_t *const k = a.k + (head_of(id) * s.page + in_page(u)) * DP + lc * DP + lq * 16;
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int j = 0; j < DP / 64; ++j) kr[tt][j] = piece<FM::ONCE>(k + tt * 16 * DP + j * 64);
  };
  auto load_v = [&](int u, int id) {
    const uint8_t *const v = a.v + (head_of(id) * s.page + in_page(u)) * VP + lc * UNIT + lq * 16;
#pragma unroll
    for (int i = 0; i < VP / 16; ++i) vr[i] = piece<FM::ONCE>(v + i * 16 * UNIT);
  };
  // scales of the four blocks of 16 of a group
  auto load_scales = [&](int u, int id) {
    const size_t at = head_of(id) * scales_per_page;
    const Constant<uint32_t> k = (Constant<uint32_t>)(uintptr_t)(a.ks + at), v = (Constant<uint32_t>)(uintptr_t)(a.vs + at);
    Scales r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = (in_page(u) + i * 16) >> a.block_bits;
      r.k[i] = k[j];
      r.v[i] = v[j];
    }
    return r;
  };
  int id = 0, next = 0;
  Scales sc = {};
  if (u_from < u_to) {
    id = page_at(u_from);
    next = page_at(u_from + STEP);
    load_k(u_from, id);
    load_v(u_from, id);
    sc = load_scales(u_from, id);
  }

  h8 q[NQ][DP / 32], ql[F32 ? NQ : 1][F32 ? DP / 32 : 1];
  float qf[NQ];
  float *const rows = lds + (SHARE ? 0 : wave * 16 * FM::QLD);
#pragma unroll
  for (int n0 = 0; n0 < NQ; n0 += SHARE ? NQ : 1) {
    if (n0) ask_queries(n0);
    int turned_at = -1;
    float cs[PP], sn[PP];
#pragma unroll
    for (int k = 0; k < MINE; ++k) {
      const int at = row_of(column(n0, k));
      if (at != turned_at) {
        turned_at = at;
#pragma unroll
        for (int p = 0; p < PP; ++p) {
          float quarters;
          int whole;
          quarters_of(turn[p], pos + at, quarters, whole);
          turned(quarters, whole, cs[p], sn[p]);
        }
      }
#pragma unroll
      for (int p = 0; p < PP; ++p) {
        if (lane + 64 * p >= DP / 2) continue;
        const int2 d = pair_of(lane + 64 * p, s.rot, s.pairs);
        const float u = qx[k][p][0], v = qx[k][p][1];
        const bool turns = lane + 64 * p < s.rot / 2;
        float *const row = rows + (k * NTH + q_first) * FM::QLD;
        row[d.x] = turns ? u * cs[p] - v * sn[p] : u;
        row[d.y] = turns ? u * sn[p] + v * cs[p] : v;
      }
    }
    __syncthreads();
#pragma unroll
    for (int n = n0; n < (SHARE ? NQ : n0 + 1); ++n) {
      uint32_t most = 0;  // bits of the largest magnitude; those of what is not finite are above those of all that is
      const float *const mine = rows + ((n - n0) * 16 + lc) * FM::QLD + lq * 16;
#pragma unroll
      for (int j = 0; j < DP / 64; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) most = max(most, kx_f32_bits(mine[j * 64 + e]) & 0x7fffffffu);
      most = quarters_max(most);
      const int e = max((int)(most >> 23) - 141, -100);  // the largest element becomes 2^14 or more: f16 has 2^-24 beside it
      // a query that is not finite has infinite scores or none, and NaN for their softmax: NaN in all elements, where minus infinity would hide its positions
      const float down = most >= 0x7f800000u ? __builtin_nanf("") : s.scale == 0.0f ? 0.0f : __builtin_copysignf(kx_bits_f32(scale_bits(-e)), s.scale);
      qf[n] = kx_bits_f32(scale_bits(e)) * __builtin_fabsf(s.scale) * 1.44269504088896341f;
#pragma unroll
      for (int j = 0; j < DP / 64; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float x = mine[j * 64 + e] * down;
          const _Float16 h = (_Float16)x;
          q[n][2 * j + (e >> 3)][e & 7] = h;
          if constexpr (F32) ql[n][2 * j + (e >> 3)][e & 7] = (_Float16)(x - (float)h);
        }
    }
    __syncthreads();
  }

  f4 o[NQ][VP / 16];
  float m[NQ], l[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m[n] = NONE;
    l[n] = 0.0f;
#pragma unroll
    for (int v = 0; v < VP / 16; ++v) o[n][v] = f4{0, 0, 0, 0};
  }

  // a group, SUB blocks of 16 at a time
  constexpr int SUB = FM::SUB;
  int most_scale = kxpage::LEAST;  // largest exponent of the values' scales so far
  for (int u = u_from; u < u_to; u += STEP) {
    const bool there = page_ok(id, a.pages);
    const int base = u * UNIT, after = page_at(u + 2 * STEP);
    const bool whole = there & (base + UNIT - 1 <= hi_min) & (base >= lo_most);  // every column sees all of it
    uint32_t ks[4], vs[4];
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
      ks[tt] = sc.k[tt];
      vs[tt] = sc.v[tt];
    }
    bool nan = false;
    if (!whole) {
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {  // blocks that no column sees may hold anything
        const bool unseen = !there | (base + tt * 16 > hi_max) | (base + tt * 16 + 15 < lo_tile);
        ks[tt] = unseen ? 0x3f800000u : ks[tt];
        vs[tt] = unseen ? 0x3f800000u : vs[tt];
      }
      if (!there && lane == 0) atomicOr(a.fault, BAD_PAGE);
#pragma unroll
      for (int d = 0; d < 4; ++d) {  // values that no column sees, and NaN, become zero
        const int b = base + (d >> 1) * 32 + (d & 1) * 16 + lq * 4;
        const int to = max(min(hi_max - b + 1, 4), 0), from = max(min(lo_tile - b, 4), 0);
        const uint32_t keep = !there ? 0u : (to == 4 ? ~0u : (1u << 8 * to) - 1u) & (from == 4 ? 0u : ~0u << 8 * from);
#pragma unroll
        for (int i = 0; i < VP / 16; ++i) {
          uint32_t &w = d == 0 ? vr[i].x : d == 1 ? vr[i].y : d == 2 ? vr[i].z : vr[i].w;
          w &= keep;
          const uint32_t bad = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
          w &= ~((bad >> 7) * 0xffu);
          nan |= bad != 0;
        }
      }
    }
#pragma unroll
    for (int t0 = 0; t0 < 4; t0 += SUB) {
      f4 x[NQ][SUB];
#pragma unroll
      for (int tt = 0; tt < SUB; ++tt) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) x[n][tt] = f4{0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < DP / 64; ++j) {
          const h8 k0 = unpacked(kr[t0 + tt][j].x, kr[t0 + tt][j].y), k1 = unpacked(kr[t0 + tt][j].z, kr[t0 + tt][j].w);
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            x[n][tt] = mfma(k0, q[n][2 * j], x[n][tt]);
            x[n][tt] = mfma(k1, q[n][2 * j + 1], x[n][tt]);
            if constexpr (F32) {
              x[n][tt] = mfma(k0, ql[n][2 * j], x[n][tt]);
              x[n][tt] = mfma(k1, ql[n][2 * j + 1], x[n][tt]);
            }
          }
        }
      }
      if (t0 + SUB == 4 && u + STEP < u_to) {
        load_k(u + STEP, next);
        sc = load_scales(u + STEP, next);
      }
      int least_scale = scale_exponent(vs[t0]);
      most_scale = max(most_scale, least_scale);
#pragma unroll
      for (int tt = 1; tt < SUB; ++tt) {
        most_scale = max(most_scale, scale_exponent(vs[t0 + tt]));
        least_scale = min(least_scale, scale_exponent(vs[t0 + tt]));
      }
      const bool far = most_scale - least_scale > FAR;
      typedef std::conditional_t<F32, b8, h8> P8;
      P8 ph[NQ][SUB / 2], pm[F32 ? NQ : 1][SUB / 2], pl[F32 ? NQ : 1][SUB / 2];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        if (!whole) {
          // positions of the lane's tokens that its column sees, counted from its first token
          const int from = there ? lo[n] - (base + t0 * 16 + lq * 4) : 1 << 30, to = hi[n] - (base + t0 * 16 + lq * 4);
#pragma unroll
          for (int tt = 0; tt < SUB; ++tt)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[n][tt][i] = ((tt * 16 + i > to) | (tt * 16 + i < from)) ? -__builtin_inff() : x[n][tt][i];
        }
        // x = score f + b, which grows with the score: the largest of a block's by its largest score.  f is above zero, so that -inf stays
        float most = NONE, f[SUB];
#pragma unroll
        for (int tt = 0; tt < SUB; ++tt) {
          f[tt] = fmaxf(qf[n] * kx_bits_f32(ks[t0 + tt]), 1e-37f);
          const float score = fmaxf(fmaxf(x[n][tt][0], x[n][tt][1]), fmaxf(x[n][tt][2], x[n][tt][3]));
          most = fmaxf(most, __builtin_fmaf(score, f[tt], (float)scale_exponent(vs[t0 + tt])));
        }
        most = fmaxf(m[n], quarters_max(most));
        if (far || __builtin_amdgcn_ballot_w64(most > m[n] + GROWTH)) {
          const float less = m[n] - most, shrink = exp2_(less);
          m[n] = most;
          l[n] = lowered(l[n], less);
#pragma unroll
          for (int v = 0; v < VP / 16; ++v) o[n][v] *= shrink;
          if (far) {
#pragma unroll
            for (int tt = 0; tt < SUB; ++tt)
#pragma unroll
              for (int i = 0; i < 4; ++i)  // the weight, and what will be added below instead of it
                l[n] += exp2_(__builtin_fmaf(x[n][tt][i], f[tt], -m[n])) -
                        unscaled(exp2_(__builtin_fmaf(x[n][tt][i], f[tt], (float)(scale_exponent(vs[t0 + tt]) + ROOM) - m[n])), vs[t0 + tt]);
          }
        }
#pragma unroll
        for (int tt = 0; tt < SUB; ++tt) {
          f4 p;
          const float less = (float)(scale_exponent(vs[t0 + tt]) + ROOM) - m[n];
#pragma unroll
          for (int i = 0; i < 4; ++i) p[i] = exp2_(__builtin_fmaf(x[n][tt][i], f[tt], less));
          l[n] += unscaled((p[0] + p[1]) + (p[2] + p[3]), vs[t0 + tt]);
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            auto put = [&](P8 &to, auto w) {
              to[(tt & 1) * 4 + i] = w[0];
              to[(tt & 1) * 4 + i + 1] = w[1];
            };
            if constexpr (F32) {  // three bf16 hold a float
              float a = p[i], b = p[i + 1];
              auto next = [&](P8 &to) {
                const b2 w = __builtin_convertvector((f2{a, b}), b2);
                put(to, w);
                a -= (float)w[0], b -= (float)w[1];
              };
              next(ph[n][tt >> 1]);
              next(pm[n][tt >> 1]);
              next(pl[n][tt >> 1]);
            } else {
              put(ph[n][tt >> 1], halves_of(p[i], p[i + 1]));
            }
          }
        }
      }
#pragma unroll
      for (int i = 0; i < VP / 16; ++i)
#pragma unroll
        for (int h = 0; h < SUB / 2; ++h) {
          const uint32_t lo = t0 / 2 + h == 0 ? vr[i].x : vr[i].z, hi = t0 / 2 + h == 0 ? vr[i].y : vr[i].w;
          P8 v;
          if constexpr (F32) v = unpacked_down_wide(lo, hi);
          else v = unpacked_down(lo, hi);
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            o[n][i] = mfma(v, ph[n][h], o[n][i]);
            if constexpr (F32) o[n][i] = mfma(v, pl[n][h], mfma(v, pm[n][h], o[n][i]));
          }
        }
    }
    if (u + STEP < u_to) load_v(u + STEP, next);
    if (!whole)
      if (__builtin_amdgcn_ballot_w64(nan)) {  // NaN among the values: the columns that see it, which products of ones and zeros say, have it
        const uint8_t *const v = a.v + (head_of(id) * s.page + in_page(u)) * VP + lc * UNIT + lq * 16;
        h8 sees[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int j = base + (e >> 2) * 16 + lq * 4 + (e & 3);
            sees[n][e >> 3][e & 7] = ((j <= hi[n]) & (j >= lo[n])) ? (_Float16)1.0f : (_Float16)0.0f;
          }
#pragma unroll
        for (int i = 0; i < VP / 16; ++i) {
          uint4 w = *(const uint4 *)(v + i * 16 * UNIT);
          auto ones = [](uint32_t w) { return ((((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0x38u; };
          const h8 v0 = unpacked(ones(w.x), ones(w.y)), v1 = unpacked(ones(w.z), ones(w.w));
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            const f4 seen = mfma(v1, sees[n][1], mfma(v0, sees[n][0], f4{0, 0, 0, 0}));
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n][i][e] = seen[e] > 0.0f ? __builtin_nanf("") : o[n][i][e];
          }
        }
      }
    id = next;
    next = after;
  }
#pragma unroll
  for (int n = 0; n < NQ; ++n) l[n] = quarters_sum(l[n]);

  // results: four neighbouring dimensions of a column at a time
  float *const part = a.part + (size_t)(task * s.kv_heads + head) * a.splits * FM::PART;
  auto give = [&](int c, int d, f4 y) {  // column c of the sequence, dimensions d .. d + 3
    const int at = row_of(c);
    const size_t to = (size_t)(t.r.first + at) * a.out_ld + (size_t)(head * g + c - at * g) * s.vdim + d;
    if (a.wide_v) {
      if (d >= s.vdim) return;
      if constexpr (F32) *(f4 *)((float *)a.out + to) = y;
      else *(uint2 *)((uint16_t *)a.out + to) = make_uint2(kx_bf16_rne(y[0]) | (uint32_t)kx_bf16_rne(y[1]) << 16, kx_bf16_rne(y[2]) | (uint32_t)kx_bf16_rne(y[3]) << 16);
      return;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (d + e < s.vdim) {
        if constexpr (F32) ((float *)a.out)[to + e] = y[e];
        else ((uint16_t *)a.out)[to + e] = kx_bf16_rne(y[e]);
      }
  };
  auto hand = [&](int c, int d, f4 y) {  // column c of the workgroup
    uint64_t *const to = (uint64_t *)(part + split * FM::PART + (size_t)c * VP + d);
    kx_arrive_store(to, (uint64_t)kx_f32_bits(y[0]) | (uint64_t)kx_f32_bits(y[1]) << 32);
    kx_arrive_store(to + 1, (uint64_t)kx_f32_bits(y[2]) | (uint64_t)kx_f32_bits(y[3]) << 32);
  };
  auto hand_stats = [&](int c, float m, float l) {
    kx_arrive_store((uint64_t *)(part + split * FM::PART + (size_t)COLS * VP) + c, (uint64_t)kx_f32_bits(m) | (uint64_t)kx_f32_bits(l) << 32);
  };
  if constexpr (SHARE) {
    float2 *const stats = (float2 *)(lds + NW * 16 * FM::OLD);  // [NW][TILE]
    if (lq == 0) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) stats[wave * TILE + n * 16 + lc] = make_float2(m[n], l[n]);
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int h = 0; h < VP / 64; ++h) {
#pragma unroll
        for (int i = 0; i < 4; ++i) *(f4 *)(lds + (wave * 16 + lc) * FM::OLD + i * 16 + lq * 4) = o[n][h * 4 + i];
        __syncthreads();
        for (int i = threadIdx.x; i < 256; i += FM::THREADS) {
          const int c = i >> 4, d = (i & 15) * 4;
          float2 st[NW];
          float most = NONE, sum = 0.0f;
#pragma unroll
          for (int w = 0; w < NW; ++w) {
            st[w] = stats[w * TILE + n * 16 + c];
            most = fmaxf(most, st[w].x);
          }
          f4 y = {0, 0, 0, 0};
#pragma unroll
          for (int w = 0; w < NW; ++w) {
            const float f = exp2_(st[w].x - most);
            sum += lowered(st[w].y, st[w].x - most);
            const f4 x = *(const f4 *)(lds + (w * 16 + c) * FM::OLD + d);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf(x[e], f, y[e]);
          }
          const int cc = w0 + n * 16 + c;
          if (cc < R) {
            if (used == 1) {
              const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
              give(cc, h * 64 + d, y * f);
            } else {
              hand(n * 16 + c, h * 64 + d, y);
              if (h == 0 && d == 0) hand_stats(n * 16 + c, most, sum);
            }
          }
        }
        __syncthreads();
      }
  } else if (!idle) {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int c = c0 + n * 16 + lc;
      if (c >= R) continue;
      if (used == 1) {
        const float f = l[n] == 0.0f ? 0.0f : 1.0f / l[n];
#pragma unroll
        for (int i = 0; i < VP / 16; ++i) give(c, i * 16 + lq * 4, o[n][i] * f);
      } else {
#pragma unroll
        for (int i = 0; i < VP / 16; ++i) hand(c - w0, i * 16 + lq * 4, o[n][i]);
        if (lq == 0) hand_stats(c - w0, m[n], l[n]);
      }
    }
  }
  if (used == 1) return;
  kx_arrive_writes_done();
  __syncthreads();
  int *const arrived = a.arrived + task * s.kv_heads + head;
  if (threadIdx.x == 0) last = kx_arrive_is_last(arrived, used);
  __syncthreads();
  if (!last) return;
  if (threadIdx.x == 0) kx_arrive_reset(arrived);
  // sums of the parts: a lane four dimensions of ITEMS columns, AT_ONCE parts at a time; the first of them are asked for before the weights are worked out, 16
  // lanes a column
  const int cols = min(COLS, R - w0);
  float2 *const st = (float2 *)lds;  // [used][COLS]
  auto stat_of = [&](int i) { return kx_arrive_load((const uint64_t *)(part + (size_t)(i / COLS) * FM::PART + (size_t)COLS * VP) + i % COLS); };
  auto keep = [&](int i, uint64_t w) { st[i] = make_float2(kx_bits_f32((uint32_t)w), kx_bits_f32((uint32_t)(w >> 32))); };
  const bool first_stat = (int)threadIdx.x < used * COLS && (int)threadIdx.x % COLS < cols;
  const uint64_t first_word = first_stat ? stat_of(threadIdx.x) : 0;
  auto weights = [&]() {
    if (first_stat) keep(threadIdx.x, first_word);
    for (int i = threadIdx.x + FM::THREADS; i < used * COLS; i += FM::THREADS)
      if (i % COLS < cols) keep(i, stat_of(i));
    __syncthreads();
    for (int c = threadIdx.x >> 4; c < cols; c += FM::THREADS / 16) {
      float most = NONE, sum = 0.0f;
      for (int p = lc; p < used; p += 16) most = fmaxf(most, st[p * COLS + c].x);
#pragma unroll
      for (int d = 1; d < 16; d <<= 1) most = fmaxf(most, __shfl_xor(most, d));
      for (int p = lc; p < used; p += 16) sum += lowered(st[p * COLS + c].y, st[p * COLS + c].x - most);
#pragma unroll
      for (int d = 1; d < 16; d <<= 1) sum += __shfl_xor(sum, d);
      const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
      for (int p = lc; p < used; p += 16) st[p * COLS + c].x = exp2_(st[p * COLS + c].x - most) * f;
    }
    __syncthreads();
  };
  auto add_up = [&](auto items_, auto at_once_) {
    constexpr int ITEMS = items_(), AT_ONCE = at_once_();
    const int items = cols * (VP / 4);
    bool weighed = false;
    for (int i0 = threadIdx.x; i0 - (int)threadIdx.x < items; i0 += ITEMS * FM::THREADS) {
      f4 y[ITEMS];
#pragma unroll
      for (int n = 0; n < ITEMS; ++n) y[n] = f4{0, 0, 0, 0};
      for (int p0 = 0; p0 < used; p0 += AT_ONCE) {
        uint64_t w[ITEMS][AT_ONCE][2];
#pragma unroll
        for (int n = 0; n < ITEMS; ++n) {
          const uint64_t *const from = (const uint64_t *)(part + (size_t)min(i0 + n * FM::THREADS, items - 1) * 4);
#pragma unroll
          for (int k = 0; k < AT_ONCE; ++k)
            if (p0 + k < used) {
              const size_t at = (size_t)(p0 + k) * (FM::PART / 2);
              w[n][k][0] = kx_arrive_load(from + at);
              w[n][k][1] = kx_arrive_load(from + at + 1);
            }
        }
        if (!weighed) {
          weights();
          weighed = true;
        }
#pragma unroll
        for (int n = 0; n < ITEMS; ++n) {
          const int c = min((i0 + n * FM::THREADS) / (VP / 4), cols - 1);
          float f[AT_ONCE];
#pragma unroll
          for (int k = 0; k < AT_ONCE; ++k) f[k] = st[min(p0 + k, used - 1) * COLS + c].x;
#pragma unroll
          for (int k = 0; k < AT_ONCE; ++k) {
            if (p0 + k >= used) break;
            y[n][0] = __builtin_fmaf(kx_bits_f32((uint32_t)w[n][k][0]), f[k], y[n][0]);
            y[n][1] = __builtin_fmaf(kx_bits_f32((uint32_t)(w[n][k][0] >> 32)), f[k], y[n][1]);
            y[n][2] = __builtin_fmaf(kx_bits_f32((uint32_t)w[n][k][1]), f[k], y[n][2]);
            y[n][3] = __builtin_fmaf(kx_bits_f32((uint32_t)(w[n][k][1] >> 32)), f[k], y[n][3]);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < ITEMS; ++n) {
        const int i = i0 + n * FM::THREADS;
        if (i < items) give(w0 + i / (VP / 4), i % (VP / 4) * 4, y[n]);
      }
    }
  };
  if (used <= 8) add_up(std::integral_constant<int, 2>(), std::integral_constant<int, 8>());
  else add_up(std::integral_constant<int, 1>(), std::integral_constant<int, 16>());
}

template <class FM>
int launch(KxPagedArgs a, int g, hipStream_t st) {
  const int cus = std::max(1, kx_device_cus()), kv = a.s.kv_heads;
  // tasks: at most a partly filled one of every sequence and the full ones
  const long tasks = std::min<long>((long)std::min(a.batch, a.tokens) + (long)a.tokens * g / FM::COLS, (long)a.arrivals / kv);
  const long rows = std::max<long>(1, (a.tokens + a.batch - 1) / a.batch);
  const long most = a.s.size ? std::min<long>(a.longest, (long)a.s.size + rows - 1 + UNIT) : a.longest;
  const int units = (int)((std::max<long>(most, 1) + UNIT - 1) / UNIT);
  const long busy = (long)std::min(a.batch, a.tokens) * ((rows * g + FM::COLS - 1) / FM::COLS) * kv;  // workgroups of whole sequences
  const long room = std::min<long>({(long)(a.part_floats / FM::PART) / std::max<long>(1, tasks * kv), STATS / FM::COLS, units});
  // a workgroup for each that the card holds; one a CU where a few long sequences fill it evenly: 1 x 131072 56.0 -> 51.9 us, 2 x 131072 87.3 -> 82.7, but 16 x 8192
  // 41.5 -> 42.4 and 40 x 8192 94 -> 126, whose sequences differ in length
  const long slots = (long)cus * (FM::ONCE && busy * 8 <= cus ? 1 : FM::WAVES), want = (slots + busy - 1) / busy;
  // Where waves share columns, a part has a group for each at least, and where more than 256 columns of parts are for one workgroup to add up, eight.  Where
  // they do not, adding up 128 columns takes as long as 12 groups, and a part has 20: 256 rows after 7744, 6 parts 251 -> 129 us, 100 rows after 7900 237 -> 89,
  // but 300 rows after 1700 in 2 parts 72 -> 79, 100 rows after 500 32 -> 38.
  const long most_parts = FM::SHARE ? std::max<long>(std::min<long>(units / FM::NW, 256 / FM::COLS), units / (FM::NW * 8)) : units / 20;
  a.splits = (int)std::max<long>(1, std::min({room, want, most_parts}));
  a.chunk = (units + a.splits - 1) / a.splits;
  a.by_splits = divider(a.splits);
  // a sequence longer than `longest` has longer parts
  attend_k<FM><<<dim3((unsigned)(tasks * a.splits * kv)), FM::THREADS, 0, st>>>(a);
  KX_LAUNCH_CHECK();
  return KX_OK;
}

template <int DP, int VP, bool F32>
int launch_columns(const KxPagedArgs &a, hipStream_t st) {
  const int g = a.s.heads / a.s.kv_heads;
  const long columns = (long)a.tokens * g / std::min(a.batch, a.tokens);  // of a sequence, on average
  constexpr int NQ = DP == 256 ? 1 : 2;  // the widest rows leave registers for one block of columns
  // a cache that no level of caches holds is read past them where one workgroup reads each of its positions: 269 MB 61.8 -> 51.9 us with fewer parts, 56.0 with as
  // many, 640 MB 127 -> 124; with 131 MB, which the last level holds from one call to the next in a program of one layer, it takes 33.3 us instead of 31.3
  const size_t seen = a.s.size ? std::min(a.longest, a.s.size) : a.longest;
  if (columns <= 16 && kxonce::latent((size_t)std::min(a.batch, a.tokens) * seen * a.s.kv_heads * (DP + VP))) return launch<Form<DP, VP, 1, true, F32, true>>(a, g, st);
  if (columns <= 16) return launch<Form<DP, VP, 1, true, F32>>(a, g, st);
  if (columns <= 64) return launch<Form<DP, VP, NQ, true, F32>>(a, g, st);
  return launch<Form<DP, VP, NQ, false, F32>>(a, g, st);
}
template <bool F32>
int launch_widths(const KxPagedArgs &a, hipStream_t st) {
  if (a.s.dp == 64) return launch_columns<64, 64, F32>(a, st);
  if (a.s.dp == 128) return launch_columns<128, 128, F32>(a, st);
  if (a.s.dp == 192) return launch_columns<192, 128, F32>(a, st);
  return launch_columns<256, 256, F32>(a, st);
}

}  // namespace

int kx_paged_arrivals(const KxPagedSpec &s, int max_batch, int max_tokens) {
  const long tasks = (long)std::min(max_batch, max_tokens) + (long)max_tokens * (s.heads / s.kv_heads) / 16;
  return (int)std::min<long>(tasks * s.kv_heads, 0x7fffffff);
}
// room for a part of each of 512 workgroups of 64 columns of 128 dimensions, or for four parts of every column, those of partly filled blocks among them, in calls
// whose sequences have more than 64; 128 MB at most
size_t kx_paged_part_floats(const KxPagedSpec &s, int max_batch, int max_tokens) {
  const size_t g = (size_t)(s.heads / s.kv_heads), least = (size_t)512 * 64 * 130, most = (size_t)1 << 25;
  const size_t sequences = std::min<size_t>((size_t)std::min(max_batch, max_tokens), (size_t)max_tokens * g / 64 + 1);
  return std::max(least, std::min(most, 4 * (size_t)(s.vp + 2) * ((size_t)max_tokens * (size_t)s.heads + 128 * (size_t)s.kv_heads * sequences)));
}
int kx_paged_attend_launch(bool f32, const KxPagedArgs &a, hipStream_t st) { return f32 ? launch_widths<true>(a, st) : launch_widths<false>(a, st); }

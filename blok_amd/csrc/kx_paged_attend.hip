// kx_paged_attend.hip -- attention of the newest positions of a ragged batch over a paged cache of 8-bit keys and values (kx_paged.h).  No counterpart
// in the reference, whose attention goes over 32-bit tiles of one sequence (tiled_attention, src/kimi_exec.cu:692-716).
//
// With codes k, v and scales 2^a, 2^b of a token's blocks, and all in powers of two: x_t = (q . k_t) 2^a scale log2(e) + b,
//   out = sum_t 2^(x_t - M) v_t / sum_t 2^(x_t - b - M),  M the largest x so far.
// The values' scale is a part of the exponent, so that the products with the values are of codes as they are and the largest weight is 1.
// A wave has 16 NQ columns -- a column is a query head of a row, all of them of one head of keys -- and goes through groups of 64 tokens on its own:
//   S^T = K Q^T (v_mfma_f32_16x16x32_f16) leaves each lane scores of one column and of 4 tokens of each block of 16, which is the operand that
//   O^T += V^T P^T wants, with the values' tokens in the order of kxpage::place_of.  Nothing passes through LDS or between lanes but the largest x.
// Codes become f16 in registers, exactly; a query is divided by a power of two and rounded to f16, weights likewise (2^-12 of each, against the 2^-9 of
// the bf16 result; in the 32-bit format both are the sum of two f16, 2^-22).  Sums, M and denominators are 32-bit.
// Two forms: few columns a sequence (SHARE): the waves of a workgroup take groups of tokens in turn and are added up in LDS; many: every wave has columns
// of its own.  In both the positions may be split between workgroups, and the last one in adds the parts (kx_arrive.h), in order.
#include <algorithm>
#include "kx_arrive.h"
#include "kx_common.h"
#include "kx_math.h"
#include "kx_paged.h"

namespace {

using namespace kxpage;

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr float NONE = -1e30f;  // M where nothing has been seen
constexpr int STATS = 4096;     // columns times parts of a task

__device__ __forceinline__ h8 unpacked(uint32_t lo, uint32_t hi) {
  const h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.0f, true);
  const h2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.0f, true);
  return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ f4 mfma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
// over the four quarters of the wave
__device__ __forceinline__ float quarters_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float quarters_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

template <int DP_, int VP_, int NQ_, bool SHARE_, bool F32_>
struct Form {
  static constexpr int DP = DP_, VP = VP_, NQ = NQ_, NW = 4, THREADS = NW * 64, TILE = 16 * NQ;  // columns of a wave
  static constexpr bool SHARE = SHARE_, F32 = F32_;
  static constexpr int COLS = SHARE ? TILE : NW * TILE;                         // of a workgroup
  static constexpr size_t PART = (size_t)COLS * (VP + 2);                       // floats of a part: sums, then M and denominator
  static constexpr int REGISTERS = NQ * (DP / 8 * (F32 ? 2 : 1) + VP / 4 + 16) + DP / 4 + VP / 4;
  static constexpr int WAVES = REGISTERS > 200 ? 1 : 2;                         // per SIMD
  static constexpr int QLD = DP + 4, OLD = 68;                                  // floats of a row in LDS: a query; 64 sums of a column
  static constexpr int Q_FLOATS = (SHARE ? 1 : NW) * 16 * QLD, O_FLOATS = NW * 16 * OLD + 2 * NW * TILE;
  static constexpr int LDS = Q_FLOATS > O_FLOATS ? Q_FLOATS : O_FLOATS;
};

template <class FM>
__global__ void __launch_bounds__(FM::THREADS, FM::WAVES) attend_k(KxPagedArgs a) {
  constexpr int DP = FM::DP, VP = FM::VP, NQ = FM::NQ, NW = FM::NW, TILE = FM::TILE, COLS = FM::COLS;
  constexpr bool SHARE = FM::SHARE, F32 = FM::F32;
  __shared__ __attribute__((aligned(16))) float lds[FM::LDS > 2 * STATS ? FM::LDS : 2 * STATS];
  __shared__ int last;
  const KxPagedSpec &s = a.s;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lc = lane & 15, lq = lane >> 4;
  const int g = s.heads / s.kv_heads, head = blockIdx.x % s.kv_heads, rest = blockIdx.x / s.kv_heads, split = rest % a.splits, task = rest / a.splits;
  const Task t = find_task(a, task, [&](const Rows &r) { return (r.n * g + COLS - 1) / COLS; });
  if (!t.r.n) return;
  const int R = t.r.n * g, pos = t.r.pos;
  auto low = [&](int hi) { return s.size ? max(hi - s.size + 1, 0) : 0; };
  // the workgroup's units and its part of them
  const int w0 = t.index * COLS, hi_all = pos + (min(w0 + COLS, R) - 1) / g, first = low(pos + w0 / g) / UNIT, units = hi_all / UNIT - first + 1;
  const int chunk = max(a.chunk, (units + a.splits - 1) / a.splits), used = (units + chunk - 1) / chunk;
  if (split >= used) return;
  // the wave's columns
  const int c0 = w0 + (SHARE ? 0 : wave * TILE);
  const bool idle = c0 >= R;
  const int hi_min = pos + min(c0, R - 1) / g, hi_max = pos + min(c0 + TILE - 1, R - 1) / g;
  int hi[NQ], lo[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    hi[n] = pos + min(c0 + n * 16 + lc, R - 1) / g;
    lo[n] = low(hi[n]);
  }

  // queries: turned by their positions into LDS, 16 columns at a time, and from there to the lanes in the order of the keys' loads
  h8 q[NQ][DP / 32], ql[F32 ? NQ : 1][F32 ? DP / 32 : 1];
  float qf[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    float *const rows = lds + (SHARE ? 0 : wave * 16 * FM::QLD);
    for (int i = SHARE ? threadIdx.x : lane; i < 16 * (DP / 2); i += SHARE ? FM::THREADS : 64) {
      const int c = min(c0 + n * 16 + i / (DP / 2), R - 1), p = i % (DP / 2), at = c / g;
      const int2 d = pair_of(p, s.rot, s.pairs);
      const float *const x = a.proj + (size_t)(t.r.first + at) * a.proj_ld + a.q_off + (size_t)(head * g + c - at * g) * s.dim;
      float u = d.x < s.dim ? x[d.x] : 0.0f, v = d.y < s.dim ? x[d.y] : 0.0f;
      if (p < s.rot / 2) {
        float quarters, cs, sn;
        int whole;
        quarters_of(a.turn[p], pos + at, quarters, whole);
        turned(quarters, whole, cs, sn);
        const float y = u * cs - v * sn;
        v = u * sn + v * cs;
        u = y;
      }
      rows[i / (DP / 2) * FM::QLD + d.x] = u;
      rows[i / (DP / 2) * FM::QLD + d.y] = v;
    }
    __syncthreads();
    float most = 0.0f;
    const float *const mine = rows + lc * FM::QLD + lq * 16;
#pragma unroll
    for (int j = 0; j < DP / 64; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float x = __builtin_fabsf(mine[j * 64 + e]);
        most = fmaxf(most, x < __builtin_inff() ? x : 0.0f);
      }
    most = quarters_max(most);
    const int e = max(min((int)(kx_f32_bits(most) >> 23) - 126, 120), -100);
    const float down = kx_bits_f32(scale_bits(-e));
    qf[n] = kx_bits_f32(scale_bits(e)) * s.scale * 1.44269504088896341f;
#pragma unroll
    for (int j = 0; j < DP / 64; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float x = mine[j * 64 + e] * down;
        const _Float16 h = (_Float16)x;
        q[n][2 * j + (e >> 3)][e & 7] = h;
        if constexpr (F32) ql[n][2 * j + (e >> 3)][e & 7] = (_Float16)(x - (float)h);
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

  const int u_to = min(first + min((split + 1) * chunk, units), hi_max / UNIT + 1);
  const int u_from = max(first + split * chunk, low(hi_min) / UNIT) + (SHARE ? wave : 0);
  constexpr int STEP = SHARE ? NW : 1;
  const int *const table = a.table + (size_t)t.seq * a.table_ld;
  const int lo_tile = low(hi_min), lo_most = low(hi_max);
  uint4 kr[4][DP / 64];
  auto page_at = [&](int u) { return __builtin_amdgcn_readfirstlane(table[min(u, u_to - 1) * UNIT / s.page]); };
  auto head_of = [&](int id) { return (size_t)(page_ok(id, a.pages) ? id : 0) * s.kv_heads + head; };
  auto load_k = [&](int u, int id) {
    const uint8_t *const k = a.k + (head_of(id) * s.page + u * UNIT % s.page) * DP + lc * DP + lq * 16;
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int j = 0; j < DP / 64; ++j) kr[tt][j] = *(const uint4 *)(k + tt * 16 * DP + j * 64);
  };
  int id = 0, next = 0;
  if (u_from < u_to && !idle) {
    id = page_at(u_from);
    next = page_at(u_from + STEP);
    load_k(u_from, id);
  }
  for (int u = u_from; u < u_to && !idle; u += STEP) {
    const bool there = page_ok(id, a.pages);
    const size_t at = head_of(id);
    const int in = u * UNIT % s.page, base = u * UNIT;
    uint4 vr[VP / 16];
    {
      const uint8_t *const v = a.v + (at * s.page + in) * VP + lc * UNIT + lq * 16;
#pragma unroll
      for (int i = 0; i < VP / 16; ++i) vr[i] = *(const uint4 *)(v + i * 16 * UNIT);
    }
    const bool whole = there && base + UNIT - 1 <= hi_min && base >= lo_most;
    float kc[4], ve[4], vi[4];
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
      const size_t sc = at * (s.page / s.block) + (in + tt * 16) / s.block;
      uint32_t ks = kx_f32_bits(a.ks[sc]), vs = kx_f32_bits(a.vs[sc]);
      // blocks that no column sees may hold anything
      if (!whole && (!there || base + tt * 16 > hi_max || base + tt * 16 + 15 < lo_tile)) ks = vs = kx_f32_bits(1.0f);
      kc[tt] = kx_bits_f32(ks);
      ve[tt] = (float)scale_exponent(vs);
      vi[tt] = kx_bits_f32(scale_bits(-scale_exponent(vs)));
    }
    f4 x[NQ][4];
#pragma unroll
    for (int tt = 0; tt < 4; ++tt) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) x[n][tt] = f4{0, 0, 0, 0};
#pragma unroll
      for (int j = 0; j < DP / 64; ++j) {
        const h8 k0 = unpacked(kr[tt][j].x, kr[tt][j].y), k1 = unpacked(kr[tt][j].z, kr[tt][j].w);
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
    id = next;
    if (u + STEP < u_to) load_k(u + STEP, id);
    next = page_at(u + 2 * STEP);
    bool nan = false;
    if (!whole) {
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
    h8 ph[NQ][2], pl[F32 ? NQ : 1][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float most = NONE;
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
        const float f = qf[n] * kc[tt];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float y = __builtin_fmaf(x[n][tt][i], f, ve[tt]);
          if (!whole) {
            const int j = base + tt * 16 + lq * 4 + i;
            if (!there || j > hi[n] || j < lo[n]) y = -__builtin_inff();
          }
          x[n][tt][i] = y;
          most = fmaxf(most, y);
        }
      }
      most = fmaxf(m[n], quarters_max(most));
      if (__builtin_amdgcn_ballot_w64(most > m[n])) {
        const float f = exp2_(m[n] - most);
        m[n] = most;
        l[n] *= f;
#pragma unroll
        for (int v = 0; v < VP / 16; ++v) o[n][v] *= f;
      }
#pragma unroll
      for (int tt = 0; tt < 4; ++tt) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = exp2_(x[n][tt][i] - m[n]);
          sum += p;
          const _Float16 h = (_Float16)p;
          ph[n][tt >> 1][(tt & 1) * 4 + i] = h;
          if constexpr (F32) pl[n][tt >> 1][(tt & 1) * 4 + i] = (_Float16)(p - (float)h);
        }
        l[n] = __builtin_fmaf(sum, vi[tt], l[n]);
      }
    }
#pragma unroll
    for (int i = 0; i < VP / 16; ++i) {
      const h8 v0 = unpacked(vr[i].x, vr[i].y), v1 = unpacked(vr[i].z, vr[i].w);
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        o[n][i] = mfma(v0, ph[n][0], o[n][i]);
        o[n][i] = mfma(v1, ph[n][1], o[n][i]);
        if constexpr (F32) {
          o[n][i] = mfma(v0, pl[n][0], o[n][i]);
          o[n][i] = mfma(v1, pl[n][1], o[n][i]);
        }
      }
    }
    if (__builtin_amdgcn_ballot_w64(nan)) {  // NaN among the values: the columns that see it have it
      const uint8_t *const v = a.v + (at * s.page + in) * VP;
#pragma unroll
      for (int i = 0; i < VP / 16; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint8_t *const row = v + (i * 16 + lq * 4 + e) * UNIT;
#pragma unroll 1
          for (int p = 0; p < UNIT; ++p)
            if ((row[p] & 0x7f) == 0x7f) {
              const int j = base + token_of(p);
#pragma unroll
              for (int n = 0; n < NQ; ++n)
                if (j <= hi[n] && j >= lo[n]) o[n][i][e] = __builtin_nanf("");
            }
        }
    }
  }
#pragma unroll
  for (int n = 0; n < NQ; ++n) l[n] = quarters_sum(l[n]);

  // results: four neighbouring dimensions of a column at a time
  float *const part = a.part + (size_t)(task * s.kv_heads + head) * a.splits * FM::PART;
  auto give = [&](int c, int d, f4 y) {  // column c of the sequence, dimensions d .. d + 3
    const int at = c / g;
    const size_t to = (size_t)(t.r.first + at) * a.out_ld + (size_t)(head * g + c - at * g) * s.vdim + d;
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
            sum = __builtin_fmaf(st[w].y, f, sum);
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
  const int cols = min(COLS, R - w0);
  float2 *const st = (float2 *)lds;  // [used][COLS]
  for (int i = threadIdx.x; i < used * COLS; i += FM::THREADS)
    if (i % COLS < cols) {
      const uint64_t w = kx_arrive_load((const uint64_t *)(part + (size_t)(i / COLS) * FM::PART + (size_t)COLS * VP) + i % COLS);
      st[i] = make_float2(kx_bits_f32((uint32_t)w), kx_bits_f32((uint32_t)(w >> 32)));
    }
  __syncthreads();
  for (int c = threadIdx.x; c < cols; c += FM::THREADS) {
    float most = NONE, sum = 0.0f;
    for (int p = 0; p < used; ++p) most = fmaxf(most, st[p * COLS + c].x);
    for (int p = 0; p < used; ++p) sum = __builtin_fmaf(st[p * COLS + c].y, exp2_(st[p * COLS + c].x - most), sum);
    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
    for (int p = 0; p < used; ++p) st[p * COLS + c].x = exp2_(st[p * COLS + c].x - most) * f;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < cols * (VP / 4); i += FM::THREADS) {
    const int c = i / (VP / 4), d = i % (VP / 4) * 4;
    const uint64_t *from = (const uint64_t *)(part + (size_t)c * VP + d);
    f4 y = {0, 0, 0, 0};
#pragma unroll 4
    for (int p = 0; p < used; ++p) {
      const uint64_t x0 = kx_arrive_load(from + p * (FM::PART / 2)), x1 = kx_arrive_load(from + p * (FM::PART / 2) + 1);
      const float f = st[p * COLS + c].x;
      y[0] = __builtin_fmaf(kx_bits_f32((uint32_t)x0), f, y[0]);
      y[1] = __builtin_fmaf(kx_bits_f32((uint32_t)(x0 >> 32)), f, y[1]);
      y[2] = __builtin_fmaf(kx_bits_f32((uint32_t)x1), f, y[2]);
      y[3] = __builtin_fmaf(kx_bits_f32((uint32_t)(x1 >> 32)), f, y[3]);
    }
    give(w0 + c, d, y);
  }
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
  const long want = ((long)cus * FM::WAVES + busy - 1) / busy;
  a.splits = (int)std::max<long>(1, std::min(room, want));
  a.chunk = (units + a.splits - 1) / a.splits;
  // a sequence longer than `longest` has longer parts
  attend_k<FM><<<dim3((unsigned)(tasks * a.splits * kv)), FM::THREADS, 0, st>>>(a);
  KX_LAUNCH_CHECK();
  return KX_OK;
}

template <int DP, int VP, bool F32>
int launch_columns(const KxPagedArgs &a, hipStream_t st) {
  const int g = a.s.heads / a.s.kv_heads;
  const long columns = (long)a.tokens * g / std::min(a.batch, a.tokens);  // of a sequence, on average
  if (columns <= 16) return launch<Form<DP, VP, 1, true, F32>>(a, g, st);
  if (columns <= 64) return launch<Form<DP, VP, 2, true, F32>>(a, g, st);
  return launch<Form<DP, VP, 2, false, F32>>(a, g, st);
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
int kx_paged_attend_launch(bool f32, const KxPagedArgs &a, hipStream_t st) { return f32 ? launch_widths<true>(a, st) : launch_widths<false>(a, st); }

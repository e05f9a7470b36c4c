// kx_paged_cache.hip -- keys and values into the pages of an 8-bit cache and out of them again (kx_paged.h).  No counterpart in the reference,
// which stores 32-bit keys and values tile by tile on a disk (KvCache, src/kimi_exec.cu:192-238).
//
// append: a workgroup has the new tokens that lie in one group of 64 of a sequence, for one head of keys and values, and each of its four waves 16 tokens in
//   a row.  Every element is read once, turned by its position in 64 bits -- two sines and cosines a lane, the others by addition of angles -- and kept as a
//   float that any rounding to 4 bits of fraction takes where it takes the exact number.  The largest magnitude of each block goes through LDS; with the
//   scales known, codes are made in registers and put together in LDS: whole rows of keys, and pieces of 16 bytes of the values, with the older ones of
//   those 16 where there are any.
// read: the same groups, codes times scales as bf16, which holds them exactly; values are turned four tokens by eight dimensions a lane.
// What bounds them: 6 prompts of up to 2048 tokens, 8 heads of 128 + 128, appended in 23 us -- 71 MB read, 18 written, 17 us for a copy of as many, with vector
// instructions in 46 % of a SIMD's cycles -- and read back in 12 us, 18 MB read and 36 written, 10.5 for a copy.  64 sequences of one row 7 and 6 us, one row 5.5 and
// 3: a chain of dependent loads.
#include <algorithm>
#include <cmath>
#include <memory>
#include <type_traits>
#include <vector>
#include "kx_common.h"
#include "kx_math.h"
#include "kx_paged.h"
#include "kx_wave.h"

namespace {

using namespace kxpage;

constexpr int THREADS = 256, FEW = 4;  // FEW: most tokens whose values are stored byte by byte

// Two numbers as floats that round to 4 bits of fraction, and lie next to a power of two times 1.75, as they do themselves: a float on a border between two
// codes has 19 zeros at its end, and only then its last bit is set where the number is not the float.
__device__ __forceinline__ float off_border(float f, double x) {
  const uint32_t u = kx_f32_bits(f);
  if (u & 0x7ffffu || (double)f == x || f != f) return f;
  return kx_bits_f32(__builtin_fabs((double)f) > __builtin_fabs(x) ? u - 1 : u | 1);
}
__device__ __forceinline__ void rounded(double x, double y, float &a, float &b) {
  a = (float)x;
  b = (float)y;
  if (__builtin_amdgcn_ballot_w64((kx_f32_bits(a) & 0x7ffffu) == 0 || (kx_f32_bits(b) & 0x7ffffu) == 0)) {
    a = off_border(a, x);
    b = off_border(b, y);
  }
}
__device__ __forceinline__ float finite(float x) { return __builtin_fabsf(x) < __builtin_inff() ? x : 0.0f; }  // largest magnitudes leave out what is not
// codes of two numbers of at most 448, in the low 16 bits; NaN of what is not finite
__device__ __forceinline__ uint32_t codes(float a, float b) { return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false) & 0xffffu; }
// the four codes of a word divided by 2^down
__device__ __forceinline__ uint32_t lowered(uint32_t w, int down) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const float f = down > 100 ? 0.0f : kx_bits_f32(scale_bits(-down));
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a[0] * f, a[1] * f, 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(b[0] * f, b[1] * f, r, true);
  return (uint32_t)r;
}

struct Unit {
  int from, to, row;  // new tokens of the group [from, to), row of the first; none: to is 0
  size_t head;        // page * kv_heads + head
  int in_page;        // position of the group in its page
  int pos, id;        // of the group; its page, which need not exist
};
__device__ __forceinline__ Unit unit_of(const KxPagedArgs &a) {
  const Task t = find_task(a, blockIdx.x, [](const Rows &r) { return units_of(r.pos, r.n); });
  Unit u;
  u.pos = (t.r.pos / UNIT + t.index) * UNIT;
  u.from = max(t.r.pos - u.pos, 0);
  u.to = t.r.n > 0 ? min(t.r.pos + t.r.n - u.pos, UNIT) : 0;
  if (!u.to) return u;
  u.row = t.r.first + u.pos + u.from - t.r.pos;
  const int page = quotient(u.pos / UNIT, a.per_page);
  u.id = a.table[(size_t)t.seq * a.table_ld + page];
  u.in_page = u.pos - page * a.s.page;
  return u;
}
__device__ __forceinline__ bool placed(const KxPagedArgs &a, Unit &u) {  // whether the page exists
  u.head = (size_t)u.id * a.s.kv_heads + blockIdx.y;
  if (page_ok(u.id, a.pages)) return true;
  if (threadIdx.x == 0) atomicOr(a.fault, BAD_PAGE);
  return false;
}
// bytes of a word of tokens t .. t + 3 that lie in [from, to)
__device__ __forceinline__ uint32_t bytes_within(int t, int from, int to) {
  const int n = max(min(to - t, 4), 0), k = max(min(from - t, 4), 0);
  return (n == 4 ? ~0u : (1u << 8 * n) - 1u) & (k == 4 ? 0u : ~0u << 8 * k);
}

template <int DP, int VP>
__global__ void __launch_bounds__(THREADS) append_k(KxPagedArgs a) {
  constexpr int PK = (DP + 127) / 128, PV = VP / 64, NW = THREADS / 64, MINE = UNIT / NW;  // of a lane: pairs of a key, elements of a value; tokens of a wave
  constexpr int LD = UNIT + 16;                                                            // bytes of a row of values in LDS
  __shared__ __attribute__((aligned(16))) uint8_t lk[UNIT * DP], lv[VP * LD];
  __shared__ float most[2][NW];
  const KxPagedSpec &s = a.s;
  Unit u = unit_of(a);
  if (!u.to) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), from = u.from, to = u.to, t0 = MINE * wave;
  const int mine_from = max(from - t0, 0), mine_to = min(to - t0, MINE);  // the wave's new tokens
  float xk[MINE][PK][2], xv[MINE][PV];
  double turn[PK];
#pragma unroll
  for (int p = 0; p < PK; ++p) turn[p] = lane + 64 * p < s.rot / 2 ? a.turn[lane + 64 * p] : 0.0;
#pragma unroll
  for (int i = 0; i < MINE; ++i) {
#pragma unroll
    for (int p = 0; p < PK; ++p) xk[i][p][0] = xk[i][p][1] = 0.0f;
#pragma unroll
    for (int p = 0; p < PV; ++p) xv[i][p] = 0.0f;
    if (i < mine_from || i >= mine_to) continue;
    const float *const row = a.proj + (size_t)(u.row + t0 + i - from) * a.proj_ld;
    const float *const rk = row + a.k_off + (size_t)blockIdx.y * s.dim, *const rv = row + a.v_off + (size_t)blockIdx.y * s.vdim;
#pragma unroll
    for (int p = 0; p < PK; ++p) {
      const int2 d = pair_of(lane + 64 * p, s.rot, s.pairs);
      if (d.x < s.dim) xk[i][p][0] = rk[d.x];
      if (d.y < s.dim) xk[i][p][1] = rk[d.y];
    }
#pragma unroll
    for (int p = 0; p < PV; ++p)
      if (lane + 64 * p < s.vdim) xv[i][p] = rv[lane + 64 * p];
  }
  if (!placed(a, u)) return;
  uint8_t *const gk = a.k + (u.head * s.page + u.in_page) * DP, *const gv = a.v + (u.head * s.page + u.in_page) * VP;
  const size_t sc = u.head * (s.page >> a.block_bits) + (u.in_page >> a.block_bits);  // scale of the group's first block
  const int b0 = from >> a.block_bits;
  const bool kept = (from & (s.block - 1)) != 0;  // the first block has older tokens
  const int old_k = kept ? scale_exponent(kx_f32_bits(a.ks[sc + b0])) : 0, old_v = kept ? scale_exponent(kx_f32_bits(a.vs[sc + b0])) : 0;

  float mk = 0.0f, mv = 0.0f;
  if (mine_from < mine_to) {
#pragma unroll
    for (int p = 0; p < PK; ++p) {
      auto eval = [&](int n, double &c, double &s) {
        const double at = turn[p] * (double)n;
        turned(at - __builtin_rint(at), c, s);
      };
      double c, n, c1 = 1.0, n1 = 0.0;
      eval(u.pos + t0 + mine_from, c, n);
      if (mine_to - mine_from > 1) eval(1, c1, n1);
      const bool turns = lane + 64 * p < s.rot / 2;
#pragma unroll
      for (int i = 0; i < MINE; ++i) {
        if (i < mine_from || i >= mine_to) continue;
        float &x = xk[i][p][0], &y = xk[i][p][1];
        if (turns) rounded(__builtin_fma(-(double)y, n, x * c), __builtin_fma((double)y, c, x * n), x, y);
        mk = fmaxf(mk, fmaxf(__builtin_fabsf(x), __builtin_fabsf(y)));
        const double d = __builtin_fma(-n, n1, c * c1);
        n = __builtin_fma(n, c1, c * n1);
        c = d;
      }
    }
#pragma unroll
    for (int i = 0; i < MINE; ++i)
#pragma unroll
      for (int p = 0; p < PV; ++p) mv = fmaxf(mv, __builtin_fabsf(xv[i][p]));
    mk = kxw::wave_max_f32(mk);
    mv = kxw::wave_max_f32(mv);
    if (!(fmaxf(mk, mv) < __builtin_inff())) {
      mk = mv = 0.0f;
#pragma unroll
      for (int i = 0; i < MINE; ++i) {
#pragma unroll
        for (int p = 0; p < PK; ++p) mk = fmaxf(mk, fmaxf(__builtin_fabsf(finite(xk[i][p][0])), __builtin_fabsf(finite(xk[i][p][1]))));
#pragma unroll
        for (int p = 0; p < PV; ++p) mv = fmaxf(mv, __builtin_fabsf(finite(xv[i][p])));
      }
      mk = kxw::wave_max_f32(mk);
      mv = kxw::wave_max_f32(mv);
    }
  }
  if (lane == 0) {
    most[0][wave] = mk;
    most[1][wave] = mv;
  }
  __syncthreads();
  // exponents of block b, before and with the new tokens
  const int bits = a.block_bits, per = s.block / MINE;
  auto exponent = [&](int which, int b, int old) {
    float m = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) m = w / per == b ? fmaxf(m, most[which][w]) : m;
    const int e = exponent_of(kx_f32_bits(m));
    return kept && b == b0 ? max(e, old) : e;
  };
  const int b = t0 >> bits, ek = exponent(0, b, old_k), ev = exponent(1, b, old_v);
  const int grown_k = kept ? exponent(0, b0, old_k) - old_k : 0, grown_v = kept ? exponent(1, b0, old_v) - old_v : 0;
  if (lane == 0 && (t0 & (s.block - 1)) == 0 && b >= b0 && b <= (to - 1) >> bits) {
    a.ks[sc + b] = kx_bits_f32(scale_bits(ek));
    a.vs[sc + b] = kx_bits_f32(scale_bits(ev));
  }

  if (grown_k) {
    uint32_t *const w = (uint32_t *)(gk + b0 * s.block * DP);
    for (int i = tid; i < (from - b0 * s.block) * (DP / 4); i += THREADS) w[i] = lowered(w[i], grown_k);
  }
  const float rk = kx_bits_f32(scale_bits(-ek)), rv = kx_bits_f32(scale_bits(-ev));
#pragma unroll
  for (int i = 0; i < MINE; ++i) {
    if (i < mine_from || i >= mine_to) continue;
    uint8_t *const row = lk + (t0 + i) * DP;
#pragma unroll
    for (int p = 0; p < PK; ++p)
      if (lane + 64 * p < DP / 2) {
        const int2 d = pair_of(lane + 64 * p, s.rot, s.pairs);
        const uint32_t c = codes(xk[i][p][0] * rk, xk[i][p][1] * rk);
        row[d.x] = (uint8_t)c;
        row[d.y] = (uint8_t)(c >> 8);
      }
  }
  const bool few = to - from <= FEW && !grown_v;
#pragma unroll
  for (int p = 0; p < PV; ++p)
#pragma unroll
    for (int i = 0; i < MINE; i += 4) {
      const uint32_t w = codes(xv[i][p] * rv, xv[i + 1][p] * rv) | codes(xv[i + 2][p] * rv, xv[i + 3][p] * rv) << 16;
      const int d = lane + 64 * p, at = place_of(t0 + i);
      if (!few) {
        *(uint32_t *)(lv + d * LD + at) = w;
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (i + r >= mine_from && i + r < mine_to) gv[d * UNIT + at + r] = (uint8_t)(w >> 8 * r);
      }
    }
  __syncthreads();
  for (int i = from * (DP / 16) + tid; i < to * (DP / 16); i += THREADS) ((uint4 *)gk)[i] = ((const uint4 *)lk)[i];
  if (few) return;
  for (int i = tid; i < VP * 4; i += THREADS) {  // 16 bytes: tokens 16 j + 4 q + 0 .. 3
    const int q = i & 3;
    uint4 *const at = (uint4 *)gv + i;
    uint4 w = *(const uint4 *)(lv + (i >> 2) * LD + q * 16);
    if (from > 0 && (from > 4 * q || to < 4 * q + 52)) {
      if (!grown_v && (from > 4 * q + 51 || to <= 4 * q)) continue;
      const uint4 old = *at;
      auto mixed = [&](uint32_t n, uint32_t o, int j) {
        const uint32_t mask = bytes_within(16 * j + 4 * q, from, to);
        return (n & mask) | ((grown_v && 16 * j >> bits == b0 ? lowered(o, grown_v) : o) & ~mask);
      };
      w = make_uint4(mixed(w.x, old.x, 0), mixed(w.y, old.y, 1), mixed(w.z, old.z, 2), mixed(w.w, old.w, 3));
    }
    *at = w;
  }
}

// eight codes times a power of two as bf16, which holds them exactly, at element d of a row of n; wide: rows and d are whole pieces of 16 bytes
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
template <bool HIGH>
__device__ __forceinline__ uint32_t values(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, scale, HIGH));
}
__device__ __forceinline__ void put(uint16_t *row, int d, int n, bool wide, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  if (wide) {
    if (d < n) *(uint4 *)(row + d) = make_uint4(x, y, z, w);
    return;
  }
  const uint32_t v[4] = {x, y, z, w};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (d + e < n) row[d + e] = (uint16_t)(v[e >> 1] >> 16 * (e & 1));
}

template <int DP, int VP>
__global__ void __launch_bounds__(THREADS) read_k(KxPagedArgs a) {
  const KxPagedSpec &s = a.s;
  Unit u = unit_of(a);
  if (!u.to || !placed(a, u)) return;
  const int tid = threadIdx.x;
  const uint8_t *const gk = a.k + (u.head * s.page + u.in_page) * DP, *const gv = a.v + (u.head * s.page + u.in_page) * VP;
  const size_t sc = u.head * (s.page >> a.block_bits) + (u.in_page >> a.block_bits);
  uint16_t *const ok = (uint16_t *)a.out + (size_t)u.row * a.out_ld + (size_t)blockIdx.y * s.dim;
  uint16_t *const ov = (uint16_t *)a.out_v + (size_t)u.row * a.out_v_ld + (size_t)blockIdx.y * s.vdim;
  for (int i = tid; i < VP / 8 * 16; i += THREADS) {  // eight words of 8 rows by eight of them a wave: whole lines of results
    const int word = (i & 7) | (i >> 6 & 1) << 3, d = ((i >> 3 & 7) | i >> 7 << 3) * 8, t = token_of(word * 4);
    if (t + 3 < u.from || t >= u.to) continue;
    uint32_t w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = *(const uint32_t *)(gv + (d + e) * UNIT + word * 4);
    const float f = a.vs[sc + (t >> a.block_bits)];
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // tokens t + 2 h and t + 2 h + 1
      uint32_t c[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) c[e] = __builtin_amdgcn_perm(w[2 * e + 1], w[2 * e], h ? 0x07030602u : 0x05010400u);
      const int at = t + 2 * h;
      if (at >= u.from && at < u.to)
        put(ov + (size_t)(at - u.from) * a.out_v_ld, d, s.vdim, a.wide_v, values<false>(c[0], f), values<false>(c[1], f), values<false>(c[2], f), values<false>(c[3], f));
      if (at + 1 >= u.from && at + 1 < u.to)
        put(ov + (size_t)(at + 1 - u.from) * a.out_v_ld, d, s.vdim, a.wide_v, values<true>(c[0], f), values<true>(c[1], f), values<true>(c[2], f), values<true>(c[3], f));
    }
  }
  for (int i = tid; i < (u.to - u.from) * (DP / 8); i += THREADS) {
    const int t = u.from + i / (DP / 8), d = i % (DP / 8) * 8;
    const uint2 c = *(const uint2 *)(gk + t * DP + d);
    const float f = a.ks[sc + (t >> a.block_bits)];
    put(ok + (size_t)(t - u.from) * a.out_ld, d, s.dim, a.wide_k, values<false>(c.x, f), values<true>(c.x, f), values<false>(c.y, f), values<true>(c.y, f));
  }
}

template <class F>
int by_widths(const KxPagedSpec &s, F f) {
  if (s.dp == 64) f(std::integral_constant<int, 64>(), std::integral_constant<int, 64>());
  else if (s.dp == 128) f(std::integral_constant<int, 128>(), std::integral_constant<int, 128>());
  else if (s.dp == 192) f(std::integral_constant<int, 192>(), std::integral_constant<int, 128>());
  else f(std::integral_constant<int, 256>(), std::integral_constant<int, 256>());
  KX_LAUNCH_CHECK();
  return KX_OK;
}
// groups of 64 that so many rows of so many sequences can lie in: n of a sequence in at most n, and in at most 2 + (n - 2) / 64
unsigned most_units(const KxPagedArgs &a) { return (unsigned)std::min(a.tokens, 2 * std::min(a.batch, a.tokens) + a.tokens / UNIT); }

}  // namespace

int kx_paged_append_launch(const KxPagedArgs &a, hipStream_t st) {
  const dim3 grid(most_units(a), a.s.kv_heads);
  return by_widths(a.s, [&](auto k, auto v) { append_k<k(), v()><<<grid, THREADS, 0, st>>>(a); });
}
int kx_paged_read_launch(const KxPagedArgs &a, hipStream_t st) {
  const dim3 grid(most_units(a), a.s.kv_heads);
  return by_widths(a.s, [&](auto k, auto v) { read_k<k(), v()><<<grid, THREADS, 0, st>>>(a); });
}

// ---- the operators of the C ABI ---------------------------------------------------------------------------------------------------------
struct kx_paged {
  KxPagedArgs a;
  bool f32 = false;
  int max_batch = 0, max_tokens = 0, device = 0;
  char *mem = nullptr;
};

namespace {

int common(const char *who, kx_paged *p, const kx_paged_cache *c, const kx_paged_rows *r, KxPagedArgs *out) {
  KX_REQUIRE(p && c && r, "%s: null argument", who);
  KX_REQUIRE(c->d_k && c->d_v && c->d_k_scale && c->d_v_scale && c->d_table && r->d_start && r->d_pos, "%s: null pointer in the cache or the rows", who);
  auto aligned = [](const void *q, size_t to) { return (uintptr_t)q % to == 0; };
  KX_REQUIRE(aligned(c->d_k, 16) && aligned(c->d_v, 16) && aligned(c->d_k_scale, 4) && aligned(c->d_v_scale, 4) && aligned(c->d_table, 4) && aligned(r->d_start, 4) && aligned(r->d_pos, 4),
             "%s: keys and values begin at multiples of 16 bytes, the other tables at multiples of 4", who);
  KX_REQUIRE(c->pages > 0 && c->table_ld > 0 && c->table_ld <= (0x7fffffff - UNIT) / p->a.s.page, "%s: pages=%d table_ld=%d of %d positions", who, c->pages, c->table_ld, p->a.s.page);
  KX_REQUIRE(r->batch > 0 && r->batch <= p->max_batch && r->tokens >= 0 && r->longest > 0, "%s: batch=%d tokens=%d longest=%d", who, r->batch, r->tokens, r->longest);
  int dev = -1;
  KX_HIP(hipGetDevice(&dev));
  KX_REQUIRE(dev == p->device, "%s: made on device %d, called on device %d", who, p->device, dev);
  *out = p->a;
  out->k = (uint8_t *)c->d_k; out->v = (uint8_t *)c->d_v; out->ks = c->d_k_scale; out->vs = c->d_v_scale;
  out->table = c->d_table; out->pages = c->pages; out->table_ld = c->table_ld;
  out->start = r->d_start; out->pos = r->d_pos; out->batch = r->batch; out->tokens = r->tokens;
  out->longest = std::min(r->longest, c->table_ld * p->a.s.page);
  return KX_OK;
}

}  // namespace

extern "C" int kx_paged_create(const kx_paged_config *c, const double *h_freq, int f32, int32_t max_batch, int32_t max_tokens, kx_paged **out) {
  KX_REQUIRE(c && out, "kx_paged_create: null argument");
  *out = nullptr;
  KX_REQUIRE(c->heads > 0 && c->kv_heads > 0 && c->kv_heads <= 65535 && c->heads % c->kv_heads == 0 && c->dim > 0 && c->vdim > 0 && kxpage::widths_of(c->dim, c->vdim).k,
             "kx_paged_create: heads=%d kv_heads=%d dim=%d vdim=%d", c->heads, c->kv_heads, c->dim, c->vdim);
  KX_REQUIRE(c->page > 0 && c->page % UNIT == 0 && c->page <= 1 << 20 && (c->block == 16 || c->block == 32 || c->block == 64), "kx_paged_create: pages of %d, blocks of %d", c->page, c->block);
  KX_REQUIRE(c->rot >= 0 && c->rot <= c->dim && c->rot % 2 == 0 && (c->pairs == 0 || c->pairs == 1) && c->size >= 0, "kx_paged_create: rot=%d pairs=%d size=%d", c->rot, c->pairs, c->size);
  KX_REQUIRE(std::isfinite(c->scale) && (!c->rot || h_freq || (std::isfinite(c->base) && c->base > 0)), "kx_paged_create: scale=%g base=%g", c->scale, c->base);
  KX_REQUIRE(max_batch > 0 && max_tokens > 0 && (int64_t)max_tokens * c->heads <= 1 << 28 && (int64_t)max_batch * c->heads <= 1 << 28, "kx_paged_create: max_batch=%d max_tokens=%d",
             max_batch, max_tokens);
  return kx_guard("kx_paged_create", [&]() -> int {
    std::vector<double> turn((size_t)std::max(c->rot / 2, 1));
    for (int d = 0; d < c->rot / 2; ++d) {
      const double f = h_freq ? h_freq[d] : std::pow(c->base, -2.0 * d / c->rot);
      KX_REQUIRE(std::isfinite(f), "kx_paged_create: frequency %d is not finite", d);
      turn[(size_t)d] = f / 6.283185307179586476925;
    }
    std::unique_ptr<kx_paged> p(new kx_paged());
    KxPagedSpec &s = p->a.s;
    s.heads = c->heads; s.kv_heads = c->kv_heads; s.dim = c->dim; s.vdim = c->vdim; s.page = c->page; s.block = c->block; s.rot = c->rot; s.pairs = c->pairs;
    s.size = c->size; s.scale = c->scale;
    const kxpage::Widths w = kxpage::widths_of(c->dim, c->vdim);
    s.dp = w.k; s.vp = w.v;
    p->a.by_g = divider(s.heads / s.kv_heads); p->a.by_kv = divider(s.kv_heads); p->a.per_page = divider(s.page / UNIT);
    p->a.block_bits = __builtin_ctz((unsigned)s.block);
    p->f32 = f32 != 0;
    p->max_batch = max_batch; p->max_tokens = max_tokens;
    p->a.arrivals = kx_paged_arrivals(s, max_batch, max_tokens);
    p->a.part_floats = kx_paged_part_floats(s, max_batch, max_tokens);
    const size_t turns = (turn.size() * 8 + 255) & ~(size_t)255, counters = ((size_t)p->a.arrivals * 4 + 4 + 255) & ~(size_t)255;
    KX_HIP(hipGetDevice(&p->device));
    if (hipMalloc((void **)&p->mem, turns + counters + p->a.part_floats * 4) != hipSuccess) {
      kx_set_error("kx_paged_create: no device memory for %zu bytes", turns + counters + p->a.part_floats * 4);
      return KX_ERR_HIP;
    }
    p->a.turn = (const double *)p->mem;
    p->a.fault = (int *)(p->mem + turns);
    p->a.arrived = p->a.fault + 1;
    p->a.part = (float *)(p->mem + turns + counters);
    hipError_t e = hipMemcpy(p->mem, turn.data(), turn.size() * 8, hipMemcpyHostToDevice);
    if (e == hipSuccess) e = hipMemset(p->a.fault, 0, counters);
    if (e == hipSuccess) e = hipStreamSynchronize(nullptr);  // calls may come on any stream
    if (e != hipSuccess) {
      (void)hipFree(p->mem);
      kx_set_error("kx_paged_create: %s", hipGetErrorString(e));
      return KX_ERR_HIP;
    }
    *out = p.release();
    return KX_OK;
  });
}
extern "C" int kx_paged_destroy(kx_paged *p) {
  if (!p) return KX_OK;
  if (p->mem) (void)hipFree(p->mem);
  delete p;
  return KX_OK;
}
extern "C" int kx_paged_append(kx_paged *p, const kx_paged_cache *cache, const kx_paged_rows *rows, const void *d_proj, int32_t proj_ld, int32_t k_off, int32_t v_off, void *stream) {
  KxPagedArgs a;
  KX_DO(common("kx_paged_append", p, cache, rows, &a));
  auto fits = [&](int off, int n) { return off >= 0 && off <= proj_ld - n; };
  KX_REQUIRE(d_proj && (uintptr_t)d_proj % 4 == 0 && fits(k_off, a.s.kv_heads * a.s.dim) && fits(v_off, a.s.kv_heads * a.s.vdim), "kx_paged_append: columns outside the rows");
  KX_REQUIRE(a.tokens <= p->max_tokens, "kx_paged_append: tokens=%d", a.tokens);
  if (!a.tokens) return KX_OK;
  a.proj = (const float *)d_proj; a.proj_ld = proj_ld; a.k_off = k_off; a.v_off = v_off;
  return kx_paged_append_launch(a, kx_stream(stream));
}
extern "C" int kx_paged_read(kx_paged *p, const kx_paged_cache *cache, const kx_paged_rows *rows, void *d_k, int32_t k_ld, void *d_v, int32_t v_ld, void *stream) {
  KxPagedArgs a;
  KX_DO(common("kx_paged_read", p, cache, rows, &a));
  KX_REQUIRE(d_k && d_v && (uintptr_t)d_k % 2 == 0 && (uintptr_t)d_v % 2 == 0 && k_ld >= a.s.kv_heads * a.s.dim && v_ld >= a.s.kv_heads * a.s.vdim, "kx_paged_read: k_ld=%d v_ld=%d", k_ld, v_ld);
  if (!a.tokens) return KX_OK;
  a.out = d_k; a.out_ld = k_ld; a.out_v = d_v; a.out_v_ld = v_ld;
  a.wide_k = (uintptr_t)d_k % 16 == 0 && k_ld % 8 == 0 && a.s.dim % 8 == 0;
  a.wide_v = (uintptr_t)d_v % 16 == 0 && v_ld % 8 == 0 && a.s.vdim % 8 == 0;
  return kx_paged_read_launch(a, kx_stream(stream));
}
extern "C" int kx_paged_attend(kx_paged *p, const kx_paged_cache *cache, const kx_paged_rows *rows, const void *d_proj, int32_t proj_ld, int32_t q_off, void *d_out, int32_t out_ld, void *stream) {
  KxPagedArgs a;
  KX_DO(common("kx_paged_attend", p, cache, rows, &a));
  KX_REQUIRE(d_proj && (uintptr_t)d_proj % 4 == 0 && q_off >= 0 && q_off <= proj_ld - a.s.heads * a.s.dim, "kx_paged_attend: columns outside the rows");
  KX_REQUIRE(d_out && (uintptr_t)d_out % (p->f32 ? 4 : 2) == 0 && out_ld >= a.s.heads * a.s.vdim, "kx_paged_attend: out_ld=%d", out_ld);
  KX_REQUIRE(a.tokens <= p->max_tokens, "kx_paged_attend: tokens=%d", a.tokens);
  if (!a.tokens) return KX_OK;
  a.proj = (const float *)d_proj; a.proj_ld = proj_ld; a.q_off = q_off;
  a.out = d_out; a.out_ld = out_ld;
  a.wide_v = (uintptr_t)d_out % (p->f32 ? 16 : 8) == 0 && out_ld % 4 == 0 && a.s.vdim % 4 == 0;
  return kx_paged_attend_launch(p->f32, a, kx_stream(stream));
}
extern "C" int kx_paged_faults(kx_paged *p, int32_t *h_bits, void *stream) {
  KX_REQUIRE(p && h_bits, "kx_paged_faults: null argument");
  int dev = -1;
  KX_HIP(hipGetDevice(&dev));
  KX_REQUIRE(dev == p->device, "kx_paged_faults: made on device %d, called on device %d", p->device, dev);
  KX_HIP(hipStreamSynchronize(kx_stream(stream)));
  KX_HIP(hipMemcpy(h_bits, p->a.fault, 4, hipMemcpyDeviceToHost));
  if (*h_bits) {
    KX_HIP(hipMemset(p->a.fault, 0, 4));
    KX_HIP(hipStreamSynchronize(nullptr));  // the next call may come on any stream
  }
  return KX_OK;
}

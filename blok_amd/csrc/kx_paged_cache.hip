// kx_paged_cache.hip -- keys and values into the pages of an 8-bit cache and out of them again (kx_paged.h).  No counterpart in the reference,
// which stores 32-bit keys and values tile by tile on a disk (KvCache, src/kimi_exec.cu:192-238).
//
// append: a workgroup has the new tokens that lie in one group of 64 of a sequence, for one head of keys and values.  Every element is read once, turned by
//   its position in 64 bits and kept as a float whose last bit says whether anything was cut off; rounding that to 4 bits of fraction at any scale is
//   one rounding of the exact number.  The largest magnitude of each block goes through LDS; with the scales known, codes are made in registers.
//   A few tokens whose blocks keep their scales are stored byte by byte (a byte of a row of 64 for each value: 128 of them for a decoded token).
//   Otherwise the group is put together in LDS, with the tokens that it keeps, and written in whole pieces of 16 bytes.
// read: the same groups, codes times scales as bf16, which holds them exactly.
#include <algorithm>
#include <cmath>
#include <memory>
#include <type_traits>
#include <vector>
#include "kx_common.h"
#include "kx_math.h"
#include "kx_paged.h"

namespace {

using namespace kxpage;

constexpr int THREADS = 256, FEW = 4;  // FEW: most tokens that are stored byte by byte

// x with its last bits cut off, and the last that is left set where that changed anything
__device__ __forceinline__ float sticky(double x) {
  float f = (float)x;
  if ((double)f != x && f == f) {
    uint32_t u = kx_f32_bits(f);
    if (__builtin_fabs((double)f) > __builtin_fabs(x)) --u;
    f = kx_bits_f32(u | 1u);
  }
  return f;
}
__device__ __forceinline__ uint32_t magnitude(float x) {  // bits of |x|; 0 for what is not finite
  const uint32_t u = kx_f32_bits(x) & 0x7fffffffu;
  return u >= 0x7f800000u ? 0u : u;
}
// codes of two numbers at the scale whose reciprocal is given, in the low 16 bits
__device__ __forceinline__ uint32_t codes(float a, float b, float inverse) {
  auto scaled = [&](float x) { return (kx_f32_bits(x) & 0x7f800000u) == 0x7f800000u ? __builtin_nanf("") : x * inverse; };
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(scaled(a), scaled(b), 0, false) & 0xffffu;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, d));
  return v;
}
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
  int seq, from, to, row;  // new tokens of the group [from, to), rows of the first
  size_t head;             // (page * kv_heads + head)
  int in_page;             // position of the group in its page
  int pos;                 // of the group
  bool ok;
};
__device__ __forceinline__ Unit unit_of(const KxPagedArgs &a) {
  const Task t = find_task(a, blockIdx.x, [](const Rows &r) { return units_of(r.pos, r.n); });
  Unit u;
  u.ok = t.r.n > 0;
  if (!u.ok) return u;
  u.seq = t.seq;
  u.pos = (t.r.pos / UNIT + t.index) * UNIT;
  u.from = max(t.r.pos - u.pos, 0);
  u.to = min(t.r.pos + t.r.n - u.pos, UNIT);
  u.row = t.r.first + u.pos + u.from - t.r.pos;
  const int id = a.table[(size_t)t.seq * a.table_ld + u.pos / a.s.page];
  if (!page_ok(id, a.pages)) {
    if (threadIdx.x == 0) atomicOr(a.fault, BAD_PAGE);
    u.ok = false;
    return u;
  }
  u.head = (size_t)id * a.s.kv_heads + blockIdx.y;
  u.in_page = u.pos % a.s.page;
  return u;
}

template <int DP, int VP>
__global__ void __launch_bounds__(THREADS) append_k(KxPagedArgs a) {
  constexpr int PK = (DP + 127) / 128, PV = (VP + 127) / 128;  // pairs of a lane
  __shared__ __attribute__((aligned(16))) uint8_t lk[UNIT * DP], lv[VP * UNIT];
  __shared__ uint32_t most[4][8];
  const KxPagedSpec &s = a.s;
  const Unit u = unit_of(a);
  if (!u.ok) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, from = u.from, to = u.to;
  uint8_t *const gk = a.k + (u.head * s.page + u.in_page) * DP, *const gv = a.v + (u.head * s.page + u.in_page) * VP;
  const size_t sc = u.head * (s.page / s.block) + u.in_page / s.block;  // scale of the group's first block
  const int b0 = from / s.block;
  const bool kept = from % s.block != 0;  // the first block has older tokens
  const int old_k = kept ? scale_exponent(kx_f32_bits(a.ks[sc + b0])) : 0, old_v = kept ? scale_exponent(kx_f32_bits(a.vs[sc + b0])) : 0;

  // wave w has tokens w, w + 4, ... of the group; four of them are in a block of 16
  float xk[16][PK][2], xv[16][PV][2];
  double turn[PK];
#pragma unroll
  for (int p = 0; p < PK; ++p) turn[p] = lane + 64 * p < s.rot / 2 ? a.turn[lane + 64 * p] : 0.0;
  uint32_t mk[4] = {0, 0, 0, 0}, mv[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int t = wave + 4 * i;
    const bool mine = t >= from && t < to;
    const float *row = a.proj + (size_t)(u.row + (mine ? t - from : 0)) * a.proj_ld;
    const float *rk = row + a.k_off + (size_t)blockIdx.y * s.dim, *rv = row + a.v_off + (size_t)blockIdx.y * s.vdim;
#pragma unroll
    for (int p = 0; p < PK; ++p) {
      const int2 d = pair_of(lane + 64 * p, s.rot, s.pairs);
      xk[i][p][0] = mine && d.x < s.dim ? rk[d.x] : 0.0f;
      xk[i][p][1] = mine && d.y < s.dim ? rk[d.y] : 0.0f;
    }
#pragma unroll
    for (int p = 0; p < PV; ++p) {
      const int d = 2 * (lane + 64 * p);
      xv[i][p][0] = mine && d < s.vdim ? rv[d] : 0.0f;
      xv[i][p][1] = mine && d + 1 < s.vdim ? rv[d + 1] : 0.0f;
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int t = wave + 4 * i;
    if (t < from || t >= to) continue;
#pragma unroll
    for (int p = 0; p < PK; ++p) {
      if (lane + 64 * p < s.rot / 2) {
        double c, n;
        const double at = turn[p] * (double)(u.pos + t);
        turned(at - __builtin_rint(at), c, n);
        const double x = xk[i][p][0], y = xk[i][p][1];
        xk[i][p][0] = sticky(x * c - y * n);
        xk[i][p][1] = sticky(x * n + y * c);
      }
      mk[i >> 2] = max(mk[i >> 2], max(magnitude(xk[i][p][0]), magnitude(xk[i][p][1])));
    }
#pragma unroll
    for (int p = 0; p < PV; ++p) mv[i >> 2] = max(mv[i >> 2], max(magnitude(xv[i][p][0]), magnitude(xv[i][p][1])));
  }
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    mk[g] = wave_max(mk[g]);
    mv[g] = wave_max(mv[g]);
  }
  if (lane == 0) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      most[wave][g] = mk[g];
      most[wave][4 + g] = mv[g];
    }
  }
  __syncthreads();
  // exponents of the blocks that the group's four blocks of 16 lie in
  int ek[4], ev[4];
  const int per = s.block / 16;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    uint32_t k = 0, v = 0;
#pragma unroll
    for (int h = 0; h < 4; ++h)
      if (h / per == g / per) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          k = max(k, most[w][h]);
          v = max(v, most[w][4 + h]);
        }
      }
    ek[g] = exponent_of(k);
    ev[g] = exponent_of(v);
    if (kept && g / per == b0) {
      ek[g] = max(ek[g], old_k);
      ev[g] = max(ev[g], old_v);
    }
  }
  // the exponents of the first block that the group writes to
  const int g0 = b0 * per, ek0 = g0 == 0 ? ek[0] : g0 == 1 ? ek[1] : g0 == 2 ? ek[2] : ek[3], ev0 = g0 == 0 ? ev[0] : g0 == 1 ? ev[1] : g0 == 2 ? ev[2] : ev[3];
  const int grown_k = kept ? ek0 - old_k : 0, grown_v = kept ? ev0 - old_v : 0;
  if (tid < 4 && tid % per == 0 && tid / per >= b0 && tid / per <= (to - 1) / s.block) {
    const int k = tid == 0 ? ek[0] : tid == 1 ? ek[1] : tid == 2 ? ek[2] : ek[3], v = tid == 0 ? ev[0] : tid == 1 ? ev[1] : tid == 2 ? ev[2] : ev[3];
    a.ks[sc + tid / per] = kx_bits_f32(scale_bits(k));
    a.vs[sc + tid / per] = kx_bits_f32(scale_bits(v));
  }
  const bool few = to - from <= FEW && !grown_k && !grown_v;
  if (!few) {
    if (from > 0) {  // what the group keeps
      for (int i = tid; i < from * DP / 16; i += THREADS) ((uint4 *)lk)[i] = ((const uint4 *)gk)[i];
      for (int i = tid; i < VP * UNIT / 16; i += THREADS) ((uint4 *)lv)[i] = ((const uint4 *)gv)[i];
      __syncthreads();
      if (grown_k)
        for (int i = tid + b0 * s.block * DP / 4; i < from * DP / 4; i += THREADS) ((uint32_t *)lk)[i] = lowered(((uint32_t *)lk)[i], grown_k);
      if (grown_v)
        for (int i = tid; i < VP * UNIT / 4; i += THREADS) {  // a word has four tokens of one block of 16
          const int t = token_of(i * 4 % UNIT);
          if (t / s.block == b0) ((uint32_t *)lv)[i] = lowered(((uint32_t *)lv)[i], grown_v);
        }
    } else {
      for (int i = tid; i < VP * UNIT / 16; i += THREADS) ((uint4 *)lv)[i] = make_uint4(0, 0, 0, 0);
    }
    __syncthreads();
  }
  uint8_t *const tk = few ? gk : lk, *const tv = few ? gv : lv;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int t = wave + 4 * i;
    if (t < from || t >= to) continue;
    const float rk = kx_bits_f32(scale_bits(-ek[i >> 2])), rv = kx_bits_f32(scale_bits(-ev[i >> 2]));
    const int at = place_of(t);
#pragma unroll
    for (int p = 0; p < PK; ++p)
      if (lane + 64 * p < DP / 2) {
        const int2 d = pair_of(lane + 64 * p, s.rot, s.pairs);
        const uint32_t c = codes(xk[i][p][0], xk[i][p][1], rk);
        if (d.y == d.x + 1) {
          *(uint16_t *)(tk + t * DP + d.x) = (uint16_t)c;
        } else {
          tk[t * DP + d.x] = (uint8_t)c;
          tk[t * DP + d.y] = (uint8_t)(c >> 8);
        }
      }
#pragma unroll
    for (int p = 0; p < PV; ++p)
      if (lane + 64 * p < VP / 2) {
        const int d = 2 * (lane + 64 * p);
        const uint32_t c = codes(xv[i][p][0], xv[i][p][1], rv);
        tv[d * UNIT + at] = (uint8_t)c;
        tv[(d + 1) * UNIT + at] = (uint8_t)(c >> 8);
      }
  }
  if (few) return;
  __syncthreads();
  const int low = grown_k ? b0 * s.block : from;
  for (int i = tid + low * DP / 16; i < to * DP / 16; i += THREADS) ((uint4 *)gk)[i] = ((const uint4 *)lk)[i];
  for (int i = tid; i < VP * UNIT / 16; i += THREADS) ((uint4 *)gv)[i] = ((const uint4 *)lv)[i];
}

// bf16 of a code times a power of two: exact where the result is a bf16 number
__device__ __forceinline__ uint16_t value(uint32_t code, float scale) { return kx_bf16_rne(__builtin_amdgcn_cvt_f32_fp8((int)code, 0) * scale); }

template <int DP, int VP>
__global__ void __launch_bounds__(THREADS) read_k(KxPagedArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t lv[VP * UNIT];
  const KxPagedSpec &s = a.s;
  const Unit u = unit_of(a);
  if (!u.ok) return;
  const int tid = threadIdx.x;
  const uint8_t *const gk = a.k + (u.head * s.page + u.in_page) * DP, *const gv = a.v + (u.head * s.page + u.in_page) * VP;
  const size_t sc = u.head * (s.page / s.block) + u.in_page / s.block;
  uint16_t *const ok = (uint16_t *)a.out + (size_t)u.row * a.out_ld + (size_t)blockIdx.y * s.dim;
  uint16_t *const ov = (uint16_t *)a.out_v + (size_t)u.row * a.out_v_ld + (size_t)blockIdx.y * s.vdim;
  for (int i = tid; i < VP * UNIT / 16; i += THREADS) ((uint4 *)lv)[i] = ((const uint4 *)gv)[i];
  for (int i = tid; i < (u.to - u.from) * (DP / 2); i += THREADS) {
    const int t = u.from + i / (DP / 2), d = i % (DP / 2) * 2;
    const uint32_t c = *(const uint16_t *)(gk + t * DP + d);
    const float f = a.ks[sc + t / s.block];
    uint16_t *const to = ok + (size_t)(t - u.from) * a.out_ld + d;
    if (d < s.dim) to[0] = value(c, f);
    if (d + 1 < s.dim) to[1] = value(c >> 8, f);
  }
  __syncthreads();
  for (int i = tid; i < (u.to - u.from) * VP; i += THREADS) {
    const int t = u.from + i / VP, d = i % VP;
    if (d < s.vdim) ov[(size_t)(t - u.from) * a.out_v_ld + d] = value(lv[d * UNIT + place_of(t)], a.vs[sc + t / s.block]);
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
// groups of 64 that so many rows of so many sequences can lie in: n of a sequence in at most 2 + (n - 2) / 64
unsigned most_units(const KxPagedArgs &a) { return (unsigned)(2 * std::min(a.batch, a.tokens) + a.tokens / UNIT); }

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

// floats for the sums of parts: 256 CUs times two workgroups with 64 columns of 128 dimensions each
constexpr size_t PART_FLOATS = (size_t)512 * 64 * 130;

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
    p->a.part_floats = PART_FLOATS;
    const size_t turns = (turn.size() * 8 + 255) & ~(size_t)255, counters = ((size_t)p->a.arrivals * 4 + 4 + 255) & ~(size_t)255;
    KX_HIP(hipGetDevice(&p->device));
    if (hipMalloc((void **)&p->mem, turns + counters + PART_FLOATS * 4) != hipSuccess) {
      kx_set_error("kx_paged_create: no device memory for %zu bytes", turns + counters + PART_FLOATS * 4);
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
  return kx_paged_attend_launch(p->f32, a, kx_stream(stream));
}
extern "C" int kx_paged_faults(kx_paged *p, int32_t *h_bits, void *stream) {
  KX_REQUIRE(p && h_bits, "kx_paged_faults: null argument");
  KX_HIP(hipStreamSynchronize(kx_stream(stream)));
  KX_HIP(hipMemcpy(h_bits, p->a.fault, 4, hipMemcpyDeviceToHost));
  if (*h_bits) KX_HIP(hipMemset(p->a.fault, 0, 4));
  return KX_OK;
}

// kx_fp8.hip -- products with matrices of 8-bit elements that have a scale for each block of 128 x 128 (kx_fp8.h).
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies a block of 128 columns of 16 rows and 16 tokens, and takes the tokens' 2^e for nothing; the matrix's scale, any
// float, is one multiplication and addition for each sum of a block.  It adds the products of a block with fewer than 24 bits: 1.4e-5 of a block's sum on
// average (normal codes of three magnitudes), as v_mfma_f32_16x16x32_fp8_fp8 does, a hundredth of what rounding to bf16 is off.  Results in 32 bits
// go through f16, which holds the codes exactly, and v_mfma_f32_16x16x32_f16 at half the rate (6e-9 on the same sums).
#include <algorithm>
#include <atomic>
#include <memory>
#include <type_traits>
#include "kx_common.h"
#include "kx_fp8.h"
#include "kx_fp8_tile.h"
#include "kx_math.h"
#include "kx_paged_place.h"
#include "kx_read_once.h"
#include "kx_wave.h"

namespace {

using namespace kxfp8;

// element i of a row of the given format
__device__ __forceinline__ float element(const void *x, size_t i, bool f32) { return f32 ? ((const float *)x)[i] : kx_bf16_f32(((const uint16_t *)x)[i]); }
__device__ __forceinline__ uint32_t magnitude(float x) {
  const uint32_t u = kx_f32_bits(x) & 0x7fffffffu;
  return u >= 0x7f800000u ? 0u : u;
}
__device__ __forceinline__ float scaled(float x, float inverse) { return (kx_f32_bits(x) & 0x7f800000u) == 0x7f800000u ? __builtin_nanf("") : x * inverse; }
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float inverse) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(scaled(a, inverse), scaled(b, inverse), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(scaled(c, inverse), scaled(d, inverse), r, true);
}

__device__ __forceinline__ i8v pieces(const uint8_t *p, const uint8_t *q) {  // a lane's 32 codes of a block
  const i4v a = *(const i4v *)p, b = *(const i4v *)q;
  return i8v{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

__device__ __forceinline__ uint32_t row_max(uint32_t v) {  // over 16 lanes
#define KXF_STEP(C) v = max(v, (uint32_t)kxw::dpp_keep_i<C>((int)v))
  KXF_STEP(kxw::DPP_QUAD_XOR1);
  KXF_STEP(kxw::DPP_QUAD_XOR2);
  KXF_STEP(kxw::DPP_ROW_HALF_MIRROR);
  KXF_STEP(kxw::DPP_ROW_MIRROR);
#undef KXF_STEP
  return v;
}
// 8 columns of a row from c on, zero beyond cols; vector: rows of whole 16-byte pieces at multiples of 16
template <bool F32>
__device__ __forceinline__ void load8(const void *x, size_t row, int c, int cols, bool vector, float (&v)[8]) {
  if (vector && c + 8 <= cols) {
    if constexpr (F32) {
      const float4 *const p = (const float4 *)((const float *)x + row + c);
      const float4 u = p[0], w = p[1];
      v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w, v[4] = w.x, v[5] = w.y, v[6] = w.z, v[7] = w.w;
    } else {
      const uint4 u = *(const uint4 *)((const uint16_t *)x + row + c);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = kx_bits_f32(w[i] << 16);
        v[2 * i + 1] = kx_bits_f32(w[i] & 0xffff0000u);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? element(x, row + c + i, F32) : 0.0f;
  }
}

// Rows of x as codes and exponents: 16 lanes have a block of 128 columns, 8 of them each.
template <bool F32>
__global__ void __launch_bounds__(256) fp8_rows_k(KxFp8Args a, int vector) {
  const int lane = threadIdx.x & 15, b = blockIdx.x * 16 + (threadIdx.x >> 4), c = b * 128 + lane * 8;
  if (b >= a.blocks) return;
  for (int t = blockIdx.y; t < a.tokens; t += gridDim.y) {
    float v[8];
    load8<F32>(a.x, (size_t)t * a.x_ld, c, a.cols, vector, v);
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, magnitude(v[i]));
    m = row_max(m);
    const int e = kxpage::exponent_of(m);
    const float inverse = kx_bits_f32(kxpage::scale_bits(-e));
    *(uint2 *)(a.xc + (size_t)t * a.blocks * 128 + c) = make_uint2(codes4(v[0], v[1], v[2], v[3], inverse), codes4(v[4], v[5], v[6], v[7], inverse));
    if (lane == 0) a.xe[exponent_at(b, t, a.groups)] = (uint8_t)(e + 127);
  }
}

template <bool ONCE>
__device__ __forceinline__ void copy_row(const uint8_t *at, uint32_t to) {
  if constexpr (ONCE) kx_copy16_to_lds_once(at, to);
  else kx_copy16_to_lds(at, to);
}
template <bool F32>
__device__ __forceinline__ void store4(const KxFp8Args &a, int t, int r, int rows, f4 y) {  // four rows of a token
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (r + e < rows) {
      if constexpr (F32) ((float *)a.out)[(size_t)t * a.out_ld + r + e] = y[e];
      else ((uint16_t *)a.out)[(size_t)t * a.out_ld + r + e] = kx_bf16_rne(y[e]);
    }
}

// Up to 32 tokens: what counts is that the matrix is on its way at once and then flows.  A workgroup has an equal share of the rows, goes through them in tiles of 16 RT rows,
// and its KW waves have the blocks of columns in turn.  A wave copies its blocks, R ahead and from one tile into the next, to a ring in LDS of its own and
// reads them from there as operands: whole lines of 128 bytes, 8 rows an instruction, 16-byte pieces xor-ed by the row, no barrier.  The sums of the KW waves
// meet in LDS at the end of a tile.
//   CT = 0: up to 4 tokens, which the workgroup rounds to 8 bits itself while the first blocks come, and keeps in LDS: one launch.
//   CT > 0: 16 CT rounded tokens, copied block by block with the matrix.
template <int CT_, int RT_, int KW_, int R_>
struct Stream {
  static constexpr bool SELF = CT_ == 0;
  static constexpr int CT = SELF ? 1 : CT_, RT = RT_, KW = KW_, R = R_, THREADS = KW * 64, ROWS = 16 * RT;
  static constexpr int BLOCK = RT * 2048 + (SELF ? 0 : CT * 2048), COPIES = 2 * RT + (SELF ? 0 : 2 * CT), RING = KW * R * BLOCK, SUMS = RT * CT * KW * 1024;
  static_assert(RT * CT <= KW, "a wave for each block of sums");
  static int x_bytes(const KxFp8Args &a) { return SELF ? a.tokens * (a.blocks * 128 + 16) + a.blocks * 4 : a.blocks * 64; }  // tokens and exponents, or exponents alone
  static int lds(const KxFp8Args &a, int bands) { return RING + 2 * SUMS + ((x_bytes(a) + 15) & ~15) + bands * a.blocks * 4; }
};
template <class N, bool F32, bool X32, bool ONCE>
__global__ void __launch_bounds__(N::THREADS, 2) fp8_stream_k(KxFp8Args a, int vector, int x_bytes) {
  constexpr int CT = N::CT, RT = N::RT, KW = N::KW, R = N::R;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
  const int lane = threadIdx.x & 63, kw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, kq = lane >> 4, sub = lane >> 3, piece = ((lane & 7) ^ sub) * 16;
  // the share in units of four rows, which have one scale
  const int units = (a.rows + 3) / 4, lo = kxtile::cut(units, blockIdx.x, gridDim.x) * 4, hi = min(kxtile::cut(units, blockIdx.x + 1, gridDim.x) * 4, a.rows);
  const int tiles = (hi - lo + N::ROWS - 1) / N::ROWS, mine = (a.blocks - kw + KW - 1) / KW, xld = a.blocks * 128 + 16;
  f4 *const sums = (f4 *)(lds + N::RING);
  uint8_t *const xs = lds + N::RING + 2 * N::SUMS, *const es = N::SELF ? xs + a.tokens * xld : xs;
  float *const sc = (float *)(xs + x_bytes);

  // the next block to copy: block k KW + kw of the tile whose rows begin at w
  const uint8_t *w[2 * RT], *x[N::SELF ? 1 : 2 * CT];
  int next_k = 0, next_row = lo, asked = 0;
  auto rows_at = [&](int row) {
#pragma unroll
    for (int i = 0; i < 2 * RT; ++i) w[i] = a.w + (size_t)min(row + i * 8 + sub, hi - 1) * a.ld + kw * 128 + piece;
  };
  rows_at(lo);
  if constexpr (!N::SELF) {
#pragma unroll
    for (int i = 0; i < 2 * CT; ++i) x[i] = a.xc + (size_t)min(i * 8 + sub, a.tokens - 1) * (a.blocks * 128) + kw * 128 + piece;
  }
  const int total = tiles * mine;
  auto copy = [&]() {
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + (kw * R + asked % R) * N::BLOCK);
    const size_t at = (size_t)next_k * (KW * 128);
#pragma unroll
    for (int i = 0; i < 2 * RT; ++i) copy_row<ONCE>(w[i] + at, to + i * 1024);
    if constexpr (!N::SELF) {
#pragma unroll
      for (int i = 0; i < 2 * CT; ++i) kx_copy16_to_lds(x[i] + at, to + RT * 2048 + i * 1024);
    }
    ++asked;
    if (++next_k == mine) {
      next_k = 0;
      next_row += N::ROWS;
      rows_at(min(next_row, hi - 1));
    }
  };
  while (asked < min(R, total)) copy();

  // scales of the share's rows, and the tokens
  const int band = lo / 128, bands = (hi - 1) / 128 - band + 1;
  for (int i = threadIdx.x; i < bands * a.blocks; i += N::THREADS) sc[i] = a.w_scale[(size_t)band * a.blocks + i];
  if constexpr (N::SELF) {
    // 16 lanes a block of a token, 8 columns each; four of these are asked for before the first is used
    constexpr int U = 4;
    const int items = a.blocks * a.tokens;
    for (int i0 = threadIdx.x >> 4; i0 < items; i0 += U * (N::THREADS / 16)) {
      float v[U][8];
      int t[U], b[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = min(i0 + u * (N::THREADS / 16), items - 1);
        b[u] = a.tokens == 1 ? i : a.tokens == 2 ? i >> 1 : a.tokens == 4 ? i >> 2 : i / 3;
        t[u] = i - b[u] * a.tokens;
        load8<X32>(a.x, (size_t)t[u] * a.x_ld, b[u] * 128 + lr * 8, a.cols, vector, v[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, magnitude(v[u][i]));
        m = row_max(m);
        const int e = kxpage::exponent_of(m);
        const float inverse = kx_bits_f32(kxpage::scale_bits(-e));
        *(uint2 *)(xs + t[u] * xld + b[u] * 128 + lr * 8) =
            make_uint2(codes4(v[u][0], v[u][1], v[u][2], v[u][3], inverse), codes4(v[u][4], v[u][5], v[u][6], v[u][7], inverse));
        if (lr == 0) es[b[u] * 4 + t[u]] = (uint8_t)(e + 127);
      }
    }
  } else {
    for (int i = threadIdx.x; i < a.blocks * 4; i += N::THREADS) ((uint4 *)es)[i] = *(const uint4 *)(a.xe + exponent_at(i / 4, 0, a.groups) + i % 4 * 16);
  }
  __syncthreads();

  const int p0 = (kq ^ (lr & 7)) * 16, p1 = ((4 + kq) ^ (lr & 7)) * 16, token = min(lr, a.tokens - 1);
  int read = 0;
  for (int tile = 0; tile < tiles; ++tile) {
    const int r0 = lo + tile * N::ROWS;
    const float *scales[RT];  // of the lane's rows
#pragma unroll
    for (int r = 0; r < RT; ++r) scales[r] = sc + (min(r0 + r * 16 + kq * 4, hi - 1) / 128 - band) * a.blocks;
    f4 acc[RT][CT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int c = 0; c < CT; ++c) acc[r][c] = f4{0, 0, 0, 0};
    for (int b = kw; b < a.blocks; b += KW) {
      // copies of a wave come in order: a block has when no more than those behind it are on their way
      if (total - read >= R) kx_wait_copies<N::COPIES * (R - 1)>();
      else kx_wait_copies<0>();
      const uint8_t *const at = lds + (kw * R + read % R) * N::BLOCK + lr * 128;
      ++read;
      i8v wv[RT], xv[CT];
      float s[RT];
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        wv[r] = pieces(at + r * 2048 + p0, at + r * 2048 + p1);
        s[r] = scales[r][b];
      }
      uint32_t e;
      if constexpr (N::SELF) {
        xv[0] = pieces(xs + token * xld + b * 128 + kq * 16, xs + token * xld + b * 128 + kq * 16 + 64);
        e = es[b * 4 + token];
      } else {
#pragma unroll
        for (int c = 0; c < CT; ++c) xv[c] = pieces(at + RT * 2048 + c * 2048 + p0, at + RT * 2048 + c * 2048 + p1);
        e = *(const uint32_t *)(es + b * 64 + lr * 4);
      }
      __builtin_amdgcn_sched_barrier(0);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // its place is read: the next block's copies may go there
      if (asked < total) copy();
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const f4 p = F32 ? block16(halves(wv[r]), halves(xv[c])) : block8<false>(wv[r], xv[c], c, (int)e);
          const float f = F32 ? s[r] * power(e >> 8 * c & 0xffu) : s[r];
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[r][c][i] = __builtin_fmaf(p[i], f, acc[r][c][i]);
        }
    }
    f4 *const mine_at = sums + (tile & 1) * (N::SUMS / 16);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int c = 0; c < CT; ++c) mine_at[((r * CT + c) * KW + kw) * 64 + lane] = acc[r][c];
    kx_lds_barrier();
    if (kw < RT * CT) {
      f4 y = mine_at[kw * KW * 64 + lane];
#pragma unroll
      for (int v = 1; v < KW; ++v) y += mine_at[(kw * KW + v) * 64 + lane];
      const int t = kw % CT * 16 + lr;
      if (t < a.tokens) store4<F32>(a, t, r0 + kw / CT * 16 + kq * 4, hi, y);
    }
  }
}

// 33 to 64 tokens, and fewer beside long rows, already rounded: 16 CT of them, and 16 rows of the matrix for each of NW waves, and a part of the columns a workgroup.  A step is a block of
// columns: every wave copies its rows of it and a share of the tokens to LDS, R - 1 steps ahead, and one barrier a step says that all of it has come and that
// the place of the step before is free.  Sums of parts are added by the last workgroup in (kx_arrive.h), in order.
template <int CT_, int NW_, int R_>
struct Narrow {
  static constexpr int CT = CT_, NW = NW_, R = R_, THREADS = NW * 64, ROWS = 16 * NW, TOKENS = 16 * CT, AHEAD = 64;
  static constexpr int STEP = NW * 2048 + CT * 2048, XC = (2 * CT + NW - 1) / NW, COPIES = 2 + XC, LDS = R * STEP + AHEAD * 64;
};
template <class N, bool F32, bool ONCE>
__global__ void __launch_bounds__(N::THREADS, 2) fp8_narrow_k(KxFp8Args a, int parts) {
  constexpr int CT = N::CT, NW = N::NW, R = N::R;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  __shared__ int last;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, kq = lane >> 4, sub = lane >> 3;
  const int group = blockIdx.x / parts, part = blockIdx.x - group * parts, r0 = group * N::ROWS;
  const int b0 = kxtile::cut(a.blocks, part, parts), b1 = kxtile::cut(a.blocks, part + 1, parts);
  uint8_t *const es = lds + R * N::STEP;
  const uint8_t *w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) w[i] = a.w + (size_t)min(r0 + wave * 16 + i * 8 + sub, a.rows - 1) * a.ld + ((lane & 7) ^ sub) * 16;
  const uint8_t *x[N::XC];
#pragma unroll
  for (int i = 0; i < N::XC; ++i) x[i] = a.xc + (size_t)min((i * NW + wave) % (2 * CT) * 8 + sub, a.tokens - 1) * (a.blocks * 128) + ((lane & 7) ^ sub) * 16;
  auto copy = [&](int b) {
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + (b - b0) % R * N::STEP);
#pragma unroll
    for (int i = 0; i < 2; ++i) copy_row<ONCE>(w[i] + (size_t)b * 128, to + wave * 2048 + i * 1024);
#pragma unroll
    for (int i = 0; i < N::XC; ++i) kx_copy16_to_lds(x[i] + (size_t)b * 128, __builtin_amdgcn_readfirstlane(to + NW * 2048 + (i * NW + wave) % (2 * CT) * 1024));
  };
  const float *const ws = a.w_scale + (size_t)(r0 / 128) * a.blocks;
  const int p0 = (kq ^ (lr & 7)) * 16, p1 = ((4 + kq) ^ (lr & 7)) * 16;
  f4 acc[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) acc[c] = f4{0, 0, 0, 0};
  for (int b = b0; b < min(b0 + R - 1, b1); ++b) copy(b);
  float scales = 0.0f;
  for (int b = b0; b < b1; ++b) {
    const int q = (b - b0) % N::AHEAD;
    if (q == 0) {  // exponents of the tokens and scales of the rows, for the next blocks
      const int n = min(N::AHEAD, b1 - b);
      if (b > b0) __syncthreads();
      for (int i = threadIdx.x; i < n * 4; i += N::THREADS) ((uint4 *)es)[i] = *(const uint4 *)(a.xe + exponent_at(b + i / 4, 0, a.groups) + i % 4 * 16);
      scales = ws[b + min(lane, n - 1)];
    }
    // copies of a wave come in order: the step's have when no more than those behind it are on their way
    if (b1 - b >= R - 1) kx_wait_copies<N::COPIES * (R - 2)>();
    else kx_wait_copies<0>();
    kx_lds_barrier();
    if (b + R - 1 < b1) copy(b + R - 1);
    const uint8_t *const at = lds + (b - b0) % R * N::STEP, *const wr = at + wave * 2048 + lr * 128, *const xr = at + NW * 2048 + lr * 128;
    const i8v wv = pieces(wr + p0, wr + p1);
    const uint32_t e = *(const uint32_t *)(es + q * 64 + lr * 4);
    i8v xv[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) xv[c] = pieces(xr + c * 2048 + p0, xr + c * 2048 + p1);
    const float s = kx_bits_f32((uint32_t)__builtin_amdgcn_readlane((int)kx_f32_bits(scales), q));
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const f4 p = F32 ? block16(halves(wv), halves(xv[c])) : block8<false>(wv, xv[c], c, (int)e);
      const float f = F32 ? s * power(e >> 8 * c & 0xffu) : s;
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[c][i] = __builtin_fmaf(p[i], f, acc[c][i]);
    }
  }
  if (parts == 1) {
#pragma unroll
    for (int c = 0; c < CT; ++c)
      if (c * 16 + lr < a.tokens) store4<F32>(a, c * 16 + lr, r0 + wave * 16 + kq * 4, a.rows, acc[c]);
    return;
  }
  const size_t size = (size_t)a.tokens * N::ROWS;  // floats of a part
  uint64_t *const sums = (uint64_t *)(a.part + (size_t)group * parts * size);
#pragma unroll
  for (int c = 0; c < CT; ++c)
    if (c * 16 + lr < a.tokens) {
      uint64_t *const to = sums + (part * size + (c * 16 + lr) * N::ROWS + wave * 16 + kq * 4) / 2;
#pragma unroll
      for (int i = 0; i < 2; ++i) kx_arrive_store(to + i, (uint64_t)kx_f32_bits(acc[c][2 * i]) | (uint64_t)kx_f32_bits(acc[c][2 * i + 1]) << 32);
    }
  kx_arrive_writes_done();
  __syncthreads();
  if (threadIdx.x == 0) last = kx_arrive_is_last(a.arrived + group, parts);
  __syncthreads();
  if (!last) return;
  if (threadIdx.x == 0) kx_arrive_reset(a.arrived + group);
  for (int i = threadIdx.x; i < (int)(size / 4); i += N::THREADS) {
    f4 y = {0, 0, 0, 0};
    for (int p = 0; p < parts; p += 8) {
      uint64_t u[8][2];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (p + k < parts) {
          u[k][0] = kx_arrive_load(sums + ((p + k) * size) / 2 + i * 2);
          u[k][1] = kx_arrive_load(sums + ((p + k) * size) / 2 + i * 2 + 1);
        }
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (p + k < parts) y += f4{kx_bits_f32((uint32_t)u[k][0]), kx_bits_f32((uint32_t)(u[k][0] >> 32)), kx_bits_f32((uint32_t)u[k][1]), kx_bits_f32((uint32_t)(u[k][1] >> 32))};
    }
    store4<F32>(a, i / (N::ROWS / 4), r0 + i % (N::ROWS / 4) * 4, a.rows, y);
  }
}

// Whether the matrix passes the memory-side cache by (kx_read_once.h); the model's size is not known here, a matrix of 24 MB is taken for one of a large one's.
bool read_once(const KxFp8Args &a) { return (size_t)a.rows * a.ld >= kxonce::MATRIX; }
bool in_pieces(const KxFp8Args &a) { return (uintptr_t)a.x % 16 == 0 && (size_t)a.x_ld * (a.x_f32 ? 4 : 2) % 16 == 0; }

constexpr int LDS = 160 * 1024;  // of a CU
template <class K>
int allow_lds(K kernel, int bytes, std::atomic<bool> &done) {  // setting it twice from two threads is harmless
  if (!done) {
    KX_HIP(hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
    done = true;
  }
  return KX_OK;
}
// bytes of LDS with the scales of a share's rows, which matrices of millions of rows have too many of
template <class N>
int stream_lds(const KxFp8Args &a, int grid) {
  const int share = kx_cdiv(kx_cdiv(a.rows, 4), grid) * 4;
  return N::lds(a, (share + 126) / 128 + 1);
}
template <class N, bool F32, bool X32, bool ONCE>
int launch_stream(const KxFp8Args &a, int grid, hipStream_t st) {
  static std::atomic<bool> attr{false};
  KX_DO(allow_lds(fp8_stream_k<N, F32, X32, ONCE>, LDS, attr));
  fp8_stream_k<N, F32, X32, ONCE><<<(unsigned)grid, N::THREADS, stream_lds<N>(a, grid), st>>>(a, in_pieces(a), (N::x_bytes(a) + 15) & ~15);
  KX_LAUNCH_CHECK();
  return KX_OK;
}
template <class N>
int launch_stream(const KxFp8Args &a, int grid, hipStream_t st) {
  const bool once = read_once(a);
  if (N::SELF && a.x_f32) {
    if (a.out_f32) return once ? launch_stream<N, true, N::SELF, true>(a, grid, st) : launch_stream<N, true, N::SELF, false>(a, grid, st);
    return once ? launch_stream<N, false, N::SELF, true>(a, grid, st) : launch_stream<N, false, N::SELF, false>(a, grid, st);
  }
  if (a.out_f32) return once ? launch_stream<N, true, false, true>(a, grid, st) : launch_stream<N, true, false, false>(a, grid, st);
  return once ? launch_stream<N, false, false, true>(a, grid, st) : launch_stream<N, false, false, false>(a, grid, st);
}
template <class N, bool F32, bool ONCE>
int launch_narrow(const KxFp8Args &a, hipStream_t st) {
  const int cus = std::max(1, kx_device_cus()), groups = kx_cdiv(a.rows, N::ROWS), room = (int)std::min<size_t>(64, a.part_floats / ((size_t)groups * a.tokens * N::ROWS));
  const int parts = std::max(1, std::min({2 * cus / groups, a.blocks / 4, room, groups <= a.arrivals ? 64 : 1}));
  static std::atomic<bool> attr{false};
  KX_DO(allow_lds(fp8_narrow_k<N, F32, ONCE>, N::LDS, attr));
  fp8_narrow_k<N, F32, ONCE><<<(unsigned)(groups * parts), N::THREADS, N::LDS, st>>>(a, parts);
  KX_LAUNCH_CHECK();
  return KX_OK;
}
template <class N>
int launch_narrow(const KxFp8Args &a, hipStream_t st) {
  if (a.out_f32) return read_once(a) ? launch_narrow<N, true, true>(a, st) : launch_narrow<N, true, false>(a, st);
  return read_once(a) ? launch_narrow<N, false, true>(a, st) : launch_narrow<N, false, false>(a, st);
}

// Tiles of kx_fp8_tile.h.
template <int RI, bool F32>
__global__ void __launch_bounds__(512, 2) fp8_tile_k(KxFp8Args a, kxtile::Share share) {
  typedef Tile<RI, F32> TL;
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int tm = (a.tokens + TL::BM - 1) / TL::BM, xld = a.blocks * 128;
  const kxtile::Place place = kxtile::place_of(blockIdx.x, tm * ((a.rows + TL::BN - 1) / TL::BN), share);
  const int m0 = place.tile % tm * TL::BM, n0 = place.tile / tm * TL::BN, bands = (a.rows + 127) / 128;
  typename TL::Sums acc;
  TL::run(lds, kxtile::cut(a.blocks, place.part, place.of), kxtile::cut(a.blocks, place.part + 1, place.of),
          a.xc + (size_t)m0 * xld, xld, a.tokens - m0, a.w + (size_t)n0 * a.ld, a.ld, a.rows - n0,
          [&](int b) { return a.xe + exponent_at(b, m0, a.groups); }, a.w_scale + (size_t)min(n0 / 128 + TL::group(), bands - 1) * a.blocks, acc);
  if (place.of > 1 &&
      !kxtile::gather<TL>(lds, acc, a.part + (size_t)(place.tile - share.whole) * place.of * TL::PART, a.arrived + place.tile - share.whole, place.of, place.part))
    return;
  auto at = [&](int i, int v) { return (size_t)min(m0 + TL::row(i, v), a.tokens - 1) * a.out_ld; };
  auto in = [&](int i, int v) { return m0 + TL::row(i, v) < a.tokens; };
  if constexpr (F32) {
#pragma unroll
    for (int i = 0; i < TL::MI; ++i)
#pragma unroll
      for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int j = 0; j < TL::NI; ++j)
          if (in(i, v) && n0 + TL::col(j) < a.rows) ((float *)a.out)[at(i, v) + n0 + TL::col(j)] = acc[i][j][v];
  } else {
    // a result is 2 bytes and a block of 16 columns 32 bytes of a row: two lanes exchange theirs of two blocks, so that a store takes 64 bytes of each row
    const uint32_t odd = threadIdx.x & 1, order = odd ? 0x03020706u : 0x05040100u;
    uint16_t *const out = (uint16_t *)a.out;
#pragma unroll
    for (int i = 0; i < TL::MI; ++i)
#pragma unroll
      for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int j = 0; j < TL::NI; j += 2) {
          const uint32_t p = (uint32_t)kx_bf16_rne(acc[i][j][v]) | (uint32_t)kx_bf16_rne(acc[i][j + 1][v]) << 16;
          const uint32_t q = kx_f32_bits(kxw::dpp_f<kxw::DPP_QUAD_XOR1>(kx_bits_f32(p))), y = __builtin_amdgcn_perm(q, p, order);
          const int n = n0 + (odd ? TL::col(j + 1) - 1 : TL::col(j));
          if (!in(i, v)) continue;
          if (a.pairs && n + 1 < a.rows) {
            *(uint32_t *)(out + at(i, v) + n) = y;
          } else {
            if (n < a.rows) out[at(i, v) + n] = (uint16_t)y;
            if (n + 1 < a.rows) out[at(i, v) + n + 1] = (uint16_t)(y >> 16);
          }
        }
  }
}

template <int RI, bool F32>
int launch_tiles(const KxFp8Args &a, kxtile::Share share, hipStream_t st) {
  typedef Tile<RI, F32> TL;
  static std::atomic<bool> attr{false};
  KX_DO(allow_lds(fp8_tile_k<RI, F32>, TL::LDS, attr));
  fp8_tile_k<RI, F32><<<dim3(share.grid(kx_cdiv(a.tokens, TL::BM) * kx_cdiv(a.rows, TL::BN))), TL::THREADS, TL::LDS, st>>>(a, share);
  KX_LAUNCH_CHECK();
  return KX_OK;
}
// The tile that is sooner by estimates in us, and how it is shared out: rounds of one workgroup per CU, and for parts of the columns what handing over their sums takes.
// us with the rows before it, tiles of 256 / 128 / 64 tokens: 2048 x 18432 x 7168 296 / 323 / 514, 2048 x 7168 x 8192 128 / 153 / 237, 2048 x 2112 x 7168 80 / 74 / 79 (the
// estimate takes the first), 1024 x 12288 x 1536 41 / 46 / 49, 512 x 7168 x 8192 79 / 54 / 57, 256 x 7168 x 2048 43 / 28 / 22, 128 x 18432 x 7168 77 / 56 / 63, 128 x 7168 x 8192 69 /
// 42 / 30, 96 x 2112 x 7168 65 / 38 / 26; 32-bit results 2048 x 7168 x 8192 - / 280 / 339, 333 x 4103 x 2000 - / 36 / 27.
template <bool F32>
int tiles(const KxFp8Args &a, hipStream_t st) {
  const int cus = std::max(1, kx_device_cus());
  constexpr int LARGEST = F32 ? 2 : 4;
  double best = 1e30;
  int ri = 1;
  kxtile::Share share = {0, 1};
  for (int r = LARGEST; r >= 1; r /= 2) {
    const double block = F32 ? (r == 2 ? 2.0 : 1.27) : r == 4 ? 1.95 : r == 2 ? 1.3 : 0.83;
    const int bm = 64 * r;
    const long n = (long)kx_cdiv(a.tokens, bm) * kx_cdiv(a.rows, 256);
    auto rounds = [&](long wgs, double per) { return (double)((wgs + cus - 1) / cus) * (4.0 + block * per); };
    auto time = [&](long whole, long rest, int p) { return rounds(whole, a.blocks) + (rest ? rounds(rest * p, (double)a.blocks / p) + 1.5 + 2.4 * r * p : 0.0); };
    double t;
    const kxtile::Share s = kxtile::share(n, cus, std::min(16, a.blocks / 4), (long)(a.part_floats / ((size_t)bm * 256)), a.arrivals, time, &t);
    if (t < best) best = t, ri = r, share = s;
  }
  if constexpr (!F32)
    if (ri == 4) return launch_tiles<4, F32>(a, share, st);
  return ri == 2 ? launch_tiles<2, F32>(a, share, st) : launch_tiles<1, F32>(a, share, st);
}

}  // namespace

// us, measured with matrices in turn.  One workgroup of eight waves a CU: 1 x 7168 x 8192 12.8, 1 x 18432 x 7168 23.4 (5.6 TB/s), 1 x 163840 x 7168 174 (6.75 TB/s), 24 x 7168 x
// 8192 18.4; two of four 13.4, 24.9, 176 and 18.3, and 4 x 7168 x 8192 19.1 instead of 15.2; workgroups of 16 rows instead of shares of all 14.9, 34.9, 243.  16 tokens beside
// tiles of 32 rows 27.5 at 18432 x 7168, 29.2 beside 16; 8 at 7168 x 8192, where a share is 28 rows, 18.1 and 14.6.  Rounding the tokens in a launch of its own takes 3 to 4.
// The tiles of 64 tokens take over where they are as soon: 128 x 7168 x 8192 29.7, 64 of fp8_narrow_k 29.9, 32 of it 23.9.
int kx_fp8_launch(const KxFp8Args &a, hipStream_t st) {
  const int cus = std::max(1, kx_device_cus()), stream = std::min(kx_cdiv(a.rows, 16), cus);
  if (a.tokens <= 4 && a.tokens * a.blocks <= 256 && stream_lds<Stream<0, 1, 8, 4>>(a, stream) <= LDS) return launch_stream<Stream<0, 1, 8, 4>>(a, stream, st);
  const dim3 rows(kx_cdiv(a.blocks, 16), std::min(a.tokens, 65535));
  if (a.x_f32) fp8_rows_k<true><<<rows, 256, 0, st>>>(a, in_pieces(a));
  else fp8_rows_k<false><<<rows, 256, 0, st>>>(a, in_pieces(a));
  KX_LAUNCH_CHECK();
  if (a.tokens <= 32 && a.blocks <= 160 && std::max(stream_lds<Stream<2, 1, 8, 2>>(a, stream), stream_lds<Stream<1, 2, 8, 2>>(a, cus)) <= LDS) {
    if (a.tokens > 16) return launch_stream<Stream<2, 1, 8, 2>>(a, stream, st);
    if (a.rows < 64 * cus) return launch_stream<Stream<1, 1, 8, 3>>(a, stream, st);
    return launch_stream<Stream<1, 2, 8, 2>>(a, cus, st);
  }
  if (a.tokens <= 32) return launch_narrow<Narrow<2, 4, 6>>(a, st);
  if (a.tokens <= 64) return launch_narrow<Narrow<4, 4, 4>>(a, st);
  return a.out_f32 ? tiles<true>(a, st) : tiles<false>(a, st);
}

// ---- the operator of the C ABI ----------------------------------------------------------------------------------------------------------
struct kx_fp8 {
  KxFp8Args a;
  int max_tokens = 0, max_blocks = 0, device = 0;
  uint8_t *mem = nullptr;
};
// floats for the sums of parts: of up to 64 tokens, and of a tile of 256 x 256 on each of 256 CUs
static constexpr size_t FP8_FEW_PARTS = (size_t)4 << 20, FP8_PARTS = (size_t)256 * 256 * 256;
static constexpr int FP8_ARRIVALS = 512;

extern "C" int kx_fp8_create(int32_t max_tokens, int32_t max_cols, kx_fp8 **out) {
  KX_REQUIRE(out, "kx_fp8_create: null argument");
  *out = nullptr;
  KX_REQUIRE(max_tokens > 0 && max_cols > 0 && max_tokens <= 1 << 22 && max_cols <= 1 << 17, "kx_fp8_create: max_tokens=%d max_cols=%d", max_tokens, max_cols);
  return kx_guard("kx_fp8_create", [&]() -> int {
    std::unique_ptr<kx_fp8> p(new kx_fp8());
    p->max_tokens = max_tokens;
    p->max_blocks = kx_cdiv(max_cols, 128);
    KX_HIP(hipGetDevice(&p->device));
    const size_t groups = (size_t)kx_cdiv(max_tokens, 256) * 4;
    size_t at = 0;
    auto take = [&](size_t n) { const size_t from = at; at += (n + 255) & ~(size_t)255; return from; };
    const size_t xc = take((size_t)max_tokens * p->max_blocks * 128), xe = take(groups * 64 * p->max_blocks), arrived = take(FP8_ARRIVALS * 4), part = take((max_tokens > 64 ? FP8_PARTS : FP8_FEW_PARTS) * 4);
    if (hipMalloc((void **)&p->mem, at) != hipSuccess) {
      kx_set_error("kx_fp8_create: no device memory for %zu bytes", at);
      return KX_ERR_HIP;
    }
    p->a.xc = p->mem + xc;
    p->a.xe = p->mem + xe;
    p->a.arrived = (int *)(p->mem + arrived);
    p->a.part = (float *)(p->mem + part);
    p->a.arrivals = FP8_ARRIVALS;
    p->a.part_floats = max_tokens > 64 ? FP8_PARTS : FP8_FEW_PARTS;
    hipError_t e = hipMemset(p->a.arrived, 0, FP8_ARRIVALS * 4);
    if (e == hipSuccess) e = hipStreamSynchronize(nullptr);  // calls may come on any stream
    if (e != hipSuccess) {
      (void)hipFree(p->mem);
      kx_set_error("kx_fp8_create: %s", hipGetErrorString(e));
      return KX_ERR_HIP;
    }
    *out = p.release();
    return KX_OK;
  });
}
extern "C" int kx_fp8_destroy(kx_fp8 *p) {
  if (!p) return KX_OK;
  if (p->mem) (void)hipFree(p->mem);
  delete p;
  return KX_OK;
}
extern "C" int kx_fp8_run(kx_fp8 *p, const kx_fp8_args *x, void *stream) {
  KX_REQUIRE(p && x && x->d_w && x->d_w_scale && x->d_x && x->d_out, "kx_fp8_run: null argument");
  KX_REQUIRE(x->tokens >= 0 && x->tokens <= p->max_tokens && x->rows > 0 && x->cols > 0 && x->cols <= p->max_blocks * 128, "kx_fp8_run: tokens=%d rows=%d cols=%d", x->tokens, x->rows, x->cols);
  KX_REQUIRE(x->rows <= 1 << 25, "kx_fp8_run: rows=%d", x->rows);  // shares of rows are worked out in 32 bits (kxtile::cut)
  KxFp8Args a = p->a;
  a.blocks = kx_cdiv(x->cols, 128);
  KX_REQUIRE(x->ld % 128 == 0 && x->ld >= a.blocks * 128 && x->ld < 1 << 24 && x->x_ld >= x->cols && x->out_ld >= x->rows, "kx_fp8_run: ld=%d x_ld=%d out_ld=%d", x->ld, x->x_ld, x->out_ld);
  const size_t xs = x->x_f32 ? 4 : 2, os = x->out_f32 ? 4 : 2;
  KX_REQUIRE((uintptr_t)x->d_w % 16 == 0 && (uintptr_t)x->d_w_scale % 4 == 0 && (uintptr_t)x->d_x % xs == 0 && (uintptr_t)x->d_out % os == 0, "kx_fp8_run: the matrix begins at a multiple of 16 bytes, rows at one of an element");
  int dev = -1;
  KX_HIP(hipGetDevice(&dev));
  KX_REQUIRE(dev == p->device, "kx_fp8_run: made on device %d, called on device %d", p->device, dev);
  if (!x->tokens) return KX_OK;
  a.w = (const uint8_t *)x->d_w; a.w_scale = x->d_w_scale; a.x = x->d_x; a.out = x->d_out;
  a.tokens = x->tokens; a.rows = x->rows; a.cols = x->cols; a.ld = x->ld; a.x_ld = x->x_ld; a.out_ld = x->out_ld;
  a.x_f32 = x->x_f32 != 0; a.out_f32 = x->out_f32 != 0;
  a.groups = kx_cdiv(a.tokens, 256) * 4;
  a.pairs = x->out_ld % 2 == 0 && (uintptr_t)x->d_out % 4 == 0;
  return kx_fp8_launch(a, kx_stream(stream));
}

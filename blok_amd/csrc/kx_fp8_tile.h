// kx_fp8_tile.h -- a tile of a product of 8-bit rows with an 8-bit matrix (kx_fp8.h) whose two groups of four waves take turns as those of
// kx_gemm_turns.h do: while one multiplies, the other reads its next operands from LDS and asks for copies.
//
// A block of 128 columns is 128 bytes of a row, so staged rows, the order of the copies and the turns are those of 64 columns of bf16, with one difference:
// every sum of a block is multiplied by the matrix's scale and added (4 instructions of 4 cycles beside a product of 32), which the wave does
// for the product before the last while the matrix core has the next.  The tokens' exponents ride along in LDS, 32 blocks at a time and twice, and
// go into the product as they are.
// With EXACT the codes become f16 in registers, a row's block at a time, and the tokens' 2^e is a factor of the scale.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "kx_gemm_tile.h"

namespace kxfp8 {

typedef int i8v __attribute__((ext_vector_type(8)));
typedef int i4v __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ h8 unpacked(uint32_t lo, uint32_t hi) {
  const h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.0f, true);
  const h2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.0f, true);
  return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// The sums of a block: rows of the first operand times rows of the second, of 128 columns, 32 of them a lane.  Byte `which` of e is the exponent, + 127, of
// the lane's row of the first (FIRST) or second operand.
template <bool FIRST>
__device__ __forceinline__ f4 block8(i8v a, i8v b, int which, int e) {
  const f4 z = {0, 0, 0, 0};
  constexpr int one = 127;
#define KXF_CASE(n) case n: return FIRST ? __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, z, 0, 0, n, e, 0, one) : __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, z, 0, 0, 0, one, n, e)
  switch (which) {
    KXF_CASE(0);
    KXF_CASE(1);
    KXF_CASE(2);
    default: KXF_CASE(3);
  }
#undef KXF_CASE
}
struct Half {  // a lane's 32 codes as f16
  h8 p[4];
};
__device__ __forceinline__ Half halves(i8v a) {
  return {{unpacked((uint32_t)a[0], (uint32_t)a[1]), unpacked((uint32_t)a[2], (uint32_t)a[3]), unpacked((uint32_t)a[4], (uint32_t)a[5]), unpacked((uint32_t)a[6], (uint32_t)a[7])}};
}
__device__ __forceinline__ f4 block16(const Half &a, const Half &b) {
  f4 p = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.p[0], b.p[0], f4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
  for (int i = 1; i < 4; ++i) p = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.p[i], b.p[i], p, 0, 0, 0);
  return p;
}
__device__ __forceinline__ float power(uint32_t e) { return __builtin_bit_cast(float, e << 23); }  // 2^(e - 127)
// Where the exponent of token t lies behind those of its block of columns: the tokens of 64 that a lane's place stands for are one word.
__host__ __device__ __forceinline__ size_t exponent_at(size_t block, int t, int groups) { return (block * groups + t / 64) * 64 + (t & 15) * 4 + (t >> 4 & 3); }

// kx_copy16_to_lds of a place that is told by a wave's address and a lane's 32-bit offset from it: half the registers
__device__ __forceinline__ void copy16(const uint8_t *base, uint32_t offset, uint32_t lds_base) {
  const uint64_t at = (uint64_t)(uintptr_t)base;
  const uint64_t wave = (uint64_t)__builtin_amdgcn_readfirstlane((int)(at >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
  uint32_t m0_saved;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b32 m0, %0"
               : "=&s"(m0_saved)
               : "s"(lds_base), "v"(offset), "s"(wave)
               : "memory");
}

// Tiles of 64 RI tokens x 256 rows of the matrix; element v of sums (i, j) is matrix row col(j), token row(i, v).
template <int RI, bool EXACT>
struct Tile {
  typedef f4 Block;
  static constexpr int V = 4, THREADS = 512, BM = 64 * RI, BN = 256, MI = RI, NI = 8;
  static constexpr int XS = BM * 128, WS = BN * 128, AHEAD = 32, ES = AHEAD * BM, LDS = 2 * (XS + WS + ES);
  static constexpr size_t PART = (size_t)BM * BN;
  typedef Block Sums[MI][NI];
  static __device__ __forceinline__ int group() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 8); }
  static __device__ __forceinline__ int member() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6 & 3); }
  static __device__ __forceinline__ int col(int j) { return group() * 128 + j * 16 + (threadIdx.x & 15); }
  static __device__ __forceinline__ int row(int i, int v) { return member() * (16 * RI) + i * 16 + 4 * (threadIdx.x >> 4 & 3) + v; }
  static __device__ __forceinline__ void turn() {
    kx_lds_barrier();
    __builtin_amdgcn_sched_barrier(0);
  }
  // Blocks kb0 .. kb1 - 1 (kb0 < kb1) of 128 columns.  x, w: the tile's first rows, x_ld and w_ld bytes (below 2^24) from one to the next, and how many there are of
  // each (of those past the end the last one is read again); exps(b): the exponents of the tile's tokens for block b, readable up to the last block;
  // scales: of the group's rows, by block
  template <class Exps>
  static __device__ __forceinline__ void run(uint8_t *lds, int kb0, int kb1, const uint8_t *x_rows, int x_ld, int tokens, const uint8_t *w_rows, int w_ld, int w_count, Exps exps,
                                             const float *scales, Sums &acc) {
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t *)lds;
    const int lane = threadIdx.x & 63, sub = lane >> 3, g = group(), me = member(), lr = lane & 15, kq = lane >> 4, n = kb1 - kb0;
    constexpr int XW = 2 * XS, E = 2 * (XS + WS);
    const uint8_t *const rows = (g ? w_rows : x_rows) + (size_t)kb0 * 128;
    const int row_ld = g ? w_ld : x_ld, last = (g ? w_count : min(tokens, BM)) - 1, piece = ((lane & 7) ^ sub) * 16;
    auto copy = [&](int b, int base, int i) {
      int r = sub;
      if constexpr (RI == 4) asm volatile("" : "+v"(r));  // places are worked out where they are used: eight of them do not fit the registers
      copy16(rows + (size_t)b * 128, __umul24(min((i * 4 + me) * 8 + r, last), row_ld) + piece, __builtin_amdgcn_readfirstlane(lds0 + base + (i * 4 + me) * 1024));
    };
    auto copy_exps = [&](int chunk) {  // by group 0; with fewer than four kilobytes some of them twice
#pragma unroll
      for (int i = 0; i < (RI + 1) / 2; ++i) {
        const int at = ((i * 4 + me) & (2 * RI - 1)) * 1024, byte = at + lane * 16;
        kx_copy16_to_lds(exps(min(kb0 + chunk * AHEAD + byte / BM, kb1 - 1)) + byte % BM, __builtin_amdgcn_readfirstlane(lds0 + E + (chunk & 1) * ES + at));
      }
    };
    const uint8_t *const xs = lds + (me * (16 * RI) + lr) * 128, *const ws = lds + XW + (g * 128 + lr) * 128;
    const uint8_t *const es = lds + E + me * (16 * RI) / 64 * 64 + (EXACT ? kq * 16 : lr * 4);
    const int shift = me * RI % 4 * 8;
    const __attribute__((address_space(4))) float *const sc = (const __attribute__((address_space(4))) float *)(uintptr_t)scales;
    const int p[2] = {(kq ^ (lr & 7)) * 16, ((4 + kq) ^ (lr & 7)) * 16};
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j) acc[i][j] = Block{0.0f, 0.0f, 0.0f, 0.0f};
    i8v x[MI], w[NI];
    uint32_t ex[EXACT ? 4 : 1];
    float scale = 0.0f;
    auto read = [&](int q, int xo, int wo) {
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const i4v u = *(const i4v *)(xs + xo + p[q] + i * 2048);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i][4 * q + e] = u[e];
      }
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const i4v u = *(const i4v *)(ws + wo + p[q] + j * 2048);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[j][4 * q + e] = u[e];
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    auto read_scales = [&](int b) {
      const uint8_t *const at = es + (b / AHEAD & 1) * ES + b % AHEAD * BM;
      if constexpr (EXACT) {
#pragma unroll
        for (int v = 0; v < 4; ++v) ex[v] = *(const uint32_t *)(at + v * 4);
      } else {
        ex[0] = *(const uint32_t *)at;
      }
      scale = sc[kb0 + b];
    };
    // A turn's products lie between empty statements that take its operands and its sums: the compiler orders products, which touch no memory, as it likes, and
    // had most of them behind the barrier that ends the turn, where the other group's are (2.6 us a block of a 256 x 256 tile with few bits set, 2.0 of random ones since).
    auto multiply = [&]() {
#pragma unroll
      for (int i = 0; i < MI; ++i) asm volatile("" : "+v"(x[i]));
#pragma unroll
      for (int j = 0; j < NI; ++j) asm volatile("" : "+v"(w[j]));
      if constexpr (EXACT) {
        float f[MI][4];
        Half xh[MI];
#pragma unroll
        for (int i = 0; i < MI; ++i) {
#pragma unroll
          for (int v = 0; v < 4; ++v) f[i][v] = scale * power(ex[v] >> shift >> 8 * i & 0xffu);
          xh[i] = halves(x[i]);
        }
#pragma unroll
        for (int j = 0; j < NI; ++j) {
          const Half wh = halves(w[j]);
#pragma unroll
          for (int i = 0; i < MI; ++i) {
            const f4 s = block16(xh[i], wh);
#pragma unroll
            for (int v = 0; v < 4; ++v) acc[i][j][v] = __builtin_fmaf(s[v], f[i][v], acc[i][j][v]);
          }
        }
      } else {
        constexpr int N = MI * NI, LAG = 2;
        const int e = (int)(ex[0] >> shift);
        f4 s[LAG + 1];
#pragma unroll
        for (int k = 0; k < N + LAG; ++k) {
          if (k < N) s[k % (LAG + 1)] = block8<true>(x[k / NI], w[k % NI], k / NI, e);
          if (k >= LAG) {
            const int d = k - LAG;
#pragma unroll
            for (int v = 0; v < 4; ++v) acc[d / NI][d % NI][v] = __builtin_fmaf(s[d % (LAG + 1)][v], scale, acc[d / NI][d % NI][v]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) asm volatile("" : "+v"(acc[i][j]));
      __builtin_amdgcn_sched_barrier(0);
    };
    if (g == 0) {
      copy_exps(0);
#pragma unroll
      for (int i = 0; i < 2 * RI; ++i) copy(0, 0, i);
      kx_wait_copies<0>();
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) copy(0, XW, i);
      if (n > 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) copy(1, XW + WS, i);
        kx_wait_copies<4>();
      } else {
        kx_wait_copies<0>();
      }
    }
    turn();
    if (g == 1) turn();
    for (int b = 0; b < n; ++b) {
      const int at = b & 1, other = at ^ 1;
      if (g == 0 && b % AHEAD == 0 && b + AHEAD < n) copy_exps(b / AHEAD + 1);
      read_scales(b);
      read(0, at * XS, at * WS);
      if (b + 1 < n) {
        if (g == 0) {
#pragma unroll
          for (int i = 0; i < RI; ++i) copy(b + 1, other * XS, i);
        } else {
#pragma unroll
          for (int i = 4; i < 8; ++i) copy(b + 1, XW + other * WS, i);
        }
      }
      read(1, at * XS, at * WS);
      if (g == 0) {
        if (b + 1 < n)
#pragma unroll
          for (int i = RI; i < 2 * RI; ++i) copy(b + 1, other * XS, i);
      } else if (b + 2 < n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) copy(b + 2, XW + at * WS, i);
        kx_wait_copies<8>();  // group 0's half of block b + 1, asked for a block ago, has come
      } else {
        kx_wait_copies<0>();
      }
      turn();
      multiply();
      if (g == 1 && b + 2 < n) kx_wait_copies<4>();  // its own half of block b + 1
      else kx_wait_copies<0>();
      turn();
    }
    if (g == 0) turn();
  }
};

}  // namespace kxfp8

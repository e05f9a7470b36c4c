// kx_fp8.h -- products with matrices of 8-bit elements that have a scale for each block of 128 x 128 (kx_fp8.hip).  No counterpart in the
// reference, whose matrices are bf16 or 4-bit (src/kimi_exec.cu:272-323).
//
//   y[t][r] = sum over blocks b of 128 columns of  w_scale[r / 128][b] * 2^e[t][b] * sum of the block's x codes times w codes
// with e[t][b] the least whole number from -100 on that keeps the largest magnitude of row t's block within 448 * 2^e, and the x codes
// x / 2^e rounded to e4m3.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

struct KxFp8Args {
  const uint8_t *w = nullptr;       // e4m3 [rows][ld], zero beyond cols
  const float *w_scale = nullptr;   // [ceil(rows / 128)][blocks]
  const void *x = nullptr;          // [tokens][x_ld] float or bf16
  void *out = nullptr;              // [tokens][out_ld] float or bf16
  int tokens = 0, rows = 0, cols = 0, ld = 0, x_ld = 0, out_ld = 0;
  bool x_f32 = false, out_f32 = false;
  int blocks = 0;                   // of 128 columns
  uint8_t *xc = nullptr;            // scratch: codes [tokens][blocks * 128]
  uint8_t *xe = nullptr;            // scratch: e + 127, [blocks][groups of 64 tokens][64] (kxfp8::exponent_at)
  int groups = 0;                   // of 64 tokens, a multiple of 4
  float *part = nullptr;            // scratch: sums of parts, and who has handed his in
  size_t part_floats = 0;
  int *arrived = nullptr;
  int arrivals = 0;
  bool pairs = false;               // two neighbouring bf16 results can be stored together
};
int kx_fp8_launch(const KxFp8Args &a, hipStream_t st);

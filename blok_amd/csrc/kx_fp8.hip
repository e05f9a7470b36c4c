// kx_fp8.hip -- products with matrices of 8-bit elements that have a scale for each block of 128 x 128 (kx_fp8.h).
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies a block of 128 columns of 16 rows and 16 tokens, and takes the tokens' 2^e for nothing; the matrix's scale, any
// float, is one multiplication and addition for each sum of a block.  It adds the products of a block with fewer than 24 bits: 1.4e-5 of a block's sum on
// average (normal codes of three magnitudes), as v_mfma_f32_16x16x32_fp8_fp8 does, a hundredth of what rounding to bf16 is off.  Results in 32 bits
// go through f16, which holds the codes exactly, and v_mfma_f32_16x16x32_f16 at half the rate (6e-9 on the same sums).
#include <algorithm>
#include <memory>
#include <type_traits>
#include "kx_common.h"
#include "kx_fp8.h"
#include "kx_math.h"
#include "kx_paged_place.h"

namespace {

typedef int i8v __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

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

__device__ __forceinline__ h8 unpacked(uint32_t lo, uint32_t hi) {
  const h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)lo, 1.0f, true);
  const h2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)hi, 1.0f, true);
  return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// The sums of a block of 128 columns, 32 of them a lane in two pieces; in 8 bits times the tokens' 2^(e - 127), exactly without it.
struct Piece {
  uint4 a, b;
};
__device__ __forceinline__ f4 block8(const Piece &w, const Piece &x, int e) {
  const i8v u = {(int)w.a.x, (int)w.a.y, (int)w.a.z, (int)w.a.w, (int)w.b.x, (int)w.b.y, (int)w.b.z, (int)w.b.w};
  const i8v v = {(int)x.a.x, (int)x.a.y, (int)x.a.z, (int)x.a.w, (int)x.b.x, (int)x.b.y, (int)x.b.z, (int)x.b.w};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(u, v, f4{0, 0, 0, 0}, 0, 0, 0, 127, 0, e);
}
__device__ __forceinline__ f4 block16(const Piece &w, const Piece &x) {
  f4 p = __builtin_amdgcn_mfma_f32_16x16x32_f16(unpacked(w.a.x, w.a.y), unpacked(x.a.x, x.a.y), f4{0, 0, 0, 0}, 0, 0, 0);
  p = __builtin_amdgcn_mfma_f32_16x16x32_f16(unpacked(w.a.z, w.a.w), unpacked(x.a.z, x.a.w), p, 0, 0, 0);
  p = __builtin_amdgcn_mfma_f32_16x16x32_f16(unpacked(w.b.x, w.b.y), unpacked(x.b.x, x.b.y), p, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(unpacked(w.b.z, w.b.w), unpacked(x.b.z, x.b.w), p, 0, 0, 0);
}

// Rows of x as codes and exponents: half a wave has a block of 128 columns, 4 of them a lane.
__global__ void __launch_bounds__(256) fp8_rows_k(KxFp8Args a) {
  const long item = (long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31, t = (int)(item / a.blocks), b = (int)(item % a.blocks), c = b * 128 + lane * 4;
  if (t >= a.tokens) return;
  const size_t row = (size_t)t * a.x_ld;
  float v[4];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = c + i < a.cols ? element(a.x, row + c + i, a.x_f32) : 0.0f;
    m = max(m, magnitude(v[i]));
  }
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
  const int e = kxpage::exponent_of(m);
  *(uint32_t *)(a.xc + (size_t)t * a.blocks * 128 + c) = codes4(v[0], v[1], v[2], v[3], kx_bits_f32(kxpage::scale_bits(-e)));
  if (lane == 0) a.xe[(size_t)t * ((a.blocks + 3) & ~3) + b] = (uint8_t)(e + 127);
}

// 16 rows of the matrix times 16 CT tokens a workgroup, its waves the blocks of columns in turn; their sums are added in LDS.
template <int CT, int NW, bool F32>
__global__ void __launch_bounds__(NW * 64) fp8_skinny_k(KxFp8Args a) {
  __shared__ f4 sums[NW][CT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lq = lane >> 4;
  const int r0 = blockIdx.x * 16, t0 = blockIdx.y * 16 * CT, xld = a.blocks * 128, eld = (a.blocks + 3) & ~3;
  const uint8_t *const w = a.w + (size_t)min(r0 + lr, a.rows - 1) * a.ld + lq * 16;
  const float *const ws = a.w_scale + (size_t)(r0 / 128) * a.blocks;
  f4 acc[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) acc[c] = f4{0, 0, 0, 0};
  for (int b = wave; b < a.blocks; b += NW) {
    const Piece wp = {*(const uint4 *)(w + b * 128), *(const uint4 *)(w + b * 128 + 64)};
    const float s = ws[b];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const int t = min(t0 + c * 16 + lr, a.tokens - 1), e = a.xe[(size_t)t * eld + b];
      const uint8_t *const x = a.xc + (size_t)t * xld + b * 128 + lq * 16;
      const Piece xp = {*(const uint4 *)x, *(const uint4 *)(x + 64)};
      const f4 p = F32 ? block16(wp, xp) : block8(wp, xp, e);
      const float f = F32 ? s * kx_bits_f32((uint32_t)e << 23) : s;
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[c][i] = __builtin_fmaf(p[i], f, acc[c][i]);
    }
  }
#pragma unroll
  for (int c = 0; c < CT; ++c) sums[wave][c][lane] = acc[c];
  __syncthreads();
  for (int i = threadIdx.x; i < CT * 64; i += NW * 64) {
    f4 y = {0, 0, 0, 0};
#pragma unroll
    for (int v = 0; v < NW; ++v) y += sums[v][i >> 6][i & 63];
    const int t = t0 + (i >> 6) * 16 + (i & 15), r = r0 + (i >> 4 & 3) * 4;
    if (t >= a.tokens) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (r + e < a.rows) {
        if constexpr (F32) ((float *)a.out)[(size_t)t * a.out_ld + r + e] = y[e];
        else ((uint16_t *)a.out)[(size_t)t * a.out_ld + r + e] = kx_bf16_rne(y[e]);
      }
  }
}

}  // namespace

int kx_fp8_launch(const KxFp8Args &a, hipStream_t st) {
  fp8_rows_k<<<(unsigned)(((long)a.tokens * a.blocks + 7) / 8), 256, 0, st>>>(a);
  KX_LAUNCH_CHECK();
  auto skinny = [&](auto f32) {
    if (a.tokens <= 16) fp8_skinny_k<1, 8, f32()><<<dim3(kx_cdiv(a.rows, 16)), 512, 0, st>>>(a);
    else fp8_skinny_k<4, 4, f32()><<<dim3(kx_cdiv(a.rows, 16), kx_cdiv(a.tokens, 64)), 256, 0, st>>>(a);
  };
  if (a.out_f32) skinny(std::true_type());
  else skinny(std::false_type());
  KX_LAUNCH_CHECK();
  return KX_OK;
}

// ---- the operator of the C ABI ----------------------------------------------------------------------------------------------------------
struct kx_fp8 {
  int max_tokens = 0, max_blocks = 0, device = 0;
  uint8_t *mem = nullptr;
};
extern "C" int kx_fp8_create(int32_t max_tokens, int32_t max_cols, kx_fp8 **out) {
  KX_REQUIRE(out, "kx_fp8_create: null argument");
  *out = nullptr;
  KX_REQUIRE(max_tokens > 0 && max_cols > 0 && max_tokens <= 1 << 24 && max_cols <= 1 << 24, "kx_fp8_create: max_tokens=%d max_cols=%d", max_tokens, max_cols);
  return kx_guard("kx_fp8_create", [&]() -> int {
    std::unique_ptr<kx_fp8> p(new kx_fp8());
    p->max_tokens = max_tokens;
    p->max_blocks = kx_cdiv(max_cols, 128);
    KX_HIP(hipGetDevice(&p->device));
    const size_t bytes = (size_t)max_tokens * (p->max_blocks * 128 + ((p->max_blocks + 3) & ~3));
    if (hipMalloc((void **)&p->mem, bytes) != hipSuccess) {
      kx_set_error("kx_fp8_create: no device memory for %zu bytes", bytes);
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
  KxFp8Args a;
  a.blocks = kx_cdiv(x->cols, 128);
  KX_REQUIRE(x->ld % 128 == 0 && x->ld >= a.blocks * 128 && x->x_ld >= x->cols && x->out_ld >= x->rows, "kx_fp8_run: ld=%d x_ld=%d out_ld=%d", x->ld, x->x_ld, x->out_ld);
  const size_t xs = x->x_f32 ? 4 : 2, os = x->out_f32 ? 4 : 2;
  KX_REQUIRE((uintptr_t)x->d_w % 16 == 0 && (uintptr_t)x->d_w_scale % 4 == 0 && (uintptr_t)x->d_x % xs == 0 && (uintptr_t)x->d_out % os == 0, "kx_fp8_run: the matrix begins at a multiple of 16 bytes, rows at one of an element");
  int dev = -1;
  KX_HIP(hipGetDevice(&dev));
  KX_REQUIRE(dev == p->device, "kx_fp8_run: made on device %d, called on device %d", p->device, dev);
  if (!x->tokens) return KX_OK;
  a.w = (const uint8_t *)x->d_w; a.w_scale = x->d_w_scale; a.x = x->d_x; a.out = x->d_out;
  a.tokens = x->tokens; a.rows = x->rows; a.cols = x->cols; a.ld = x->ld; a.x_ld = x->x_ld; a.out_ld = x->out_ld;
  a.x_f32 = x->x_f32 != 0; a.out_f32 = x->out_f32 != 0;
  a.xc = p->mem;
  a.xe = p->mem + (size_t)p->max_tokens * p->max_blocks * 128;
  return kx_fp8_launch(a, kx_stream(stream));
}

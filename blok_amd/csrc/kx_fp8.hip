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

__device__ __forceinline__ i8v piece(const uint8_t *at) {  // a lane's 32 codes of a block, in two pieces
  const uint4 a = *(const uint4 *)at, b = *(const uint4 *)(at + 64);
  return i8v{(int)a.x, (int)a.y, (int)a.z, (int)a.w, (int)b.x, (int)b.y, (int)b.z, (int)b.w};
}

// Rows of x as codes and exponents: 16 lanes have a block of 128 columns, 8 of them each; VECTOR: rows of whole 16-byte pieces at multiples of 16.
template <bool F32, bool VECTOR>
__global__ void __launch_bounds__(256) fp8_rows_k(KxFp8Args a) {
  const int lane = threadIdx.x & 15, b = blockIdx.x * 16 + (threadIdx.x >> 4), c = b * 128 + lane * 8;
  if (b >= a.blocks) return;
  for (int t = blockIdx.y; t < a.tokens; t += gridDim.y) {
    const size_t row = (size_t)t * a.x_ld;
    float v[8];
    if (VECTOR && c + 8 <= a.cols) {
      if constexpr (F32) {
        const float4 *const p = (const float4 *)((const float *)a.x + row + c);
        const float4 u = p[0], w = p[1];
        v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w, v[4] = w.x, v[5] = w.y, v[6] = w.z, v[7] = w.w;
      } else {
        const uint4 u = *(const uint4 *)((const uint16_t *)a.x + row + c);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[2 * i] = kx_bits_f32(w[i] << 16);
          v[2 * i + 1] = kx_bits_f32(w[i] & 0xffff0000u);
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = c + i < a.cols ? element(a.x, row + c + i, F32) : 0.0f;
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, magnitude(v[i]));
#pragma unroll
    for (int d = 8; d >= 1; d >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, d));
    const int e = kxpage::exponent_of(m);
    const float inverse = kx_bits_f32(kxpage::scale_bits(-e));
    *(uint2 *)(a.xc + (size_t)t * a.blocks * 128 + c) = make_uint2(codes4(v[0], v[1], v[2], v[3], inverse), codes4(v[4], v[5], v[6], v[7], inverse));
    if (lane == 0) a.xe[exponent_at(b, t, a.groups)] = (uint8_t)(e + 127);
  }
}

// 16 rows of the matrix times 16 CT tokens a workgroup, its waves the blocks of columns in turn; their sums are added in LDS.
template <int CT, int NW, bool F32>
__global__ void __launch_bounds__(NW * 64) fp8_skinny_k(KxFp8Args a) {
  __shared__ f4 sums[NW][CT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lr = lane & 15, lq = lane >> 4;
  const int r0 = blockIdx.x * 16, t0 = blockIdx.y * 16 * CT, xld = a.blocks * 128;
  const uint8_t *const w = a.w + (size_t)min(r0 + lr, a.rows - 1) * a.ld + lq * 16;
  const float *const ws = a.w_scale + (size_t)(r0 / 128) * a.blocks;
  f4 acc[CT];
#pragma unroll
  for (int c = 0; c < CT; ++c) acc[c] = f4{0, 0, 0, 0};
  for (int b = wave; b < a.blocks; b += NW) {
    const i8v wp = piece(w + b * 128);
    const uint32_t e = *(const uint32_t *)(a.xe + exponent_at(b, t0 + lr, a.groups));
    const float s = ws[b];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      const i8v xp = piece(a.xc + (size_t)min(t0 + c * 16 + lr, a.tokens - 1) * xld + b * 128 + lq * 16);
      const f4 p = F32 ? block16(halves(wp), halves(xp)) : block8<false>(wp, xp, c, (int)e);
      const float f = F32 ? s * power(e >> 8 * c & 0xffu) : s;
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
  static std::atomic<bool> attr{false};  // setting it twice from two threads is harmless
  if (!attr) {
    KX_HIP(hipFuncSetAttribute((const void *)fp8_tile_k<RI, F32>, hipFuncAttributeMaxDynamicSharedMemorySize, TL::LDS));
    attr = true;
  }
  fp8_tile_k<RI, F32><<<dim3(share.grid(kx_cdiv(a.tokens, TL::BM) * kx_cdiv(a.rows, TL::BN))), TL::THREADS, TL::LDS, st>>>(a, share);
  KX_LAUNCH_CHECK();
  return KX_OK;
}
// The tile that is sooner by estimates in us, and how it is shared out: rounds of one workgroup per CU, and for parts of the columns what handing over their sums takes.
// us, tiles of 256 / 128 / 64 tokens: 2048 x 18432 x 7168 323 / 346 / 523, 2048 x 7168 x 8192 143 / 166 / 246, 2048 x 2112 x 7168 89 / 86 / 89, 1024 x 12288 x 1536 42 / 47 /
// 51, 512 x 7168 x 8192 80 / 58 / 59, 256 x 7168 x 2048 53 / 34 / 22, 128 x 18432 x 7168 77 / 56 / 61, 128 x 7168 x 8192 94 / 47 / 30, 96 x 2112 x 7168 81 / 42 / 25; 32-bit
// results 2048 x 7168 x 8192 - / 288 / 349, 333 x 4103 x 2000 - / 37 / 31.
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

int kx_fp8_launch(const KxFp8Args &a, hipStream_t st) {
  const bool vector = (uintptr_t)a.x % 16 == 0 && (size_t)a.x_ld * (a.x_f32 ? 4 : 2) % 16 == 0;
  const dim3 rows(kx_cdiv(a.blocks, 16), std::min(a.tokens, 65535));
  if (a.x_f32) vector ? fp8_rows_k<true, true><<<rows, 256, 0, st>>>(a) : fp8_rows_k<true, false><<<rows, 256, 0, st>>>(a);
  else vector ? fp8_rows_k<false, true><<<rows, 256, 0, st>>>(a) : fp8_rows_k<false, false><<<rows, 256, 0, st>>>(a);
  KX_LAUNCH_CHECK();
  if (a.tokens > 64) return a.out_f32 ? tiles<true>(a, st) : tiles<false>(a, st);
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
  KxFp8Args a;
  int max_tokens = 0, max_blocks = 0, device = 0;
  uint8_t *mem = nullptr;
};
// sums of parts for a tile of 256 x 256 on each of 256 CUs
static constexpr size_t FP8_PARTS = (size_t)256 * 256 * 256;
static constexpr int FP8_ARRIVALS = 256;

extern "C" int kx_fp8_create(int32_t max_tokens, int32_t max_cols, kx_fp8 **out) {
  KX_REQUIRE(out, "kx_fp8_create: null argument");
  *out = nullptr;
  KX_REQUIRE(max_tokens > 0 && max_cols > 0 && max_tokens <= 1 << 22 && max_cols < 1 << 23, "kx_fp8_create: max_tokens=%d max_cols=%d", max_tokens, max_cols);
  return kx_guard("kx_fp8_create", [&]() -> int {
    std::unique_ptr<kx_fp8> p(new kx_fp8());
    p->max_tokens = max_tokens;
    p->max_blocks = kx_cdiv(max_cols, 128);
    KX_HIP(hipGetDevice(&p->device));
    const size_t groups = (size_t)kx_cdiv(max_tokens, 256) * 4;
    size_t at = 0;
    auto take = [&](size_t n) { const size_t from = at; at += (n + 255) & ~(size_t)255; return from; };
    const size_t xc = take((size_t)max_tokens * p->max_blocks * 128), xe = take(groups * 64 * p->max_blocks), arrived = take(FP8_ARRIVALS * 4), part = take(max_tokens > 64 ? FP8_PARTS * 4 : 0);
    if (hipMalloc((void **)&p->mem, at) != hipSuccess) {
      kx_set_error("kx_fp8_create: no device memory for %zu bytes", at);
      return KX_ERR_HIP;
    }
    p->a.xc = p->mem + xc;
    p->a.xe = p->mem + xe;
    p->a.arrived = (int *)(p->mem + arrived);
    p->a.part = (float *)(p->mem + part);
    p->a.arrivals = FP8_ARRIVALS;
    p->a.part_floats = max_tokens > 64 ? FP8_PARTS : 0;
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

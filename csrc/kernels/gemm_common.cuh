// Pieces shared by the one-CTA and the CTA-pair grouped GEMM kernels: tile walk and epilogues.
#pragma once
#include "api.h"
#include "sm100_ptx.cuh"
#include "tile_walker.h"

namespace fastb {
namespace gemm {

constexpr int BN = 256, BK = 64, UMMA_K = 16;

static_assert(BK == kWalkBK, "the tile walker counts reduction steps of BK");

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&v);
}
// What pack_bf16 takes from the two, as bf16: both together have 16 bits of a value. An infinity leaves nothing.
__device__ __forceinline__ uint32_t pack_rest(float a, float b) {
  const float x = __bfloat162float(__float2bfloat16_rn(a)), y = __bfloat162float(__float2bfloat16_rn(b));
  return pack_bf16(fabsf(x) < INFINITY ? a - x : 0.0f, fabsf(y) < INFINITY ? b - y : 0.0f);
}
// 1 / (1 + exp(-x)) and x times that. Built with --use_fast_math (FASTB_FAST_MATH): two operations of the special-function unit; a division, approximate
// too, takes more of them, for divisors above 2^126, whose reciprocal is zero anyway. Built without: the rounded division.
#ifdef FASTB_FAST_MATH
__device__ __forceinline__ float sigmoid(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + __expf(-x)));
  return r;
}
__device__ __forceinline__ float silu(float x) { return x * sigmoid(x); }
#else
__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + __expf(-x)); }
__device__ __forceinline__ float silu(float x) { return x / (1.0f + __expf(-x)); }
#endif
// max(x, 0); NaN stays NaN (fmaxf would make it 0, and a diverged row look healthy).
__device__ __forceinline__ float relu(float x) {
  float r;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(x));
  return r;
}
// The normal distribution's tail: Phi(-|z|) = e q, e = exp(-z^2 / 2). q is half the scaled complementary error function of |z| / sqrt(2), here t times a polynomial of
// t = 1 / (1 + a |z|), the form of Abramowitz and Stegun, Handbook of Mathematical Functions, 7.1.26. Its coefficients were fitted for the least RELATIVE error (a linear
// programme over 6000 points up to |z| = 13.6, where e ends): 4.2e-6 in fp32 arithmetic, so that far negative values are rounded once too. (The handbook's, fitted for the
// absolute error, are 1 % off at z = -8 and 2 % at -10.) The exponential serves the density as well. (The general error function made the activation's
// backward pass a matter of arithmetic: 294 us for 8192 x 14336, where memory wants 107.)
__device__ __forceinline__ float normal_tail(float z) {
  const float t = __fdividef(1.0f, fmaf(0.308298558f, fabsf(z), 1.0f));
  return t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, -0.0752880722f, 0.188464284f), 0.00832129549f), 0.13617529f), 0.119090386f), 0.123234853f);
}
// z Phi(z) and its derivative. Of a far negative z the tail is multiplied by z before the exponential, which alone is down at the smallest normal numbers there.
__device__ __forceinline__ float gelu(float z) {
  const float e = __expf(-0.5f * z * z), q = normal_tail(z);
  return z < 0.0f ? z * q * e : z * fmaf(-q, e, 1.0f);
}
__device__ __forceinline__ float gelu_slope(float z) {
  const float e = __expf(-0.5f * z * z), q = normal_tail(z), d = 0.39894228f * z;
  return z < 0.0f ? e * (d + q) : fmaf(e, d - q, 1.0f);
}
__device__ __forceinline__ uint4 pack8(const uint32_t* r) {
  return make_uint4(pack_bf16(__uint_as_float(r[0]), __uint_as_float(r[1])), pack_bf16(__uint_as_float(r[2]), __uint_as_float(r[3])),
                    pack_bf16(__uint_as_float(r[4]), __uint_as_float(r[5])), pack_bf16(__uint_as_float(r[6]), __uint_as_float(r[7])));
}

// One thread = one output row: reads its 256 fp32 accumulators from TMEM (t_row = TMEM address of
// the row's first column) and writes bf16 to global. `zero` writes zeros without touching TMEM.
__device__ __forceinline__ void epilogue_store_row(__nv_bfloat16* crow, uint32_t t_row, bool zero) {
#pragma unroll 1
  for (int c = 0; c < BN / 32; ++c) {
    uint32_t r[32];
    if (!zero) { ptx::tmem_ld_32x32(t_row + c * 32, r); ptx::tmem_wait_ld(); }
    else {
#pragma unroll
      for (int i = 0; i < 32; ++i) r[i] = 0;
    }
    uint4* dst = reinterpret_cast<uint4*>(crow + c * 32);
#pragma unroll
    for (int q = 0; q < 4; ++q) dst[q] = pack8(r + 8 * q);
  }
}

// The same as fp32 sums, [64 groups of four columns][128 rows]: `at` is row r of the first group. A warp's stores are contiguous; row by row in global memory
// every one of them touched 32 lines.
__device__ __forceinline__ void epilogue_sums(float4* at, uint32_t t_row, bool zero) {
#pragma unroll 1
  for (int c = 0; c < BN / 32; ++c) {
    uint32_t r[32];
    if (!zero) { ptx::tmem_ld_32x32(t_row + c * 32, r); ptx::tmem_wait_ld(); }
    else {
#pragma unroll
      for (int i = 0; i < 32; ++i) r[i] = 0;
    }
#pragma unroll
    for (int q = 0; q < 8; ++q)
      __stcg(at + (c * 8 + q) * 128, make_float4(__uint_as_float(r[4 * q]), __uint_as_float(r[4 * q + 1]), __uint_as_float(r[4 * q + 2]), __uint_as_float(r[4 * q + 3])));
  }
}

// SwiGLU: the 256 columns of a tile are [128 gate | 128 up] of the same 128 features.
__device__ __forceinline__ void epilogue_swiglu_row(__nv_bfloat16* arow, __nv_bfloat16* gurow, uint32_t t_row) {
#pragma unroll 1
  for (int c = 0; c < BN / 64; ++c) {
    uint32_t g[32], u[32];
    ptx::tmem_ld_32x32(t_row + c * 32, g);
    ptx::tmem_ld_32x32(t_row + BN / 2 + c * 32, u);
    ptx::tmem_wait_ld();
    uint4* dst = reinterpret_cast<uint4*>(arow + c * 32);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float o[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = silu(__uint_as_float(g[8 * q + i])) * __uint_as_float(u[8 * q + i]);
      dst[q] = make_uint4(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]), pack_bf16(o[4], o[5]), pack_bf16(o[6], o[7]));
    }
    if (gurow) {
      uint4* dg = reinterpret_cast<uint4*>(gurow + c * 32);
      uint4* du = reinterpret_cast<uint4*>(gurow + BN / 2 + c * 32);
#pragma unroll
      for (int q = 0; q < 4; ++q) { dg[q] = pack8(g + 8 * q); du[q] = pack8(u + 8 * q); }
    }
  }
}

}  // namespace gemm
}  // namespace fastb

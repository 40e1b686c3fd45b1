// Rows in e4m3 with one fp32 scale per 128 elements, as the dispatch sends them.
#pragma once
#include <cuda_fp8.h>
#include <cuda_runtime.h>

namespace fastb {

// Scale of 128 elements whose largest magnitude is amax: amax / 448 rounded UP to the next value a bf16 can hold. Quantised values still fit
// e4m3, and a receiver that multiplies in bf16 (the expert GEMM's converter warps) reproduces value x scale without a second rounding.
__device__ __forceinline__ float e4m3_scale(float amax) {
  return __uint_as_float((__float_as_uint(fmaxf(amax, 1e-12f) * (1.0f / 448.0f)) + 0xFFFFu) & 0xFFFF0000u);
}
// inv = 1 / scale
__device__ __forceinline__ unsigned short e4m3_pair(float a, float b, float inv) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a * inv, b * inv), __NV_SATFINITE, __NV_E4M3);
}

}  // namespace fastb

// Tensor maps of bf16 matrices for TMA loads and stores.
#pragma once
#include <cuda.h>

#include "py_types.h"

namespace fastb_py {

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                   const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                   CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_tiled() {
  static EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    cuda_check(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q), "cudaGetDriverEntryPoint");
    TORCH_CHECK(p != nullptr && q == cudaDriverEntryPointSuccess, "cuTensorMapEncodeTiled is not available in this driver");
    return reinterpret_cast<EncodeTiledFn>(p);
  }();
  return fn;
}

inline CUtensorMap bf16_map(int rank, int64_t ptr, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box, CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B) {
  TORCH_CHECK(ptr % 16 == 0, "tensor map base must be 16-byte aligned");
  for (int i = 0; i + 1 < rank; ++i) TORCH_CHECK(strides[i] % 16 == 0, "tensor map strides must be multiples of 16 bytes");
  alignas(64) CUtensorMap m;
  cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const auto encode = [&] {
    return encode_tiled()(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, reinterpret_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = encode();
  if (r == CUDA_ERROR_INVALID_CONTEXT) {   // a thread that has called the driver for nothing else yet, as the autograd engine's may be
    int dev = 0;
    cuda_check(cudaGetDevice(&dev), "cudaGetDevice");
    cuda_check(cudaSetDevice(dev), "cudaSetDevice");
    r = encode();
  }
  TORCH_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed with code ", static_cast<int>(r));
  return m;
}
inline CUtensorMap bf16_map_2d(const torch::Tensor& t, int box_rows) {
  TORCH_CHECK(t.is_cuda() && t.scalar_type() == torch::kBFloat16 && t.dim() == 2 && t.stride(1) == 1, "expected a CUDA bf16 matrix with contiguous rows");
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(t.size(1)), static_cast<cuuint64_t>(t.size(0))}, strides[1] = {static_cast<cuuint64_t>(t.stride(0)) * 2};
  const cuuint32_t box[2] = {64u, static_cast<cuuint32_t>(box_rows)};
  return bf16_map(2, reinterpret_cast<int64_t>(t.data_ptr()), dims, strides, box);
}

}  // namespace fastb_py

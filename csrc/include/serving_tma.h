// Tensor maps of the serving operators (host): any rank, any swizzle.
#pragma once

#include "tma_host.h"

namespace raiccl {

// dims / box innermost first; strides[i] is the byte stride of dims[i + 1].
inline CUtensorMap make_tmap(const void* base, bool bf16, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                             const cuuint32_t* box, CUtensorMapSwizzle swizzle) {
  const cuuint32_t ones[5] = {1, 1, 1, 1, 1};
  CUtensorMap map;
  const CUresult r = tensor_map_encoder()(
      &map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, rank, const_cast<void*>(base), dims,
      strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw std::runtime_error("cuTensorMapEncodeTiled failed with code " + std::to_string((int)r));
  return map;
}

}  // namespace raiccl

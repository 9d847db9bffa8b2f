// Host side of the TMA descriptors: the driver's encoder, found without linking libcuda
// (the library must load on hosts without a driver).
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace grinqh {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn tmap_encoder() {
  static const EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
                    q == cudaDriverEntryPointSuccess;
    return ok ? reinterpret_cast<EncodeTiledFn>(p) : nullptr;
  }();
  return fn;
}

// 16-bit heads [tokens, heads, dim] (strides in elements) as boxes of 64 channels x
// `box_heads` x `box_tokens`, 128-byte swizzle; tokens past the end read as zero.
inline int tmap_heads(CUtensorMap* map, bool bf16, const void* base, int64_t tokens, int64_t heads, int64_t dim,
                      int64_t token_stride, int64_t head_stride, uint32_t box_heads, uint32_t box_tokens,
                      const char* what) {
  const EncodeTiledFn enc = tmap_encoder();
  if (!enc) return set_error(GRINQH_ERR_CUDA, "cuTensorMapEncodeTiled is unavailable");
  // a stride that no index is multiplied with may hold anything
  if (heads == 1) head_stride = dim;
  if (tokens == 1) token_stride = heads * dim;
  GRINQH_REQUIRE(head_stride > 0 && token_stride > 0, "the strides of %s must be positive (got %lld, %lld)", what,
                 (long long)token_stride, (long long)head_stride);
  const cuuint64_t gdim[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)tokens};
  const cuuint64_t gstride[2] = {(cuuint64_t)head_stride * 2, (cuuint64_t)token_stride * 2};
  const cuuint32_t box[3] = {64, box_heads, box_tokens}, step[3] = {1, 1, 1};
  const CUresult r = enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                         const_cast<void*>(base), gdim, gstride, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return set_error(GRINQH_ERR_INVALID, "cuTensorMapEncodeTiled(%s) failed (%d)", what, (int)r);
  return GRINQH_OK;
}

}  // namespace grinqh

// Host-side TMA tensor-map encoding (cuTensorMapEncodeTiled through the runtime's driver entry
// point, so the library links against the CUDA runtime only).
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace yb {

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn tmap_encode_fn() {
  static EncodeTiledFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return (EncodeTiledFn) nullptr;
    return reinterpret_cast<EncodeTiledFn>(p);
  }();
  return fn;
}

// Row-major fp16 matrix [rows][cols] read in boxes of box_rows x box_cols elements (box_cols * 2
// <= 128 bytes) with the 128-byte swizzle; rows beyond the matrix read as zeros.
inline bool tmap_f16_2d_sw128(CUtensorMap* m, const __half* base, long long rows, int cols, int box_cols,
                              int box_rows) {
  EncodeTiledFn enc = tmap_encode_fn();
  if (!enc || box_cols * 2 > 128) return false;
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)cols * 2};
  const cuuint32_t box[2] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<__half*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// 3-D fp16 or bf16 tensor, dims and box innermost first (box[0] * 2 <= 128 bytes, 128-byte swizzle),
// strides in elements of the two outer dimensions; elements outside read as zeros.
inline bool tmap_16_3d_sw128(CUtensorMap* m, const void* base, bool bf16, const long long (&dim)[3],
                             const long long (&stride)[2], const int (&box)[3]) {
  EncodeTiledFn enc = tmap_encode_fn();
  if (!enc || box[0] * 2 > 128) return false;
  const cuuint64_t dims[3] = {(cuuint64_t)dim[0], (cuuint64_t)dim[1], (cuuint64_t)dim[2]};
  const cuuint64_t strides[2] = {(cuuint64_t)stride[0] * 2, (cuuint64_t)stride[1] * 2};
  const cuuint32_t b[3] = {(cuuint32_t)box[0], (cuuint32_t)box[1], (cuuint32_t)box[2]};
  const cuuint32_t estr[3] = {1, 1, 1};
  return enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
             const_cast<void*>(base), dims, strides, b, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace yb

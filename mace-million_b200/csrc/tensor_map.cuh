// Tensor maps of row-major matrices for TMA loads (SWIZZLE_128B), encoded by the driver's entry point.
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace mb {

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
inline EncodeTiled encode_tiled() {
  static EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      p = nullptr;
    return (EncodeTiled)p;
  }();
  return fn;
}

// Map of a tensor of `rank` (at most 4) dimensions (inner to outer), strides of the outer ones and the box in elements of `size` bytes;
// elements outside are zero
inline int tensor_map(const char* who, CUtensorMap* m, CUtensorMapDataType type, int size, int rank, const void* p,
                      const int64_t* dims, const int64_t* strides, const int* box) {
  EncodeTiled enc = encode_tiled();
  if (!enc) {
    set_error("%s: the driver has no cuTensorMapEncodeTiled", who);
    return MB_E_CUDA;
  }
  cuuint64_t d[4], s[3];
  cuuint32_t b[4], es[4] = {1, 1, 1, 1};
  for (int i = 0; i < rank; ++i) {
    d[i] = (cuuint64_t)dims[i];
    b[i] = (cuuint32_t)box[i];
    if (i) s[i - 1] = (cuuint64_t)strides[i - 1] * size;
  }
  const CUresult rc = enc(m, type, rank, const_cast<void*>(p), d, s, b, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (rc != CUDA_SUCCESS) {
    set_error("%s: cuTensorMapEncodeTiled failed (%d)", who, (int)rc);
    return MB_E_CUDA;
  }
  return 0;
}
inline int tensor_map_2d(const char* who, CUtensorMap* m, CUtensorMapDataType type, int size, const void* p, int64_t cols,
                         int64_t rows, int64_t ld, int box_cols, int box_rows) {
  const int64_t dims[2] = {cols, rows}, str[1] = {ld};
  const int box[2] = {box_cols, box_rows};
  return tensor_map(who, m, type, size, 2, p, dims, str, box);
}

}  // namespace mb

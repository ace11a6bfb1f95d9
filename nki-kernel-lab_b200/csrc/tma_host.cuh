// tma_host.cuh - host-side creation of TMA tensor maps (cuTensorMapEncodeTiled),
// reached through the runtime's driver entry-point query so the library needs no
// link-time dependency on libcuda.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace nkl {

inline PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = []() -> PFN_cuTensorMapEncodeTiled_v12000 {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}

// Tiled map over a rank-`rank` bf16 tensor. dims/box are innermost-first; strides
// (bytes) are for dims 1..rank-1. 128-byte swizzle, zero fill out of bounds.
inline int make_tensor_map(CUtensorMap* map, CUtensorMapDataType type, CUtensorMapSwizzle swizzle, const void* base,
                           int rank, const uint64_t* dims, const uint64_t* strides_bytes, const uint32_t* box,
                           const char* what) {
  auto enc = tensor_map_encoder();
  if (!enc) return fail(NKL_ERR_CUDA, "%s: cuTensorMapEncodeTiled unavailable", what);
  uint32_t elem_strides[5] = {1, 1, 1, 1, 1};
  CUresult r = enc(map, type, (cuuint32_t)rank, const_cast<void*>(base), reinterpret_cast<const cuuint64_t*>(dims),
                   reinterpret_cast<const cuuint64_t*>(strides_bytes), reinterpret_cast<const cuuint32_t*>(box),
                   elem_strides, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(NKL_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed (%d)", what, (int)r);
  return NKL_OK;
}

inline int make_tensor_map_bf16(CUtensorMap* map, const void* base, int rank, const uint64_t* dims,
                                const uint64_t* strides_bytes, const uint32_t* box, const char* what) {
  return make_tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, CU_TENSOR_MAP_SWIZZLE_128B, base, rank, dims,
                         strides_bytes, box, what);
}

// The same over bytes: rows of 128 or 64, swizzled over as many.
inline int make_tensor_map_u8(CUtensorMap* map, const void* base, int rank, const uint64_t* dims,
                              const uint64_t* strides_bytes, const uint32_t* box, const char* what) {
  return make_tensor_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8,
                         box[0] == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, base, rank, dims,
                         strides_bytes, box, what);
}

}  // namespace nkl

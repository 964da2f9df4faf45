// The driver's tensor-map encoder, looked up once (the library links no
// libcuda).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <mutex>

namespace laya {

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Null when the driver lacks the entry point.
inline EncodeTiledFn get_encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// False when the driver lacks the encoder or rejects the geometry.
inline bool encode_map(CUtensorMap* m, CUtensorMapDataType type, int rank, const void* ptr, const cuuint64_t* dims,
                       const cuuint64_t* strides, const cuuint32_t* box, CUtensorMapSwizzle swizzle) {
  const cuuint32_t estr[3] = {1, 1, 1};
  EncodeTiledFn enc = get_encode_fn();
  return enc && enc(m, type, rank, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Rows of `esize`-byte elements (1: bytes, 2: bf16, 4: fp32), `ld` elements
// apart: box of 128 bytes x box_rows, 128-byte swizzle.
inline bool rows_map(CUtensorMap* m, const void* ptr, int rows, int cols, long long ld, int esize, int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * esize};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / esize), (cuuint32_t)box_rows};
  const CUtensorMapDataType type = esize == 4   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : esize == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                : CU_TENSOR_MAP_DATA_TYPE_UINT8;
  return encode_map(m, type, 2, ptr, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// [slots][rows][cols] bf16 (the matrices of an adapter pool): box of box_cols x
// box_rows of one slot; whatever lies past the ends reads as zeros.
inline bool slots_map(CUtensorMap* m, const void* ptr, int slots, int rows, int cols, int box_cols, int box_rows,
                      CUtensorMapSwizzle swizzle) {
  const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)slots};
  const cuuint64_t strides[2] = {(cuuint64_t)cols * 2, (cuuint64_t)rows * cols * 2};
  const cuuint32_t box[3] = {(cuuint32_t)box_cols, (cuuint32_t)box_rows, 1};
  return encode_map(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, ptr, dims, strides, box, swizzle);
}

}  // namespace laya

#include "tensor_map.h"

#include <stdexcept>

#include "engine.h"

namespace t0b {
namespace {

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The library does not link against the driver, so that it loads without one.
EncodeTiled Encoder() {
  static const EncodeTiled function = [] {
    void* entry = nullptr;
    cudaDriverEntryPointQueryResult found;
    Check(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &entry, cudaEnableDefault, &found), "tensor map entry point");
    if (found != cudaDriverEntryPointSuccess || entry == nullptr) {
      throw std::runtime_error("the driver has no cuTensorMapEncodeTiled");
    }
    return reinterpret_cast<EncodeTiled>(entry);
  }();
  return function;
}

CUtensorMap Encode(CUtensorMapDataType type, int item, const void* data, int64_t columns, int64_t rows, int64_t depth,
                   int64_t row_stride, int64_t depth_stride, int box_columns, int box_rows) {
  const cuuint64_t sizes[3] = {static_cast<cuuint64_t>(columns), static_cast<cuuint64_t>(rows),
                               static_cast<cuuint64_t>(depth)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(row_stride) * item, static_cast<cuuint64_t>(depth_stride) * item};
  const cuuint32_t boxes[3] = {static_cast<cuuint32_t>(box_columns), static_cast<cuuint32_t>(box_rows), 1};
  const cuuint32_t steps[3] = {1, 1, 1};
  CUtensorMap map;
  const CUresult status = Encoder()(&map, type, depth != 0 ? 3 : 2, const_cast<void*>(data), sizes, strides, boxes,
                                    steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (status != CUDA_SUCCESS) throw std::runtime_error("cuTensorMapEncodeTiled failed");
  return map;
}

}  // namespace

CUtensorMap EncodeHalves(bool bf16, const void* data, int64_t columns, int64_t rows, int64_t depth,
                         int64_t row_stride, int64_t depth_stride, int box) {
  return Encode(bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, data, columns, rows,
                depth, row_stride, depth_stride, 64, box);
}

CUtensorMap EncodeBytes(const void* data, int64_t columns, int64_t rows, int box_columns, int box_rows) {
  return Encode(CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, data, columns, rows, 0, columns, 0, box_columns, box_rows);
}

}  // namespace t0b

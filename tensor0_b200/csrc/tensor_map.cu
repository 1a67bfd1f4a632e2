#include "tensor_map.h"

#include <stdexcept>
#include <string>

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

// sizes and boxes by dimension, innermost first; strides of the outer ones in bytes.
CUtensorMap Encode(CUtensorMapDataType type, const void* data, int rank, const cuuint64_t* sizes,
                   const cuuint64_t* strides, const cuuint32_t* boxes) {
  const cuuint32_t steps[4] = {1, 1, 1, 1};
  CUtensorMap map;
  const auto encode = [&] {
    return Encoder()(&map, type, rank, const_cast<void*>(data), sizes, strides, boxes, steps,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult status = encode();
  if (status == CUDA_ERROR_INVALID_CONTEXT || status == CUDA_ERROR_NOT_INITIALIZED) {
    // A thread that has not used the device: unlike the runtime's functions, the
    // driver's do not make the device's context current themselves.
    int device = 0;
    Check(cudaGetDevice(&device), "current device");
    Check(cudaSetDevice(device), "device context");
    status = encode();
  }
  if (status != CUDA_SUCCESS) throw std::runtime_error("cuTensorMapEncodeTiled failed with error " + std::to_string(status));
  return map;
}

CUtensorMapDataType HalfType(bool bf16) {
  return bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

cuuint64_t Size(int64_t n) { return static_cast<cuuint64_t>(n); }

}  // namespace

CUtensorMap EncodeHalves(bool bf16, const void* data, int64_t columns, int64_t rows, int64_t depth,
                         int64_t row_stride, int64_t depth_stride, int box) {
  const cuuint64_t sizes[3] = {Size(columns), Size(rows), Size(depth)};
  const cuuint64_t strides[2] = {Size(row_stride) * 2, Size(depth_stride) * 2};
  const cuuint32_t boxes[3] = {64, static_cast<cuuint32_t>(box), 1};
  return Encode(HalfType(bf16), data, depth != 0 ? 3 : 2, sizes, strides, boxes);
}

CUtensorMap EncodeBlocks(bool bf16, const void* data, int64_t columns, int64_t rows, int64_t depth,
                         int64_t row_stride, int64_t depth_stride, int box_rows, int box_blocks) {
  const cuuint64_t sizes[4] = {64, Size(rows), Size(columns / 64), Size(depth)};
  const cuuint64_t strides[3] = {Size(row_stride) * 2, 128, Size(depth_stride) * 2};
  const cuuint32_t boxes[4] = {64, static_cast<cuuint32_t>(box_rows), static_cast<cuuint32_t>(box_blocks), 1};
  return Encode(HalfType(bf16), data, depth != 0 ? 4 : 3, sizes, strides, boxes);
}

CUtensorMap EncodeBytes(const void* data, int64_t columns, int64_t rows, int box_columns, int box_rows) {
  const cuuint64_t sizes[2] = {Size(columns), Size(rows)}, strides[1] = {Size(columns)};
  const cuuint32_t boxes[2] = {static_cast<cuuint32_t>(box_columns), static_cast<cuuint32_t>(box_rows)};
  return Encode(CU_TENSOR_MAP_DATA_TYPE_UINT8, data, 2, sizes, strides, boxes);
}

}  // namespace t0b

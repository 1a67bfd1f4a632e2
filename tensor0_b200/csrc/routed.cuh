// Device helpers shared by the routed operators.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <cstddef>
#include <cstdint>
#include <mutex>
#include <utility>

#include "engine.h"

namespace t0b {

// XLA_FFI_DataType codes of the types these operators take.
constexpr int32_t kTypeF16 = 10, kTypeF32 = 11, kTypeBf16 = 16;

__device__ __forceinline__ float ToFloat(float v) { return v; }
__device__ __forceinline__ float ToFloat(__half v) { return __half2float(v); }
__device__ __forceinline__ float ToFloat(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T> __device__ __forceinline__ T FromFloat(float v);
template <> __device__ __forceinline__ float FromFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ __half FromFloat<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 FromFloat<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two floats rounded into one 32-bit word (the first in the low half).
template <typename T> __device__ __forceinline__ uint32_t Pack2(float a, float b) {
  const T lo = FromFloat<T>(a), hi = FromFloat<T>(b);
  return static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(&lo)) |
         (static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(&hi)) << 16);
}
template <> __device__ __forceinline__ uint32_t Pack2<__half>(float a, float b) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t Pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename T> __device__ __forceinline__ float2 Unpack2(uint32_t v);
template <> __device__ __forceinline__ float2 Unpack2<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
template <> __device__ __forceinline__ float2 Unpack2<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

// Eight neighbouring values of a row as floats.  Vector: one 16-byte access
// (p is 16-byte aligned and all eight lie in the row); otherwise value by
// value, `count` of them (the others read as 0 and are not written).
template <typename T, bool Vector>
__device__ __forceinline__ void Load8(const T* p, int count, float (&v)[8]) {
  if constexpr (Vector) {
    if (count <= 0) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = 0.0f;
      return;
    }
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = Unpack2<T>(w[i]);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < count ? ToFloat(p[i]) : 0.0f;
  }
}

template <typename T, bool Vector>
__device__ __forceinline__ void Store8(T* p, int count, const float (&v)[8]) {
  if constexpr (Vector) {
    if (count <= 0) return;
    *reinterpret_cast<uint4*>(p) = make_uint4(Pack2<T>(v[0], v[1]), Pack2<T>(v[2], v[3]), Pack2<T>(v[4], v[5]),
                                              Pack2<T>(v[6], v[7]));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i < count) p[i] = FromFloat<T>(v[i]);
    }
  }
}

// An expert's first row as read from the device, kept inside the rows there are.
__device__ __forceinline__ int64_t RowBound(int32_t offset, int64_t entries) {
  return offset < 0 ? 0 : offset < entries ? offset : entries;
}

// Brief kernels follow one another closely: each lets the next one start (and
// set itself up) while it runs, and waits for the one before it to have ended,
// with its writes, before it touches memory.  Every block of every kernel waits,
// so that a kernel's end implies the end of all before it.
__device__ __forceinline__ void LetNextStart() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void WaitForPrevious() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Launches a kernel that begins with these two.  brief: it may start while the
// kernel before it runs.  That takes 2 us off calls of 4 to 8 us that follow one
// another (a route of 8 tokens 4.2 us instead of 6.1, a product of 64 6.3 instead of
// 8.2), and costs long ones a few percent (the product and sum of 8192 tokens 196 us
// instead of 189), so those do without.
template <typename... Parameters, typename... Arguments>
void LaunchRouted(const char* what, bool brief, void (*kernel)(Parameters...), dim3 blocks, unsigned threads, std::size_t smem,
                  cudaStream_t stream, Arguments&&... arguments) {
  cudaLaunchAttribute overlap{};
  overlap.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  overlap.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config{};
  config.gridDim = blocks;
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  config.attrs = &overlap;
  config.numAttrs = brief ? 1 : 0;
  Check(cudaLaunchKernelEx(&config, kernel, std::forward<Arguments>(arguments)...), what);
  g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
}

// Whether a kernel of that many blocks is over in about one turn.
inline bool BriefGrid(int64_t blocks);

// The current device, and its streaming multiprocessors (asked for once).
constexpr int kMaxDevices = 64;

inline int CurrentDevice() {
  int device = 0;
  return cudaGetDevice(&device) == cudaSuccess && device >= 0 && device < kMaxDevices ? device : 0;
}

inline int RoutedSmCount() {
  static std::atomic<int> counts[kMaxDevices];
  const int device = CurrentDevice();
  int count = counts[device].load(std::memory_order_relaxed);
  if (count == 0) {
    if (cudaDeviceGetAttribute(&count, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || count < 1) return 148;
    counts[device].store(count, std::memory_order_relaxed);
  }
  return count;
}

inline bool BriefGrid(int64_t blocks) { return blocks <= 2 * RoutedSmCount(); }

// Lets kernel `kKernel` use `bytes` of dynamic shared memory on the current
// device; asked for once per device and size, since the call costs as much as
// a launch's share of a small operator.  Under a lock, so that the limit only
// grows: another thread's smaller size neither takes it back nor is recorded
// over a larger one.
template <auto kKernel>
void AllowShared(int bytes) {
  static std::atomic<int> allowed[kMaxDevices];
  static std::mutex setting;
  const int device = CurrentDevice();
  if (bytes <= 48 * 1024 || allowed[device].load(std::memory_order_acquire) >= bytes) return;
  const std::lock_guard<std::mutex> lock(setting);
  if (allowed[device].load(std::memory_order_relaxed) >= bytes) return;
  Check(cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), "kernel shared memory");
  allowed[device].store(bytes, std::memory_order_release);
}

}  // namespace t0b

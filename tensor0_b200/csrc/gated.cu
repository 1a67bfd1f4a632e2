// Gated activation between a routed layer's two products, with its input kept
// for the backward pass in 8 bits.
//
//   h = [g | u],  a = w silu(g) u,  silu(g) = g s,  s = 1 / (1 + exp(-g))
//   checkpoint: groups of `group` neighbours within g and within u;
//     m = max |h|,  scale = m (1/127),  code = round(h * (127 (1/m))), half to even
//     m < 2^-100: all zeros.  A NaN or infinity makes its group NaN on loading.
//   backward, from g' u' = code * scale:
//     dg = w da u' (s + silu (1 - s)),  du = w da silu,
//     dw = sum over the row of da silu u',  a' = w silu u' (for the next weight gradient)
// w is the row's routing weight (1 without a routing); rows that belong to no
// expert are not read, and zeros are written for them.
#include <algorithm>

#include "engine.h"
#include "layout.h"
#include "routed.cuh"
#include "routed.h"

namespace t0b {
namespace {

constexpr uint32_t kFull = 0xffffffffu;
constexpr int kGatedThreads = 256;
constexpr float kSmallest = 0x1p-100f;   // 127 / m and m / 127 stay normal numbers above it

__device__ __forceinline__ float Sigmoid(float g) { return __fdividef(1.0f, 1.0f + __expf(-g)); }

// Row p's routing weight; false if the row belongs to no expert.
__device__ __forceinline__ bool RowWeight(const GatedArgs& a, int64_t p, float* weight, int64_t* entry) {
  *weight = 1.0f;
  *entry = p;
  if (a.rows == nullptr) return true;
  *entry = a.rows[p];
  if (p >= a.offsets[a.experts] || *entry < 0 || *entry >= a.rows_count) return false;
  *weight = a.weights[*entry];
  return true;
}

// Codes of eight values and, by the group's first lane, the group's scale.
// A NaN's magnitude bits are above infinity's, so the integer maximum keeps it.
template <bool Vector>
__device__ __forceinline__ void StoreCodes(const float (&v)[8], int count, int lanes, int lane, int8_t* codes,
                                           float* scale) {
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) bits = max(bits, __float_as_uint(v[i]) & 0x7fffffffu);
  for (int d = lanes >> 1; d > 0; d >>= 1) bits = max(bits, __shfl_xor_sync(kFull, bits, d));
  const float largest = __uint_as_float(bits);
  const bool none = largest < kSmallest;
  const float per_unit = none ? 0.0f : __frcp_rn(largest) * 127.0f;
  if (count <= 0) return;
  if ((lane & (lanes - 1)) == 0) *scale = none ? 0.0f : largest * (1.0f / 127.0f);
  int q[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) q[i] = max(-127, min(127, __float2int_rn(v[i] * per_unit)));
  if constexpr (Vector) {
    uint2 packed;
    packed.x = (q[0] & 255) | ((q[1] & 255) << 8) | ((q[2] & 255) << 16) | (q[3] << 24);
    packed.y = (q[4] & 255) | ((q[5] & 255) << 8) | ((q[6] & 255) << 16) | (q[7] << 24);
    *reinterpret_cast<uint2*>(codes) = packed;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i < count) codes[i] = static_cast<int8_t>(q[i]);
    }
  }
}

template <bool Vector>
__device__ __forceinline__ void LoadCodes(const int8_t* codes, const float* scale, int count, float (&v)[8]) {
  if (count <= 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    return;
  }
  const float unit = *scale;
  if constexpr (Vector) {
    const uint2 packed = *reinterpret_cast<const uint2*>(codes);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t word = i < 4 ? packed.x : packed.y;
      v[i] = static_cast<float>(static_cast<int8_t>(word >> (8 * (i & 3)))) * unit;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < count ? static_cast<float>(codes[i]) * unit : 0.0f;
  }
}

// A warp takes 256 columns of one row, of both halves.
template <typename T, bool Vector>
__global__ void __launch_bounds__(kGatedThreads) GatedSave(GatedArgs a, int64_t chunks) {
  const int lane = threadIdx.x & 31, lanes = a.group / 8;
  const int groups = (a.width + a.group - 1) / a.group;
  const int64_t units = a.rows_count * chunks, step = int64_t{gridDim.x} * (kGatedThreads / 32);
  for (int64_t unit = int64_t{blockIdx.x} * (kGatedThreads / 32) + (threadIdx.x >> 5); unit < units; unit += step) {
    const int64_t p = unit / chunks;
    const int column = static_cast<int>(unit - p * chunks) * 256 + lane * 8;
    const int count = a.width - column;
    float weight;
    int64_t entry;
    const bool present = RowWeight(a, p, &weight, &entry);
    const T* row = static_cast<const T*>(a.h) + p * a.h_stride + column;
    float g[8], u[8], out[8];
    Load8<T, Vector>(row, present ? count : 0, g);
    Load8<T, Vector>(row + a.width, present ? count : 0, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = present ? weight * (g[i] * Sigmoid(g[i])) * u[i] : 0.0f;
    Store8<T, Vector>(static_cast<T*>(a.a) + p * a.width + column, count, out);
    int8_t* codes = a.codes + p * 2 * a.width + column;
    float* scales = a.scales + p * 2 * groups + column / a.group;
    StoreCodes<Vector>(g, count, lanes, lane, codes, scales);
    StoreCodes<Vector>(u, count, lanes, lane, codes + a.width, scales + groups);
  }
}

// A warp takes a row: the routing weight's gradient is the row's sum.
template <typename T, bool Vector>
__global__ void __launch_bounds__(kGatedThreads) GatedBackward(GatedArgs a) {
  const int lane = threadIdx.x & 31;
  const int groups = (a.width + a.group - 1) / a.group;
  const int64_t step = int64_t{gridDim.x} * (kGatedThreads / 32);
  for (int64_t p = int64_t{blockIdx.x} * (kGatedThreads / 32) + (threadIdx.x >> 5); p < a.rows_count; p += step) {
    float weight;
    int64_t entry;
    const bool present = RowWeight(a, p, &weight, &entry);
    float dot = 0.0f;
    for (int column = lane * 8; column < a.width; column += 256) {
      const int count = a.width - column;
      const int8_t* codes = a.codes + p * 2 * a.width + column;
      const float* scales = a.scales + p * 2 * groups + column / a.group;
      float g[8], u[8], da[8], dg[8], du[8], out[8];
      LoadCodes<Vector>(codes, scales, present ? count : 0, g);
      LoadCodes<Vector>(codes + a.width, scales + groups, present ? count : 0, u);
      Load8<T, Vector>(static_cast<const T*>(a.a_grad) + p * a.a_grad_stride + column, present ? count : 0, da);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float s = Sigmoid(g[i]), silu = g[i] * s;
        const float wda = weight * da[i];
        dg[i] = wda * u[i] * (s + silu * (1.0f - s));
        du[i] = wda * silu;
        out[i] = weight * silu * u[i];
        dot += da[i] * silu * u[i];
      }
      T* h_grad = static_cast<T*>(a.h_grad) + p * 2 * a.width + column;
      Store8<T, Vector>(h_grad, count, dg);
      Store8<T, Vector>(h_grad + a.width, count, du);
      Store8<T, Vector>(static_cast<T*>(a.a) + p * a.width + column, count, out);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(kFull, dot, d);
    if (lane == 0 && a.weights_grad != nullptr && entry >= 0 && entry < a.rows_count) a.weights_grad[entry] = dot;
  }
}

template <typename T, bool Vector>
__global__ void __launch_bounds__(kGatedThreads) CheckpointLoad(GatedArgs a, T* values, int64_t chunks) {
  const int lane = threadIdx.x & 31;
  const int groups = (a.width + a.group - 1) / a.group;
  const int64_t units = a.rows_count * 2 * chunks, step = int64_t{gridDim.x} * (kGatedThreads / 32);
  for (int64_t unit = int64_t{blockIdx.x} * (kGatedThreads / 32) + (threadIdx.x >> 5); unit < units; unit += step) {
    const int64_t half = unit / chunks;   // 2 p for g, 2 p + 1 for u
    const int column = static_cast<int>(unit - half * chunks) * 256 + lane * 8;
    float v[8];
    LoadCodes<Vector>(a.codes + half * a.width + column, a.scales + half * groups + column / a.group,
                      a.width - column, v);
    if constexpr (sizeof(T) == 2) {
      Store8<T, Vector>(values + half * a.width + column, a.width - column, v);
    } else {
      Store8<T, false>(values + half * a.width + column, a.width - column, v);
    }
  }
}

bool Aligned(const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

unsigned Blocks(int64_t units) {
  return static_cast<unsigned>(std::min<int64_t>((units + kGatedThreads / 32 - 1) / (kGatedThreads / 32), 1 << 20));
}

template <typename T>
void Save(const GatedArgs& a, cudaStream_t stream) {
  const int64_t chunks = (a.width + 255) / 256;
  const bool vector = a.width % 8 == 0 && a.h_stride % 8 == 0 && Aligned(a.h, 16) && Aligned(a.a, 16) && Aligned(a.codes, 8);
  const unsigned blocks = Blocks(a.rows_count * chunks);
  if (vector) GatedSave<T, true><<<blocks, kGatedThreads, 0, stream>>>(a, chunks);
  else GatedSave<T, false><<<blocks, kGatedThreads, 0, stream>>>(a, chunks);
}

template <typename T>
void Backward(const GatedArgs& a, cudaStream_t stream) {
  const bool vector = a.width % 8 == 0 && a.a_grad_stride % 8 == 0 && Aligned(a.a_grad, 16) && Aligned(a.a, 16) &&
                      Aligned(a.h_grad, 16) && Aligned(a.codes, 8);
  const unsigned blocks = Blocks(a.rows_count);
  if (vector) GatedBackward<T, true><<<blocks, kGatedThreads, 0, stream>>>(a);
  else GatedBackward<T, false><<<blocks, kGatedThreads, 0, stream>>>(a);
}

template <typename T>
void Load(const GatedArgs& a, void* values, cudaStream_t stream) {
  const int64_t chunks = (a.width + 255) / 256;
  const bool vector = a.width % 8 == 0 && Aligned(values, 16) && Aligned(a.codes, 8);
  const unsigned blocks = Blocks(a.rows_count * 2 * chunks);
  if (vector) CheckpointLoad<T, true><<<blocks, kGatedThreads, 0, stream>>>(a, static_cast<T*>(values), chunks);
  else CheckpointLoad<T, false><<<blocks, kGatedThreads, 0, stream>>>(a, static_cast<T*>(values), chunks);
}

void Launched() {
  Check(cudaGetLastError(), "gated activation launch");
  g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
}

}  // namespace

void LaunchGatedSave(int32_t dtype, const GatedArgs& args, cudaStream_t stream) {
  if (dtype == kTypeF16) Save<__half>(args, stream);
  else if (dtype == kTypeBf16) Save<__nv_bfloat16>(args, stream);
  else throw InvalidArgument("gated activations take F16 or BF16");
  Launched();
}

void LaunchGatedBackward(int32_t dtype, const GatedArgs& args, cudaStream_t stream) {
  if (dtype == kTypeF16) Backward<__half>(args, stream);
  else if (dtype == kTypeBf16) Backward<__nv_bfloat16>(args, stream);
  else throw InvalidArgument("gated activations take F16 or BF16");
  Launched();
}

void LaunchCheckpointLoad(int32_t dtype, const GatedArgs& args, void* values, cudaStream_t stream) {
  if (dtype == kTypeF16) Load<__half>(args, values, stream);
  else if (dtype == kTypeBf16) Load<__nv_bfloat16>(args, values, stream);
  else if (dtype == kTypeF32) Load<float>(args, values, stream);
  else throw InvalidArgument("checkpoints load as F32, F16 or BF16");
  Launched();
}

}  // namespace t0b

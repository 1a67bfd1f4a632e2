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
//
// Measured, replayed with three inputs by turns: saving 12294 rows of 1416 (f16,
// groups of 64) 35 us, 141 MB, and loading them 21 us, 106 MB: bound by instructions
// as much as by memory.  The gradient of 65536 rows of 2048 (bf16) 225 us, 1.35 GB,
// 0.91 of the copy bandwidth; the activation alone 144 us, 0.81 GB, 0.85.  Widths that
// 8 does not divide take 1.2 to 1.7 times as long.
#include <algorithm>
#include <type_traits>

#include "engine.h"
#include "layout.h"
#include "routed.cuh"
#include "routed.h"

namespace t0b {
namespace {

constexpr uint32_t kFull = 0xffffffffu;
constexpr int kGatedThreads = 256;
constexpr const char* kLaunch = "gated activation launch";
constexpr float kSmallest = 0x1p-100f;   // 127 / m and m / 127 stay normal numbers above it

// 1 / (1 + exp(-g)), off by a few units in the last place of 1 + exp(-g).
// Without .ftz each of the two special functions takes a comparison and a scaling
// more.  What they flush, below 2^-126, is far below F16 (four instructions).  BF16
// reaches down to 2^-133, which silu passes at g = -97 only: there the sum is held
// as 2^-15 (1 + exp(-g)), which is below 2^126 down to g = -97.7, and the reciprocal
// is scaled back by a product that keeps subnormal numbers.
template <typename T>
__device__ __forceinline__ float Sigmoid(float g) {
  float e, r;
  if constexpr (std::is_same<T, __half>::value) {
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return r;
  } else {
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(g, -1.4426950408889634f, -15.0f)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(0x1p-15f + e));
    return r * 0x1p-15f;
  }
}

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

// A warp works on 256 columns of a row, eight per lane: neighbours in one
// 16-byte access (Vector) where the rows allow it, otherwise every 32nd column,
// so that a 2-byte access is still one 64-byte run of the warp.
template <bool Vector>
__device__ __forceinline__ int Column(int lane, int i) { return Vector ? lane * 8 + i : lane + 32 * i; }

// Eight values as they lie in memory, fetched ahead of their use.  `row`: the
// 256 columns' first, `left`: columns of the row from there on.
template <typename T, bool Vector>
struct Raw8 {
  uint32_t w[Vector ? 4 : 8];   // two values each, or one
  __device__ __forceinline__ void Fetch(const T* row, int left, int lane) {
    if constexpr (Vector) {
      uint4 q = make_uint4(0u, 0u, 0u, 0u);
      if (lane * 8 < left) q = __ldcs(reinterpret_cast<const uint4*>(row + lane * 8));
      w[0] = q.x; w[1] = q.y; w[2] = q.z; w[3] = q.w;
    } else {
      const uint16_t* p = reinterpret_cast<const uint16_t*>(row) + lane;
      if (left >= 256) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = __ldcs(p + 32 * i);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = lane + 32 * i < left ? __ldcs(p + 32 * i) : 0u;
      }
    }
  }
  __device__ __forceinline__ void Values(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (Vector) v[i] = (i & 1) == 0 ? Unpack2<T>(w[i / 2]).x : Unpack2<T>(w[i / 2]).y;
      else v[i] = Unpack2<T>(w[i]).x;
    }
  }
};

template <typename T, bool Vector>
__device__ __forceinline__ void StoreRow(T* row, int left, int lane, const float (&v)[8]) {
  if constexpr (Vector) {
    Store8<T, true>(row + lane * 8, left - lane * 8, v);
  } else {
    T* p = row + lane;
    if (left >= 256) {
#pragma unroll
      for (int i = 0; i < 8; ++i) p[32 * i] = FromFloat<T>(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (lane + 32 * i < left) p[32 * i] = FromFloat<T>(v[i]);
      }
    }
  }
}

template <bool Vector>
struct RawCodes {
  uint32_t w[Vector ? 2 : 8];   // four codes each, or one
  float unit[Vector ? 1 : 8];
  // `scales`: of the 256 columns' first group.
  __device__ __forceinline__ void Fetch(const int8_t* row, const float* scales, int shift, int left, int lane) {
    if constexpr (Vector) {
      unit[0] = 0.0f;
      w[0] = w[1] = 0u;
      if (lane * 8 >= left) return;
      unit[0] = scales[(lane * 8) >> shift];
      const uint2 q = __ldcs(reinterpret_cast<const uint2*>(row + lane * 8));
      w[0] = q.x;
      w[1] = q.y;
    } else {
      const uint8_t* p = reinterpret_cast<const uint8_t*>(row) + lane;
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = lane + 32 * i < left ? __ldcs(p + 32 * i) : 0u;
#pragma unroll
      for (int i = 0; i < 8; ++i) {   // one per group
        const bool next = i == 0 || ((32 * i) & ((1 << shift) - 1)) == 0;
        unit[i] = i != 0 && !next ? unit[i != 0 ? i - 1 : 0] : 32 * i < left ? scales[(32 * i) >> shift] : 0.0f;
      }
    }
  }
  // A byte c + 128 in the low bits of 2^23 is 2^23 + 128 + c: exact, without a conversion.
  __device__ __forceinline__ void Values(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t biased = w[Vector ? i >> 2 : i] ^ (Vector ? 0x80808080u : 0x80u);
      const uint32_t word = __byte_perm(biased, 0x4b000000u, 0x7650 | (Vector ? i & 3 : 0));
      v[i] = (__uint_as_float(Vector ? word : (biased | 0x4b000000u)) - 8388736.0f) * unit[Vector ? 0 : i];
    }
  }
};

// A group's units per value and its scale, from the largest magnitude's bits.
// An infinity's group has the scale NaN: an infinite scale would make -inf of a
// code below 0, which is what a value that has no code may leave.
struct GroupScale {
  float per_unit, scale;
  __device__ __forceinline__ explicit GroupScale(uint32_t bits) {
    const float largest = __uint_as_float(bits);
    const bool none = largest < kSmallest;
    per_unit = none ? 0.0f : __frcp_rn(largest) * 127.0f;
    scale = none ? 0.0f : largest * (1.0f / 127.0f);
    if (bits >= 0x7f800000u) scale = __uint_as_float(0x7fc00000u);
  }
};

// |v * per_unit| is at most 127 and two roundings, so adding 1.5 * 2^23 rounds
// it to a whole number, half to even, in the low byte (a group that is not
// finite loads as NaN whatever its codes are).
__device__ __forceinline__ uint32_t Code(float v, float per_unit) {
  return __float_as_uint(__fadd_rn(__fmul_rn(v, per_unit), 12582912.0f));
}

// Two 16-bit values' larger magnitudes, NaN before everything.
template <typename T>
__device__ __forceinline__ uint32_t Larger2(uint32_t a, uint32_t b) {
  using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
  const T2 r = __hmax2_nan(__habs2(*reinterpret_cast<const T2*>(&a)), __habs2(*reinterpret_cast<const T2*>(&b)));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Codes of the warp's 256 columns and the scales of their groups of 1 << kShift.
template <typename T, bool Vector, int kShift>
__device__ __forceinline__ void StoreCodes(const Raw8<T, Vector>& raw, const float (&v)[8], int left, int lane,
                                           int8_t* codes, float* scales) {
  if constexpr (Vector) {
    constexpr int kLanes = 1 << (kShift - 3);   // of a group
    uint32_t most = Larger2<T>(Larger2<T>(raw.w[0], raw.w[1]), Larger2<T>(raw.w[2], raw.w[3]));
#pragma unroll
    for (int d = kLanes >> 1; d > 0; d >>= 1) most = Larger2<T>(most, __shfl_xor_sync(kFull, most, d));
    const float2 halves = Unpack2<T>(Larger2<T>(most, most >> 16));
    const GroupScale group(__float_as_uint(halves.x) & 0x7fffffffu);
    if (lane * 8 >= left) return;
    if ((lane & (kLanes - 1)) == 0) scales[lane / kLanes] = group.scale;
    uint32_t q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = Code(v[i], group.per_unit);
    uint2 packed;
    packed.x = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
    packed.y = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
    __stcs(reinterpret_cast<uint2*>(codes + lane * 8), packed);
  } else {
    // 32 neighbours per i; a group is 1, 2 or 4 of these.  Magnitudes compare as
    // their bits do, where a NaN's are above infinity's.
    constexpr int kRuns = 1 << (kShift - 5);
    int8_t* p = codes + lane;
#pragma unroll
    for (int i = 0; i < 8; i += kRuns) {
      uint32_t most = 0;
#pragma unroll
      for (int j = 0; j < kRuns; ++j) most = max(most, raw.w[i + j] & 0x7fffu);
      const GroupScale group(__float_as_uint(Unpack2<T>(__reduce_max_sync(kFull, most)).x));
      if (lane == 0 && 32 * i < left) scales[i / kRuns] = group.scale;
#pragma unroll
      for (int j = 0; j < kRuns; ++j) {
        const int8_t code = static_cast<int8_t>(Code(v[i + j], group.per_unit) & 255u);
        if (lane + 32 * (i + j) < left) p[32 * (i + j)] = code;
      }
    }
  }
}

// A warp takes 256 columns of a row at a time, every `parts`-th; blockIdx.y is
// the part: few rows are split over their columns.  Bound by its instructions
// as much as by memory (46 of them for a gate and an up value before the group
// was a constant here and the rows' addresses were carried along).
// Value by value there are too many registers for fetching ahead and for enough
// warps; the warps are worth more.
template <typename T, bool Vector, int kShift>
__global__ void __launch_bounds__(kGatedThreads, Vector ? 0 : 4) GatedSave(GatedArgs a) {
  LetNextStart();
  WaitForPrevious();
  const int lane = threadIdx.x & 31;
  const int groups = (a.width + (1 << kShift) - 1) >> kShift;
  const int stride = static_cast<int>(gridDim.y) * 256, begin = static_cast<int>(blockIdx.y) * 256;
  const int64_t step = int64_t{gridDim.x} * (kGatedThreads / 32);
  for (int64_t p = int64_t{blockIdx.x} * (kGatedThreads / 32) + (threadIdx.x >> 5); p < a.rows_count; p += step) {
    float weight;
    int64_t entry;
    const bool present = RowWeight(a, p, &weight, &entry);
    const T* h = static_cast<const T*>(a.h) + p * a.h_stride + begin;
    T* out_row = static_cast<T*>(a.a) + p * a.width + begin;
    int8_t* codes = a.codes + p * 2 * a.width + begin;
    float* scales = a.scales + p * 2 * groups + (begin >> kShift);
    Raw8<T, Vector> next_g, next_u;
    const auto fetch = [&](int left) {
      next_g.Fetch(h, present ? left : 0, lane);
      next_u.Fetch(h + a.width, present ? left : 0, lane);
      h += stride;
    };
    if (Vector) fetch(a.width - begin);
    for (int left = a.width - begin; left > 0; left -= stride) {
      if (!Vector) fetch(left);
      const Raw8<T, Vector> raw_g = next_g, raw_u = next_u;
      if (Vector && left > stride) fetch(left - stride);
      float g[8], u[8], out[8];
      raw_g.Values(g);
      raw_u.Values(u);
      // A row that is not present is zeros, whose activation is zero.
#pragma unroll
      for (int i = 0; i < 8; ++i) out[i] = (weight * g[i]) * Sigmoid<T>(g[i]) * u[i];
      StoreRow<T, Vector>(out_row, left, lane, out);
      if (a.codes != nullptr) {   // null: the activation alone
        StoreCodes<T, Vector, kShift>(raw_g, g, left, lane, codes, scales);
        StoreCodes<T, Vector, kShift>(raw_u, u, left, lane, codes + a.width, scales + groups);
      }
      out_row += stride;
      codes += stride;
      scales += stride >> kShift;
    }
  }
}

// A warp takes a row: the routing weight's gradient is the row's sum.
template <typename T, bool Vector>
__global__ void __launch_bounds__(kGatedThreads, Vector ? 0 : 3) GatedBackward(GatedArgs a) {
  LetNextStart();
  WaitForPrevious();
  const int lane = threadIdx.x & 31, shift = 31 - __clz(a.group);
  const int groups = (a.width + a.group - 1) >> shift;
  const int64_t step = int64_t{gridDim.x} * (kGatedThreads / 32);
  for (int64_t p = int64_t{blockIdx.x} * (kGatedThreads / 32) + (threadIdx.x >> 5); p < a.rows_count; p += step) {
    float weight;
    int64_t entry;
    const bool present = RowWeight(a, p, &weight, &entry);
    const int8_t* code_row = a.codes + p * 2 * a.width;
    const float* scale_row = a.scales + p * 2 * groups;
    const T* grad_row = static_cast<const T*>(a.a_grad) + p * a.a_grad_stride;
    T* h_row = static_cast<T*>(a.h_grad) + p * 2 * a.width;
    T* out_row = static_cast<T*>(a.a) + p * a.width;
    RawCodes<Vector> next_g, next_u;
    Raw8<T, Vector> next_da;
    const auto fetch = [&](int base) {
      const int left = present ? a.width - base : 0;
      next_g.Fetch(code_row + base, scale_row + (base >> shift), shift, left, lane);
      next_u.Fetch(code_row + a.width + base, scale_row + groups + (base >> shift), shift, left, lane);
      next_da.Fetch(grad_row + base, left, lane);
    };
    if (Vector) fetch(0);
    float dot = 0.0f;
    for (int base = 0; base < a.width; base += 256) {
      if (!Vector) fetch(base);
      const int left = a.width - base;
      float g[8], u[8], da[8], dg[8], du[8], out[8];
      next_g.Values(g);
      next_u.Values(u);
      next_da.Values(da);
      if (Vector && base + 256 < a.width) fetch(base + 256);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float s = Sigmoid<T>(g[i]), silu = g[i] * s;
        const float wda = weight * da[i], silu_u = silu * u[i];
        dg[i] = wda * u[i] * fmaf(silu, 1.0f - s, s);
        du[i] = wda * silu;
        out[i] = weight * silu_u;
        dot = fmaf(da[i], silu_u, dot);
      }
      StoreRow<T, Vector>(h_row + base, left, lane, dg);
      StoreRow<T, Vector>(h_row + a.width + base, left, lane, du);
      StoreRow<T, Vector>(out_row + base, left, lane, out);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(kFull, dot, d);
    if (lane == 0 && a.weights_grad != nullptr && entry >= 0 && entry < a.rows_count) a.weights_grad[entry] = dot;
  }
}

template <typename T, bool Vector>
__global__ void __launch_bounds__(kGatedThreads) CheckpointLoad(GatedArgs a, T* values) {
  LetNextStart();
  WaitForPrevious();
  const int lane = threadIdx.x & 31, shift = 31 - __clz(a.group);
  const int groups = (a.width + a.group - 1) >> shift, stride = static_cast<int>(gridDim.y) * 256;
  const int64_t halves = a.rows_count * 2, step = int64_t{gridDim.x} * (kGatedThreads / 32);
  // Half 2 p is row p's gate, 2 p + 1 its up.
  for (int64_t half = int64_t{blockIdx.x} * (kGatedThreads / 32) + (threadIdx.x >> 5); half < halves; half += step) {
    const int8_t* code_row = a.codes + half * a.width;
    const float* scale_row = a.scales + half * groups;
    const int begin = static_cast<int>(blockIdx.y) * 256;
    RawCodes<Vector> next;
    const auto fetch = [&](int base) {
      next.Fetch(code_row + base, scale_row + (base >> shift), shift, a.width - base, lane);
    };
    if (Vector) fetch(begin);
    for (int base = begin; base < a.width; base += stride) {
      if (!Vector) fetch(base);
      float v[8];
      next.Values(v);
      if (Vector && base + stride < a.width) fetch(base + stride);
      T* row = values + half * a.width + base;
      const int left = a.width - base;
      if constexpr (Vector && sizeof(T) == 4) {
        if (lane * 8 < left) {
          reinterpret_cast<float4*>(row + lane * 8)[0] = make_float4(v[0], v[1], v[2], v[3]);
          reinterpret_cast<float4*>(row + lane * 8)[1] = make_float4(v[4], v[5], v[6], v[7]);
        }
      } else {
        StoreRow<T, Vector>(row, left, lane, v);
      }
    }
  }
}

bool Aligned(const void* p, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// A warp per row, and where that leaves the device empty also a part of each
// row's columns per warp.
dim3 RowBlocks(int64_t rows, int width) {
  const int64_t blocks = std::min<int64_t>((rows + kGatedThreads / 32 - 1) / (kGatedThreads / 32), 1 << 20);
  const int64_t room = int64_t{RoutedSmCount()} * 8 / blocks;   // blocks that run at once, for each of these
  const int64_t parts = std::min<int64_t>((width + 255) / 256, std::max<int64_t>(1, room));
  return dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(std::min<int64_t>(parts, 65535)));
}

template <typename T, int kShift>
void SaveGroups(const GatedArgs& a, cudaStream_t stream) {
  const bool vector = a.width % 8 == 0 && a.h_stride % 8 == 0 && Aligned(a.h, 16) && Aligned(a.a, 16) && Aligned(a.codes, 8);
  const dim3 blocks = RowBlocks(a.rows_count, a.width);
  if (vector) LaunchRouted(kLaunch, BriefGrid(int64_t{blocks.x} * blocks.y), GatedSave<T, true, kShift>, blocks, kGatedThreads, 0, stream, a);
  else LaunchRouted(kLaunch, BriefGrid(int64_t{blocks.x} * blocks.y), GatedSave<T, false, kShift>, blocks, kGatedThreads, 0, stream, a);
}

template <typename T>
void Save(const GatedArgs& a, cudaStream_t stream) {
  if (a.group == 128) SaveGroups<T, 7>(a, stream);
  else if (a.group == 64) SaveGroups<T, 6>(a, stream);
  else SaveGroups<T, 5>(a, stream);
}

template <typename T>
void Backward(const GatedArgs& a, cudaStream_t stream) {
  const bool vector = a.width % 8 == 0 && a.a_grad_stride % 8 == 0 && Aligned(a.a_grad, 16) && Aligned(a.a, 16) &&
                      Aligned(a.h_grad, 16) && Aligned(a.codes, 8);
  const unsigned blocks = RowBlocks(a.rows_count, 1).x;
  if (vector) LaunchRouted(kLaunch, BriefGrid(blocks), GatedBackward<T, true>, blocks, kGatedThreads, 0, stream, a);
  else LaunchRouted(kLaunch, BriefGrid(blocks), GatedBackward<T, false>, blocks, kGatedThreads, 0, stream, a);
}

template <typename T>
void Load(const GatedArgs& a, void* values, cudaStream_t stream) {
  const bool vector = a.width % 8 == 0 && Aligned(values, 16) && Aligned(a.codes, 8);
  const dim3 blocks = RowBlocks(a.rows_count * 2, a.width);
  T* to = static_cast<T*>(values);
  if (vector) LaunchRouted(kLaunch, BriefGrid(int64_t{blocks.x} * blocks.y), CheckpointLoad<T, true>, blocks, kGatedThreads, 0, stream, a, to);
  else LaunchRouted(kLaunch, BriefGrid(int64_t{blocks.x} * blocks.y), CheckpointLoad<T, false>, blocks, kGatedThreads, 0, stream, a, to);
}

}  // namespace

void LaunchGatedSave(int32_t dtype, const GatedArgs& args, cudaStream_t stream) {
  if (dtype == kTypeF16) Save<__half>(args, stream);
  else if (dtype == kTypeBf16) Save<__nv_bfloat16>(args, stream);
  else throw InvalidArgument("gated activations take F16 or BF16");
}

void LaunchGatedBackward(int32_t dtype, const GatedArgs& args, cudaStream_t stream) {
  if (dtype == kTypeF16) Backward<__half>(args, stream);
  else if (dtype == kTypeBf16) Backward<__nv_bfloat16>(args, stream);
  else throw InvalidArgument("gated activations take F16 or BF16");
}

void LaunchCheckpointLoad(int32_t dtype, const GatedArgs& args, void* values, cudaStream_t stream) {
  if (dtype == kTypeF16) Load<__half>(args, values, stream);
  else if (dtype == kTypeBf16) Load<__nv_bfloat16>(args, values, stream);
  else if (dtype == kTypeF32) Load<float>(args, values, stream);
  else throw InvalidArgument("checkpoints load as F32, F16 or BF16");
}

}  // namespace t0b

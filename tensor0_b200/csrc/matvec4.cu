// Products of single tokens with 4-bit weights: for each expert-ordered row p,
//   y[p][n] = sum over groups of scale[e][n][group] * sum over k of (q[e][n][k] - 8) x[r(p)][k]
// q holds two weights per byte, the even one in the low half.
//
// Bound by the weights' bytes, half a byte each: 2.5 instructions per weight
// are all that fits beside them, so the products run on the tensor cores
// (mma.sync: 16 weight rows x 8 token rows x 16 deep; its rate is far above
// what memory feeds) and the scale multiplies a group's 32-bit sum, so that
// q - 8 enters exactly and nothing is rounded before the result.
//
// A block has 32 weight rows of one expert: eight warps, two 16-row tiles times
// four parts of the deep axis that are summed in shared memory in a fixed
// order.  An expert's weights are read once for every eight of its rows.
#include <algorithm>

#include "engine.h"
#include "layout.h"
#include "routed.cuh"
#include "routed.h"

namespace t0b {
namespace {

constexpr uint32_t kFull = 0xffffffffu;
constexpr int kMvThreads = 256, kMvRows = 32, kMvParts = 4;
constexpr int kMvStep = 128;            // deep values of one step of a warp: 32 of each lane's row
constexpr int kMvAhead = 4;             // steps whose weights are loaded ahead
constexpr int kMvChunk = 4096;          // deep values of x in shared memory at a time

// Row stride of x in shared memory, in units of 8 values: 4 more than a
// multiple of 8, so that two rows' 16-byte reads use different banks.
__host__ __device__ constexpr int MvStride(int inner) {
  return (inner < kMvChunk ? (inner + kMvStep - 1) / kMvStep * kMvStep : kMvChunk) / 8 + 4;
}

// Where unit u (8 values) of a row of x lies: the four lanes that share a
// weight row read four units 1, 2 or 4 apart, which this spreads over the banks.
__device__ __forceinline__ int MvUnit(int u) { return u ^ ((u >> 2) & 3); }

template <typename T>
__device__ __forceinline__ void Mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

// Weights i and i + 4 of a word, minus 8, exactly: a nibble in the low bits of
// 1024 (F16) or 128 (BF16) adds its value.
template <typename T>
__device__ __forceinline__ uint32_t Weights2(uint32_t word, int i) {
  const uint32_t bits = (word >> (4 * i)) & 0x000f000fu;
  if constexpr (std::is_same<T, __half>::value) {
    const uint32_t v = bits | 0x64006400u;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&v), __float2half2_rn(1032.0f));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const uint32_t v = bits | 0x43004300u;
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), __float2bfloat162_rn(136.0f));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}

// One step's weights of a lane: 32 deep neighbours of two weight rows, and the
// scales of the group that holds them.
struct MvLoad {
  uint4 top, bottom;
  float scale_top, scale_bottom;
};

// Swap words between lanes so that each of the step's groups is spread over
// the four lanes of a weight row: a matrix instruction then stays in one group.
template <int kGroups>
__device__ __forceinline__ void Spread(uint4& w, int t) {
  if constexpr (kGroups >= 2) {   // lanes t and t ^ 2 swap halves
    const bool high = (t & 2) != 0;
    const uint32_t s0 = __shfl_xor_sync(kFull, high ? w.x : w.z, 2), s1 = __shfl_xor_sync(kFull, high ? w.y : w.w, 2);
    if (high) { w.x = s0; w.y = s1; } else { w.z = s0; w.w = s1; }
  }
  if constexpr (kGroups == 4) {   // lanes t and t ^ 1 swap within the halves
    const bool odd = (t & 1) != 0;
    const uint32_t s0 = __shfl_xor_sync(kFull, odd ? w.x : w.y, 1), s1 = __shfl_xor_sync(kFull, odd ? w.z : w.w, 1);
    if (odd) { w.x = s0; w.z = s1; } else { w.y = s0; w.w = s1; }
  }
}

// Unit of x (8 values, from the step's first) that multiplies word w of lane t.
template <int kGroups>
__device__ __forceinline__ int StepUnit(int t, int w) {
  if constexpr (kGroups == 1) return 4 * t + w;
  // Words 0, 1 are group 0 (lanes 0, 1 their first half, lanes 2, 3 its second), words 2, 3 group 1.
  if constexpr (kGroups == 2) return 8 * (w >> 1) + 4 * (t & 1) + 2 * (t >> 1) + (w & 1);
  return 4 * w + t;   // word w is group w
}

template <typename T, int kGroup>
__global__ void __launch_bounds__(kMvThreads, 2) Matvec(MatvecArgs a, int row_blocks, bool vector) {
  constexpr int kGroups = kMvStep / kGroup;
  extern __shared__ uint4 mv_x[];
  __shared__ float sums[kMvThreads / 32][16][9];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3, part = warp & (kMvParts - 1), tile = warp / kMvParts;
  const int which = blockIdx.x / row_blocks, row0 = (blockIdx.x % row_blocks) * kMvRows;
  // The block's expert: the `which`-th that has rows.
  int expert = -1, seen = 0;
  for (int e0 = 0; e0 < a.experts && expert < 0; e0 += 32) {
    const int e = e0 + lane;
    const bool some = e < a.experts && RowBound(a.offsets[e + 1], a.entries) > RowBound(a.offsets[e], a.entries);
    const uint32_t present = __ballot_sync(kFull, some);
    const bool mine = some && seen + __popc(present & ((1u << lane) - 1)) == which;
    const uint32_t found = __ballot_sync(kFull, mine);
    if (found != 0u) expert = e0 + __ffs(found) - 1;
    seen += __popc(present);
  }
  if (which == 0) {   // rows without an expert
    T* out = static_cast<T*>(a.out);
    const int columns = min(kMvRows, a.outer - row0);
    const int64_t from = RowBound(a.offsets[a.experts], a.entries);
    for (int64_t i = tid; i < (a.entries - from) * columns; i += kMvThreads) {
      out[(from + i / columns) * a.outer + row0 + i % columns] = FromFloat<T>(0.0f);
    }
  }
  if (expert < 0) return;
  const int64_t begin = RowBound(a.offsets[expert], a.entries), end = RowBound(a.offsets[expert + 1], a.entries);
  const int groups = a.inner / kGroup, steps = (a.inner + kMvStep - 1) / kMvStep, stride = MvStride(a.inner);
  const int top = min(row0 + tile * 16 + g, a.outer - 1), bottom = min(row0 + tile * 16 + g + 8, a.outer - 1);
  const int64_t first = int64_t{expert} * a.outer;
  const uint8_t* codes_top = a.codes + (first + top) * (a.inner / 2);
  const uint8_t* codes_bottom = a.codes + (first + bottom) * (a.inner / 2);
  const T* scales_top = static_cast<const T*>(a.scales) + (first + top) * groups;
  const T* scales_bottom = static_cast<const T*>(a.scales) + (first + bottom) * groups;
  const auto load = [&](int step, MvLoad& l) {
    const int k = step * kMvStep + t * 32;
    const bool inside = step < steps && k < a.inner;
    l.top = l.bottom = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);   // zeros
    l.scale_top = l.scale_bottom = 0.0f;
    if (inside) {
      l.top = __ldcs(reinterpret_cast<const uint4*>(codes_top + k / 2));
      l.bottom = __ldcs(reinterpret_cast<const uint4*>(codes_bottom + k / 2));
      l.scale_top = ToFloat(scales_top[k / kGroup]);
      l.scale_bottom = ToFloat(scales_bottom[k / kGroup]);
    }
  };
  for (int64_t p0 = begin; p0 < end; p0 += 8) {
    const int rows = static_cast<int>(min(int64_t{8}, end - p0));
    MvLoad ahead[kMvAhead];
#pragma unroll
    for (int i = 0; i < kMvAhead; ++i) load(part + i * kMvParts, ahead[i]);
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = 0; k0 < a.inner; k0 += kMvChunk) {
      // x of these rows, in the order the tensor cores take the weights' nibbles.
      const int units = (min(kMvChunk, a.inner - k0) + kMvStep - 1) / kMvStep * (kMvStep / 8);
      __syncthreads();
      for (int i = tid; i < rows * units; i += kMvThreads) {
        const int n = i / units, u = i % units;
        const int64_t r = a.gather != 0 ? a.rows[p0 + n] / a.top_k : p0 + n;
        const int k = k0 + u * 8;
        uint32_t v[4] = {0u, 0u, 0u, 0u};
        if (k < a.inner && r >= 0 && r < a.x_rows) {   // 8 divides inner
          const T* x = static_cast<const T*>(a.x) + r * a.x_stride + k;
          if (vector) {
            const uint4 q = *reinterpret_cast<const uint4*>(x);
            v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
          } else {
            const uint16_t* bits = reinterpret_cast<const uint16_t*>(x);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = bits[2 * j] | (static_cast<uint32_t>(bits[2 * j + 1]) << 16);
          }
        }
        mv_x[n * stride + MvUnit(u)] = make_uint4(__byte_perm(v[0], v[2], 0x5410), __byte_perm(v[0], v[2], 0x7632),
                                                  __byte_perm(v[1], v[3], 0x5410), __byte_perm(v[1], v[3], 0x7632));
      }
      __syncthreads();
      const uint4* x = mv_x + (g < rows ? g : 0) * stride;
      const int last = min(steps, (k0 + kMvChunk) / kMvStep);
      for (int step0 = k0 / kMvStep + part; step0 < last; step0 += kMvAhead * kMvParts) {
#pragma unroll
        for (int i = 0; i < kMvAhead; ++i) {
          const int step = step0 + i * kMvParts;
          if (step >= last) break;   // chunks are whole rounds, so only the row's end comes here
          MvLoad l = ahead[i];
          load(step + kMvAhead * kMvParts, ahead[i]);
          Spread<kGroups>(l.top, t);
          Spread<kGroups>(l.bottom, t);
          const uint32_t wt[4] = {l.top.x, l.top.y, l.top.z, l.top.w};
          const uint32_t wb[4] = {l.bottom.x, l.bottom.y, l.bottom.z, l.bottom.w};
          const int unit0 = (step * kMvStep - k0) / 8;
#pragma unroll
          for (int n = 0; n < kGroups; ++n) {
            float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = n * 4 / kGroups; w < (n + 1) * 4 / kGroups; ++w) {
              const uint4 b = x[MvUnit(unit0 + StepUnit<kGroups>(t, w))];
              const uint32_t a0[4] = {Weights2<T>(wt[w], 0), Weights2<T>(wb[w], 0), Weights2<T>(wt[w], 1), Weights2<T>(wb[w], 1)};
              Mma<T>(c, a0, b.x, b.y);
              const uint32_t a1[4] = {Weights2<T>(wt[w], 2), Weights2<T>(wb[w], 2), Weights2<T>(wt[w], 3), Weights2<T>(wb[w], 3)};
              Mma<T>(c, a1, b.z, b.w);
            }
            const int owner = (lane & ~3) | (n * 4 / kGroups);
            const float st = kGroups == 1 ? l.scale_top : __shfl_sync(kFull, l.scale_top, owner);
            const float sb = kGroups == 1 ? l.scale_bottom : __shfl_sync(kFull, l.scale_bottom, owner);
            acc[0] = fmaf(st, c[0], acc[0]);
            acc[1] = fmaf(st, c[1], acc[1]);
            acc[2] = fmaf(sb, c[2], acc[2]);
            acc[3] = fmaf(sb, c[3], acc[3]);
          }
        }
      }
    }
    // acc: weight rows g and g + 8, token rows 2 t and 2 t + 1.
    sums[warp][g][2 * t] = acc[0];
    sums[warp][g][2 * t + 1] = acc[1];
    sums[warp][g + 8][2 * t] = acc[2];
    sums[warp][g + 8][2 * t + 1] = acc[3];
    __syncthreads();
    const int n = tid >> 5, row = tid & 31;   // token row, weight row
    if (n < rows && row0 + row < a.outer) {
      float sum = 0.0f;
#pragma unroll
      for (int q = 0; q < kMvParts; ++q) sum += sums[(row >> 4) * kMvParts + q][row & 15][n];
      static_cast<T*>(a.out)[(p0 + n) * a.outer + row0 + row] = FromFloat<T>(sum);
    }
  }
}

template <typename T, int kGroup>
void Launch(const MatvecArgs& a, cudaStream_t stream) {
  const int row_blocks = (a.outer + kMvRows - 1) / kMvRows;
  const int64_t blocks = std::min<int64_t>(a.experts, a.entries) * row_blocks;
  if (blocks >= int64_t{1} << 31) throw InvalidArgument("4-bit product is too large");
  // A token has an expert at most once, so an expert has at most that many rows.
  const int rows = static_cast<int>(std::min<int64_t>(8, a.entries));
  const int smem = rows * MvStride(a.inner) * 16;
  const bool vector = a.x_stride % 8 == 0 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0;
  Check(cudaFuncSetAttribute(Matvec<T, kGroup>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
        "4-bit product shared memory");
  Matvec<T, kGroup><<<static_cast<unsigned>(blocks), kMvThreads, smem, stream>>>(a, row_blocks, vector);
  Check(cudaGetLastError(), "4-bit product launch");
  g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
}

template <typename T>
void ByGroup(const MatvecArgs& a, cudaStream_t stream) {
  if (a.group == 128) Launch<T, 128>(a, stream);
  else if (a.group == 64) Launch<T, 64>(a, stream);
  else Launch<T, 32>(a, stream);
}

}  // namespace

void LaunchMatvec(int32_t dtype, const MatvecArgs& args, cudaStream_t stream) {
  if (dtype == kTypeF16) ByGroup<__half>(args, stream);
  else if (dtype == kTypeBf16) ByGroup<__nv_bfloat16>(args, stream);
  else throw InvalidArgument("4-bit products take F16 or BF16");
}

}  // namespace t0b

// Products of single tokens with 4-bit weights: for each expert-ordered row p,
//   y[p][n] = sum over groups of scale[e][n][group] * sum over k of (q[e][n][k] - 8) x[r(p)][k]
// q holds two weights per byte, the even one in the low half.
//
// Bound by the weights' bytes, half a byte each, beside which a scheduler has
// about 12 weights per instruction: the products run on the tensor cores
// (mma.sync: 16 weight rows x 8 token rows x 16 deep; its rate is far above
// what memory feeds), and a nibble becomes a 16-bit float by masking alone:
//   F16:  bits of a subnormal, q 2^-24 (nibbles 0, 4, ...) or 16 q 2^-24; the
//         two kinds have accumulators of their own
//   BF16: the top of the fraction of 16 + q
// Both are exact.  What is added to each weight (8 too much, or 24) is taken
// off by starting a group's 32-bit sum at minus that times the sum of x, and
// the scale multiplies the group's sum, so nothing is rounded before the result.
//
// A block is eight warps: 16-row tiles of one expert's weights times kParts
// parts of the deep axis that are summed in shared memory in a fixed order.  An
// expert's weights are read once for every eight of its rows.
#include <algorithm>

#include "engine.h"
#include "layout.h"
#include "routed.cuh"
#include "routed.h"

namespace t0b {
namespace {

constexpr uint32_t kFull = 0xffffffffu;
constexpr int kMvThreads = 256, kMvWarps = kMvThreads / 32;
constexpr int kMvStep = 128;            // deep values of one step of a warp
constexpr int kMvAhead = 4;             // steps whose weights are loaded ahead
constexpr int kMvChunk = 4096;          // deep values of x in shared memory at a time

// Row stride of x in shared memory, in units of 8 values: 4 more than a
// multiple of 8, so that two rows' 16-byte reads use different banks.
__host__ __device__ constexpr int MvStride(int inner) {
  return (inner < kMvChunk ? (inner + kMvStep - 1) / kMvStep * kMvStep : kMvChunk) / 8 + 4;
}

// Where unit u (8 values) of a row of x lies: the four lanes that share a
// weight row read units 1 or 2 apart, which this spreads over the banks.
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

// Weights i and i + 4 of a word as the tensor cores take them.
__device__ __forceinline__ uint32_t Mask2(uint32_t word, uint32_t mask, uint32_t with) {
  return (word & mask) | with;
}

// The partial sums of one group: 16 weight rows x 8 token rows.
template <typename T>
struct MvSum {
  float c[4], wide[4];   // wide: F16 weights that stand for 16 times their value
  // Start at minus the excess of the weights times the token rows' sums.
  __device__ __forceinline__ void Start(float2 excess) {
    c[0] = c[2] = excess.x;
    c[1] = c[3] = excess.y;
#pragma unroll
    for (int i = 0; i < 4; ++i) wide[i] = 0.0f;
  }
  // A word of each of the two weight rows, eight deep values.
  __device__ __forceinline__ void Add(uint32_t top, uint32_t bottom, const uint4& x) {
    if constexpr (std::is_same<T, __half>::value) {
      const uint32_t t8 = top >> 8, b8 = bottom >> 8;
      const uint32_t plain[4] = {top & 0x000f000fu, bottom & 0x000f000fu, t8 & 0x000f000fu, b8 & 0x000f000fu};
      const uint32_t times16[4] = {top & 0x00f000f0u, bottom & 0x00f000f0u, t8 & 0x00f000f0u, b8 & 0x00f000f0u};
      Mma<T>(c, plain, x.x, x.z);
      Mma<T>(wide, times16, x.y, x.w);
    } else {
      const uint32_t one = 0x00780078u, base = 0x41804180u;
      const uint32_t first[4] = {Mask2(top << 3, one, base), Mask2(bottom << 3, one, base), Mask2(top >> 1, one, base),
                                 Mask2(bottom >> 1, one, base)};
      const uint32_t second[4] = {Mask2(top >> 5, one, base), Mask2(bottom >> 5, one, base), Mask2(top >> 9, one, base),
                                  Mask2(bottom >> 9, one, base)};
      Mma<T>(c, first, x.x, x.y);
      Mma<T>(c, second, x.z, x.w);
    }
  }
  __device__ __forceinline__ float Value(int i) const {
    if constexpr (std::is_same<T, __half>::value) return fmaf(wide[i], 0.0625f, c[i]);
    return c[i];
  }
};

// The sum of x times this starts a group; the last factor restores the size.
template <typename T> constexpr float kMvExcess = std::is_same<T, __half>::value ? -8.0f * 0x1p-24f : -24.0f;
template <typename T> constexpr float kMvSize = std::is_same<T, __half>::value ? 0x1p24f : 1.0f;

// One step's weights of a lane: of each half (64 deep values) 16 neighbours of
// two weight rows, and the scales of the group that holds them.
struct MvLoad {
  uint2 top[2], bottom[2];
  float scale_top[2], scale_bottom[2];
};

// Groups of 32: lanes t and t ^ 2 swap a word, so that each of a half's two
// groups is spread over the four lanes and a matrix instruction stays in one.
__device__ __forceinline__ void Swap(uint2& w, int t) {
  const bool high = (t & 2) != 0;
  const uint32_t other = __shfl_xor_sync(kFull, high ? w.x : w.y, 2);
  if (high) w.x = other; else w.y = other;
}

template <typename T, int kGroup, int kParts>
__global__ void __launch_bounds__(kMvThreads, 2) Matvec(MatvecArgs a, int row_blocks, int max_rows, bool vector) {
  constexpr int kRows = 16 * kMvWarps / kParts;   // weight rows of a block
  extern __shared__ uint4 mv_x[];
  __shared__ float sums[kMvWarps][16][9];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3, part = warp % kParts, tile = warp / kParts;
  const int which = blockIdx.x / row_blocks, row0 = (blockIdx.x % row_blocks) * kRows;
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
    const int columns = min(kRows, a.outer - row0);
    const int64_t from = RowBound(a.offsets[a.experts], a.entries);
    for (int64_t i = tid; i < (a.entries - from) * columns; i += kMvThreads) {
      out[(from + i / columns) * a.outer + row0 + i % columns] = FromFloat<T>(0.0f);
    }
  }
  if (expert < 0) return;
  const int64_t begin = RowBound(a.offsets[expert], a.entries), end = RowBound(a.offsets[expert + 1], a.entries);
  const int groups = a.inner / kGroup, steps = (a.inner + kMvStep - 1) / kMvStep, stride = MvStride(a.inner);
  const int group_stride = (stride - 4) * 8 / kGroup;
  float* x_sums = reinterpret_cast<float*>(mv_x + max_rows * stride);   // [token row][group of the chunk]
  const int top = min(row0 + tile * 16 + g, a.outer - 1), bottom = min(row0 + tile * 16 + g + 8, a.outer - 1);
  const int64_t first = int64_t{expert} * a.outer;
  const uint8_t* codes_top = a.codes + (first + top) * (a.inner / 2) + t * 8;
  const uint8_t* codes_bottom = a.codes + (first + bottom) * (a.inner / 2) + t * 8;
  const T* scales_top = static_cast<const T*>(a.scales) + (first + top) * groups;
  const T* scales_bottom = static_cast<const T*>(a.scales) + (first + bottom) * groups;
  const auto load = [&](int step, MvLoad& l) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = step * kMvStep + h * 64;
      l.top[h] = l.bottom[h] = make_uint2(0u, 0u);
      if (k + t * 16 < a.inner) {   // false past the last step; 16 divides inner
        l.top[h] = __ldcs(reinterpret_cast<const uint2*>(codes_top + k / 2));
        l.bottom[h] = __ldcs(reinterpret_cast<const uint2*>(codes_bottom + k / 2));
      }
      if (kGroup < 128 || h == 0) {
        const int group = (k + t * 16) / kGroup;
        const bool inside = group < groups;   // past the row's end: weights that count for nothing
        l.scale_top[h] = inside ? ToFloat(scales_top[group]) : 0.0f;
        l.scale_bottom[h] = inside ? ToFloat(scales_bottom[group]) : 0.0f;
      }
    }
  };
  // Units of x that multiply a half's words x and y.  (A step begins at a
  // multiple of 16 units, which MvUnit leaves alone.)
  int unit_x[2], unit_y[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    unit_x[h] = MvUnit(8 * h + (kGroup == 32 ? 2 * (t & 1) + (t >> 1) : 2 * t));
    unit_y[h] = MvUnit(8 * h + (kGroup == 32 ? 4 + 2 * (t & 1) + (t >> 1) : 2 * t + 1));
  }
  for (int64_t p0 = begin; p0 < end; p0 += 8) {
    const int rows = static_cast<int>(min(int64_t{max_rows}, end - p0));
    MvLoad ahead[kMvAhead];
#pragma unroll
    for (int i = 0; i < kMvAhead; ++i) load(part + i * kParts, ahead[i]);
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = 0; k0 < a.inner; k0 += kMvChunk) {
      // x of these rows, in the order the tensor cores take the weights'
      // nibbles, and its sums by group.
      const int units = (min(kMvChunk, a.inner - k0) + kMvStep - 1) / kMvStep * (kMvStep / 8);
      __syncthreads();
      for (int n = 0; n < rows; ++n) {
        const int64_t r = a.gather != 0 ? a.rows[p0 + n] / a.top_k : p0 + n;
        for (int u0 = 0; u0 < units; u0 += kMvThreads) {
          const int u = u0 + tid, k = k0 + u * 8;
          uint32_t v[4] = {0u, 0u, 0u, 0u};
          if (u < units && k < a.inner && r >= 0 && r < a.x_rows) {   // 8 divides inner
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
          float sum = 0.0f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = Unpack2<T>(v[j]);
            sum += f.x + f.y;
          }
#pragma unroll
          for (int d = kGroup / 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kFull, sum, d);
          if (u < units) {   // units are a multiple of 16: whole groups
            mv_x[n * stride + MvUnit(u)] = make_uint4(__byte_perm(v[0], v[2], 0x5410), __byte_perm(v[0], v[2], 0x7632),
                                                      __byte_perm(v[1], v[3], 0x5410), __byte_perm(v[1], v[3], 0x7632));
            if (u % (kGroup / 8) == 0) x_sums[n * group_stride + u / (kGroup / 8)] = kMvExcess<T> * sum;
          }
        }
      }
      __syncthreads();
      const uint4* x = mv_x + (g < rows ? g : 0) * stride;
      const float* even = x_sums + (2 * t < rows ? 2 * t : 0) * group_stride;
      const float* odd = x_sums + (2 * t + 1 < rows ? 2 * t + 1 : 0) * group_stride;
      const int last = min(steps, (k0 + kMvChunk) / kMvStep);
      for (int step0 = k0 / kMvStep + part; step0 < last; step0 += kMvAhead * kParts) {
#pragma unroll
        for (int i = 0; i < kMvAhead; ++i) {
          const int step = step0 + i * kParts;
          if (step >= last) break;   // chunks are whole rounds, so only the row's end comes here
          MvLoad l = ahead[i];
          load(step + kMvAhead * kParts, ahead[i]);
          const int from = step * kMvStep - k0;
          const auto excess = [&](int group) { return make_float2(even[from / kGroup + group], odd[from / kGroup + group]); };
          const auto scaled = [&](const MvSum<T>& c, float st, float sb) {
            acc[0] = fmaf(st, c.Value(0), acc[0]);
            acc[1] = fmaf(st, c.Value(1), acc[1]);
            acc[2] = fmaf(sb, c.Value(2), acc[2]);
            acc[3] = fmaf(sb, c.Value(3), acc[3]);
          };
          MvSum<T> c;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint4 bx = x[from / 8 + unit_x[h]], by = x[from / 8 + unit_y[h]];
            if constexpr (kGroup == 32) {
              Swap(l.top[h], t);
              Swap(l.bottom[h], t);
              c.Start(excess(2 * h));
              c.Add(l.top[h].x, l.bottom[h].x, bx);
              scaled(c, __shfl_sync(kFull, l.scale_top[h], lane & ~3), __shfl_sync(kFull, l.scale_bottom[h], lane & ~3));
              c.Start(excess(2 * h + 1));
              c.Add(l.top[h].y, l.bottom[h].y, by);
              scaled(c, __shfl_sync(kFull, l.scale_top[h], lane | 3), __shfl_sync(kFull, l.scale_bottom[h], lane | 3));
            } else {
              if (kGroup == 64 || h == 0) c.Start(excess(kGroup == 64 ? h : 0));
              c.Add(l.top[h].x, l.bottom[h].x, bx);
              c.Add(l.top[h].y, l.bottom[h].y, by);
              if (kGroup == 64) scaled(c, l.scale_top[h], l.scale_bottom[h]);
              else if (h == 1) scaled(c, l.scale_top[0], l.scale_bottom[0]);
            }
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
    for (int i = tid; i < rows * kRows; i += kMvThreads) {
      const int n = i / kRows, row = i % kRows;   // token row, weight row
      if (row0 + row >= a.outer) continue;
      float sum = 0.0f;
#pragma unroll
      for (int q = 0; q < kParts; ++q) sum += sums[(row >> 4) * kParts + q][row & 15][n];
      static_cast<T*>(a.out)[(p0 + n) * a.outer + row0 + row] = FromFloat<T>(sum * kMvSize<T>);
    }
  }
}

template <typename T, int kGroup, int kParts>
void Launch(const MatvecArgs& a, cudaStream_t stream) {
  constexpr int kRows = 16 * kMvWarps / kParts;
  const int row_blocks = (a.outer + kRows - 1) / kRows;
  const int64_t blocks = std::min<int64_t>(a.experts, a.entries) * row_blocks;
  if (blocks >= int64_t{1} << 31) throw InvalidArgument("4-bit product is too large");
  const int rows = static_cast<int>(std::min<int64_t>(8, a.entries)), stride = MvStride(a.inner);
  const int smem = rows * (stride * 16 + (stride - 4) * 8 / kGroup * 4);
  const bool vector = a.x_stride % 8 == 0 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0;
  AllowShared<Matvec<T, kGroup, kParts>>(smem);
  Matvec<T, kGroup, kParts><<<static_cast<unsigned>(blocks), kMvThreads, smem, stream>>>(a, row_blocks, rows, vector);
  Check(cudaGetLastError(), "4-bit product launch");
  g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
}

template <typename T, int kGroup>
void ByParts(const MatvecArgs& a, cudaStream_t stream) {
  // Fewer parts read longer runs of the deep axis per warp; more parts give
  // more blocks.
  const int64_t blocks = std::min<int64_t>(a.experts, a.entries) * ((a.outer + 127) / 128);
  const int resident = RoutedSmCount() * 2;
  if (blocks >= 2 * resident) Launch<T, kGroup, 1>(a, stream);
  else if (blocks >= resident) Launch<T, kGroup, 2>(a, stream);
  else Launch<T, kGroup, 4>(a, stream);
}

template <typename T>
void ByGroup(const MatvecArgs& a, cudaStream_t stream) {
  if (a.group == 128) ByParts<T, 128>(a, stream);
  else if (a.group == 64) ByParts<T, 64>(a, stream);
  else ByParts<T, 32>(a, stream);
}

}  // namespace

void LaunchMatvec(int32_t dtype, const MatvecArgs& args, cudaStream_t stream) {
  if (dtype == kTypeF16) ByGroup<__half>(args, stream);
  else if (dtype == kTypeBf16) ByGroup<__nv_bfloat16>(args, stream);
  else throw InvalidArgument("4-bit products take F16 or BF16");
}

}  // namespace t0b

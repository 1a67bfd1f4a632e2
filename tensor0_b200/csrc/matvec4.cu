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
// parts of the deep axis that are summed in shared memory in a fixed order; a
// ninth brings the weights by TMA, three 16 KB stages ahead.  (Loaded straight
// into registers, each warp's load touched eight rows, 42 wavefronts for 1024
// weights with the scales: the load path was the bound at twice the time.)  An
// expert's weights are read once for every eight of its rows.
#include <algorithm>

#include "engine.h"
#include "layout.h"
#include "routed.cuh"
#include "routed.h"
#include "tcgen05.cuh"
#include "tensor_map.h"

namespace t0b {
namespace {

constexpr uint32_t kFull = 0xffffffffu;
constexpr int kMvWarps = 8, kMvThreads = kMvWarps * 32;   // computing; one more warp loads
constexpr int kMvBox = 256;             // deep values of a row in one box: 128 bytes
constexpr int kMvStages = 3;
constexpr uint32_t kMvStageBytes = 16 * kMvWarps * 128;   // kParts boxes of all the block's rows
constexpr int kMvChunk = 2048;          // deep values of x and of the scales in shared memory at a time

// Row stride of x in shared memory, in units of 8 values: 4 more than a
// multiple of 8, so that two rows' 16-byte reads use different banks.
constexpr int kMvStride = kMvChunk / 8 + 4;

// Where unit u (8 values) of a row of x lies: the four lanes that share a
// weight row read units 1 or 2 apart, which this spreads over the banks.
__device__ __forceinline__ int MvUnit(int u) { return u ^ ((u >> 2) & 3); }

// The computing warps' barrier.
__device__ __forceinline__ void MvSync() { asm volatile("bar.sync 1, %0;" ::"n"(kMvThreads) : "memory"); }

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

// Groups of 32: lanes t and t ^ 2 swap a word, so that each of a half's two
// groups is spread over the four lanes and a matrix instruction stays in one.
__device__ __forceinline__ void Swap(uint2& w, int t) {
  const bool high = (t & 2) != 0;
  const uint32_t other = __shfl_xor_sync(kFull, high ? w.x : w.y, 2);
  if (high) w.x = other; else w.y = other;
}

struct MvShared {
  uint64_t full[kMvStages], empty[kMvStages];
  volatile int failed;
  float sums[kMvWarps][16][9];
};

template <typename T, int kGroup, int kParts>
__global__ void __launch_bounds__(kMvThreads + 32, 2)
    Matvec(MatvecArgs a, const __grid_constant__ CUtensorMap map, int row_blocks, int max_rows, bool vector) {
  constexpr int kRows = 16 * kMvWarps / kParts;   // weight rows of a block
  constexpr int kSpan = kParts * kMvBox;          // deep values of a stage
  constexpr int kChunkGroups = kMvChunk / kGroup, kScaleStride = kChunkGroups + 2;
  extern __shared__ unsigned char mv_raw[];
  __shared__ MvShared s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int which = blockIdx.x / row_blocks, row0 = (blockIdx.x % row_blocks) * kRows;
  const uint32_t ring = (SharedAddress(mv_raw) + 1023u) & ~1023u;
  uint4* x_values = reinterpret_cast<uint4*>(mv_raw + (ring - SharedAddress(mv_raw)) + kMvStages * kMvStageBytes);
  float* x_sums = reinterpret_cast<float*>(x_values + max_rows * kMvStride);   // [token row][group of the chunk]
  uint16_t* scales = reinterpret_cast<uint16_t*>(x_sums + max_rows * kChunkGroups);   // [weight row][group of the chunk]
  if (tid == 0) {
    for (int i = 0; i < kMvStages; ++i) {
      BarrierInit(SharedAddress(&s.full[i]), 1);
      BarrierInit(SharedAddress(&s.empty[i]), kMvWarps);
    }
    s.failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
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
    for (int64_t i = tid; i < (a.entries - from) * columns; i += blockDim.x) {
      out[(from + i / columns) * a.outer + row0 + i % columns] = FromFloat<T>(0.0f);
    }
  }
  if (expert < 0) return;
  const int64_t begin = RowBound(a.offsets[expert], a.entries), end = RowBound(a.offsets[expert + 1], a.entries);
  const int spans = (a.inner + kSpan - 1) / kSpan;
  const int64_t first = int64_t{expert} * a.outer;

  if (warp == kMvWarps) {   // loads: one thread
    if (lane != 0) return;
    uint32_t fill = 0;
    bool ok = true;
    for (int64_t p0 = begin; p0 < end && ok; p0 += 8) {
      for (int span = 0; span < spans; ++span, ++fill) {
        const uint32_t stage = fill % kMvStages, full = SharedAddress(&s.full[stage]);
        if (fill >= kMvStages) {
          ok = BarrierWait(SharedAddress(&s.empty[stage]), (fill / kMvStages + 1) & 1, &s.failed);
          if (!ok) break;
        }
        // Boxes that begin in the row at all.
        const int boxes = min(kParts, (a.inner - span * kSpan + kMvBox - 1) / kMvBox);
        BarrierExpect(full, boxes * (kMvStageBytes / kParts));
        for (int box = 0; box < boxes; ++box) {
          LoadTile2(ring + stage * kMvStageBytes + box * (kMvStageBytes / kParts), &map, full,
                    (span * kSpan + box * kMvBox) / 2, static_cast<int>(first) + row0);
        }
      }
    }
    // Whoever gives up, the copies in flight land before the block ends.
    for (uint32_t f = fill - min(fill, static_cast<uint32_t>(kMvStages)); f < fill; ++f) {
      BarrierWait(SharedAddress(&s.full[f % kMvStages]), (f / kMvStages) & 1, nullptr);
    }
    return;
  }

  const int g = lane >> 2, t = lane & 3, part = warp % kParts, tile = warp / kParts;
  // Rows of the tile in the tensor cores' order: lanes that read together take
  // every second row, whose swizzled 16-byte places differ.
  const int top = tile * 16 + 2 * (g & 3) + (g >> 2), bottom = top + 8;
  const uint32_t swizzle = static_cast<uint32_t>(top & 7);
  const int groups = a.inner / kGroup;
  // Units of x that multiply a half's (64 deep values) words x and y, for even and odd halves.
  int unit_x[2], unit_y[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    unit_x[h] = MvUnit(8 * h + (kGroup == 32 ? 2 * (t & 1) + (t >> 1) : 2 * t));
    unit_y[h] = MvUnit(8 * h + (kGroup == 32 ? 4 + 2 * (t & 1) + (t >> 1) : 2 * t + 1));
  }
  uint32_t fill = 0;
  bool ok = true;
  for (int64_t p0 = begin; p0 < end; p0 += 8) {
    const int rows = static_cast<int>(min(int64_t{max_rows}, end - p0));
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k0 = 0; k0 < a.inner; k0 += kMvChunk) {
      // x of these rows, in the order the tensor cores take the weights'
      // nibbles, its sums by group, and the weight rows' scales.
      const int units = (min(kMvChunk, a.inner - k0) + 127) / 128 * 16;
      const int chunk_groups = min(kChunkGroups, groups - k0 / kGroup);
      MvSync();
      for (int i = tid; i < kRows * kChunkGroups; i += kMvThreads) {
        const int row = i / kChunkGroups, group = i % kChunkGroups;
        const bool inside = group < chunk_groups && row0 + row < a.outer;
        scales[row * kScaleStride + group] =
            inside ? static_cast<const uint16_t*>(a.scales)[(first + row0 + row) * groups + k0 / kGroup + group] : 0;
      }
      for (int n = 0; n < rows; ++n) {
        const int64_t r = a.gather != 0 ? a.rows[p0 + n] / a.top_k : p0 + n;
        const int u = tid, k = k0 + u * 8;   // a chunk has one unit per thread
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
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = Unpack2<T>(v[j]);
          sum += f.x + f.y;
        }
#pragma unroll
        for (int d = kGroup / 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kFull, sum, d);
        if (u < units) {   // units are a multiple of 16: whole groups
          x_values[n * kMvStride + MvUnit(u)] = make_uint4(__byte_perm(v[0], v[2], 0x5410), __byte_perm(v[0], v[2], 0x7632),
                                                           __byte_perm(v[1], v[3], 0x5410), __byte_perm(v[1], v[3], 0x7632));
          if (u % (kGroup / 8) == 0) x_sums[n * kChunkGroups + u / (kGroup / 8)] = kMvExcess<T> * sum;
        }
      }
      MvSync();
      const uint4* x = x_values + (g < rows ? g : 0) * kMvStride;
      const float* even = x_sums + (2 * t < rows ? 2 * t : 0) * kChunkGroups;
      const float* odd = x_sums + (2 * t + 1 < rows ? 2 * t + 1 : 0) * kChunkGroups;
      const uint16_t* scales_top = scales + top * kScaleStride;
      const uint16_t* scales_bottom = scales + bottom * kScaleStride;
      const int last = min(a.inner, k0 + kMvChunk);
      for (int k1 = k0; k1 < last; k1 += kSpan, ++fill) {
        const uint32_t stage = fill % kMvStages;
        ok = ok && BarrierWait(SharedAddress(&s.full[stage]), (fill / kMvStages) & 1, &s.failed);
        ok = __all_sync(kFull, ok);
        const int k = k1 + part * kMvBox;
        if (ok && k < last) {   // `last` is the row's end, or this part begins before the chunk's
          const uint32_t box = ring + stage * kMvStageBytes + part * (kMvStageBytes / kParts);
          const int halves = min(kMvBox / 64, (last - k + 63) / 64), from = k - k0;
          const auto scaled = [&](const MvSum<T>& c, int group) {
            const uint16_t raw_top = scales_top[group], raw_bottom = scales_bottom[group];
            const float st = ToFloat(*reinterpret_cast<const T*>(&raw_top)), sb = ToFloat(*reinterpret_cast<const T*>(&raw_bottom));
            acc[0] = fmaf(st, c.Value(0), acc[0]);
            acc[1] = fmaf(st, c.Value(1), acc[1]);
            acc[2] = fmaf(sb, c.Value(2), acc[2]);
            acc[3] = fmaf(sb, c.Value(3), acc[3]);
          };
          MvSum<T> c;
#pragma unroll
          for (int h = 0; h < kMvBox / 64; ++h) {
            if (h >= halves) break;
            uint2 wt, wb;
            const uint32_t place = ((2 * h + (t >> 1)) ^ swizzle) * 16 + (t & 1) * 8;
            asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(wt.x), "=r"(wt.y) : "r"(box + top * 128 + place));
            asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(wb.x), "=r"(wb.y) : "r"(box + bottom * 128 + place));
            const int unit0 = from / 8 + (h >> 1) * 16, group = (from + h * 64) / kGroup;
            const uint4 bx = x[unit0 + unit_x[h & 1]], by = x[unit0 + unit_y[h & 1]];
            if constexpr (kGroup == 32) {
              Swap(wt, t);
              Swap(wb, t);
              c.Start(make_float2(even[group], odd[group]));
              c.Add(wt.x, wb.x, bx);
              scaled(c, group);
              c.Start(make_float2(even[group + 1], odd[group + 1]));
              c.Add(wt.y, wb.y, by);
              scaled(c, group + 1);
            } else {
              if (kGroup == 64 || (h & 1) == 0) c.Start(make_float2(even[group], odd[group]));
              c.Add(wt.x, wb.x, bx);
              c.Add(wt.y, wb.y, by);
              if (kGroup == 64 || (h & 1) == 1) scaled(c, group);
            }
          }
        }
        __syncwarp();
        if (lane == 0) BarrierArrive(SharedAddress(&s.empty[stage]));
      }
    }
    if (!ok) acc[0] = acc[1] = acc[2] = acc[3] = __uint_as_float(0x7fc00000u);   // a wait gave up: no partial sums
    // acc: this lane's top and bottom row, token rows 2 t and 2 t + 1.
    s.sums[warp][top & 15][2 * t] = acc[0];
    s.sums[warp][top & 15][2 * t + 1] = acc[1];
    s.sums[warp][bottom & 15][2 * t] = acc[2];
    s.sums[warp][bottom & 15][2 * t + 1] = acc[3];
    MvSync();
    for (int i = tid; i < rows * kRows; i += kMvThreads) {
      const int n = i / kRows, row = i % kRows;   // token row, weight row
      if (row0 + row >= a.outer) continue;
      float sum = 0.0f;
#pragma unroll
      for (int q = 0; q < kParts; ++q) sum += s.sums[(row >> 4) * kParts + q][row & 15][n];
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
  if (int64_t{a.experts} * a.outer >= int64_t{1} << 31) throw InvalidArgument("4-bit product is too large");
  const int rows = static_cast<int>(std::min<int64_t>(8, a.entries));
  constexpr int kChunkGroups = kMvChunk / kGroup;
  const int smem = 1024 + kMvStages * kMvStageBytes + rows * (kMvStride * 16 + kChunkGroups * 4) +
                   kRows * (kChunkGroups + 2) * 2;
  const bool vector = a.x_stride % 8 == 0 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0;
  const CUtensorMap map = EncodeBytes(a.codes, a.inner / 2, int64_t{a.experts} * a.outer, 128, kRows);
  AllowShared<Matvec<T, kGroup, kParts>>(smem);
  Matvec<T, kGroup, kParts><<<static_cast<unsigned>(blocks), kMvThreads + 32, smem, stream>>>(a, map, row_blocks, rows, vector);
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

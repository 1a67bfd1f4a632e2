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
// Values that these sums do not hold, infinities or BF16 ones from 2^115 (4e34) on, are
// rare: eight token rows with one among them are computed again, by the formula as
// it stands (MvAgain; 16 tokens to 4 of 64 experts at 4096 x 2048 with an infinity
// each 1.4 ms).  Looking for them costs 0.2 us of a small call, 1 % of a large one.
//
// Two blocks per streaming multiprocessor walk tasks: some weight rows of one
// expert and eight of its token rows.  Eight warps compute: 16-row tiles times
// kParts parts of the deep axis, summed in shared memory in a fixed order.  One
// warp brings the weights by TMA, three 16 KB stages ahead, and four warps lay
// out x and the scales of the next 1024 deep values meanwhile, so that the
// computing warps wait for neither.  (Weights loaded straight into registers
// touch eight rows per instruction: the load path was the bound at twice the
// time.)  An expert's weights are read once for every eight of its rows.
//
// Measured, replayed with three inputs by turns: one token to 8 of 64 experts at
// 2048 x 1024 6.7 us; 16 tokens to 4 of 64 at 4096 x 2048 44 us, 180 MB (4.1 TB/s):
// 656 tasks on 296 blocks are three rounds for 2.2, and the computing warps issue in
// two of three cycles.
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
constexpr int kMvWarps = 8, kMvThreads = kMvWarps * 32;   // computing
constexpr int kMvBox = 256;             // deep values of a row in one box: 128 bytes
constexpr int kMvStages = 3;
constexpr uint32_t kMvStageBytes = 16 * kMvWarps * 128;   // kParts boxes of all the block's rows
constexpr int kMvChunk = 1024;          // deep values of x and of the scales laid out at a time
constexpr int kMvLayout = 128;          // threads that lay them out

// Row stride of x in shared memory, in units of 8 values: 4 more than a
// multiple of 8, so that two rows' 16-byte reads use different banks.
constexpr int kMvStride = kMvChunk / 8 + 4;

// Where unit u (8 values) of a row of x lies: the four lanes that share a
// weight row read units 1 or 2 apart, which this spreads over the banks.
__device__ __forceinline__ int MvUnit(int u) { return u ^ ((u >> 2) & 3); }

// The computing warps' barrier.
__device__ __forceinline__ void MvSync() { asm volatile("bar.sync 1, %0;" ::"n"(kMvThreads) : "memory"); }

// d = a b + c.
template <typename T>
__device__ __forceinline__ void Mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1,
                                    float c2, float c3) {
  if constexpr (std::is_same<T, __half>::value) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
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
  // A word of each of the two weight rows, eight deep values.  The group's
  // first word starts from `excess`, minus what the weights have too much.
  template <bool kFirst>
  __device__ __forceinline__ void Add(uint32_t top, uint32_t bottom, const uint4& x, float2 excess) {
    const float c0 = kFirst ? excess.x : c[0], c1 = kFirst ? excess.y : c[1];
    const float c2 = kFirst ? excess.x : c[2], c3 = kFirst ? excess.y : c[3];
    if constexpr (std::is_same<T, __half>::value) {
      const uint32_t t8 = top >> 8, b8 = bottom >> 8;
      const uint32_t plain[4] = {top & 0x000f000fu, bottom & 0x000f000fu, t8 & 0x000f000fu, b8 & 0x000f000fu};
      const uint32_t times16[4] = {top & 0x00f000f0u, bottom & 0x00f000f0u, t8 & 0x00f000f0u, b8 & 0x00f000f0u};
      Mma<T>(c, plain, x.x, x.z, c0, c1, c2, c3);
      if constexpr (kFirst) Mma<T>(wide, times16, x.y, x.w, 0.0f, 0.0f, 0.0f, 0.0f);
      else Mma<T>(wide, times16, x.y, x.w, wide[0], wide[1], wide[2], wide[3]);
    } else {
      const uint32_t one = 0x00780078u, base = 0x41804180u;
      const uint32_t first[4] = {Mask2(top << 3, one, base), Mask2(bottom << 3, one, base), Mask2(top >> 1, one, base),
                                 Mask2(bottom >> 1, one, base)};
      const uint32_t second[4] = {Mask2(top >> 5, one, base), Mask2(bottom >> 5, one, base), Mask2(top >> 9, one, base),
                                  Mask2(bottom >> 9, one, base)};
      Mma<T>(c, first, x.x, x.y, c0, c1, c2, c3);
      Mma<T>(c, second, x.z, x.w, c[0], c[1], c[2], c[3]);
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

// Added to a 16-bit magnitude it sets the top bit of one that is too large for the
// sums: an infinity or NaN, and of BF16 what 128 weights of up to 31 could take
// past 2^127.  (F16 values that are finite stay far below.)
template <typename T> constexpr uint32_t kMvAbove = std::is_same<T, __half>::value ? 0x0400u : 0x0700u;
template <typename T> __device__ __forceinline__ uint32_t MvAbove(const uint4& q) {
  constexpr uint32_t kMagnitudes = 0x7fff7fffu, kAdd = kMvAbove<T> * 0x10001u;
  return (((q.x & kMagnitudes) + kAdd) | ((q.y & kMagnitudes) + kAdd) | ((q.z & kMagnitudes) + kAdd) |
          ((q.w & kMagnitudes) + kAdd)) & 0x80008000u;
}

// Groups of 32: lanes t and t ^ 2 swap a word, so that each of a half's two
// groups is spread over the four lanes and a matrix instruction stays in one.
__device__ __forceinline__ void Swap(uint2& w, int t) {
  const bool high = (t & 2) != 0;
  const uint32_t other = __shfl_xor_sync(kFull, high ? w.x : w.y, 2);
  if (high) w.x = other; else w.y = other;
}

struct MvShared {
  uint64_t full[kMvStages], empty[kMvStages], laid[2], used[2], seen, stored;
  volatile int failed;
  volatile int above;                // x has values too large for the sums
  int present;                       // experts that have rows
  int experts[kRouteMaxExperts];     // and which
  float sums[kMvWarps][16][9];
};

// One task: kRows weight rows from row0 of an expert, token rows [begin, end).
struct MvTask {
  int64_t first, begin, end;   // first: the expert's first weight row
  int row0;
};

// One of four warps: its share of a task's weight rows times eight token rows, if
// one of these has a value that is too large for the sums, by the formula as it
// stands and straight from memory.  Lanes take every 32nd eight of the deep values.
template <typename T, int kGroup, int kRows>
__device__ __forceinline__ void MvAgain(const MatvecArgs& a, const MvTask& task, int64_t p0, int warp) {
  const int lane = threadIdx.x & 31, groups = a.inner / kGroup, rows = static_cast<int>(min(int64_t{8}, task.end - p0));
  const uint16_t* mine = nullptr;   // lane n: token row n, null if there is none
  if (lane < rows) {
    const int64_t token = a.gather != 0 ? a.rows[p0 + lane] / a.top_k : p0 + lane;
    if (token >= 0 && token < a.x_rows) mine = static_cast<const uint16_t*>(a.x) + token * a.x_stride;
  }
  uint32_t above = 0;
#pragma unroll 1
  for (int n = 0; n < rows; ++n) {
    const uint16_t* x = reinterpret_cast<const uint16_t*>(__shfl_sync(kFull, reinterpret_cast<unsigned long long>(mine), n));
    if (x == nullptr) continue;
#pragma unroll 1
    for (int k = lane; k < a.inner; k += 32) above |= ((x[k] & 0x7fffu) + kMvAbove<T>) & 0x8000u;
  }
  if (!__any_sync(kFull, above != 0u)) return;
#pragma unroll 1
  for (int row = task.row0 + warp; row < min(task.row0 + kRows, a.outer); row += kMvLayout / 32) {
    const uint32_t* codes = reinterpret_cast<const uint32_t*>(a.codes + (task.first + row) * (a.inner / 2));
    const T* scales = static_cast<const T*>(a.scales) + (task.first + row) * groups;
#pragma unroll 1
    for (int n = 0; n < rows; ++n) {
      const uint16_t* x = reinterpret_cast<const uint16_t*>(__shfl_sync(kFull, reinterpret_cast<unsigned long long>(mine), n));
      float sum = 0.0f;
#pragma unroll 1
      for (int u = lane; u < a.inner / 8 && x != nullptr; u += 32) {
        const uint32_t word = codes[u];
        const float scale = ToFloat(scales[u / (kGroup / 8)]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {   // weights are exact in 32 bits
          sum = fmaf(static_cast<float>(static_cast<int>((word >> (4 * i)) & 15u) - 8) * scale, Unpack2<T>(x[u * 8 + i]).x, sum);
        }
      }
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kFull, sum, d);
      if (lane == 0) static_cast<T*>(a.out)[(p0 + n) * a.outer + row] = FromFloat<T>(sum);
    }
  }
}

template <typename T, int kGroup, int kParts>
__global__ void __launch_bounds__(kMvThreads + 32 + kMvLayout, 2)
    Matvec(MatvecArgs a, const __grid_constant__ CUtensorMap map, int row_blocks, int max_rows, bool vector,
           bool vector_scales) {
  constexpr int kRows = 16 * kMvWarps / kParts;   // weight rows of a task
  constexpr int kSpan = kParts * kMvBox;          // deep values of a stage
  constexpr int kChunkGroups = kMvChunk / kGroup, kScaleStride = kChunkGroups + 2;
  extern __shared__ unsigned char mv_raw[];
  __shared__ MvShared s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t ring = (SharedAddress(mv_raw) + 1023u) & ~1023u;
  // Two of each: x [token row][unit], its sums [pair of token rows][group][2], scales [weight row][group].
  uint4* x_values = reinterpret_cast<uint4*>(mv_raw + (ring - SharedAddress(mv_raw)) + kMvStages * kMvStageBytes);
  const int x_size = max_rows * kMvStride, sum_size = (max_rows + 1) / 2 * 2 * kChunkGroups;
  float* x_sums = reinterpret_cast<float*>(x_values + 2 * x_size);
  uint16_t* scales = reinterpret_cast<uint16_t*>(x_sums + 2 * sum_size);
  LetNextStart();
  if (tid == 0) {
    for (int i = 0; i < kMvStages; ++i) {
      BarrierInit(SharedAddress(&s.full[i]), 1);
      BarrierInit(SharedAddress(&s.empty[i]), kMvWarps);
    }
    for (int i = 0; i < 2; ++i) {
      BarrierInit(SharedAddress(&s.laid[i]), kMvLayout);
      BarrierInit(SharedAddress(&s.used[i]), kMvWarps);
    }
    s.failed = 0;
    BarrierInit(SharedAddress(&s.seen), kMvLayout / 32);
    BarrierInit(SharedAddress(&s.stored), kMvWarps);
    s.above = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid == 32) PrefetchMap(&map);
  WaitForPrevious();
  if (warp == 0) {
    int seen = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
      const int e = e0 + lane;
      const bool some = e < a.experts && RowBound(a.offsets[e + 1], a.entries) > RowBound(a.offsets[e], a.entries);
      const uint32_t present = __ballot_sync(kFull, some);
      if (some) s.experts[seen + __popc(present & ((1u << lane) - 1))] = e;
      seen += __popc(present);
    }
    if (lane == 0) s.present = seen;
  }
  __syncthreads();
  const int tasks = s.present * row_blocks;
  const auto task_at = [&](int index) {
    const int which = index / row_blocks, e = s.experts[which];
    MvTask task;
    task.row0 = (index - which * row_blocks) * kRows;
    task.first = int64_t{e} * a.outer;
    task.begin = RowBound(a.offsets[e], a.entries);
    task.end = RowBound(a.offsets[e + 1], a.entries);
    return task;
  };

  if (warp == kMvWarps) {   // weights: one thread
    if (lane != 0) return;
    const int spans = (a.inner + kSpan - 1) / kSpan;
    uint32_t fill = 0;
    bool ok = true;
    for (int index = blockIdx.x; index < tasks && ok; index += gridDim.x) {
      const MvTask task = task_at(index);
      for (int64_t p0 = task.begin; p0 < task.end && ok; p0 += 8) {
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
                      (span * kSpan + box * kMvBox) / 2, static_cast<int>(task.first) + task.row0);
          }
        }
      }
    }
    // Whoever gives up, the copies in flight land before the block ends.
    for (uint32_t f = fill - min(fill, static_cast<uint32_t>(kMvStages)); f < fill; ++f) {
      BarrierWait(SharedAddress(&s.full[f % kMvStages]), (f / kMvStages) & 1, nullptr);
    }
    return;
  }

  const int groups = a.inner / kGroup;
  if (warp > kMvWarps) {
    // x of a task's token rows in the order the tensor cores take the weights'
    // nibbles, its sums by group, and the weight rows' scales.
    const int lt = tid - kMvThreads - 32;
    {   // rows without an expert: zeros
      const int64_t from = RowBound(a.offsets[a.experts], a.entries) * a.outer, to = a.entries * int64_t{a.outer};
      T* out = static_cast<T*>(a.out);
      for (int64_t i = from + int64_t{blockIdx.x} * kMvLayout + lt; i < to; i += int64_t{gridDim.x} * kMvLayout) {
        out[i] = FromFloat<T>(0.0f);
      }
    }
    uint32_t turn = 0, above = 0;
    for (int index = blockIdx.x; index < tasks; index += gridDim.x) {
      const MvTask task = task_at(index);
      const uint16_t* source = static_cast<const uint16_t*>(a.scales) + (task.first + task.row0) * groups;
      const int weight_rows = min(kRows, a.outer - task.row0);
      for (int64_t p0 = task.begin; p0 < task.end; p0 += 8) {
        const int rows = static_cast<int>(min(int64_t{max_rows}, task.end - p0));
        int64_t token = -1;   // lane n: x's row of token row n, -1 if there is none
        if (lane < rows) {
          token = a.gather != 0 ? a.rows[p0 + lane] / a.top_k : p0 + lane;
          if (token >= a.x_rows) token = -1;
        }
        for (int k0 = 0; k0 < a.inner; k0 += kMvChunk, ++turn) {
          const uint32_t buffer = turn & 1;
          if (turn >= 2) {
            const bool ok = BarrierWait(SharedAddress(&s.used[buffer]), ((turn >> 1) + 1) & 1, &s.failed);
            if (!__all_sync(kFull, ok)) return;
          }
          uint4* x_out = x_values + buffer * x_size;
          float* sum_out = x_sums + buffer * sum_size;
          uint16_t* scale_out = scales + buffer * (kRows * kScaleStride);
          const int units = (min(kMvChunk, a.inner - k0) + 127) / 128 * 16;
          const int chunk_groups = min(kChunkGroups, groups - k0 / kGroup);
          // Loads first, as many at once as there are registers for.
          constexpr int kQuads = kChunkGroups / 4, kStep = kMvLayout / kQuads, kLoads = (kRows + kStep - 1) / kStep;
          const int quad = lt % kQuads;
          uint2 quads[kLoads < 8 ? kLoads : 8];
          const auto fetch_quads = [&](int from) {
#pragma unroll
            for (int i = 0; i < (kLoads < 8 ? kLoads : 8); ++i) {
              const int row = lt / kQuads + (from + i) * kStep;
              quads[i] = make_uint2(0u, 0u);
              if (quad * 4 < chunk_groups && row < weight_rows) {
                quads[i] = *reinterpret_cast<const uint2*>(source + row * int64_t{groups} + k0 / kGroup + quad * 4);
              }
            }
          };
          const auto store_quads = [&](int from) {
#pragma unroll
            for (int i = 0; i < (kLoads < 8 ? kLoads : 8); ++i) {
              const int row = lt / kQuads + (from + i) * kStep;
              if (row >= kRows) break;
              uint32_t* to = reinterpret_cast<uint32_t*>(scale_out + row * kScaleStride + quad * 4);
              to[0] = quads[i].x;
              to[1] = quads[i].y;
            }
          };
          if (vector_scales) {
            fetch_quads(0);
          } else {
            for (int i = lt; i < kRows * kChunkGroups; i += kMvLayout) {
              const int row = i / kChunkGroups, group = i % kChunkGroups;
              const bool inside = group < chunk_groups && row < weight_rows;
              scale_out[row * kScaleStride + group] = inside ? source[row * int64_t{groups} + k0 / kGroup + group] : 0;
            }
          }
          constexpr int kUnits = kMvChunk / 8 / kMvLayout;   // of a row, per thread
          for (int n0 = 0; n0 < rows; n0 += 2) {
            uint4 v[2][kUnits];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              const int64_t r = __shfl_sync(kFull, token, n0 + n);
              const T* x = static_cast<const T*>(a.x) + r * a.x_stride + k0;
#pragma unroll
              for (int i = 0; i < kUnits; ++i) {
                const int u = i * kMvLayout + lt;
                v[n][i] = make_uint4(0u, 0u, 0u, 0u);
                if (r >= 0 && k0 + u * 8 < a.inner) {   // 8 divides inner
                  if (vector) {
                    v[n][i] = *reinterpret_cast<const uint4*>(x + u * 8);
                  } else {
                    const uint16_t* bits = reinterpret_cast<const uint16_t*>(x + u * 8);
                    uint32_t w[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j] = bits[j];
                    v[n][i] = make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
                  }
                }
              }
            }
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              if (n0 + n >= rows) break;
#pragma unroll
              for (int i = 0; i < kUnits; ++i) {
                const int u = i * kMvLayout + lt;
                const uint4 q = v[n][i];
                above |= MvAbove<T>(q);
                const float2 f0 = Unpack2<T>(q.x), f1 = Unpack2<T>(q.y), f2 = Unpack2<T>(q.z), f3 = Unpack2<T>(q.w);
                float sum = ((f0.x + f0.y) + (f1.x + f1.y)) + ((f2.x + f2.y) + (f3.x + f3.y));
#pragma unroll
                for (int d = kGroup / 16; d > 0; d >>= 1) sum += __shfl_xor_sync(kFull, sum, d);
                if (u < units) {   // units are a multiple of 16: whole groups
                  x_out[(n0 + n) * kMvStride + MvUnit(u)] =
                      make_uint4(__byte_perm(q.x, q.z, 0x5410), __byte_perm(q.x, q.z, 0x7632),
                                 __byte_perm(q.y, q.w, 0x5410), __byte_perm(q.y, q.w, 0x7632));
                  if (u % (kGroup / 8) == 0) {
                    sum_out[(((n0 + n) >> 1) * kChunkGroups + u / (kGroup / 8)) * 2 + (n & 1)] = kMvExcess<T> * sum;
                  }
                }
              }
            }
          }
          if (vector_scales) {
            store_quads(0);
            if constexpr (kLoads > 8) {
#pragma unroll 1
              for (int from = 8; from < kLoads; from += 8) {
                fetch_quads(from);
                store_quads(from);
              }
            }
          }
          BarrierArrive(SharedAddress(&s.laid[buffer]));
        }
      }
    }
    // Token rows with values too large for the sums: again, over what the computing
    // warps have stored by then.
    if (__any_sync(kFull, above != 0u) && lane == 0) s.above = 1;
    __syncwarp();
    if (lane == 0) BarrierArrive(SharedAddress(&s.seen));
    bool all = BarrierWait(SharedAddress(&s.seen), 0, &s.failed);
    if (!__all_sync(kFull, all) || s.above == 0) return;
    all = BarrierWait(SharedAddress(&s.stored), 0, &s.failed);
    if (!__all_sync(kFull, all)) return;
    for (int index = blockIdx.x; index < tasks; index += gridDim.x) {
      const MvTask task = task_at(index);
      for (int64_t p0 = task.begin; p0 < task.end; p0 += 8) MvAgain<T, kGroup, kRows>(a, task, p0, lt >> 5);
    }
    return;
  }

  const int g = lane >> 2, t = lane & 3, part = warp % kParts, tile = warp / kParts;
  // Rows of the tile in the tensor cores' order: lanes that read together take
  // every second row, whose swizzled 16-byte places differ.
  const int top = tile * 16 + 2 * (g & 3) + (g >> 2), bottom = top + 8;
  const uint32_t swizzle = static_cast<uint32_t>(top & 7);
  // Units of x that multiply a half's (64 deep values) words x and y, for even and odd halves.
  int unit_x[2], unit_y[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    unit_x[h] = MvUnit(8 * h + (kGroup == 32 ? 2 * (t & 1) + (t >> 1) : 2 * t));
    unit_y[h] = MvUnit(8 * h + (kGroup == 32 ? 4 + 2 * (t & 1) + (t >> 1) : 2 * t + 1));
  }
  uint32_t fill = 0, turn = 0;
  bool ok = true;
  for (int index = blockIdx.x; index < tasks; index += gridDim.x) {
    const MvTask task = task_at(index);
    for (int64_t p0 = task.begin; p0 < task.end; p0 += 8) {
      const int rows = static_cast<int>(min(int64_t{max_rows}, task.end - p0));
      float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int k0 = 0; k0 < a.inner; k0 += kMvChunk, ++turn) {
        const uint32_t buffer = turn & 1;
        ok = ok && BarrierWait(SharedAddress(&s.laid[buffer]), (turn >> 1) & 1, &s.failed);
        const uint4* x = x_values + buffer * x_size + (g < rows ? g : 0) * kMvStride;
        const float2* excess = reinterpret_cast<const float2*>(x_sums + buffer * sum_size) + (2 * t < rows ? t : 0) * kChunkGroups;
        const uint16_t* scales_top = scales + buffer * (kRows * kScaleStride) + top * kScaleStride;
        const uint16_t* scales_bottom = scales_top + 8 * kScaleStride;
        const int last = min(a.inner, k0 + kMvChunk);
        for (int k1 = k0; k1 < last; k1 += kSpan, ++fill) {
          const uint32_t stage = fill % kMvStages;
          ok = ok && BarrierWait(SharedAddress(&s.full[stage]), (fill / kMvStages) & 1, &s.failed);
          ok = __all_sync(kFull, ok);
          const int k = k1 + part * kMvBox;
          if (ok && k < last) {
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
                c.template Add<true>(wt.x, wb.x, bx, excess[group]);
                scaled(c, group);
                c.template Add<true>(wt.y, wb.y, by, excess[group + 1]);
                scaled(c, group + 1);
              } else {
                if (kGroup == 64 || (h & 1) == 0) c.template Add<true>(wt.x, wb.x, bx, excess[group]);
                else c.template Add<false>(wt.x, wb.x, bx, float2{});
                c.template Add<false>(wt.y, wb.y, by, float2{});
                if (kGroup == 64 || (h & 1) == 1) scaled(c, group);
              }
            }
          }
          __syncwarp();
          if (lane == 0) BarrierArrive(SharedAddress(&s.empty[stage]));
        }
        if (lane == 0) BarrierArrive(SharedAddress(&s.used[buffer]));
      }
      if (!ok) acc[0] = acc[1] = acc[2] = acc[3] = __uint_as_float(0x7fc00000u);   // a wait gave up: no partial sums
      // acc: this lane's top and bottom row, token rows 2 t and 2 t + 1.
      if (kParts == 1) __syncwarp(); else MvSync();
      s.sums[warp][top & 15][2 * t] = acc[0];
      s.sums[warp][top & 15][2 * t + 1] = acc[1];
      s.sums[warp][bottom & 15][2 * t] = acc[2];
      s.sums[warp][bottom & 15][2 * t + 1] = acc[3];
      T* out = static_cast<T*>(a.out) + p0 * a.outer + task.row0;
      if constexpr (kParts == 1) {   // a warp has its rows to itself
        __syncwarp();
        const int row = lane & 15;
        for (int n = lane >> 4; n < rows && task.row0 + tile * 16 + row < a.outer; n += 2) {
          out[n * int64_t{a.outer} + tile * 16 + row] = FromFloat<T>(s.sums[warp][row][n] * kMvSize<T>);
        }
      } else {
        MvSync();
        for (int i = tid; i < rows * kRows; i += kMvThreads) {
          const int n = i / kRows, row = i % kRows;   // token row, weight row
          if (task.row0 + row >= a.outer) continue;
          float sum = 0.0f;
#pragma unroll
          for (int q = 0; q < kParts; ++q) sum += s.sums[(row >> 4) * kParts + q][row & 15][n];
          out[n * int64_t{a.outer} + row] = FromFloat<T>(sum * kMvSize<T>);
        }
      }
    }
  }
  __syncwarp();
  if (lane == 0) BarrierArrive(SharedAddress(&s.stored));
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
  const int smem = 1024 + kMvStages * kMvStageBytes +
                   2 * (rows * kMvStride * 16 + (rows + 1) / 2 * 2 * kChunkGroups * 4 + kRows * (kChunkGroups + 2) * 2);
  const bool vector = a.x_stride % 8 == 0 && reinterpret_cast<uintptr_t>(a.x) % 16 == 0;
  const bool vector_scales = a.inner / kGroup % 4 == 0 && reinterpret_cast<uintptr_t>(a.scales) % 8 == 0;
  const CUtensorMap map = EncodeBytes(a.codes, a.inner / 2, int64_t{a.experts} * a.outer, 128, kRows);
  AllowShared<Matvec<T, kGroup, kParts>>(smem);
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(blocks, RoutedSmCount() * 2));
  LaunchRouted("4-bit product launch", BriefGrid(blocks), Matvec<T, kGroup, kParts>, grid, kMvThreads + 32 + kMvLayout, smem, stream, a, map,
               row_blocks, rows, vector, vector_scales);
}

template <typename T, int kGroup>
void ByParts(const MatvecArgs& a, cudaStream_t stream) {
  // Fewer parts read longer runs of the deep axis per warp; more parts give
  // more blocks.  Replayed, with 1, 2 and 4 parts, tokens to top_k of experts:
  //    1 to 8 of  64, 2048 x 1024:  10.2   8.7   6.5 us (4 taken)
  //    4 to 8 of  64, 2048 x 1024:  15.1  14.9  16.7    (4)
  //    8 to 4 of  32, 4096 x 2048:  37.2  38.3  42.3    (2)
  //    8 to 8 of 128, 2048 x 1024:  25.1  25.8  28.1    (2)
  //   16 to 4 of  64, 4096 x 2048:  43.4  47.5  61.3    (1)
  //   16 to 8 of 128, 2048 x 1024:  33.0  35.0  42.8    (1)
  // It goes by blocks and not by the rounds they make: 64 tokens to 1 of 16 at
  // 4096 x 1500 take 36.3 us with 2 parts and 47.5 with the 4 taken.
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

// Routed products on the tcgen05 tensor cores, for operands whose rows start
// on 16-byte boundaries.
//
// A block owns one streaming multiprocessor and walks 128 x kWide output
// tiles.  Warp 0 loads 64-deep slices into a ring of shared-memory stages by
// TMA.  One thread of warp 1 issues the matrix instructions into one of two
// accumulators in tensor memory, and warps 2 to 5 round and store the other one
// meanwhile.  Where rows are gathered, warps 6 to 13 copy them by their indices
// with 16-byte asynchronous copies, straight from the token rows: no ordered
// copy of the input is made.  (TMA's own four-row gather was measured at about
// 100 cycles an instruction, 512 bytes each: 1.8 us a slice against 0.28 us of
// matrix instructions.  Four copying warps took 348 us for a weight gradient with
// gathered y where eight take 303, and one microsecond longer for small calls;
// sixteen were slower again.)
//
//   product:     A = rows of x (deep-major), B = W[e] as it lies (wide-major)
//   transposed:  A = rows of x (deep-major), B = W[e]^T: W[e] as it lies (deep-major)
//   weight grad: A = x^T, B = y: rows are the deep axis, both as they lie (wide-major)
//
// A tile's rows past its expert's last are computed from whatever lies in
// shared memory and not stored (experts with few rows load few).  In the weight
// gradient they would enter the sum: the matrix warp zeroes them in shared
// memory, in both operands, so that a value that is not finite stays with its
// own expert.
//
// Measured, bf16, replayed with three inputs by turns: 32768 rows of 64 experts,
// 1024 x 2048, 136 us (1.0 PFLOP/s, 0.61 of the matrix rate; every second expert's
// last tile is half empty); of 32 experts at 2048 x 2048 223 us (1.23 PFLOP/s),
// transposed 248; that weight gradient 245 us, with gathered rows 272 (x) or 309 (y).
// 9222 rows of 40 experts at 1000 x 1416 57 us, where reading the weights takes 17.
// What bounds: the slices' latency against four stages, and at few rows per expert
// the weights' bytes.
// Slower: two blocks sharing 256 x 256 tiles (cta_group::2), 265 us where this
// took 232, for the tiles' empty halves and the blocks' handshakes; eight storing
// warps, 34 us instead of 30 for the weight gradient of 64 rows of 32 experts,
// 2048 x 1024, and no gain for large ones.
#include <algorithm>

#include "engine.h"
#include "layout.h"
#include "routed.cuh"
#include "routed.h"
#include "tcgen05.cuh"
#include "tensor_map.h"

namespace t0b {
namespace {

constexpr int kTileRows = 128, kDeep = 64, kRowBox = 32;   // kRowBox: rows of x that one copy brings
constexpr int kTcThreads = 192, kGatherThreads = 256;      // roles; copying threads where rows are gathered
constexpr int kGatherRows = kGatherThreads / 8;            // rows that they copy at a time
constexpr uint32_t kSwizzleRow = 128;                      // bytes of 64 16-bit values
constexpr uint32_t kABytes = kTileRows * kSwizzleRow;      // one stage of A
constexpr uint32_t kBlockBytes = kDeep * kSwizzleRow;      // 64 x 64 values
constexpr int kMaxStages = 8;
constexpr uint32_t kStagingBytes = 32 * kSwizzleRow;       // of one storing warp

struct TcArgs {
  // a_few: products, kRowBox rows at a time.  Wide-major operands whose width
  // is whole blocks of 64 columns have one box for all of a tile's blocks
  // (blocked): a copy costs by its number as well as by its bytes.
  CUtensorMap a, a_few, b;
  int a_blocked, b_blocked;
  const uint16_t *a_data, *b_data;   // gathered operands
  int64_t a_rows, a_stride, b_rows, b_stride;
  const int32_t* rows;
  const int32_t* offsets;
  void* out;
  int64_t entries;
  int experts, top_k, inner, outer;
  int gather_a, gather_b, bf16;
};

template <int kWide>
struct TcShape {
  static constexpr uint32_t kBBytes = kWide * kSwizzleRow;
  static constexpr uint32_t kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = kWide == 256 ? 4 : kWide == 128 ? 6 : 8;
  static constexpr uint32_t kRing = kStages * kStageBytes;
};

struct TcShared {
  uint64_t full[kMaxStages], empty[kMaxStages], done[2], drained[2], drain;
  uint32_t tmem;
  volatile int failed;
  int row_begin[kRouteMaxExperts + 1];
  int tile_begin[kRouteMaxExperts + 1];
};

// Where a tile lies: output rows [m0, m0 + 128) of expert e (of its rows, or
// of `inner` in the weight gradient), columns from n0.
struct TcTile {
  int e, m0, n0, rows;   // rows: what the expert has of the tile axis
  int begin, count;      // the expert's first row and its rows
};

template <int kKind, int kWide>
struct TcWalk {
  const TcArgs& a;
  const TcShared& s;
  int e = 0;
  __device__ TcWalk(const TcArgs& args, const TcShared& shared) : a(args), s(shared) {}
  __device__ TcTile At(int tile) {
    while (s.tile_begin[e + 1] <= tile) ++e;
    TcTile t;
    t.e = e;
    t.begin = s.row_begin[e];
    t.count = max(0, s.row_begin[e + 1] - t.begin);
    t.rows = kKind == kProductWeightGrad ? a.inner : t.count;
    const int local = tile - s.tile_begin[e], tiles_m = (t.rows + kTileRows - 1) / kTileRows;
    t.m0 = local % tiles_m * kTileRows;
    t.n0 = local / tiles_m * kWide;
    return t;
  }
  __device__ int Slices(const TcTile& t) const {
    const int deep = kKind == kProductWeightGrad ? t.count : kKind == kProduct ? a.inner : a.outer;
    return (deep + kDeep - 1) / kDeep;
  }
};

// Copies 16 bytes of row `r` into a swizzled tile of 128-byte rows, chunk c of
// eight; zeros if !inside.
__device__ __forceinline__ void CopyChunk(uint32_t tile, int r, int c, const uint16_t* source, bool inside) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
               ::"r"(tile + r * kSwizzleRow + ((c ^ (r & 7)) << 4)), "l"(source), "r"(inside ? 16 : 0) : "memory");
}

template <int kKind, int kWide, bool kGather>
__global__ void __launch_bounds__(kTcThreads + (kGather ? kGatherThreads : 0), 1) TcProduct(const __grid_constant__ TcArgs a) {
  using Shape = TcShape<kWide>;
  extern __shared__ unsigned char tc_raw[];
  __shared__ TcShared s;
  const uint32_t ring = (SharedAddress(tc_raw) + 1023u) & ~1023u;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int width = kKind == kProductTransposed ? a.inner : a.outer;
  const int tiles_n = (width + kWide - 1) / kWide;
  constexpr uint32_t kTmemColumns = 2 * kWide;

  LetNextStart();
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(SharedAddress(&s.tmem)),
                 "r"(kTmemColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (tid == 0) {
    for (int i = 0; i < Shape::kStages; ++i) {
      BarrierInit(SharedAddress(&s.full[i]), 1 + (kGather ? kGatherThreads : 0));
      BarrierInit(SharedAddress(&s.empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      BarrierInit(SharedAddress(&s.done[i]), 1);
      BarrierInit(SharedAddress(&s.drained[i]), 128);
    }
    BarrierInit(SharedAddress(&s.drain), 1);
    s.failed = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid == 32) {   // a gathered operand has no map
    if (!kGather || a.gather_a == 0) PrefetchMap(&a.a);
    if (!kGather || a.gather_b == 0) PrefetchMap(&a.b);
  }
  WaitForPrevious();
  for (int e = tid; e <= a.experts; e += blockDim.x) {
    s.row_begin[e] = static_cast<int>(RowBound(a.offsets[e], a.entries));
  }
  __syncthreads();
  if (warp == 0) {   // tiles before each expert
    int carry = 0;
    for (int e0 = 0; e0 < a.experts; e0 += 32) {
      const int e = e0 + lane;
      int tiles = 0;
      if (e < a.experts) {
        const int rows = kKind == kProductWeightGrad ? a.inner : max(0, s.row_begin[e + 1] - s.row_begin[e]);
        tiles = (rows + kTileRows - 1) / kTileRows * tiles_n;
      }
      int sum = tiles;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += other;
      }
      if (e < a.experts) s.tile_begin[e] = carry + sum - tiles;
      carry += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) s.tile_begin[a.experts] = carry;
  }
  TmemFenceBefore();
  __syncthreads();
  TmemFenceAfter();
  const uint32_t tmem = s.tmem;
  const int tiles = s.tile_begin[a.experts];
  TcWalk<kKind, kWide> walk(a, s);

  if (warp == 0) {
    // Loads.  `fill` counts the stages filled since the start.
    uint32_t fill = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
      const TcTile t = walk.At(tile);
      const int slices = walk.Slices(t);
      // Column blocks of 64 that lie in the operand at all.
      const int a_blocks = kKind == kProductWeightGrad ? min(2, (a.inner - t.m0 + 63) / 64) : 1;
      const int b_blocks = min(kWide / 64, (width - t.n0 + 63) / 64);
      const int row_boxes = (min(kTileRows, t.count - t.m0) + kRowBox - 1) / kRowBox;   // products
      const uint32_t a_bytes = kKind != kProductWeightGrad ? row_boxes * (kRowBox * kSwizzleRow)
                               : a.a_blocked != 0          ? kABytes
                                                           : a_blocks * kBlockBytes;
      const uint32_t b_bytes = kKind == kProductTransposed || a.b_blocked != 0 ? Shape::kBBytes : b_blocks * kBlockBytes;
      const bool load_a = !kGather || a.gather_a == 0, load_b = !kGather || a.gather_b == 0;
      const uint32_t bytes = (load_a ? a_bytes : 0) + (load_b ? b_bytes : 0);
      for (int k = 0; k < slices; ++k, ++fill) {
        const int stage = static_cast<int>(fill % Shape::kStages);
        const uint32_t a_smem = ring + stage * Shape::kStageBytes, b_smem = a_smem + kABytes;
        const uint32_t full = SharedAddress(&s.full[stage]);
        const int k0 = k * kDeep;
        if (fill >= Shape::kStages) {
          ok = BarrierWait(SharedAddress(&s.empty[stage]), (fill / Shape::kStages + 1) & 1, &s.failed);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        }
        const bool first = ElectOne();
        if (first) BarrierExpect(full, bytes);
        __syncwarp();
        if constexpr (kKind == kProductWeightGrad) {
          if (load_a) {
            if (a.a_blocked != 0) {
              if (first) LoadTile3(a_smem, &a.a, full, 0, t.begin + k0, t.m0 / 64);
            } else if (lane < a_blocks) {
              LoadTile2(a_smem + lane * kBlockBytes, &a.a, full, t.m0 + lane * 64, t.begin + k0);
            }
          }
          if (load_b) {
            if (a.b_blocked != 0) {
              if (first) LoadTile3(b_smem, &a.b, full, 0, t.begin + k0, t.n0 / 64);
            } else if (lane < b_blocks) {
              LoadTile2(b_smem + lane * kBlockBytes, &a.b, full, t.n0 + lane * 64, t.begin + k0);
            }
          }
        } else {
          if (load_a) {
            if (row_boxes == kTileRows / kRowBox) {
              if (first) LoadTile2(a_smem, &a.a, full, k0, t.begin + t.m0);
            } else if (lane < row_boxes) {
              LoadTile2(a_smem + lane * (kRowBox * kSwizzleRow), &a.a_few, full, k0, t.begin + t.m0 + lane * kRowBox);
            }
          }
          if constexpr (kKind == kProduct) {
            if (a.b_blocked != 0) {
              if (first) LoadTile4(b_smem, &a.b, full, 0, k0, t.n0 / 64, t.e);
            } else if (lane < b_blocks) {
              LoadTile3(b_smem + lane * kBlockBytes, &a.b, full, t.n0 + lane * 64, k0, t.e);
            }
          } else {
            if (first) LoadTile3(b_smem, &a.b, full, k0, t.n0, t.e);
          }
        }
      }
    }
    // Whoever gives up, the copies in flight land before the block ends.
    for (uint32_t f = fill - min(fill, static_cast<uint32_t>(Shape::kStages)); f < fill; ++f) {
      BarrierWait(SharedAddress(&s.full[f % Shape::kStages]), (f / Shape::kStages) & 1, nullptr);
    }
  } else if (warp == 1) {
    // Matrix instructions, issued by one lane.
    constexpr uint32_t a_major = kKind == kProductWeightGrad ? 1u : 0u, b_major = kKind == kProductTransposed ? 0u : 1u;
    const uint32_t format = a.bf16 != 0 ? 1u : 0u;
    const uint32_t idesc = (1u << 4) | (format << 7) | (format << 10) | (a_major << 15) | (b_major << 16) |
                           ((kWide >> 3) << 17) | ((kTileRows >> 4) << 24);
    uint32_t fill = 0, turn = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
      const TcTile t = walk.At(tile);
      const int slices = walk.Slices(t);
      if (slices == 0) continue;
      const uint32_t buffer = turn & 1;
      if (turn >= 2) ok = BarrierWait(SharedAddress(&s.drained[buffer]), ((turn >> 1) + 1) & 1, &s.failed);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      TmemFenceAfter();
      const uint32_t accumulator = tmem + buffer * kWide;
      for (int k = 0; k < slices; ++k, ++fill) {
        const int stage = static_cast<int>(fill % Shape::kStages);
        ok = BarrierWait(SharedAddress(&s.full[stage]), (fill / Shape::kStages) & 1, &s.failed);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        const uint32_t a_smem = ring + stage * Shape::kStageBytes, b_smem = a_smem + kABytes;
        if constexpr (kGather) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        // The last slice: what is left of the sum, in steps of 16.
        const int deep = (kKind == kProductWeightGrad ? t.count : kKind == kProduct ? a.inner : a.outer) - k * kDeep;
        const int steps = min(kDeep, deep + 15) / 16;
        if constexpr (kKind == kProductWeightGrad) {
          if (steps * 16 > deep) {   // rows of the next expert: zero, in every column block of both operands
            for (int block = 0; block < 2 + kWide / 64; ++block) {
              const uint32_t to = a_smem + block * kBlockBytes + steps * (16 * kSwizzleRow);
              for (uint32_t at = to - (steps * 16 - deep) * kSwizzleRow + lane * 16; at < to; at += 512) {
                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
              }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
          }
        }
        TmemFenceAfter();
        if (ElectOne()) {
          const uint64_t left = a_major ? WideMajor(a_smem, kBlockBytes) : DeepMajor(a_smem);
          const uint64_t right = b_major ? WideMajor(b_smem, kBlockBytes) : DeepMajor(b_smem);
          constexpr uint32_t left_step = (a_major ? 16 * kSwizzleRow : 32) >> 4, right_step = (b_major ? 16 * kSwizzleRow : 32) >> 4;
          if (steps == kDeep / 16) {
#pragma unroll
            for (int step = 0; step < kDeep / 16; ++step) {
              MmaHalf(accumulator, left + step * left_step, right + step * right_step, idesc, k == 0 && step == 0 ? 0u : 1u);
            }
          } else {
#pragma unroll 1
            for (int step = 0; step < steps; ++step) {
              MmaHalf(accumulator, left + step * left_step, right + step * right_step, idesc, k == 0 && step == 0 ? 0u : 1u);
            }
          }
          MmaCommit(SharedAddress(&s.empty[stage]));
          if (k == slices - 1) MmaCommit(SharedAddress(&s.done[buffer]));
        }
        __syncwarp();
      }
      ++turn;
    }
    if (!ok) {
      if (ElectOne()) MmaCommit(SharedAddress(&s.drain));
      BarrierWait(SharedAddress(&s.drain), 0, nullptr);
    }
  } else if (warp < 6) {
    // Rounding and stores: a warp has 32 rows of the tile, 64 columns at a time.
    const int quarter = warp & 3;
    const uint32_t staging = ring + Shape::kRing + quarter * kStagingBytes;
    uint16_t* out = static_cast<uint16_t*>(a.out);
    uint32_t turn = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
      const TcTile t = walk.At(tile);
      const bool empty = walk.Slices(t) == 0;
      const uint32_t buffer = turn & 1;
      if (!empty) {
        ok = ok && BarrierWait(SharedAddress(&s.done[buffer]), (turn >> 1) & 1, &s.failed);
        TmemFenceAfter();
      }
      const uint32_t source = tmem + buffer * kWide + (static_cast<uint32_t>(quarter * 32) << 16);
      const int columns = min(kWide, width - t.n0), m0 = t.m0 + quarter * 32;
      uint16_t* rows = out + (kKind == kProductWeightGrad ? static_cast<int64_t>(t.e) * a.inner
                                                          : static_cast<int64_t>(t.begin)) * width;
      for (int c = 0; c < columns; c += 64) {
        uint32_t r[2][32], w[32];
        if (!__all_sync(0xffffffffu, ok)) {   // a wait gave up: no partial sums
          ok = false;
#pragma unroll
          for (int i = 0; i < 32; ++i) w[i] = 0x7fff7fffu;
        } else if (empty) {
#pragma unroll
          for (int i = 0; i < 32; ++i) w[i] = 0u;
        } else {
          TmemLoad(source + c, r[0]);
          TmemLoad(source + c + 32, r[1]);
          TmemLoadWait();
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float lo = __uint_as_float(r[i >> 4][(2 * i) & 31]), hi = __uint_as_float(r[i >> 4][(2 * i + 1) & 31]);
            w[i] = a.bf16 != 0 ? Pack2<__nv_bfloat16>(lo, hi) : Pack2<__half>(lo, hi);
          }
        }
        // Through shared memory, so that a store writes whole 128-byte rows.
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};"
                       ::"r"(staging + lane * kSwizzleRow + ((q ^ (lane & 7)) << 4)), "r"(w[4 * q]), "r"(w[4 * q + 1]),
                       "r"(w[4 * q + 2]), "r"(w[4 * q + 3]) : "memory");
        }
        __syncwarp();
        const int column = t.n0 + c + (lane & 7) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = i * 4 + (lane >> 3);
          uint4 v;
          asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                       : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                       : "r"(staging + row * kSwizzleRow + (((lane & 7) ^ (row & 7)) << 4)) : "memory");
          if (m0 + row < t.rows && column < width) {
            *reinterpret_cast<uint4*>(rows + static_cast<int64_t>(m0 + row) * width + column) = v;
          }
        }
      }
      if (!empty) {
        TmemFenceBefore();
        BarrierArrive(SharedAddress(&s.drained[buffer]));
        ++turn;
      }
    }
    if constexpr (kKind != kProductWeightGrad) {   // rows without an expert
      const int64_t from = int64_t{s.row_begin[a.experts]} * width / 8, to = a.entries * width / 8;
      uint4* zeros = reinterpret_cast<uint4*>(a.out);
      for (int64_t i = from + blockIdx.x * 128 + (tid - 64); i < to; i += int64_t{gridDim.x} * 128) {
        zeros[i] = make_uint4(0, 0, 0, 0);
      }
    }
  } else if constexpr (kGather) {
    // Gathered rows: eight threads copy 128 bytes of a row, a thread the same
    // chunk of rows r0, r0 + 32, ...  A thread's arrival at the stage's barrier
    // follows its copies by itself; the matrix warp then orders them before the
    // tensor cores' reads.
    const int g = tid - kTcThreads, c = g & 7, r0 = g >> 3;
    uint32_t fill = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
      const TcTile t = walk.At(tile);
      const int slices = walk.Slices(t), last = t.begin + t.count - 1;
      const int valid = t.count - t.m0;   // rows of the tile (products)
      const uint16_t* source[kTileRows / kGatherRows];   // where they lie
      int next[kDeep / kGatherRows];   // entries of the next slice's rows (weight gradient), used a slice later
      auto slice_rows = [&](int k) {
#pragma unroll
        for (int i = 0; i < kDeep / kGatherRows; ++i) {
          next[i] = a.rows[min(t.begin + k * kDeep + r0 + kGatherRows * i, last)];
        }
      };
      if constexpr (kKind != kProductWeightGrad) {
#pragma unroll
        for (int i = 0; i < kTileRows / kGatherRows; ++i) {
          const int64_t row = a.rows[min(t.begin + t.m0 + r0 + kGatherRows * i, last)] / a.top_k;
          source[i] = a.a_data + (row >= 0 && row < a.a_rows ? row : 0) * a.a_stride + c * 8;
        }
      } else if (slices > 0) {
        slice_rows(0);
      }
      for (int k = 0; k < slices; ++k, ++fill) {
        const int stage = static_cast<int>(fill % Shape::kStages);
        const uint32_t a_smem = ring + stage * Shape::kStageBytes, b_smem = a_smem + kABytes;
        if (fill >= Shape::kStages) {
          ok = BarrierWait(SharedAddress(&s.empty[stage]), (fill / Shape::kStages + 1) & 1, &s.failed);
          if (!ok) break;
        }
        if constexpr (kKind != kProductWeightGrad) {
          const int deep = kKind == kProduct ? a.inner : a.outer;
          const bool inside = k * kDeep + c * 8 < deep;
#pragma unroll
          for (int i = 0; i < kTileRows / kGatherRows; ++i) {
            const int r = r0 + kGatherRows * i;
            if (r < valid) CopyChunk(a_smem, r, c, inside ? source[i] + k * kDeep : a.a_data, inside);
          }
        } else {
          int64_t row[kDeep / kGatherRows];
#pragma unroll
          for (int i = 0; i < kDeep / kGatherRows; ++i) row[i] = next[i] / a.top_k;
          if (k + 1 < slices) slice_rows(k + 1);
          auto copy = [&](uint32_t tile_smem, const uint16_t* data, int64_t rows, int64_t stride, int column, int columns,
                          int blocks) {
            const uint16_t* from[kDeep / kGatherRows];   // null: no such row
#pragma unroll
            for (int i = 0; i < kDeep / kGatherRows; ++i) {
              from[i] = row[i] >= 0 && row[i] < rows ? data + row[i] * stride + column + c * 8 : nullptr;
            }
            for (int block = 0; block < blocks; ++block) {
              const bool in_row = column + block * 64 + c * 8 < columns;
#pragma unroll
              for (int i = 0; i < kDeep / kGatherRows; ++i) {
                const bool inside = in_row && from[i] != nullptr;
                CopyChunk(tile_smem + block * kBlockBytes, r0 + kGatherRows * i, c, inside ? from[i] + block * 64 : data,
                          inside);
              }
            }
          };
          if (a.gather_a != 0) copy(a_smem, a.a_data, a.a_rows, a.a_stride, t.m0, a.inner, 2);
          if (a.gather_b != 0) copy(b_smem, a.b_data, a.b_rows, a.b_stride, t.n0, a.outer, kWide / 64);
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];"
                     ::"r"(SharedAddress(&s.full[stage])) : "memory");
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  TmemFenceBefore();
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemColumns));
  }
}

template <int kKind, int kWide, bool kGather>
void LaunchTc(const ProductArgs& p, bool bf16, int64_t tiles, int sms, cudaStream_t stream) {
  using Shape = TcShape<kWide>;
  TcArgs a{};
  const int x_width = kKind == kProductTransposed ? p.outer : p.inner;
  if (p.gather_x == 0) {
    if constexpr (kKind == kProductWeightGrad) {
      a.a_blocked = p.inner % 64 == 0 ? 1 : 0;
      a.a = a.a_blocked != 0 ? EncodeBlocks(bf16, p.x, p.inner, p.x_rows, 0, p.x_stride, 0, kDeep, kTileRows / 64)
                             : EncodeHalves(bf16, p.x, p.inner, p.x_rows, 0, p.x_stride, 0, kDeep);
    } else {
      a.a = EncodeHalves(bf16, p.x, x_width, p.x_rows, 0, p.x_stride, 0, kTileRows);
      a.a_few = EncodeHalves(bf16, p.x, x_width, p.x_rows, 0, p.x_stride, 0, kRowBox);
    }
  }
  const int64_t matrix = int64_t{p.inner} * p.outer;
  a.b_blocked = kKind != kProductTransposed && p.outer % 64 == 0 ? 1 : 0;
  if constexpr (kKind == kProductWeightGrad) {
    if (p.gather_w != 0) a.b_blocked = 0;
    else if (a.b_blocked != 0) a.b = EncodeBlocks(bf16, p.w, p.outer, p.w_rows, 0, p.w_stride, 0, kDeep, kWide / 64);
    else a.b = EncodeHalves(bf16, p.w, p.outer, p.w_rows, 0, p.w_stride, 0, kDeep);
  } else if (a.b_blocked != 0) {
    a.b = EncodeBlocks(bf16, p.w, p.outer, p.inner, p.experts, p.outer, matrix, kDeep, kWide / 64);
  } else {
    a.b = EncodeHalves(bf16, p.w, p.outer, p.inner, p.experts, p.outer, matrix, kKind == kProduct ? kDeep : kWide);
  }
  a.a_data = static_cast<const uint16_t*>(p.x);
  a.a_rows = p.x_rows;
  a.a_stride = p.x_stride;
  a.b_data = static_cast<const uint16_t*>(p.w);
  a.b_rows = p.w_rows;
  a.b_stride = p.w_stride;
  a.rows = p.rows;
  a.offsets = p.offsets;
  a.out = p.out;
  a.entries = p.entries;
  a.experts = p.experts;
  a.top_k = p.top_k;
  a.inner = p.inner;
  a.outer = p.outer;
  a.gather_a = p.gather_x;
  a.gather_b = p.gather_w;
  a.bf16 = bf16 ? 1 : 0;
  constexpr int smem = static_cast<int>(Shape::kRing + 4 * kStagingBytes) + 1024;
  AllowShared<TcProduct<kKind, kWide, kGather>>(smem);
  const unsigned grid = static_cast<unsigned>(std::max<int64_t>(1, std::min<int64_t>(tiles, sms)));
  LaunchRouted("routed product launch", tiles <= sms, TcProduct<kKind, kWide, kGather>, grid,
               kTcThreads + (kGather ? kGatherThreads : 0), smem, stream, a);
}

template <int kKind>
void ByWidth(const ProductArgs& p, bool bf16, cudaStream_t stream) {
  const int sms = RoutedSmCount();
  const int64_t width = kKind == kProductTransposed ? p.inner : p.outer;
  // Row tiles: the experts' row counts stay on the device, so at most one
  // partial tile per expert (or per row) on top of the whole ones.
  const int64_t row_tiles = kKind == kProductWeightGrad
                                ? int64_t{p.experts} * ((p.inner + kTileRows - 1) / kTileRows)
                                : p.entries / kTileRows + std::min<int64_t>(p.experts, p.entries);
  const auto tiles = [&](int wide) { return row_tiles * ((width + wide - 1) / wide); };
  const auto launch = [&](auto wide) {
    constexpr int kWide = decltype(wide)::value;
    if (p.gather_x != 0 || p.gather_w != 0) LaunchTc<kKind, kWide, true>(p, bf16, tiles(kWide), sms, stream);
    else LaunchTc<kKind, kWide, false>(p, bf16, tiles(kWide), sms, stream);
  };
  // The widest tile that still gives every other multiprocessor one: what a
  // block brings per slice grows with the width, and narrow tiles bring the
  // rows of x more often (512 rows of 64 experts, 1024 x 1024: 27 us with 256
  // columns, 28 with 128, 33 with 64; one row of two experts, 512 x 512: 6.4, 5.4
  // and 4.9 us).  Partial row tiles count as half of one here (3000 rows of 24
  // experts, 768 x 384: 7.3 us with 128 columns, 8.7 with 256).
  const int64_t used = std::min<int64_t>(p.experts, p.entries);
  const int64_t likely = kKind == kProductWeightGrad ? row_tiles : std::max(used, p.entries / kTileRows + used / 2);
  const auto enough = [&](int wide) { return 2 * likely * ((width + wide - 1) / wide) >= sms; };
  if (enough(256)) launch(std::integral_constant<int, 256>{});
  else if (enough(128)) launch(std::integral_constant<int, 128>{});
  else launch(std::integral_constant<int, 64>{});
}

}  // namespace

// Every operand row starts on a 16-byte boundary and no tile index passes 32 bits,
// nor does one that is a turn of the blocks further.
bool TensorCoreProduct(int kind, const ProductArgs& p) {
  const auto aligned = [](const void* data) { return reinterpret_cast<uintptr_t>(data) % 16 == 0; };
  const int64_t width = kind == kProductTransposed ? p.inner : p.outer;
  const int64_t rows = kind == kProductWeightGrad ? int64_t{p.experts} * (p.inner + kTileRows) : p.entries + int64_t{p.experts} * kTileRows;
  return p.entries > 0 && p.inner % 8 == 0 && p.outer % 8 == 0 && p.x_stride % 8 == 0 &&
         (kind != kProductWeightGrad || p.w_stride % 8 == 0) && aligned(p.x) && aligned(p.w) && aligned(p.out) &&
         rows / kTileRows * ((width + 63) / 64) < (int64_t{1} << 31) - 4096;
}

void LaunchTensorCoreProduct(int kind, int32_t dtype, const ProductArgs& args, cudaStream_t stream) {
  const bool bf16 = dtype == kTypeBf16;
  if (kind == kProduct) ByWidth<kProduct>(args, bf16, stream);
  else if (kind == kProductTransposed) ByWidth<kProductTransposed>(args, bf16, stream);
  else ByWidth<kProductWeightGrad>(args, bf16, stream);
}

}  // namespace t0b

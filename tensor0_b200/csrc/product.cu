// Products over sectors chosen at run time (a router's experts), any strides
// and widths, and the sum over each token's experts.
//
//   product:      y[p] = x[r(p)] @ W[e],     p in [offsets[e], offsets[e + 1])
//   transposed:   y[p] = x[r(p)] @ W[e]^T
//   weight grad:  dW[e] = sum over p of x[r(p)]^T dy[q(p)]
// with r(p) = rows[p] / top_k (gathered token rows) or p.  Rows from
// offsets[experts] on belong to no expert; the products write zeros there.
// (The 16-byte aligned operands of product_tc.cu are the usual case; the general
// kernel here takes 9.2 ms where that takes 0.14, 32768 gathered rows of 1024 x 2048.)
// The sum of four rows of 2048 for 8192 tokens, replayed with three inputs by turns:
// 31 us, 5.4 TB/s.
#include <algorithm>

#include "engine.h"
#include "layout.h"
#include "routed.cuh"
#include "routed.h"

namespace t0b {
namespace {

// General kernel: 64 x 64 tiles on the FP32 units, 16 deep, 4 x 4 values per
// thread.  It serves operands whose rows do not start on 16-byte boundaries.
constexpr int kGenTile = 64, kGenDeep = 16, kGenThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kGenThreads) GeneralProduct(ProductArgs a, int kind) {
  __shared__ float left[kGenDeep][kGenTile + 4], right[kGenDeep][kGenTile + 4];
  LetNextStart();
  WaitForPrevious();
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const T* x = static_cast<const T*>(a.x);
  const T* w = static_cast<const T*>(a.w);
  T* out = static_cast<T*>(a.out);
  const int width = kind == kProductTransposed ? a.inner : a.outer;
  const int64_t tiles_n = (width + kGenTile - 1) / kGenTile;
  // The grid walks (expert, row tile, column tile); rows past the last expert
  // are one more expert whose products are zero.
  int64_t first = 0;
  for (int e = 0; e <= a.experts; ++e) {
    if (kind == kProductWeightGrad && e == a.experts) break;
    const int64_t begin = RowBound(a.offsets[e], a.entries);
    const int64_t end = e < a.experts ? max(begin, RowBound(a.offsets[e + 1], a.entries)) : a.entries;
    const int64_t rows = kind == kProductWeightGrad ? a.inner : end - begin;
    const int64_t deep = e == a.experts ? 0
                         : kind == kProduct ? a.inner : kind == kProductTransposed ? a.outer : end - begin;
    const int64_t tiles = (rows + kGenTile - 1) / kGenTile * tiles_n;
    int64_t tile = blockIdx.x - first % gridDim.x;
    if (tile < 0) tile += gridDim.x;
    first += tiles;
    for (; tile < tiles; tile += gridDim.x) {
      const int64_t m0 = tile / tiles_n * kGenTile, n0 = tile % tiles_n * kGenTile;
      float acc[4][4] = {};
      for (int64_t k0 = 0; k0 < deep; k0 += kGenDeep) {
        for (int i = tid; i < kGenTile * kGenDeep; i += kGenThreads) {
          // Neighbouring threads read neighbouring addresses.
          const int lk = kind == kProductWeightGrad ? i / kGenTile : i % kGenDeep;
          const int lm = kind == kProductWeightGrad ? i % kGenTile : i / kGenDeep;
          float v = 0.0f;
          if (m0 + lm < rows && k0 + lk < deep) {
            const int64_t p = begin + (kind == kProductWeightGrad ? k0 + lk : m0 + lm);
            const int64_t r = a.gather_x != 0 ? a.rows[p] / a.top_k : p;
            if (r >= 0 && r < a.x_rows) v = ToFloat(x[r * a.x_stride + (kind == kProductWeightGrad ? m0 + lm : k0 + lk)]);
          }
          left[lk][lm] = v;
          const int rk = kind == kProductTransposed ? i % kGenDeep : i / kGenTile;
          const int rn = kind == kProductTransposed ? i / kGenDeep : i % kGenTile;
          v = 0.0f;
          if (n0 + rn < width && k0 + rk < deep) {
            if (kind == kProductWeightGrad) {
              const int64_t p = begin + k0 + rk;
              const int64_t r = a.gather_w != 0 ? a.rows[p] / a.top_k : p;
              if (r >= 0 && r < a.w_rows) v = ToFloat(w[r * a.w_stride + n0 + rn]);
            } else {
              const int64_t row = kind == kProduct ? k0 + rk : n0 + rn, col = kind == kProduct ? n0 + rn : k0 + rk;
              v = ToFloat(w[(int64_t{e} * a.inner + row) * a.outer + col]);
            }
          }
          right[rk][rn] = v;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kGenDeep; ++k) {
          float l[4], r[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            l[i] = left[k][ty * 4 + i];
            r[i] = right[k][tx * 4 + i];
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(l[i], r[j], acc[i][j]);
          }
        }
        __syncthreads();
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t m = m0 + ty * 4 + i;
        if (m >= rows) continue;
        T* row = kind == kProductWeightGrad ? out + (int64_t{e} * a.inner + m) * a.outer
                                            : out + (begin + m) * a.out_stride;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (n0 + tx * 4 + j < width) row[n0 + tx * 4 + j] = FromFloat<T>(acc[i][j]);
        }
      }
    }
  }
}

// A warp sums 256 columns (blockIdx.y) of one token in 32 bits; memory bound,
// each row read once, four rows in flight.  The rows come rounded to 16 bits, so
// that they take half the traffic: their errors and the result's together are
// about 1.4 times those of one rounding, where 32-bit rows would move 268 MB more
// (41 us of copy bandwidth) for 8192 tokens of 4 rows of 2048.
template <typename T, bool Vector>
__global__ void __launch_bounds__(256) RoutedSum(RoutedSumArgs a) {
  LetNextStart();
  WaitForPrevious();
  const int column = static_cast<int>(blockIdx.y) * 256 + (threadIdx.x & 31) * 8, count = a.width - column;
  const T* y = static_cast<const T*>(a.y) + column;
  const int64_t step = int64_t{gridDim.x} * 8;
  for (int64_t t = int64_t{blockIdx.x} * 8 + (threadIdx.x >> 5); t < a.tokens; t += step) {
    float sum[8] = {};
    for (int n0 = 0; n0 < a.top_k; n0 += 4) {
      float v[4][8];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int64_t p = n0 + n < a.top_k ? a.positions[t * a.top_k + n0 + n] : -1;
        const bool some = p >= 0 && p < a.entries;
        Load8<T, Vector>(y + (some ? p : 0) * a.y_stride, some ? count : 0, v[n]);
      }
#pragma unroll
      for (int n = 0; n < 4; ++n) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += v[n][i];
      }
    }
    Store8<T, Vector>(static_cast<T*>(a.out) + t * a.out_stride + column, count, sum);
  }
}

template <typename T>
void Launch(int kind, const ProductArgs& a, cudaStream_t stream) {
  LaunchRouted("routed product launch", false, GeneralProduct<T>, static_cast<unsigned>(RoutedSmCount() * 4), kGenThreads, 0,
               stream, a, kind);
}

template <typename T>
void Sum(const RoutedSumArgs& a, cudaStream_t stream) {
  if (a.tokens == 0 || a.width == 0) return;
  const dim3 blocks(static_cast<unsigned>(std::min<int64_t>((a.tokens + 7) / 8, 1 << 20)),
                    static_cast<unsigned>((a.width + 255) / 256));   // a width is at most 2^23
  const bool vector = a.width % 8 == 0 && a.y_stride % 8 == 0 && a.out_stride % 8 == 0 &&
                      reinterpret_cast<uintptr_t>(a.y) % 16 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
  const char* what = "routed sum launch";
  const bool brief = BriefGrid(int64_t{blocks.x} * blocks.y);
  if (vector) LaunchRouted(what, brief, RoutedSum<T, true>, blocks, 256, 0, stream, a);
  else LaunchRouted(what, brief, RoutedSum<T, false>, blocks, 256, 0, stream, a);
}

}  // namespace

void LaunchProduct(int kind, int32_t dtype, const ProductArgs& args, cudaStream_t stream) {
  if (dtype != kTypeF16 && dtype != kTypeBf16) throw InvalidArgument("routed products take F16 or BF16");
  if (TensorCoreProduct(kind, args)) LaunchTensorCoreProduct(kind, dtype, args, stream);
  else if (dtype == kTypeF16) Launch<__half>(kind, args, stream);
  else Launch<__nv_bfloat16>(kind, args, stream);
}

void LaunchRoutedSum(int32_t dtype, const RoutedSumArgs& args, cudaStream_t stream) {
  if (dtype == kTypeF16) Sum<__half>(args, stream);
  else if (dtype == kTypeBf16) Sum<__nv_bfloat16>(args, stream);
  else throw InvalidArgument("routed sums take F16 or BF16");
}

}  // namespace t0b

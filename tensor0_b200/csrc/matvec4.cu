// Products of single tokens with 4-bit weights: for each expert-ordered row p,
//   y[p][n] = sum over groups of scale[e][n][group] * sum over k of (q[e][n][k] - 8) x[r(p)][k]
// q holds two weights per byte, the even one in the low half.
#include <algorithm>

#include "engine.h"
#include "layout.h"
#include "routed.cuh"
#include "routed.h"

namespace t0b {
namespace {

// A warp computes one output of one row, 256 weights (8 per lane) at a time.
template <typename T>
__global__ void __launch_bounds__(256) Matvec(MatvecArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t units = a.entries * a.outer, step = int64_t{gridDim.x} * 8;
  const int groups = a.inner / a.group;
  for (int64_t unit = int64_t{blockIdx.x} * 8 + (threadIdx.x >> 5); unit < units; unit += step) {
    const int64_t p = unit / a.outer;
    const int n = static_cast<int>(unit - p * a.outer);
    T* out = static_cast<T*>(a.out) + unit;
    int low = 0, high = a.experts;   // the expert whose rows hold p
    while (low < high) {
      const int mid = (low + high) >> 1;
      if (a.offsets[mid + 1] <= p) low = mid + 1; else high = mid;
    }
    if (low == a.experts) {
      if (lane == 0) *out = FromFloat<T>(0.0f);
      continue;
    }
    const int64_t r = a.gather != 0 ? a.rows[p] / a.top_k : p;
    if (r < 0 || r >= a.x_rows) continue;
    const T* x = static_cast<const T*>(a.x) + r * a.x_stride;
    const int64_t matrix_row = int64_t{low} * a.outer + n;
    const uint8_t* codes = a.codes + matrix_row * (a.inner / 2);
    const T* scales = static_cast<const T*>(a.scales) + matrix_row * groups;
    float sum = 0.0f;
    for (int k = lane * 8; k < a.inner; k += 256) {
      float part = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int pair = codes[k / 2 + i];
        part = fmaf(static_cast<float>((pair & 15) - 8), ToFloat(x[k + 2 * i]), part);
        part = fmaf(static_cast<float>((pair >> 4) - 8), ToFloat(x[k + 2 * i + 1]), part);
      }
      sum = fmaf(part, ToFloat(scales[k / a.group]), sum);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) *out = FromFloat<T>(sum);
  }
}

template <typename T>
void Launch(const MatvecArgs& a, cudaStream_t stream) {
  const unsigned blocks = static_cast<unsigned>(std::min<int64_t>((a.entries * a.outer + 7) / 8, 1 << 20));
  Matvec<T><<<blocks, 256, 0, stream>>>(a);
  Check(cudaGetLastError(), "4-bit product launch");
  g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
}

}  // namespace

void LaunchMatvec(int32_t dtype, const MatvecArgs& args, cudaStream_t stream) {
  if (dtype == kTypeF16) Launch<__half>(args, stream);
  else if (dtype == kTypeBf16) Launch<__nv_bfloat16>(args, stream);
  else throw InvalidArgument("4-bit products take F16 or BF16");
}

}  // namespace t0b

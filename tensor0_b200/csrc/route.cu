// Router: each token's experts and weights, and the order of the rows by
// expert; and the gradient with respect to the logits.
//
//   s = softmax(x) or sigmoid(x);  choice c = s + bias, or x itself where no
//   bias is given and groups go by their best value (softmax and sigmoid are
//   increasing, and x keeps apart what their rounding makes equal).
//   A group's score is its best c or the sum of its two best; the top groups
//   stay, then the top_k best c of what stays; ties go to the lowest index.
//   w = scale * s / (sum of the chosen s + 1e-20), or scale * s.
// A logit of -inf or NaN, and a masked token, take no expert (index -1,
// weight 0).  Under softmax a NaN or +inf logit makes the row's weights NaN.
//
// One warp holds a token: expert e is value e / 32 of lane e % 32, so loads
// coalesce.  A pick is two warp reductions: the largest choice value as an
// ordered integer, then the lowest index that holds it.
#include <algorithm>
#include <climits>

#include "engine.h"
#include "layout.h"
#include "routed.cuh"
#include "routed.h"

namespace t0b {
namespace {

constexpr uint32_t kFull = 0xffffffffu;
constexpr int kRouteThreads = 256;

// Monotone map of floats onto unsigned integers; -0 counts as +0.
__device__ __forceinline__ uint32_t Ordered(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  return u ^ ((u >> 31) != 0 ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ float WarpMax(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, d));
  return v;
}

__device__ __forceinline__ float WarpSum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(kFull, v, d);
  return v;
}

__device__ __forceinline__ double WarpSum(double v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(kFull, v, d);
  return v;
}

template <typename T, int V>
__device__ __forceinline__ void LoadLogits(const T* row, int experts, int lane, float (&x)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const int e = j * 32 + lane;
    x[j] = e < experts ? ToFloat(row[e]) : -INFINITY;
  }
}

// The scores of one token.  The softmax normaliser is summed in 64 bits and
// rounded once, so that it does not depend on the order of the terms and the
// choice of experts does not either.
template <int V>
__device__ __forceinline__ void Scores(const float (&x)[V], int experts, int lane, bool softmax, float (&s)[V]) {
  if (softmax) {
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < V; ++j) top = fmaxf(top, x[j]);
    top = WarpMax(top);
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      s[j] = j * 32 + lane < experts ? expf(x[j] - top) : 0.0f;
      sum += static_cast<double>(s[j]);
    }
    const float total = static_cast<float>(WarpSum(sum));
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] = __fdiv_rn(s[j], total);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) s[j] = __frcp_rn(1.0f + expf(-x[j]));
  }
}

// Value `index` (expert number) of a token's register array, in every lane.
template <int V>
__device__ __forceinline__ float Pick(const float (&v)[V], int index) {
  float mine = 0.0f;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (j == (index >> 5)) mine = v[j];
  }
  return __shfl_sync(kFull, mine, index & 31);
}

// Chosen experts and weights of the block's tokens.  `choices` is one row of
// experts per warp (groups only).
template <typename T, int V>
__device__ __forceinline__ void SelectTokens(const RouteArgs& a, int64_t begin, int64_t end, float* choices) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const bool by_logit = a.bias == nullptr && a.group_best == 1;
  for (int64_t t = begin + warp; t < end; t += warps) {
    int32_t* chosen = a.chosen + t * a.top_k;
    float* weights = a.weights + t * a.top_k;
    if (a.mask != nullptr && a.mask[t] == 0) {   // its logits may hold anything
      if (lane < a.top_k) {
        chosen[lane] = -1;
        weights[lane] = 0.0f;
      }
      continue;
    }
    float x[V], s[V];
    LoadLogits<T, V>(static_cast<const T*>(a.logits) + t * a.logit_stride, a.experts, lane, x);
    Scores<V>(x, a.experts, lane, a.softmax != 0, s);
    uint32_t key[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int e = j * 32 + lane;
      float c = by_logit ? x[j] : s[j];
      if (a.bias != nullptr && e < a.experts) c += a.bias[e];
      key[j] = x[j] > -INFINITY && c > -INFINITY ? Ordered(c) : 0u;
      if (a.groups > 1 && e < a.experts) {
        choices[warp * a.experts + e] = key[j] != 0u ? c : -INFINITY;
      }
    }
    if (a.groups > 1) {
      __syncwarp();
      const int size = a.experts / a.groups;
      uint32_t group_key = 0;
      if (lane < a.groups) {
        float first = -INFINITY, second = -INFINITY;
        const float* mine = choices + warp * a.experts + lane * size;
        // Lanes start at different places of their groups, which spreads the banks.
        int i = lane % size;
        for (int n = 0; n < size; ++n) {
          const float c = mine[i];
          second = fmaxf(second, fminf(first, c));
          first = fmaxf(first, c);
          if (++i == size) i = 0;
        }
        if (a.group_best == 2 && second > -INFINITY) first += second;
        group_key = Ordered(first);
      }
      __syncwarp();
      uint32_t kept = 0;
      for (int n = 0; n < a.top_groups; ++n) {
        const uint32_t best = __reduce_max_sync(kFull, group_key);
        const uint32_t holders = __ballot_sync(kFull, group_key == best && lane < a.groups);
        const int winner = __ffs(holders) - 1;
        if (winner < 0) break;
        kept |= 1u << winner;
        if (lane == winner) group_key = 0;
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int e = j * 32 + lane;
        if (e < a.experts && ((kept >> (e / size)) & 1u) == 0u) key[j] = 0u;
      }
    }
    int mine = -1;
    float score = 0.0f;
    for (int n = 0; n < a.top_k; ++n) {
      uint32_t best = 0;
      int at = 0;
      float value = 0.0f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (key[j] > best) {
          best = key[j];
          at = j;
          value = s[j];
        }
      }
      const uint32_t top = __reduce_max_sync(kFull, best);
      if (top == 0u) break;
      const unsigned index = __reduce_min_sync(kFull, best == top ? static_cast<unsigned>(at * 32 + lane) : UINT_MAX);
      value = __shfl_sync(kFull, value, index & 31);
      if (lane == n) {
        mine = static_cast<int>(index);
        score = value;
      }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (static_cast<unsigned>(j * 32 + lane) == index) key[j] = 0u;
      }
    }
    if (a.renormalize != 0) {
      const float total = WarpSum(score) + 1e-20f;
      score = __fdiv_rn(score, total);
    }
    if (lane < a.top_k) {
      chosen[lane] = mine;
      weights[lane] = mine < 0 ? 0.0f : score * a.scale;
    }
  }
}

// Entries [begin, end) into expert order, given each expert's first place for
// this block in `first` (absent entries: place `experts`).  Stable: a warp
// takes a run of entries, counts them by expert, and takes its places after
// the warps before it.
__device__ __forceinline__ void PlaceEntries(const RouteArgs& a, int64_t begin, int64_t end, const int* first,
                                             int* by_warp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int bins = a.experts + 1;
  int* mine = by_warp + warp * bins;
  for (int e = lane; e < bins; e += 32) mine[e] = 0;
  __syncwarp();
  const int64_t run = ((end - begin + warps - 1) / warps + 31) / 32 * 32;
  const int64_t from = begin + warp * run, to = from + run < end ? from + run : end;
  for (int64_t i = from + lane; i - lane < to; i += 32) {
    const bool valid = i < to;
    int e = valid ? a.chosen[i] : -2;
    if (e == -1) e = a.experts;
    const uint32_t same = __match_any_sync(kFull, e);
    if (valid && (same & ((1u << lane) - 1)) == 0) mine[e] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  for (int e = threadIdx.x; e < bins; e += blockDim.x) {
    int place = first[e];
    for (int w = 0; w < warps; ++w) {
      const int count = by_warp[w * bins + e];
      by_warp[w * bins + e] = place;
      place += count;
    }
  }
  __syncthreads();
  for (int64_t i = from + lane; i - lane < to; i += 32) {
    const bool valid = i < to;
    int e = valid ? a.chosen[i] : -2;
    if (e == -1) e = a.experts;
    const uint32_t same = __match_any_sync(kFull, e);
    const int rank = __popc(same & ((1u << lane) - 1));
    int place = 0;
    if (valid) place = mine[e] + rank;
    __syncwarp();
    if (valid) {
      if (rank == 0) mine[e] += __popc(same);
      a.rows[place] = static_cast<int32_t>(i);
      a.positions[i] = e == a.experts ? -1 : place;
    }
    __syncwarp();
  }
}

// Exclusive prefix of counts[0..n) in place, by the first warp; the total in counts[n].
__device__ __forceinline__ void PrefixByWarp(int* counts, int n) {
  if (threadIdx.x >= 32) return;
  const int lane = threadIdx.x;
  int carry = 0;
  for (int e0 = 0; e0 < n; e0 += 32) {
    const int value = e0 + lane < n ? counts[e0 + lane] : 0;
    int sum = value;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int other = __shfl_up_sync(kFull, sum, d);
      if (lane >= d) sum += other;
    }
    if (e0 + lane < n) counts[e0 + lane] = carry + sum - value;
    carry += __shfl_sync(kFull, sum, 31);
  }
  if (lane == 0) counts[n] = carry;
}

__device__ __forceinline__ void CountEntries(const RouteArgs& a, int64_t begin, int64_t end, int* bins) {
  for (int64_t i = begin + threadIdx.x; i < end; i += blockDim.x) {
    const int e = a.chosen[i];
    if (e >= 0) atomicAdd(bins + e, 1);   // whole numbers: the order of the additions does not matter
  }
}

// One block does all: few tokens, where launches cost more than the work.
template <typename T, int V>
__global__ void __launch_bounds__(1024) RouteOneBlock(RouteArgs a) {
  extern __shared__ int route_smem[];
  int* first = route_smem;                        // experts + 1
  int* by_warp = first + a.experts + 1;           // warps x (experts + 1)
  float* choices = reinterpret_cast<float*>(by_warp);   // reused: the choice is over before rows are placed
  for (int e = threadIdx.x; e <= a.experts; e += blockDim.x) first[e] = 0;
  SelectTokens<T, V>(a, 0, a.tokens, choices);
  __syncthreads();
  CountEntries(a, 0, a.tokens * a.top_k, first);
  __syncthreads();
  PrefixByWarp(first, a.experts);
  __syncthreads();
  for (int e = threadIdx.x; e <= a.experts; e += blockDim.x) a.offsets[e] = first[e];
  PlaceEntries(a, 0, a.tokens * a.top_k, first, by_warp);
}

template <typename T, int V>
__global__ void __launch_bounds__(kRouteThreads) RouteSelect(RouteArgs a, int64_t tokens_per_block) {
  extern __shared__ int route_smem[];
  int* bins = route_smem;
  float* choices = reinterpret_cast<float*>(bins + a.experts);
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) bins[e] = 0;
  const int64_t begin = blockIdx.x * tokens_per_block;
  const int64_t end = begin + tokens_per_block < a.tokens ? begin + tokens_per_block : a.tokens;
  SelectTokens<T, V>(a, begin, end, choices);
  __syncthreads();
  CountEntries(a, begin * a.top_k, end * a.top_k, bins);
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) a.counts[blockIdx.x * int64_t{a.experts} + e] = bins[e];
}

__global__ void __launch_bounds__(kRouteThreads) RoutePlace(RouteArgs a, int64_t tokens_per_block) {
  extern __shared__ int route_smem[];
  int* total = route_smem;                  // experts + 1
  int* before = total + a.experts + 1;      // experts + 1
  int* by_warp = before + a.experts + 1;
  for (int e = threadIdx.x; e <= a.experts; e += blockDim.x) total[e] = before[e] = 0;
  __syncthreads();
  // Threads share the blocks' counts: several of them sum one expert's column.
  const int lanes = a.experts < static_cast<int>(blockDim.x) ? a.experts : static_cast<int>(blockDim.x);
  const int parts = static_cast<int>(blockDim.x) / lanes;
  const int part = static_cast<int>(threadIdx.x) / lanes;
  if (part < parts) {
    for (int e = static_cast<int>(threadIdx.x) % lanes; e < a.experts; e += lanes) {
      int all = 0, mine = 0;
#pragma unroll 8
      for (unsigned b = static_cast<unsigned>(part); b < gridDim.x; b += static_cast<unsigned>(parts)) {
        const int count = a.counts[b * int64_t{a.experts} + e];
        all += count;
        mine += b < blockIdx.x ? count : 0;
      }
      atomicAdd(total + e, all);
      atomicAdd(before + e, mine);
    }
  }
  __syncthreads();
  PrefixByWarp(total, a.experts);
  __syncthreads();
  if (threadIdx.x < 32) {
    int present = 0;
    for (int e = threadIdx.x; e < a.experts; e += 32) present += before[e];
    present = __reduce_add_sync(kFull, present);
    if (threadIdx.x == 0) before[a.experts] = static_cast<int>(blockIdx.x * tokens_per_block * a.top_k) - present;
  }
  __syncthreads();
  for (int e = threadIdx.x; e <= a.experts; e += blockDim.x) {
    if (blockIdx.x == 0) a.offsets[e] = total[e];
    before[e] += total[e];
  }
  __syncthreads();
  const int64_t begin = blockIdx.x * tokens_per_block;
  const int64_t end = begin + tokens_per_block < a.tokens ? begin + tokens_per_block : a.tokens;
  PlaceEntries(a, begin * a.top_k, end * a.top_k, before, by_warp);
}

// With g = scale * (gradient of the chosen weights) and p the chosen scores:
//   renormalised: g <- (g - sum(g p) / total) / total, total = sum p + 1e-20
//   softmax: dx_j = s_j (ds_j - sum(g p)),  ds the scattered g
//   sigmoid: dx_j = ds_j s_j (1 - s_j)
// Memory bound: reads and writes each logit once; the scores are recomputed.
template <typename T, int V>
__global__ void __launch_bounds__(kRouteThreads) RouteBackward(RouteBackwardArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int64_t step = int64_t{gridDim.x} * warps;
  for (int64_t t = int64_t{blockIdx.x} * warps + warp; t < a.tokens; t += step) {
    T* out = static_cast<T*>(a.logits_grad) + t * a.experts;
    const int mine = lane < a.top_k ? a.chosen[t * a.top_k + lane] : -1;
    float g = mine >= 0 ? a.weights_grad[t * a.top_k + lane] * a.scale : 0.0f;
    if (__ballot_sync(kFull, mine >= 0) == 0u) {   // no expert: the logits may hold anything
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (j * 32 + lane < a.experts) out[j * 32 + lane] = FromFloat<T>(0.0f);
      }
      continue;
    }
    float x[V], s[V], ds[V];
    LoadLogits<T, V>(static_cast<const T*>(a.logits) + t * a.logit_stride, a.experts, lane, x);
    Scores<V>(x, a.experts, lane, a.softmax != 0, s);
    float p = 0.0f;
    for (int n = 0; n < a.top_k; ++n) {
      const int index = __shfl_sync(kFull, mine, n);
      const float value = Pick<V>(s, index < 0 ? 0 : index);
      if (lane == n && index >= 0) p = value;
    }
    if (a.renormalize != 0) {
      const float total = WarpSum(p) + 1e-20f;
      const float mean = WarpSum(g * __fdiv_rn(p, total));
      g = mine >= 0 ? __fdiv_rn(g - mean, total) : 0.0f;
    }
    const float inner = WarpSum(g * p);
#pragma unroll
    for (int j = 0; j < V; ++j) ds[j] = 0.0f;
    for (int n = 0; n < a.top_k; ++n) {
      const int index = __shfl_sync(kFull, mine, n);
      const float value = __shfl_sync(kFull, g, n);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (j * 32 + lane == index) ds[j] = value;
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int e = j * 32 + lane;
      if (e >= a.experts) continue;
      const float d = a.softmax != 0 ? s[j] * (ds[j] - inner) : ds[j] * s[j] * (1.0f - s[j]);
      out[e] = FromFloat<T>(d);
    }
  }
}

// Up to this many tokens one block does the whole call.
constexpr int64_t kOneBlockTokens = 64;

int64_t TokensPerBlock(int64_t tokens) {
  const int64_t blocks = int64_t{RoutedSmCount()} * 2;
  return std::max<int64_t>(8, (tokens + blocks - 1) / blocks);
}

template <typename T, int V>
void Route(const RouteArgs& a, cudaStream_t stream) {
  const std::size_t bins = static_cast<std::size_t>(a.experts) + 1;
  if (a.tokens <= kOneBlockTokens) {
    const unsigned warps = static_cast<unsigned>(std::min<int64_t>(32, std::max<int64_t>(1, a.tokens)));
    const std::size_t smem = (bins + warps * bins) * sizeof(int);
    AllowShared<RouteOneBlock<T, V>>(static_cast<int>(smem));
    RouteOneBlock<T, V><<<1, warps * 32, smem, stream>>>(a);
    Check(cudaGetLastError(), "router launch");
    g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
    return;
  }
  const int64_t per_block = TokensPerBlock(a.tokens);
  const unsigned blocks = static_cast<unsigned>((a.tokens + per_block - 1) / per_block);
  const int warps = kRouteThreads / 32;
  const std::size_t select = (bins + (a.groups > 1 ? warps * bins : 0)) * sizeof(int);
  RouteSelect<T, V><<<blocks, kRouteThreads, select, stream>>>(a, per_block);
  Check(cudaGetLastError(), "router launch");
  RoutePlace<<<blocks, kRouteThreads, (2 + warps) * bins * sizeof(int), stream>>>(a, per_block);
  Check(cudaGetLastError(), "row order launch");
  g_kernel_launches.fetch_add(2, std::memory_order_relaxed);
}

template <typename T, int V>
void Backward(const RouteBackwardArgs& a, cudaStream_t stream) {
  const int64_t blocks = std::min<int64_t>((a.tokens + kRouteThreads / 32 - 1) / (kRouteThreads / 32), 1 << 20);
  RouteBackward<T, V><<<static_cast<unsigned>(blocks), kRouteThreads, 0, stream>>>(a);
  Check(cudaGetLastError(), "router gradient launch");
  g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
}

template <typename T, typename Args, typename Body>
void ByExperts(const Args& a, Body&& body) {
  if (a.experts <= 32) body(std::integral_constant<int, 1>{});
  else if (a.experts <= 64) body(std::integral_constant<int, 2>{});
  else if (a.experts <= 128) body(std::integral_constant<int, 4>{});
  else if (a.experts <= 256) body(std::integral_constant<int, 8>{});
  else body(std::integral_constant<int, 16>{});
}

template <typename Body>
void ByType(int32_t dtype, Body&& body) {
  switch (dtype) {
    case kTypeF32: body(float{}); break;
    case kTypeF16: body(__half{}); break;
    case kTypeBf16: body(__nv_bfloat16{}); break;
    default: throw InvalidArgument("router logits must be F32, F16 or BF16");
  }
}

}  // namespace

std::size_t RouteWorkspace(int64_t tokens, int experts) {
  if (tokens <= kOneBlockTokens) return 0;
  const int64_t per_block = TokensPerBlock(tokens);
  return static_cast<std::size_t>((tokens + per_block - 1) / per_block) * experts * sizeof(int32_t);
}

void LaunchRoute(int32_t dtype, const RouteArgs& args, cudaStream_t stream) {
  ByType(dtype, [&](auto type) {
    using T = decltype(type);
    ByExperts<T>(args, [&](auto values) { Route<T, decltype(values)::value>(args, stream); });
  });
}

void LaunchRouteBackward(int32_t dtype, const RouteBackwardArgs& args, cudaStream_t stream) {
  ByType(dtype, [&](auto type) {
    using T = decltype(type);
    ByExperts<T>(args, [&](auto values) { Backward<T, decltype(values)::value>(args, stream); });
  });
}

}  // namespace t0b

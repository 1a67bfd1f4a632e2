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
// weight 0).  Under softmax a NaN or +inf logit makes the row's weights NaN,
// whichever experts it leaves to choose from.
//
// One warp holds a token: lane l has the V experts from l * V on.  Bound by
// instructions, not by memory, so nothing is done for all experts where it can
// be done for the chosen ones: without a bias the scores are taken of those
// alone, and where the weights are renormalised the softmax needs no sum over
// all experts.
//
// The row order takes three launches: experts counted per block of tokens, the
// counts summed over the blocks before each, entries placed.  Few tokens take
// one block that does it all.
//
// Measured, replayed with three inputs by turns: 8 tokens of 64 experts 4.0 us; 8191
// of 256 in groups with a bias 24 us (choice 17); 32768 of 128 forward and backward
// 42 to 44 us (choice 24, gradient 11 or, with cold caches, 14, where reading and
// writing the logits takes 6).  As calls one after the other: 4.2, 27 and 50 us.
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

// Sum over lanes 0 to top_k - 1 (the others hold 0), valid in those lanes.
__device__ __forceinline__ float ChosenSum(float v, int top_k) {
  if (top_k > 8) {
    v += __shfl_xor_sync(kFull, v, 16);
    v += __shfl_xor_sync(kFull, v, 8);
  }
#pragma unroll
  for (int d = 4; d > 0; d >>= 1) v += __shfl_xor_sync(kFull, v, d);
  return v;
}

// The lane's experts of a token; `vector`: as one access (rows start on
// multiples of it).
template <typename T, int V>
__device__ __forceinline__ void LoadLogits(const T* row, int experts, int lane, bool vector, float (&x)[V]) {
  constexpr int kBytes = V * static_cast<int>(sizeof(T));
  const int first = lane * V;
  if (vector && first + V <= experts) {
    alignas(16) T v[V];
    if constexpr (kBytes % 16 == 0) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4*>(v)[i] = reinterpret_cast<const uint4*>(row + first)[i];
    } else if constexpr (kBytes == 8) {
      *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(row + first);
    } else if constexpr (kBytes == 4) {
      *reinterpret_cast<uint32_t*>(v) = *reinterpret_cast<const uint32_t*>(row + first);
    } else {
      v[0] = row[first];
    }
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = ToFloat(v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = first + j < experts ? ToFloat(row[first + j]) : -INFINITY;
  }
}

template <typename T, int V>
bool VectorLogits(const void* logits, int64_t stride) {
  constexpr uintptr_t kBytes = V * sizeof(T) < 16 ? V * sizeof(T) : 16;
  return reinterpret_cast<uintptr_t>(logits) % kBytes == 0 && static_cast<uint64_t>(stride) * sizeof(T) % kBytes == 0;
}

template <typename T, int V>
__device__ __forceinline__ void StoreValues(T* row, int experts, int lane, bool vector, const float (&d)[V]) {
  constexpr int kBytes = V * static_cast<int>(sizeof(T));
  const int first = lane * V;
  alignas(16) T v[V];
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = FromFloat<T>(d[j]);
  if (vector && first + V <= experts) {
    if constexpr (kBytes % 16 == 0) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4*>(row + first)[i] = reinterpret_cast<const uint4*>(v)[i];
      return;
    } else if constexpr (kBytes == 8) {
      *reinterpret_cast<uint2*>(row + first) = *reinterpret_cast<const uint2*>(v);
      return;
    } else if constexpr (kBytes == 4) {
      *reinterpret_cast<uint32_t*>(row + first) = *reinterpret_cast<const uint32_t*>(v);
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < V; ++j) {
    if (first + j < experts) row[first + j] = v[j];
  }
}

// Largest logit of the token; exp(x - largest) is at most 1.
template <int V>
__device__ __forceinline__ float Largest(const float (&x)[V]) {
  float top = x[0];
#pragma unroll
  for (int j = 1; j < V; ++j) top = fmaxf(top, x[j]);
  return WarpMax(top);
}

// Of each group of `size` experts the best value, or the sum of its two best;
// lane g has group g's.  `values`: one row per warp of shared memory.
template <int V>
__device__ __forceinline__ float GroupScore(const float (&c)[V], int experts, int groups, int best, float* values) {
  const int lane = threadIdx.x & 31, size = experts / groups;
  float first = -INFINITY, second = -INFINITY;
  const auto add = [&](float v) {
    second = fmaxf(second, fminf(first, v));
    first = fmaxf(first, v);
  };
  // Lanes per group where a group is a power of two of whole lanes; otherwise
  // through shared memory, with as many lanes to a group as there are.
  int lanes = size / V, source;
  if (size % V == 0 && (lanes & (lanes - 1)) == 0) {
#pragma unroll
    for (int j = 0; j < V; ++j) add(c[j]);
    source = lane * lanes;
  } else {
    lanes = 1;
    while (lanes * 2 * groups <= 32) lanes *= 2;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (lane * V + j < experts) values[lane * V + j] = c[j];
    }
    __syncwarp();
    if (lane / lanes < groups) {
      for (int i = lane % lanes; i < size; i += lanes) add(values[lane / lanes * size + i]);
    }
    source = lane * lanes;
  }
  for (int d = 1; d < lanes; d <<= 1) {
    const float f = __shfl_xor_sync(kFull, first, d), s = __shfl_xor_sync(kFull, second, d);
    second = fmaxf(fmaxf(second, s), fminf(first, f));
    first = fmaxf(first, f);
  }
  if (best == 2 && second > -INFINITY) first += second;
  return __shfl_sync(kFull, first, source & 31);
}

// Batcher's merge exchange sort of a lane's numbers, largest first.
template <int V>
__device__ __forceinline__ void SortDescending(uint32_t (&k)[V]) {
#pragma unroll
  for (int p = 1; p < V; p *= 2) {
#pragma unroll
    for (int d = p; d >= 1; d /= 2) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const bool first = d == p ? j % (2 * p) < p : j >= d && (j - d) % (2 * d) < d;
        if (first && j + d < V && j / (2 * p) == (j + d) / (2 * p)) {
          const uint32_t high = max(k[j], k[j + d]), low = min(k[j], k[j + d]);
          k[j] = high;
          k[j + d] = low;
        }
      }
    }
  }
}

// The expert of slot `lane` by all bits of the choice values (0: not eligible).
// A pick is a warp reduction and a ballot: the first lane that holds the largest
// has the lowest index.
template <int V>
__device__ __forceinline__ int PickExactly(uint32_t (&key)[V], int top_k) {
  const int lane = threadIdx.x & 31;
  int mine = -1;
#pragma unroll 1
  for (int n = 0; n < top_k; ++n) {
    uint32_t best = key[0];
#pragma unroll
    for (int j = 1; j < V; ++j) best = max(best, key[j]);
    const uint32_t largest = __reduce_max_sync(kFull, best);
    if (largest == 0u) break;
    const int winner = __ffs(__ballot_sync(kFull, best == largest)) - 1;
    int at = V - 1;
#pragma unroll
    for (int j = V - 2; j >= 0; --j) at = key[j] == largest ? j : at;
    const int index = __shfl_sync(kFull, lane * V + at, winner);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (lane * V + j == index) key[j] = 0u;
    }
    if (lane == n) mine = index;
  }
  return mine;
}

// The same by one number for each expert, the choice value's high bits and the
// expert (lower ones first): every lane sorts its own, and a pick is one
// reduction and the winner's next.  Values that the high bits do not tell apart
// are next to each other in that order; *close: there is such a pair up to the
// first value not taken, and the picks may not be the ones by all bits.
template <int V>
__device__ __forceinline__ int PickPacked(const uint32_t (&key)[V], int top_k, bool* close) {
  constexpr uint32_t kIndex = 32 * V - 1;
  const int lane = threadIdx.x & 31;
  uint32_t packed[V], pick = 0u, previous = 0u;
#pragma unroll
  for (int j = 0; j < V; ++j) packed[j] = (key[j] & ~kIndex) | (kIndex - static_cast<uint32_t>(lane * V + j));
  SortDescending<V>(packed);
  *close = false;
#pragma unroll 1
  for (int n = 0; n <= top_k; ++n) {
    const uint32_t largest = __reduce_max_sync(kFull, packed[0]);
    if (largest <= kIndex) break;
    *close = *close || (largest ^ previous) <= kIndex;
    previous = largest;
    if (lane == n) pick = largest;
    const bool winner = packed[0] == largest;
#pragma unroll
    for (int j = 0; j + 1 < V; ++j) packed[j] = winner ? packed[j + 1] : packed[j];
    packed[V - 1] = winner ? 0u : packed[V - 1];
  }
  return lane < top_k && pick != 0u ? static_cast<int>(kIndex - (pick & kIndex)) : -1;
}

// Chosen experts and weights of the block's tokens.  kByLogit: the choice goes
// by the logits.
template <typename T, int V, bool kByLogit>
__device__ __forceinline__ void SelectTokens(const RouteArgs& a, int64_t begin, int64_t end, float* values, bool vector) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  // A row stride is below 2^31, and tokens * top_k by 256: 32-bit indices, which cost a
  // tenth of the instructions less than 64-bit ones.
  const int stride = static_cast<int>(a.logit_stride), last = static_cast<int>(end);
  const bool bias_vector = reinterpret_cast<uintptr_t>(a.bias) % (V * 4 < 16 ? V * 4 : 16) == 0;
  for (int t = static_cast<int>(begin) + warp; t < last; t += warps) {
    const int entry = t * a.top_k + lane;
    if (a.mask != nullptr && a.mask[t] == 0) {   // its logits may hold anything
      if (lane < a.top_k) {
        a.chosen[entry] = -1;
        a.weights[entry] = 0.0f;
      }
      continue;
    }
    const T* row = static_cast<const T*>(a.logits) + int64_t{t} * stride;
    float x[V], c[V];   // c: what the choice goes by
    LoadLogits<T, V>(row, a.experts, lane, vector, x);
    float top = 0.0f, total = 1.0f;
    bool nan = false;
    if (a.softmax != 0) {
#pragma unroll
      for (int j = 0; j < V; ++j) nan = nan || x[j] != x[j];
      nan = __any_sync(kFull, nan);
      // Where the first pick is the largest logit, it is known from there.
      if (!kByLogit || a.renormalize == 0 || a.groups > 1) top = Largest<V>(x);
    }
    if constexpr (kByLogit) {
      if (a.softmax != 0 && (a.renormalize == 0 || a.groups > 1)) {
        // With renormalised weights and one group the sum would cancel: the
        // chosen scores hold at least 1 / experts of it, beside which 1e-20 is nothing.
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) sum += lane * V + j < a.experts ? expf(x[j] - top) : 0.0f;
        total = WarpSum(sum);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) c[j] = x[j];
    } else {
      if (a.softmax != 0) {
        if (nan || top == INFINITY) {
          // No scores: the choice goes by those without the NaN logits, or by
          // their limits, equal shares for +inf and nothing for the others.
          nan = true;
          const bool infinite = top == INFINITY;
#pragma unroll
          for (int j = 0; j < V; ++j) {
            if (!(x[j] > -INFINITY)) x[j] = -INFINITY;
            else if (infinite) x[j] = x[j] == INFINITY ? 0.0f : -1e30f;
          }
          if (infinite) top = 0.0f;
        }
        // Summed in 64 bits and rounded once: the choice, which goes by these
        // scores, does not depend on the order of the terms.
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          c[j] = lane * V + j < a.experts ? expf(x[j] - top) : 0.0f;
          sum += static_cast<double>(c[j]);
        }
        total = static_cast<float>(WarpSum(sum));
#pragma unroll
        for (int j = 0; j < V; ++j) c[j] = __fdiv_rn(c[j], total);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) c[j] = __frcp_rn(1.0f + expf(-x[j]));
      }
      if (a.bias != nullptr) {
        float b[V];
        LoadLogits<float, V>(a.bias, a.experts, lane, bias_vector, b);   // -inf past the last expert
#pragma unroll
        for (int j = 0; j < V; ++j) c[j] += b[j];
      }
    }
    uint32_t key[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const bool some = x[j] > -INFINITY && c[j] > -INFINITY;
      key[j] = some ? Ordered(c[j]) : 0u;
      if (!some) c[j] = -INFINITY;
    }
    if (a.groups > 1) {
      const float score = GroupScore<V>(c, a.experts, a.groups, a.group_best, values + warp * a.experts);
      uint32_t group_key = lane < a.groups ? Ordered(score) : 0u, kept = 0;
      for (int n = 0; n < a.top_groups; ++n) {
        const uint32_t best = __reduce_max_sync(kFull, group_key);
        const int winner = __ffs(__ballot_sync(kFull, group_key == best)) - 1;
        kept |= 1u << winner;
        if (lane == winner) group_key = 0u;
      }
      // The lane's experts by their group, with one division.
      const int size = a.experts / a.groups, group = lane * V / size;
      int left = (group + 1) * size - lane * V;   // experts of this group from here on
      uint32_t bits = group < 32 ? kept >> group : 0u;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (left == 0) {
          bits >>= 1;
          left = size;
        }
        --left;
        if ((bits & 1u) == 0u) key[j] = 0u;
      }
    }
    int mine = -1;
    if constexpr (kByLogit) {
      bool close;
      mine = PickPacked<V>(key, a.top_k, &close);
      // 16-bit logits that are not equal differ in the bits that were compared.
      if (sizeof(T) == 4 && close) mine = PickExactly<V>(key, a.top_k);
    } else {
      mine = PickExactly<V>(key, a.top_k);   // (packed: 25 us for 8191 tokens instead of 23.5)
    }
    const float logit = mine >= 0 ? ToFloat(row[mine]) : -INFINITY;
    float score = 0.0f;
    if (kByLogit && a.groups == 1 && a.renormalize != 0) top = __shfl_sync(kFull, logit, 0);
    if (mine >= 0) {
      // The weights need no more than the divisions' two units in the last place.
      score = a.softmax != 0 ? __fdividef(expf(logit - top), total) : __fdividef(1.0f, 1.0f + expf(-logit));
      if (nan) score = __uint_as_float(0x7fc00000u);
    }
    // (A single choice has the weight 1 exactly.)
    if (a.renormalize != 0) score = __fdiv_rn(score, ChosenSum(score, a.top_k) + 1e-20f);
    if (lane < a.top_k) {
      a.chosen[entry] = mine;
      a.weights[entry] = mine < 0 ? 0.0f : score * a.scale;
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
template <typename T, int V, bool kByLogit>
__global__ void __launch_bounds__(1024) RouteOneBlock(RouteArgs a, bool vector) {
  extern __shared__ int route_smem[];
  LetNextStart();
  WaitForPrevious();
  int* first = route_smem;                        // experts + 1
  int* by_warp = first + a.experts + 1;           // warps x (experts + 1)
  float* values = reinterpret_cast<float*>(by_warp);   // reused: the choice is over before rows are placed
  for (int e = threadIdx.x; e <= a.experts; e += blockDim.x) first[e] = 0;
  SelectTokens<T, V, kByLogit>(a, 0, a.tokens, values, vector);
  __syncthreads();
  CountEntries(a, 0, a.tokens * a.top_k, first);
  __syncthreads();
  PrefixByWarp(first, a.experts);
  __syncthreads();
  for (int e = threadIdx.x; e <= a.experts; e += blockDim.x) a.offsets[e] = first[e];
  PlaceEntries(a, 0, a.tokens * a.top_k, first, by_warp);
}

template <typename T, int V, bool kByLogit>
__global__ void __launch_bounds__(kRouteThreads) RouteSelect(RouteArgs a, int64_t tokens_per_block, bool vector) {
  extern __shared__ int route_smem[];
  LetNextStart();
  WaitForPrevious();
  int* bins = route_smem;
  float* values = reinterpret_cast<float*>(bins + a.experts);
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) bins[e] = 0;
  const int64_t begin = blockIdx.x * tokens_per_block;
  const int64_t end = begin + tokens_per_block < a.tokens ? begin + tokens_per_block : a.tokens;
  SelectTokens<T, V, kByLogit>(a, begin, end, values, vector);
  __syncthreads();
  CountEntries(a, begin * a.top_k, end * a.top_k, bins);
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += blockDim.x) a.counts[blockIdx.x * int64_t{a.experts} + e] = bins[e];
}

// Each block's counts become the counts of the blocks before it; the totals go
// in the row after the last block's.  A block has 8 experts (a 32-byte sector of
// every row of counts), a thread a run of one expert's counts.
constexpr int kScanThreads = 1024, kScanExperts = 8;
__global__ void __launch_bounds__(kScanThreads) RouteScan(RouteArgs a, int blocks) {
  constexpr int kRuns = kScanThreads / kScanExperts, kWarps = kScanThreads / 32;
  __shared__ int sums[kWarps][kScanExperts];
  LetNextStart();
  WaitForPrevious();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int column = lane % kScanExperts, e = blockIdx.x * kScanExperts + column;
  const int run = (blocks + kRuns - 1) / kRuns, from = threadIdx.x / kScanExperts * run, to = min(blocks, from + run);
  int32_t* cells = a.counts + e;
  int sum = 0;
  if (e < a.experts) {
#pragma unroll 8
    for (int b = from; b < to; ++b) sum += cells[b * int64_t{a.experts}];
  }
  int before = sum;   // of the runs before this one in the warp, and this one
#pragma unroll
  for (int d = kScanExperts; d < 32; d *= 2) {
    const int other = __shfl_up_sync(kFull, before, d);
    if (lane >= d) before += other;
  }
  if (lane >= 32 - kScanExperts) sums[warp][column] = before;
  before -= sum;
  __syncthreads();
  int all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const int value = sums[w][column];
    before += w < warp ? value : 0;
    all += value;
  }
  if (e >= a.experts) return;
#pragma unroll 8
  for (int b = from; b < to; ++b) {
    const int count = cells[b * int64_t{a.experts}];
    cells[b * int64_t{a.experts}] = before;
    before += count;
  }
  if (threadIdx.x < kScanExperts) cells[blocks * int64_t{a.experts}] = all;
}

constexpr int kPlaceThreads = 128;
__global__ void __launch_bounds__(kPlaceThreads) RoutePlace(RouteArgs a, int64_t tokens_per_block) {
  extern __shared__ int route_smem[];
  int* first = route_smem;                  // experts + 1
  int* by_warp = first + a.experts + 1;
  LetNextStart();
  WaitForPrevious();
  const int32_t* totals = a.counts + gridDim.x * int64_t{a.experts};
  for (int e = threadIdx.x; e < a.experts; e += kPlaceThreads) first[e] = totals[e];
  __syncthreads();
  PrefixByWarp(first, a.experts);
  __syncthreads();
  const int64_t begin = blockIdx.x * tokens_per_block;
  const int64_t end = begin + tokens_per_block < a.tokens ? begin + tokens_per_block : a.tokens;
  int present = 0;   // entries with an expert before this block
  for (int e = threadIdx.x; e <= a.experts; e += kPlaceThreads) {
    if (blockIdx.x == 0) a.offsets[e] = first[e];
    if (e < a.experts) {
      const int before = a.counts[blockIdx.x * int64_t{a.experts} + e];
      present += before;
      first[e] += before;
    }
  }
  present = __reduce_add_sync(kFull, present);
  int* absent = first + a.experts;   // holds the entries that have an expert
  if ((threadIdx.x & 31) == 0) by_warp[threadIdx.x >> 5] = present;
  __syncthreads();
  if (threadIdx.x == 0) {
    int sum = 0;
    for (int w = 0; w < kPlaceThreads / 32; ++w) sum += by_warp[w];
    *absent += static_cast<int>(begin * a.top_k) - sum;
  }
  __syncthreads();
  PlaceEntries(a, begin * a.top_k, end * a.top_k, first, by_warp);
}

// With g = scale * (gradient of the chosen weights) and p the chosen scores:
//   renormalised: g <- (g - sum(g p) / total) / total, total = sum p + 1e-20
//   softmax: dx_j = s_j (ds_j - sum(g p)),  ds the scattered g
//   sigmoid: dx_j = ds_j s_j (1 - s_j)
// Reads and writes each logit once; the scores are recomputed.  (The fast
// exponential is off by 4e-6 of a score 80 below the largest, which a bias or a
// group may have chosen.)  A warp has one token: instructions bound it, and a
// loop's cost more than launching.
template <typename T, int V, bool kSoftmax>
__global__ void __launch_bounds__(kRouteThreads) RouteBackward(RouteBackwardArgs a, bool vector) {
  __shared__ __align__(16) float scattered[kRouteThreads / 32][32 * V];   // ds
  LetNextStart();
  WaitForPrevious();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = static_cast<int>(blockIdx.x) * (kRouteThreads / 32) + warp;   // there are at most 2^31 - 256 tokens
  if (t >= static_cast<int>(a.tokens)) return;
  const T* row = static_cast<const T*>(a.logits) + int64_t{t} * static_cast<int>(a.logit_stride);
  int mine = -1;
  float g = 0.0f, logit = -INFINITY, d[V];
  if (lane < a.top_k) {
    mine = a.chosen[t * a.top_k + lane];
    g = a.weights_grad[t * a.top_k + lane] * a.scale;
  }
  float* ds = scattered[warp];
#pragma unroll
  for (int j = 0; j < V; ++j) ds[j * 32 + lane] = d[j] = 0.0f;
  const bool found = mine >= 0 && mine < a.experts;
  if (__any_sync(kFull, found)) {   // otherwise the logits may hold anything
    if (found) logit = ToFloat(row[mine]);
    if (!found) g = 0.0f;
    float x[V], p;
    if constexpr (kSoftmax) {
      LoadLogits<T, V>(row, a.experts, lane, vector, x);   // -inf past the last expert
      const float top = Largest<V>(x);
      float sum = 0.0f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        x[j] = expf(x[j] - top);
        sum += x[j];
      }
      const float inverse = __fdividef(1.0f, WarpSum(sum));
      p = expf(logit - top) * inverse;
#pragma unroll
      for (int j = 0; j < V; ++j) x[j] *= inverse;
    } else {
      p = __fdividef(1.0f, 1.0f + expf(-logit));
    }
    if (a.renormalize != 0) {
      // The weight is rounded as in the forward pass: a single choice's is 1 and
      // its gradient 0, exactly.
      const float total = ChosenSum(p, a.top_k) + 1e-20f;
      const float mean = ChosenSum(g * __fdiv_rn(p, total), a.top_k);
      g = found ? __fdividef(g - mean, total) : 0.0f;
    }
    if constexpr (kSoftmax) {
      const float inner = __shfl_sync(kFull, ChosenSum(g * p, a.top_k), 0);
      __syncwarp();
      if (found) ds[mine] = g;
      __syncwarp();
#pragma unroll
      for (int j = 0; j < V; ++j) d[j] = x[j] * (ds[lane * V + j] - inner);
    } else {
      __syncwarp();
      if (found) ds[mine] = g * p * (1.0f - p);
      __syncwarp();
#pragma unroll
      for (int j = 0; j < V; ++j) d[j] = ds[lane * V + j];
    }
  }
  StoreValues<T, V>(static_cast<T*>(a.logits_grad) + int64_t{t} * a.experts, a.experts, lane, vector, d);
}

// Up to this many tokens one block does the whole call.  Replayed, one block and
// three launches, 64 experts: 8 tokens 3.9 and 7.6 us, 64 7.1 and 7.9, 96 8.8 and 8.0;
// 16 experts: 64 tokens 5.7 and 7.3, 128 8.3 and 7.5.  (With 256 experts and a bias the
// launches are ahead from 48 tokens on, 11.3 us for 14.2.)
constexpr int64_t kOneBlockTokens = 64;

// Counting blocks: enough to fill the device with warps, each with its eight
// warps' tokens at least.
int64_t TokensPerBlock(int64_t tokens) {
  const int64_t blocks = int64_t{RoutedSmCount()} * 8;
  return std::max<int64_t>(8, ((tokens + blocks - 1) / blocks + 7) / 8 * 8);
}

template <typename T, int V, bool kByLogit>
void Route(const RouteArgs& a, cudaStream_t stream) {
  const std::size_t bins = static_cast<std::size_t>(a.experts) + 1;
  const bool vector = VectorLogits<T, V>(a.logits, a.logit_stride);
  if (a.tokens <= kOneBlockTokens) {
    const unsigned warps = static_cast<unsigned>(std::min<int64_t>(32, std::max<int64_t>(1, a.tokens)));
    const std::size_t smem = (bins + warps * bins) * sizeof(int);
    AllowShared<RouteOneBlock<T, V, kByLogit>>(static_cast<int>(smem));
    LaunchRouted("router launch", true, RouteOneBlock<T, V, kByLogit>, 1, warps * 32, smem, stream, a, vector);
    return;
  }
  const int64_t per_block = TokensPerBlock(a.tokens);
  const unsigned blocks = static_cast<unsigned>((a.tokens + per_block - 1) / per_block);
  const std::size_t select = (bins + (a.groups > 1 ? kRouteThreads / 32 * bins : 0)) * sizeof(int);
  // While the choice is short, the two launches after it are worth hiding (calls one
  // after the other, 8191 tokens: 27 us instead of 31; 32768, with the gradient: 53
  // instead of 50).
  const bool close = per_block <= 16;
  LaunchRouted("router launch", BriefGrid(blocks), RouteSelect<T, V, kByLogit>, blocks, kRouteThreads, select, stream, a, per_block, vector);
  LaunchRouted("row order launch", close, RouteScan, static_cast<unsigned>((a.experts + kScanExperts - 1) / kScanExperts),
               kScanThreads, 0, stream, a, static_cast<int>(blocks));
  LaunchRouted("row order launch", close, RoutePlace, blocks, kPlaceThreads, (1 + kPlaceThreads / 32) * bins * sizeof(int),
               stream, a, per_block);
}

template <typename T, int V>
void Backward(const RouteBackwardArgs& a, cudaStream_t stream) {
  const unsigned blocks = static_cast<unsigned>((a.tokens + kRouteThreads / 32 - 1) / (kRouteThreads / 32));
  const bool vector = VectorLogits<T, V>(a.logits, a.logit_stride) && VectorLogits<T, V>(a.logits_grad, a.experts);
  const char* what = "router gradient launch";
  if (a.softmax != 0) LaunchRouted(what, BriefGrid(blocks), RouteBackward<T, V, true>, blocks, kRouteThreads, 0, stream, a, vector);
  else LaunchRouted(what, BriefGrid(blocks), RouteBackward<T, V, false>, blocks, kRouteThreads, 0, stream, a, vector);
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
  // A row of counts per block, and their totals.
  return static_cast<std::size_t>((tokens + per_block - 1) / per_block + 1) * experts * sizeof(int32_t);
}

void LaunchRoute(int32_t dtype, const RouteArgs& args, cudaStream_t stream) {
  ByType(dtype, [&](auto type) {
    using T = decltype(type);
    ByExperts<T>(args, [&](auto values) {
      constexpr int V = decltype(values)::value;
      if (args.bias == nullptr && args.group_best == 1) Route<T, V, true>(args, stream);
      else Route<T, V, false>(args, stream);
    });
  });
}

void LaunchRouteBackward(int32_t dtype, const RouteBackwardArgs& args, cudaStream_t stream) {
  ByType(dtype, [&](auto type) {
    using T = decltype(type);
    ByExperts<T>(args, [&](auto values) { Backward<T, decltype(values)::value>(args, stream); });
  });
}

}  // namespace t0b

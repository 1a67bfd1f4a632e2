// Launch interface of the routed operators: the router, the products over
// sectors chosen at run time, the gated activation with its 8-bit checkpoint
// and the 4-bit matrix-vector products.  Arguments are validated by the C
// entry points (capi_routed.cu); the launchers choose variants and enqueue.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace t0b {

constexpr int kRouteMaxExperts = 512;
constexpr int kRouteMaxTopK = 32;
constexpr int kRouteMaxGroups = 32;

struct RouteArgs {
  const void* logits;      // [tokens, experts], row stride logit_stride
  int64_t logit_stride;
  const float* bias;       // [experts] or null
  const uint8_t* mask;     // [tokens], 0 = not routed, or null
  int64_t tokens;
  int experts, top_k, groups, top_groups;
  int group_best;          // a group's score: its best choice value (1) or the sum of its two best (2)
  int softmax, renormalize;
  float scale;
  int32_t* chosen;         // [tokens, top_k]
  float* weights;          // [tokens, top_k]
  int32_t* rows;           // [tokens * top_k]
  int32_t* positions;      // [tokens, top_k]
  int32_t* offsets;        // [experts + 1]
  int32_t* counts;         // workspace [counting blocks + 1, experts]
};

struct RouteBackwardArgs {
  const void* logits;
  int64_t logit_stride;
  const int32_t* chosen;
  const float* weights_grad;
  int64_t tokens;
  int experts, top_k, softmax, renormalize;
  float scale;
  void* logits_grad;       // [tokens, experts], contiguous
};

// Workspace of one LaunchRoute call in bytes (0: none).
std::size_t RouteWorkspace(int64_t tokens, int experts);
void LaunchRoute(int32_t dtype, const RouteArgs& args, cudaStream_t stream);
void LaunchRouteBackward(int32_t dtype, const RouteBackwardArgs& args, cudaStream_t stream);

// One product per expert over the rows [offsets[e], offsets[e + 1]).
struct ProductArgs {
  const void* x;           // token rows (gather) or expert-ordered rows
  int64_t x_rows, x_stride;
  const void* w;           // weights [experts, inner, outer]; for the weight gradient: y_grad rows
  int64_t w_rows, w_stride;   // the weight gradient's y_grad only
  void* out;
  int64_t out_stride;      // elements between output rows (products)
  const int32_t* rows;     // entry of each expert-ordered row
  const int32_t* offsets;  // [experts + 1]
  int64_t entries;         // expert-ordered rows, absent ones included
  int experts, top_k, inner, outer;
  int gather_x, gather_w;  // row p of the operand is rows[p] / top_k
};

enum ProductKind : int { kProduct = 0, kProductTransposed = 1, kProductWeightGrad = 2 };
void LaunchProduct(int kind, int32_t dtype, const ProductArgs& args, cudaStream_t stream);
// The tensor-core kernel of LaunchProduct, where it takes the operands.
bool TensorCoreProduct(int kind, const ProductArgs& args);
void LaunchTensorCoreProduct(int kind, int32_t dtype, const ProductArgs& args, cudaStream_t stream);

// out[t] = sum over the token's slots of y[positions[t, slot]].
struct RoutedSumArgs {
  const void* y;
  int64_t y_stride;
  const int32_t* positions;
  int64_t tokens, entries;
  int top_k, width;
  void* out;
  int64_t out_stride;
};
void LaunchRoutedSum(int32_t dtype, const RoutedSumArgs& args, cudaStream_t stream);

struct GatedArgs {
  const void* h;           // [rows, 2 * width] (save)
  int64_t h_stride;
  int8_t* codes;           // [rows, 2 * width], contiguous
  float* scales;           // [rows, 2 * ceil(width / group)]
  int64_t rows_count;
  int width, group;
  const float* weights;    // [rows] by entry, or null: all 1
  const int32_t* rows;     // entry of each row, with weights
  const int32_t* offsets;  // rows from offsets[experts] on are absent, with weights
  int experts;
  void* a;                 // [rows, width]
  const void* a_grad;      // backward
  int64_t a_grad_stride;
  void* h_grad;            // [rows, 2 * width]
  float* weights_grad;     // [rows] by entry
};
void LaunchGatedSave(int32_t dtype, const GatedArgs& args, cudaStream_t stream);
void LaunchGatedBackward(int32_t dtype, const GatedArgs& args, cudaStream_t stream);
void LaunchCheckpointLoad(int32_t dtype, const GatedArgs& args, void* values, cudaStream_t stream);

struct MatvecArgs {
  const void* x;           // token rows (gather) or expert-ordered rows
  int64_t x_rows, x_stride;
  const uint8_t* codes;    // [experts, outer, inner / 2]
  const void* scales;      // [experts, outer, inner / group]
  const int32_t* rows;
  const int32_t* offsets;
  int64_t entries;
  int experts, top_k, inner, outer, group, gather;
  void* out;               // [entries, outer]
};
void LaunchMatvec(int32_t dtype, const MatvecArgs& args, cudaStream_t stream);

}  // namespace t0b

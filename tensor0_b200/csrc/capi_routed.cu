// C ABI of the routed operators (include/tensor0_b200.h): argument validation
// before any write, then stream-ordered launches.  No entry point
// synchronizes, allocates or reads device memory on the host.
#include "../../include/tensor0_b200.h"

#include "guard.h"
#include "routed.h"

#include <cmath>

namespace {

using t0b::Bytes;
using t0b::Disjoint;
using t0b::Guard;
using t0b::InvalidArgument;

constexpr int64_t kMaxRows = (int64_t{1} << 31) - 1;         // gated rows, row strides
// Router and products index entries in 32 bits, up to a tile of rows or a
// block's tokens past the last one.
constexpr int64_t kMaxEntries = (int64_t{1} << 31) - 256;
constexpr int32_t kMaxWidth = 1 << 23;   // blocks of 256 columns fit a grid axis

uint64_t Half(int32_t dtype, const char* what) {
  if (dtype != T0B_F16 && dtype != T0B_BF16) throw InvalidArgument(std::string(what) + " take F16 or BF16");
  return 2;
}

void Require(bool condition, const char* message) {
  if (!condition) throw InvalidArgument(message);
}

// An operand of `rows` rows: present, aligned to its element and spaced by at
// least its width.  Its extent in bytes.
uint64_t Operand(const void* data, int64_t rows, int64_t width, int64_t stride, uint64_t item, const char* what) {
  if (rows < 0 || width < 0) throw InvalidArgument(std::string(what) + " sizes must be nonnegative");
  if (stride < width) throw InvalidArgument(std::string(what) + " row stride is below the row's width");
  if (stride > kMaxRows) throw InvalidArgument(std::string(what) + " row stride must be at most 2^31 - 1");
  if (rows == 0 || width == 0) return 0;
  if (data == nullptr) throw InvalidArgument(std::string(what) + " buffer is null");
  if (reinterpret_cast<uintptr_t>(data) % item != 0) {
    throw InvalidArgument(std::string(what) + " buffer is not aligned to its element size");
  }
  uint64_t span = 0;
  if (!t0b::CheckedMul(static_cast<uint64_t>(rows - 1), static_cast<uint64_t>(stride), &span) ||
      !t0b::CheckedAdd(span, static_cast<uint64_t>(width), &span)) {
    throw InvalidArgument("buffer size exceeds addressable storage");
  }
  return Bytes(span, item);
}

uint64_t Packed(const void* data, int64_t rows, int64_t width, uint64_t item, const char* what) {
  return Operand(data, rows, width, width, item, what);
}

struct Extent {
  const void* data;
  uint64_t bytes;
};

// No output may overlap an input or another output.
void Separate(std::initializer_list<Extent> outputs, std::initializer_list<Extent> inputs) {
  for (auto out = outputs.begin(); out != outputs.end(); ++out) {
    for (const Extent& in : inputs) Disjoint(in.data, in.bytes, out->data, out->bytes);
    for (auto other = out + 1; other != outputs.end(); ++other) {
      Disjoint(other->data, other->bytes, out->data, out->bytes);
    }
  }
}

void RequireRouting(int64_t entries, int32_t experts, int32_t top_k) {
  Require(entries >= 0 && entries <= kMaxEntries, "routed entries must be at most 2^31 - 256");
  Require(experts >= 1 && experts <= t0b::kRouteMaxExperts, "routed operators take 1 to 512 experts");
  Require(top_k >= 1 && top_k <= t0b::kRouteMaxTopK, "top_k must be from 1 to 32");
  Require(entries % top_k == 0, "routed entries must be a multiple of top_k");
}

uint64_t RequireScore(int32_t dtype, int64_t tokens, int32_t experts, int32_t top_k, int32_t score, int32_t renormalize,
                      float scale) {
  Require(dtype == T0B_F32 || dtype == T0B_F16 || dtype == T0B_BF16, "router logits must be F32, F16 or BF16");
  Require(tokens >= 0, "token count must be nonnegative");
  Require(experts >= 1 && experts <= t0b::kRouteMaxExperts, "routed operators take 1 to 512 experts");
  Require(top_k >= 1 && top_k <= t0b::kRouteMaxTopK && top_k <= experts,
          "top_k must be from 1 to 32 and at most the number of experts");
  Require(tokens <= kMaxEntries / top_k, "routed entries must be at most 2^31 - 256");
  Require(score == 0 || score == 1, "router score must be 0 (softmax) or 1 (sigmoid)");
  Require(renormalize == 0 || renormalize == 1, "renormalize must be zero or one");
  Require(std::isfinite(scale), "router scale must be finite");
  return dtype == T0B_F32 ? 4 : 2;
}

void RequireGroup(int32_t width, int32_t group) {
  Require(width >= 1 && width <= kMaxWidth, "gated width must be from 1 to 2^23");
  Require(group == 32 || group == 64 || group == 128, "checkpoint group must be 32, 64 or 128");
}

// Bytes of a gated routing's arrays: its weights and its rows each, and its offsets.
struct RowWeightBytes {
  uint64_t entries = 0, offsets = 0;
};

// The routing of gated rows: all given or none.
RowWeightBytes RequireRowWeights(const float* weights, const int32_t* row_entries, const int32_t* offsets,
                                 int32_t experts, int64_t rows) {
  Require(rows >= 0 && rows <= kMaxRows, "gated rows must be at most 2^31 - 1");
  const bool some = weights != nullptr || row_entries != nullptr || offsets != nullptr;
  if (!some) return {};
  Require((weights != nullptr && row_entries != nullptr && offsets != nullptr) || rows == 0,
          "a gated routing is its weights, its rows and its offsets");
  Require(experts >= 1 && experts <= t0b::kRouteMaxExperts, "routed operators take 1 to 512 experts");
  RowWeightBytes bytes;
  bytes.entries = Packed(weights, rows, 1, 4, "weight");
  Packed(row_entries, rows, 1, 4, "row");
  if (rows != 0) bytes.offsets = Packed(offsets, experts + 1, 1, 4, "offset");
  return bytes;
}

void Product(int kind, int32_t dtype, const t0b::ProductArgs& a, uint64_t out_width, int64_t out_rows, void* stream) {
  RequireRouting(a.entries, a.experts, a.top_k);
  Require(a.inner >= 1 && a.outer >= 1 && a.inner <= kMaxWidth && a.outer <= kMaxWidth,
          "product widths must be from 1 to 2^23");
  Require((a.gather_x == 0 || a.gather_x == 1) && (a.gather_w == 0 || a.gather_w == 1), "gather must be zero or one");
  const uint64_t item = Half(dtype, "routed products");
  const int64_t matrices = int64_t{a.experts} * a.inner;
  Require(a.gather_x != 0 || a.x_rows == a.entries, "an expert-ordered operand has one row per entry");
  Require(a.gather_x == 0 || a.x_rows == a.entries / a.top_k, "a gathered operand has one row per token");
  const int x_width = kind == t0b::kProductTransposed ? a.outer : a.inner;
  const uint64_t x_bytes = Operand(a.x, a.x_rows, x_width, a.x_stride, item, "product");
  uint64_t w_bytes = 0;
  if (kind == t0b::kProductWeightGrad) {
    Require(a.gather_w != 0 || a.w_rows == a.entries, "an expert-ordered operand has one row per entry");
    Require(a.gather_w == 0 || a.w_rows == a.entries / a.top_k, "a gathered operand has one row per token");
    w_bytes = Operand(a.w, a.w_rows, a.outer, a.w_stride, item, "product");
  } else {
    w_bytes = Packed(a.w, matrices, a.outer, item, "weight");
  }
  const uint64_t out_bytes = Packed(a.out, out_rows, static_cast<int64_t>(out_width), item, "product output");
  const uint64_t row_bytes = Packed(a.rows, a.entries, 1, 4, "row");
  const uint64_t offset_bytes = Packed(a.offsets, a.experts + 1, 1, 4, "offset");
  Separate({{a.out, out_bytes}}, {{a.x, x_bytes}, {a.w, w_bytes}, {a.rows, row_bytes}, {a.offsets, offset_bytes}});
  if (out_bytes == 0) return;
  t0b::LaunchProduct(kind, dtype, a, static_cast<cudaStream_t>(stream));
}

}  // namespace

extern "C" {

size_t t0b_route_workspace(int64_t tokens, int32_t experts) {
  if (tokens < 0 || tokens > kMaxEntries || experts < 1 || experts > t0b::kRouteMaxExperts) return 0;
  return t0b::RouteWorkspace(tokens, experts);
}

int t0b_route(int32_t dtype, int64_t tokens, int32_t experts, int32_t top_k, int32_t groups, int32_t top_groups,
              int32_t group_best, int32_t score, int32_t renormalize, float scale, const void* logits,
              int64_t logit_stride, const float* bias, const uint8_t* mask, int32_t* chosen, float* weights,
              int32_t* rows, int32_t* positions, int32_t* offsets, void* workspace, size_t workspace_size,
              void* stream, char* error, size_t error_size) {
  return Guard(error, error_size, [&] {
    const uint64_t item = RequireScore(dtype, tokens, experts, top_k, score, renormalize, scale);
    Require(groups >= 1 && groups <= t0b::kRouteMaxGroups && experts % groups == 0,
            "expert groups must divide the experts evenly, 32 groups at most");
    Require(top_groups >= 1 && top_groups <= groups, "top_groups must be from 1 to the number of groups");
    Require(group_best == 1 || group_best == 2, "group_best must be 1 or 2");
    const int64_t entries = tokens * top_k;
    const uint64_t logit_bytes = Operand(logits, tokens, experts, logit_stride, item, "logits");
    const uint64_t entry_bytes = static_cast<uint64_t>(entries) * 4;
    Packed(chosen, entries, 1, 4, "choice");
    Packed(weights, entries, 1, 4, "weight");
    Packed(rows, entries, 1, 4, "row");
    Packed(positions, entries, 1, 4, "position");
    const uint64_t offset_bytes = Packed(offsets, experts + 1, 1, 4, "offset");
    const uint64_t bias_bytes = bias != nullptr ? Packed(bias, experts, 1, 4, "bias") : 0;
    const uint64_t need = t0b::RouteWorkspace(tokens, experts);
    Require(workspace_size >= need, "router workspace is too small");
    const uint64_t work_bytes = Packed(workspace, static_cast<int64_t>(need / 4), 1, 4, "router workspace");
    Separate({{chosen, entry_bytes}, {weights, entry_bytes}, {rows, entry_bytes}, {positions, entry_bytes},
              {offsets, offset_bytes}, {workspace, work_bytes}},
             {{logits, logit_bytes}, {bias, bias_bytes}, {mask, mask != nullptr ? static_cast<uint64_t>(tokens) : 0}});
    t0b::RouteArgs a{};
    a.logits = logits;
    a.logit_stride = logit_stride;
    a.bias = bias;
    a.mask = mask;
    a.tokens = tokens;
    a.experts = experts;
    a.top_k = top_k;
    a.groups = groups;
    a.top_groups = top_groups;
    a.group_best = group_best;
    a.softmax = score == 0 ? 1 : 0;
    a.renormalize = renormalize;
    a.scale = scale;
    a.chosen = chosen;
    a.weights = weights;
    a.rows = rows;
    a.positions = positions;
    a.offsets = offsets;
    a.counts = static_cast<int32_t*>(workspace);
    t0b::LaunchRoute(dtype, a, static_cast<cudaStream_t>(stream));
  });
}

int t0b_route_backward(int32_t dtype, int64_t tokens, int32_t experts, int32_t top_k, int32_t score,
                       int32_t renormalize, float scale, const void* logits, int64_t logit_stride,
                       const int32_t* chosen, const float* weights_grad, void* logits_grad, void* stream,
                       char* error, size_t error_size) {
  return Guard(error, error_size, [&] {
    const uint64_t item = RequireScore(dtype, tokens, experts, top_k, score, renormalize, scale);
    const int64_t entries = tokens * top_k;
    const uint64_t logit_bytes = Operand(logits, tokens, experts, logit_stride, item, "logits");
    const uint64_t entry_bytes = Packed(chosen, entries, 1, 4, "choice");
    Packed(weights_grad, entries, 1, 4, "weight gradient");
    const uint64_t out_bytes = Packed(logits_grad, tokens, experts, item, "logits gradient");
    Separate({{logits_grad, out_bytes}}, {{logits, logit_bytes}, {chosen, entry_bytes}, {weights_grad, entry_bytes}});
    if (tokens == 0) return;
    t0b::RouteBackwardArgs a{};
    a.logits = logits;
    a.logit_stride = logit_stride;
    a.chosen = chosen;
    a.weights_grad = weights_grad;
    a.tokens = tokens;
    a.experts = experts;
    a.top_k = top_k;
    a.softmax = score == 0 ? 1 : 0;
    a.renormalize = renormalize;
    a.scale = scale;
    a.logits_grad = logits_grad;
    t0b::LaunchRouteBackward(dtype, a, static_cast<cudaStream_t>(stream));
  });
}

int t0b_routed_product(int32_t dtype, int32_t transposed, int64_t entries, int32_t experts, int32_t top_k,
                       int32_t inner, int32_t outer, int32_t gather, const void* x, int64_t x_rows, int64_t x_stride,
                       const void* w, const int32_t* rows, const int32_t* offsets, void* output, void* stream,
                       char* error, size_t error_size) {
  return Guard(error, error_size, [&] {
    Require(transposed == 0 || transposed == 1, "transposed must be zero or one");
    const int32_t width = transposed != 0 ? inner : outer;
    t0b::ProductArgs a{};
    a.x = x;
    a.x_rows = x_rows;
    a.x_stride = x_stride;
    a.w = w;
    a.out = output;
    a.out_stride = width;
    a.rows = rows;
    a.offsets = offsets;
    a.entries = entries;
    a.experts = experts;
    a.top_k = top_k;
    a.inner = inner;
    a.outer = outer;
    a.gather_x = gather;
    Product(transposed != 0 ? t0b::kProductTransposed : t0b::kProduct, dtype, a, static_cast<uint64_t>(width), entries,
            stream);
  });
}

int t0b_routed_weight_grad(int32_t dtype, int64_t entries, int32_t experts, int32_t top_k, int32_t inner,
                           int32_t outer, int32_t gather_x, const void* x, int64_t x_rows, int64_t x_stride,
                           int32_t gather_y, const void* y, int64_t y_rows, int64_t y_stride, const int32_t* rows,
                           const int32_t* offsets, void* output, void* stream, char* error, size_t error_size) {
  return Guard(error, error_size, [&] {
    t0b::ProductArgs a{};
    a.x = x;
    a.x_rows = x_rows;
    a.x_stride = x_stride;
    a.w = y;
    a.w_rows = y_rows;
    a.w_stride = y_stride;
    a.out = output;
    a.out_stride = outer;
    a.rows = rows;
    a.offsets = offsets;
    a.entries = entries;
    a.experts = experts;
    a.top_k = top_k;
    a.inner = inner;
    a.outer = outer;
    a.gather_x = gather_x;
    a.gather_w = gather_y;
    Product(t0b::kProductWeightGrad, dtype, a, static_cast<uint64_t>(outer), int64_t{experts} * inner, stream);
  });
}

int t0b_routed_sum(int32_t dtype, int64_t tokens, int32_t top_k, int32_t width, const void* y, int64_t y_stride,
                   const int32_t* positions, void* output, void* stream, char* error, size_t error_size) {
  return Guard(error, error_size, [&] {
    const uint64_t item = Half(dtype, "routed sums");
    Require(tokens >= 0, "token count must be nonnegative");
    Require(top_k >= 1 && top_k <= t0b::kRouteMaxTopK, "top_k must be from 1 to 32");
    Require(tokens <= kMaxEntries / top_k, "routed entries must be at most 2^31 - 256");
    Require(width >= 1 && width <= kMaxWidth, "sum width must be from 1 to 2^23");
    const int64_t entries = tokens * top_k;
    const uint64_t y_bytes = Operand(y, entries, width, y_stride, item, "sum");
    const uint64_t position_bytes = Packed(positions, entries, 1, 4, "position");
    const uint64_t out_bytes = Packed(output, tokens, width, item, "sum output");
    Separate({{output, out_bytes}}, {{y, y_bytes}, {positions, position_bytes}});
    if (tokens == 0) return;
    t0b::RoutedSumArgs a{};
    a.y = y;
    a.y_stride = y_stride;
    a.positions = positions;
    a.tokens = tokens;
    a.entries = entries;
    a.top_k = top_k;
    a.width = width;
    a.out = output;
    a.out_stride = width;
    t0b::LaunchRoutedSum(dtype, a, static_cast<cudaStream_t>(stream));
  });
}

int t0b_gated_save(int32_t dtype, int64_t row_count, int32_t width, int32_t group, const void* h, int64_t h_stride,
                   const float* weights, const int32_t* row_entries, const int32_t* offsets, int32_t experts,
                   void* a, int8_t* codes, float* scales, void* stream, char* error, size_t error_size) {
  return Guard(error, error_size, [&] {
    const uint64_t item = Half(dtype, "gated activations");
    RequireGroup(width, group);
    const RowWeightBytes routing = RequireRowWeights(weights, row_entries, offsets, experts, row_count);
    const int64_t groups = (int64_t{width} + group - 1) / group;
    const uint64_t h_bytes = Operand(h, row_count, int64_t{2} * width, h_stride, item, "activation input");
    const uint64_t a_bytes = Packed(a, row_count, width, item, "activation");
    Require((codes == nullptr) == (scales == nullptr), "a checkpoint is its codes and its scales");
    const int64_t kept = codes != nullptr ? row_count : 0;
    const uint64_t code_bytes = Packed(codes, kept, int64_t{2} * width, 1, "checkpoint code");
    const uint64_t scale_bytes = Packed(scales, kept, 2 * groups, 4, "checkpoint scale");
    Separate({{a, a_bytes}, {codes, code_bytes}, {scales, scale_bytes}},
             {{h, h_bytes}, {weights, routing.entries}, {row_entries, routing.entries}, {offsets, routing.offsets}});
    if (row_count == 0) return;
    t0b::GatedArgs args{};
    args.h = h;
    args.h_stride = h_stride;
    args.codes = codes;
    args.scales = scales;
    args.rows_count = row_count;
    args.width = width;
    args.group = group;
    args.weights = weights;
    args.rows = row_entries;
    args.offsets = offsets;
    args.experts = experts;
    args.a = a;
    t0b::LaunchGatedSave(dtype, args, static_cast<cudaStream_t>(stream));
  });
}

int t0b_gated_backward(int32_t dtype, int64_t row_count, int32_t width, int32_t group, const int8_t* codes,
                       const float* scales, const void* a_grad, int64_t a_grad_stride, const float* weights,
                       const int32_t* row_entries, const int32_t* offsets, int32_t experts, void* h_grad, void* a,
                       float* weights_grad, void* stream, char* error, size_t error_size) {
  return Guard(error, error_size, [&] {
    const uint64_t item = Half(dtype, "gated activations");
    RequireGroup(width, group);
    const RowWeightBytes routing = RequireRowWeights(weights, row_entries, offsets, experts, row_count);
    const int64_t groups = (int64_t{width} + group - 1) / group;
    const uint64_t code_bytes = Packed(codes, row_count, int64_t{2} * width, 1, "checkpoint code");
    const uint64_t scale_bytes = Packed(scales, row_count, 2 * groups, 4, "checkpoint scale");
    const uint64_t grad_bytes = Operand(a_grad, row_count, width, a_grad_stride, item, "activation gradient");
    const uint64_t a_bytes = Packed(a, row_count, width, item, "activation");
    const uint64_t h_bytes = Packed(h_grad, row_count, int64_t{2} * width, item, "input gradient");
    const uint64_t w_bytes = weights_grad != nullptr ? Packed(weights_grad, row_count, 1, 4, "weight gradient") : 0;
    Separate({{a, a_bytes}, {h_grad, h_bytes}, {weights_grad, w_bytes}},
             {{codes, code_bytes}, {scales, scale_bytes}, {a_grad, grad_bytes}, {weights, routing.entries},
              {row_entries, routing.entries}, {offsets, routing.offsets}});
    if (row_count == 0) return;
    t0b::GatedArgs args{};
    args.codes = const_cast<int8_t*>(codes);
    args.scales = const_cast<float*>(scales);
    args.rows_count = row_count;
    args.width = width;
    args.group = group;
    args.weights = weights;
    args.rows = row_entries;
    args.offsets = offsets;
    args.experts = experts;
    args.a = a;
    args.a_grad = a_grad;
    args.a_grad_stride = a_grad_stride;
    args.h_grad = h_grad;
    args.weights_grad = weights_grad;
    t0b::LaunchGatedBackward(dtype, args, static_cast<cudaStream_t>(stream));
  });
}

int t0b_checkpoint_load(int32_t dtype, int64_t row_count, int32_t width, int32_t group, const int8_t* codes,
                        const float* scales, void* values, void* stream, char* error, size_t error_size) {
  return Guard(error, error_size, [&] {
    Require(dtype == T0B_F32 || dtype == T0B_F16 || dtype == T0B_BF16, "checkpoints load as F32, F16 or BF16");
    RequireGroup(width, group);
    Require(row_count >= 0 && row_count <= kMaxRows, "gated rows must be at most 2^31 - 1");
    const int64_t groups = (int64_t{width} + group - 1) / group;
    const uint64_t code_bytes = Packed(codes, row_count, int64_t{2} * width, 1, "checkpoint code");
    const uint64_t scale_bytes = Packed(scales, row_count, 2 * groups, 4, "checkpoint scale");
    const uint64_t out_bytes = Packed(values, row_count, int64_t{2} * width, dtype == T0B_F32 ? 4 : 2, "value");
    Separate({{values, out_bytes}}, {{codes, code_bytes}, {scales, scale_bytes}});
    if (row_count == 0) return;
    t0b::GatedArgs args{};
    args.codes = const_cast<int8_t*>(codes);
    args.scales = const_cast<float*>(scales);
    args.rows_count = row_count;
    args.width = width;
    args.group = group;
    t0b::LaunchCheckpointLoad(dtype, args, values, static_cast<cudaStream_t>(stream));
  });
}

int t0b_routed_matvec4(int32_t dtype, int64_t entries, int32_t experts, int32_t top_k, int32_t inner, int32_t outer,
                       int32_t group, int32_t gather, const void* x, int64_t x_rows, int64_t x_stride,
                       const uint8_t* codes, const void* scales, const int32_t* rows, const int32_t* offsets,
                       void* output, void* stream, char* error, size_t error_size) {
  return Guard(error, error_size, [&] {
    const uint64_t item = Half(dtype, "4-bit products");
    RequireRouting(entries, experts, top_k);
    Require(group == 32 || group == 64 || group == 128, "weight group must be 32, 64 or 128");
    Require(inner >= 1 && outer >= 1 && inner <= kMaxWidth && outer <= kMaxWidth, "product widths must be from 1 to 2^23");
    Require(inner % group == 0, "weight groups must divide the inner width");
    Require(gather == 0 || gather == 1, "gather must be zero or one");
    Require(x_rows == (gather != 0 ? entries / top_k : entries), "an operand has one row per token (gather) or entry");
    Require(reinterpret_cast<uintptr_t>(codes) % 16 == 0, "4-bit weights must be 16-byte aligned");
    const int64_t matrices = int64_t{experts} * outer;
    const uint64_t x_bytes = Operand(x, x_rows, inner, x_stride, item, "product");
    const uint64_t code_bytes = Packed(codes, matrices, inner / 2, 1, "4-bit weight");
    const uint64_t scale_bytes = Packed(scales, matrices, inner / group, item, "weight scale");
    const uint64_t row_bytes = Packed(rows, entries, 1, 4, "row");
    const uint64_t offset_bytes = Packed(offsets, experts + 1, 1, 4, "offset");
    const uint64_t out_bytes = Packed(output, entries, outer, item, "product output");
    Separate({{output, out_bytes}}, {{x, x_bytes}, {codes, code_bytes}, {scales, scale_bytes}, {rows, row_bytes},
                                     {offsets, offset_bytes}});
    if (entries == 0) return;
    t0b::MatvecArgs a{};
    a.x = x;
    a.x_rows = x_rows;
    a.x_stride = x_stride;
    a.codes = codes;
    a.scales = scales;
    a.rows = rows;
    a.offsets = offsets;
    a.entries = entries;
    a.experts = experts;
    a.top_k = top_k;
    a.inner = inner;
    a.outer = outer;
    a.group = group;
    a.gather = gather;
    a.out = output;
    t0b::LaunchMatvec(dtype, a, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"

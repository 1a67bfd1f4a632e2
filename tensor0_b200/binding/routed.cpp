// Python binding of the routed operators: tensors to the C entry points of
// include/tensor0_b200.h.
//
// A serving step calls these for one token, where the operators take 4 to 8 us:
// the argument checks and the call are compiled (4 to 6 us a call with its
// launch and result; the same checks in Python and ctypes took 11 to 14).  Shapes,
// types, strides, devices and autograd are checked here, values, sizes and overlaps
// by the entry points.  Every refusal is a ValueError, every other failure a
// RuntimeError.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <stdexcept>
#include <string>

#include "tensor0_b200.h"

namespace {

using at::Tensor;

struct Refusal : std::invalid_argument {
  using std::invalid_argument::invalid_argument;
};

// A C entry point's failure that is not an invalid argument.
struct Failure : std::runtime_error {
  using std::runtime_error::runtime_error;
};

// A Python error is already set.
struct Raised {};

std::string Text(at::IntArrayRef sizes) {
  std::string text = "[";
  for (size_t i = 0; i < sizes.size(); ++i) text += (i != 0 ? ", " : "") + std::to_string(sizes[i]);
  return text + "]";
}

const char* Name(at::ScalarType type) {
  switch (type) {
    case at::kFloat: return "float32";
    case at::kHalf: return "float16";
    case at::kBFloat16: return "bfloat16";
    case at::kInt: return "int32";
    case at::kBool: return "bool";
    case at::kChar: return "int8";
    case at::kByte: return "uint8";
    default: return c10::toString(type);
  }
}

const Tensor& Get(PyObject* object, const char* what) {
  if (!THPVariable_Check(object)) throw Refusal(std::string(what) + " must be a tensor");
  return THPVariable_Unpack(object);
}

long long Integer(PyObject* object) {
  const long long value = PyLong_AsLongLong(object);
  if (value == -1 && PyErr_Occurred() != nullptr) throw Raised{};
  return value;
}

int32_t Small(PyObject* object, const char* what) {
  const long long value = Integer(object);
  if (value < INT32_MIN || value > INT32_MAX) throw Refusal(std::string(what) + " is out of range");
  return static_cast<int32_t>(value);
}

float Real(PyObject* object) {
  const double value = PyFloat_AsDouble(object);
  if (value == -1.0 && PyErr_Occurred() != nullptr) throw Raised{};
  return static_cast<float>(value);
}

int32_t Flag(PyObject* object) {
  const int value = PyObject_IsTrue(object);
  if (value < 0) throw Raised{};
  return value;
}

int32_t Score(PyObject* object) {
  if (PyUnicode_Check(object)) {
    if (PyUnicode_CompareWithASCIIString(object, "softmax") == 0) return 0;
    if (PyUnicode_CompareWithASCIIString(object, "sigmoid") == 0) return 1;
  }
  throw Refusal("score must be 'softmax' or 'sigmoid'");
}

// The device of an operator's storage, from its first tensor.
class Place {
 public:
  explicit Place(const Tensor& first) {
    if (!first.is_cuda()) throw Refusal("routed storage must be a CUDA tensor (there is no CPU fallback)");
    index_ = first.get_device();
  }
  void Holds(const Tensor& tensor) const {
    if (!tensor.is_cuda()) throw Refusal("routed storage must be a CUDA tensor (there is no CPU fallback)");
    if (tensor.get_device() != index_) throw Refusal("routed operands must be on one device");
    // Recorded calls would leave this operator out of the gradient without a word.
    if (tensor.requires_grad() && c10::GradMode::is_enabled()) {
      throw Refusal("an operand requires a gradient, which routed operators do not record: call them and their backward "
                    "operators in a torch.autograd.Function, or under torch.no_grad()");
    }
  }
  // Bytes of workspace that a route needs on the device.
  size_t RouteWorkspace(int64_t tokens, int32_t experts) const {
    const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(index_));
    return t0b_route_workspace(tokens, experts);
  }
  // Runs `entry(stream, error, error size)` on the device's current stream.
  template <typename Entry>
  void Run(Entry&& entry) const {
    char error[512];
    error[0] = 0;
    int status = 0;
    {
      const c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(index_));
      void* stream = c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(index_)).stream();
      Py_BEGIN_ALLOW_THREADS
      status = entry(stream, error, sizeof(error));
      Py_END_ALLOW_THREADS
    }
    if (status == 1) throw Refusal(error);
    if (status != 0) throw Failure(error);
  }

 private:
  int64_t index_;
};

int32_t HalfCode(const Tensor& tensor, const char* what) {
  if (tensor.scalar_type() == at::kBFloat16) return T0B_BF16;
  if (tensor.scalar_type() == at::kHalf) return T0B_F16;
  throw Refusal(std::string(what) + " must be float16 or bfloat16, got " + Name(tensor.scalar_type()));
}

int32_t FloatCode(at::ScalarType type, const char* what) {
  switch (type) {
    case at::kFloat: return T0B_F32;
    case at::kHalf: return T0B_F16;
    case at::kBFloat16: return T0B_BF16;
    default: throw Refusal(std::string(what) + " must be float32, float16 or bfloat16, got " + Name(type));
  }
}

// Address of a contiguous tensor of that type and shape.
template <typename T = void>
T* Packed(const Place& place, const Tensor& tensor, at::IntArrayRef shape, at::ScalarType type, const char* what) {
  place.Holds(tensor);
  if (tensor.scalar_type() != type || tensor.sizes() != shape || !tensor.is_contiguous()) {
    throw Refusal(std::string(what) + " must be a contiguous " + Name(type) + " tensor of shape " + Text(shape) +
                  ", got " + Name(tensor.scalar_type()) + " " + Text(tensor.sizes()) + " with strides " +
                  Text(tensor.strides()));
  }
  return static_cast<T*>(tensor.data_ptr());
}

struct Rows {
  const void* data;
  int64_t stride;
};

// A matrix of that shape whose rows are contiguous.
Rows Matrix(const Place& place, const Tensor& tensor, int64_t rows, int64_t width, const char* what,
            const char* kind = nullptr) {
  place.Holds(tensor);
  if (tensor.dim() != 2 || tensor.size(0) != rows || tensor.size(1) != width) {
    throw Refusal(std::string(what) + " must be [" + std::to_string(rows) + ", " + std::to_string(width) + "]" +
                  (kind != nullptr ? std::string(" (") + kind + " rows)" : "") + ", got " + Text(tensor.sizes()));
  }
  if (width > 1 && tensor.stride(1) != 1) throw Refusal(std::string(what) + " must have contiguous rows");
  const int64_t stride = tensor.stride(0);
  return {tensor.data_ptr(), rows > 1 || stride > width ? stride : width};
}

// An operator's result: new, or `out` if that fits.
Tensor Output(const Place& place, const Tensor& like, PyObject* out, at::IntArrayRef shape, at::ScalarType type) {
  if (out == Py_None) return at::empty(shape, like.options().dtype(type));
  const Tensor& given = Get(out, "out");
  Packed(place, given, shape, type, "out");
  return given;
}

// A routing (a tuple of experts, weights, rows, positions, offsets) whose arrays agree.
struct Routing {
  const Tensor *chosen, *weights_tensor, *rows_tensor, *positions_tensor, *offsets_tensor;
  int64_t tokens, entries;
  int32_t top_k, experts;
  const int32_t *rows, *offsets;

  Routing(const Place& place, PyObject* object) {
    if (!PyTuple_Check(object) || PyTuple_GET_SIZE(object) != 5) throw Refusal("a routing has five tensors");
    chosen = &Get(PyTuple_GET_ITEM(object, 0), "routing experts");
    weights_tensor = &Get(PyTuple_GET_ITEM(object, 1), "routing weights");
    rows_tensor = &Get(PyTuple_GET_ITEM(object, 2), "routing rows");
    positions_tensor = &Get(PyTuple_GET_ITEM(object, 3), "routing positions");
    offsets_tensor = &Get(PyTuple_GET_ITEM(object, 4), "routing offsets");
    if (chosen->dim() != 2) throw Refusal("routing experts must be [tokens, top_k]");
    tokens = chosen->size(0);
    if (chosen->size(1) > INT32_MAX) throw Refusal("routing experts must be [tokens, top_k]");
    top_k = static_cast<int32_t>(chosen->size(1));
    entries = tokens * top_k;
    if (offsets_tensor->numel() < 2 || offsets_tensor->numel() > INT32_MAX) {
      throw Refusal("routing offsets must be [experts + 1]");
    }
    experts = static_cast<int32_t>(offsets_tensor->numel() - 1);
    rows = Packed<int32_t>(place, *rows_tensor, {entries}, at::kInt, "routing rows");
    offsets = Packed<int32_t>(place, *offsets_tensor, {experts + 1}, at::kInt, "routing offsets");
  }
  const int32_t* Chosen(const Place& place) const {
    return Packed<int32_t>(place, *chosen, {tokens, top_k}, at::kInt, "routing experts");
  }
  const float* Weights(const Place& place) const {
    return Packed<float>(place, *weights_tensor, {tokens, top_k}, at::kFloat, "routing weights");
  }
  const int32_t* Positions(const Place& place) const {
    return Packed<int32_t>(place, *positions_tensor, {tokens, top_k}, at::kInt, "routing positions");
  }
};

int32_t Width(int64_t width, const char* what) {
  if (width > INT32_MAX) throw Refusal(std::string(what) + " is out of range");
  return static_cast<int32_t>(width);
}

// Error boundary of a binding function: no C++ exception leaves it.
template <typename Body>
PyObject* Guarded(Py_ssize_t given, Py_ssize_t expected, Body&& body) {
  try {
    if (given != expected) throw Refusal("wrong number of arguments");
    return body();
  } catch (const Raised&) {
  } catch (const Refusal& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const Failure& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");   // its allocator's own exception type
    PyObject* type = torch != nullptr ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    if (type != nullptr) PyErr_SetString(type, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::bad_alloc&) {
    PyErr_NoMemory();
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "tensor0-b200: unknown exception");
  }
  return nullptr;
}

using Arguments = PyObject* const*;

// (logits, top_k, groups, top_groups or None, group_best, score, renormalize, scale, bias, mask, out) -> out
PyObject* Route(PyObject*, Arguments args, Py_ssize_t count) {
  return Guarded(count, 11, [&]() -> PyObject* {
    const Tensor& logits = Get(args[0], "logits");
    const Place place(logits);
    if (logits.dim() != 2) throw Refusal("logits must be [tokens, experts]");
    const int64_t tokens = logits.size(0);
    const int32_t experts = Width(logits.size(1), "expert count"), top_k = Small(args[1], "top_k");
    const int32_t code = FloatCode(logits.scalar_type(), "logits");
    const int32_t score = Score(args[5]);
    const Rows rows = Matrix(place, logits, tokens, experts, "logits");
    const int32_t groups = Small(args[2], "groups");
    const int32_t top_groups = args[3] == Py_None ? groups : Small(args[3], "top_groups");
    const int32_t best = Small(args[4], "group_best"), renormalize = Flag(args[6]);
    const float scale = Real(args[7]);
    const float* bias = nullptr;
    if (args[8] != Py_None) {
      const Tensor& given = Get(args[8], "bias");   // has no gradient: it enters the choice only
      bias = Packed<float>(place, given.requires_grad() ? given.detach() : given, {experts}, at::kFloat, "bias");
    }
    const uint8_t* mask = nullptr;
    if (args[9] != Py_None) mask = Packed<uint8_t>(place, Get(args[9], "mask"), {tokens}, at::kBool, "mask");
    const Routing out(place, args[10]);
    const int32_t* chosen = Packed<int32_t>(place, *out.chosen, {tokens, top_k}, at::kInt, "routing experts");
    const int32_t* offsets = Packed<int32_t>(place, *out.offsets_tensor, {experts + 1}, at::kInt, "routing offsets");
    const size_t size = place.RouteWorkspace(tokens, experts);
    Tensor workspace;
    if (size != 0) workspace = at::empty({static_cast<int64_t>(size)}, logits.options().dtype(at::kByte));
    void* work = size != 0 ? workspace.data_ptr() : nullptr;
    const float* weights = out.Weights(place);
    const int32_t* positions = out.Positions(place);
    place.Run([&](void* stream, char* error, size_t error_size) {
      return t0b_route(code, tokens, experts, top_k, groups, top_groups, best, score, renormalize, scale, rows.data,
                       rows.stride, bias, mask, const_cast<int32_t*>(chosen), const_cast<float*>(weights),
                       const_cast<int32_t*>(out.rows), const_cast<int32_t*>(positions),
                       const_cast<int32_t*>(offsets), work, size, stream, error, error_size);
    });
    Py_INCREF(args[10]);
    return args[10];
  });
}

// (logits, routing, weights_grad, score, renormalize, scale, out) -> logits_grad
PyObject* RouteBackward(PyObject*, Arguments args, Py_ssize_t count) {
  return Guarded(count, 7, [&]() -> PyObject* {
    const Tensor& logits = Get(args[0], "logits");
    const Place place(logits);
    if (logits.dim() != 2) throw Refusal("logits must be [tokens, experts]");
    const int64_t tokens = logits.size(0);
    const int32_t experts = Width(logits.size(1), "expert count");
    const int32_t code = FloatCode(logits.scalar_type(), "logits"), score = Score(args[3]);
    const Rows rows = Matrix(place, logits, tokens, experts, "logits");
    const Routing r(place, args[1]);
    if (r.experts != experts) {
      throw Refusal("the routing has " + std::to_string(r.experts) + " experts, the logits " + std::to_string(experts));
    }
    const int32_t* chosen = Packed<int32_t>(place, *r.chosen, {tokens, r.top_k}, at::kInt, "routing experts");
    const float* grad = Packed<float>(place, Get(args[2], "weights_grad"), {tokens, r.top_k}, at::kFloat, "weights_grad");
    const int32_t renormalize = Flag(args[4]);
    const float scale = Real(args[5]);
    const Tensor out = Output(place, logits, args[6], {tokens, experts}, logits.scalar_type());
    void* result = out.data_ptr();
    place.Run([&](void* stream, char* error, size_t error_size) {
      return t0b_route_backward(code, tokens, experts, r.top_k, score, renormalize, scale, rows.data, rows.stride,
                                chosen, grad, result, stream, error, error_size);
    });
    return THPVariable_Wrap(out);
  });
}

const char* Kind(bool gather) { return gather ? "token" : "expert-ordered"; }

// (x, w, routing, gather, transpose, out) -> rows
PyObject* RoutedMatmul(PyObject*, Arguments args, Py_ssize_t count) {
  return Guarded(count, 6, [&]() -> PyObject* {
    const Tensor &x = Get(args[0], "x"), &w = Get(args[1], "weights");
    const Place place(x);
    const Routing r(place, args[2]);
    const int32_t code = HalfCode(x, "product operands");
    if (w.dim() != 3 || w.size(0) != r.experts) {
      throw Refusal("weights must be [" + std::to_string(r.experts) + ", inner, outer]");
    }
    const int32_t inner = Width(w.size(1), "inner"), outer = Width(w.size(2), "outer");
    const int32_t gather = Flag(args[3]), transpose = Flag(args[4]);
    const void* weights = Packed(place, w, w.sizes(), x.scalar_type(), "weights");
    const int64_t x_rows = gather != 0 ? r.tokens : r.entries;
    const Rows rows = Matrix(place, x, x_rows, transpose != 0 ? outer : inner, "x", Kind(gather != 0));
    const Tensor out = Output(place, x, args[5], {r.entries, transpose != 0 ? inner : outer}, x.scalar_type());
    void* result = out.data_ptr();
    place.Run([&](void* stream, char* error, size_t error_size) {
      return t0b_routed_product(code, transpose, r.entries, r.experts, r.top_k, inner, outer, gather, rows.data, x_rows,
                                rows.stride, weights, r.rows, r.offsets, result, stream, error, error_size);
    });
    return THPVariable_Wrap(out);
  });
}

// (x, y_grad, routing, gather_x, gather_y, out) -> weights' gradient
PyObject* RoutedWeightGrad(PyObject*, Arguments args, Py_ssize_t count) {
  return Guarded(count, 6, [&]() -> PyObject* {
    const Tensor &x = Get(args[0], "x"), &y = Get(args[1], "y_grad");
    const Place place(x);
    const Routing r(place, args[2]);
    const int32_t code = HalfCode(x, "product operands");
    if (y.scalar_type() != x.scalar_type()) throw Refusal("product operands must share a dtype");
    if (x.dim() != 2 || y.dim() != 2) throw Refusal("product operands must be 2-d");
    const int32_t inner = Width(x.size(1), "inner"), outer = Width(y.size(1), "outer");
    const int32_t gather_x = Flag(args[3]), gather_y = Flag(args[4]);
    const int64_t x_rows = gather_x != 0 ? r.tokens : r.entries, y_rows = gather_y != 0 ? r.tokens : r.entries;
    const Rows left = Matrix(place, x, x_rows, inner, "x", Kind(gather_x != 0));
    const Rows right = Matrix(place, y, y_rows, outer, "y_grad", Kind(gather_y != 0));
    const Tensor out = Output(place, x, args[5], {r.experts, inner, outer}, x.scalar_type());
    void* result = out.data_ptr();
    place.Run([&](void* stream, char* error, size_t error_size) {
      return t0b_routed_weight_grad(code, r.entries, r.experts, r.top_k, inner, outer, gather_x, left.data, x_rows,
                                    left.stride, gather_y, right.data, y_rows, right.stride, r.rows, r.offsets, result,
                                    stream, error, error_size);
    });
    return THPVariable_Wrap(out);
  });
}

// (y, routing, out) -> sums
PyObject* RoutedSum(PyObject*, Arguments args, Py_ssize_t count) {
  return Guarded(count, 3, [&]() -> PyObject* {
    const Tensor& y = Get(args[0], "y");
    const Place place(y);
    const Routing r(place, args[1]);
    const int32_t code = HalfCode(y, "sum operands");
    const int32_t* positions = r.Positions(place);
    if (y.dim() != 2) throw Refusal("y must be 2-d");
    const int32_t width = Width(y.size(1), "width");
    const Rows rows = Matrix(place, y, r.entries, width, "y", Kind(false));
    const Tensor out = Output(place, y, args[2], {r.tokens, width}, y.scalar_type());
    void* result = out.data_ptr();
    place.Run([&](void* stream, char* error, size_t error_size) {
      return t0b_routed_sum(code, r.tokens, r.top_k, width, rows.data, rows.stride, positions, result, stream, error,
                            error_size);
    });
    return THPVariable_Wrap(out);
  });
}

// The routing of gated rows: all null without one.
struct RowWeights {
  const float* weights = nullptr;
  const int32_t *rows = nullptr, *offsets = nullptr;
  int32_t experts = 0;
  int64_t tokens = 0, top_k = 0;

  RowWeights(const Place& place, PyObject* object, int64_t row_count) {
    if (object == Py_None) return;
    const Routing r(place, object);
    if (r.entries != row_count) {
      throw Refusal("the routing has " + std::to_string(r.entries) + " entries, the activation " +
                    std::to_string(row_count) + " rows");
    }
    weights = r.Weights(place);
    rows = r.rows;
    offsets = r.offsets;
    experts = r.experts;
    tokens = r.tokens;
    top_k = r.top_k;
  }
};

int32_t Group(PyObject* object, const char* what) {
  const int32_t group = Small(object, what);
  if (group != 32 && group != 64 && group != 128) throw Refusal(std::string(what) + " must be 32, 64 or 128");
  return group;
}

int32_t HalfWidth(const Tensor& tensor, const char* what) {
  if (tensor.dim() != 2 || tensor.size(1) == 0 || tensor.size(1) % 2 != 0) {
    throw Refusal(std::string(what) + " must be [rows, 2 * width]");
  }
  return Width(tensor.size(1) / 2, "width");
}

// (h, routing or None, group or None, a, codes, scales; the results may be None) -> (a, codes, scales), or a
// alone without a group
PyObject* GatedSave(PyObject*, Arguments args, Py_ssize_t count) {
  return Guarded(count, 6, [&]() -> PyObject* {
    const Tensor& h = Get(args[0], "h");
    const Place place(h);
    const int32_t width = HalfWidth(h, "h"), code = HalfCode(h, "gated activations");
    const int64_t rows = h.size(0);
    const bool keep = args[2] != Py_None;
    const int32_t group = keep ? Group(args[2], "checkpoint group") : 128;
    const Rows input = Matrix(place, h, rows, 2 * int64_t{width}, "h");
    const RowWeights r(place, args[1], rows);
    const Tensor a = Output(place, h, args[3], {rows, width}, h.scalar_type());
    Tensor codes, scales;
    int8_t* code_data = nullptr;
    float* scale_data = nullptr;
    if (keep) {
      codes = Output(place, h, args[4], {rows, 2 * int64_t{width}}, at::kChar);
      scales = Output(place, h, args[5], {rows, 2 * ((int64_t{width} + group - 1) / group)}, at::kFloat);
      code_data = static_cast<int8_t*>(codes.data_ptr());
      scale_data = static_cast<float*>(scales.data_ptr());
    }
    void* result = a.data_ptr();
    place.Run([&](void* stream, char* error, size_t error_size) {
      return t0b_gated_save(code, rows, width, group, input.data, input.stride, r.weights, r.rows, r.offsets, r.experts,
                            result, code_data, scale_data, stream, error, error_size);
    });
    if (!keep) return THPVariable_Wrap(a);
    return Py_BuildValue("NNN", THPVariable_Wrap(a), THPVariable_Wrap(codes), THPVariable_Wrap(scales));
  });
}

struct Kept {
  int32_t width, group;
  int64_t rows;
  const int8_t* codes;
  const float* scales;

  // A checkpoint is a tuple of codes, scales and group.
  Kept(const Place& place, PyObject* object) {
    const Tensor& code_tensor = Get(PyTuple_GET_ITEM(object, 0), "checkpoint codes");
    group = Group(PyTuple_GET_ITEM(object, 2), "checkpoint group");
    width = HalfWidth(code_tensor, "checkpoint codes");
    rows = code_tensor.size(0);
    codes = Packed<int8_t>(place, code_tensor, code_tensor.sizes(), at::kChar, "checkpoint codes");
    scales = Packed<float>(place, Get(PyTuple_GET_ITEM(object, 1), "checkpoint scales"),
                           {rows, 2 * ((int64_t{width} + group - 1) / group)}, at::kFloat, "checkpoint scales");
  }
  static void Check(PyObject* object) {
    if (!PyTuple_Check(object) || PyTuple_GET_SIZE(object) != 3) {
      throw Refusal("a checkpoint is its codes, its scales and its group");
    }
  }
};

// (checkpoint, a_grad, routing or None) -> (h_grad, a, weights_grad)
PyObject* GatedBackward(PyObject*, Arguments args, Py_ssize_t count) {
  return Guarded(count, 3, [&]() -> PyObject* {
    Kept::Check(args[0]);
    const Tensor& grad = Get(args[1], "a_grad");
    const Place place(grad);
    const Kept kept(place, args[0]);
    const int32_t code = HalfCode(grad, "gated activations");
    const Rows input = Matrix(place, grad, kept.rows, kept.width, "a_grad");
    const RowWeights r(place, args[2], kept.rows);
    const Tensor h_grad = at::empty({kept.rows, 2 * int64_t{kept.width}}, grad.options());
    const Tensor a = at::empty({kept.rows, kept.width}, grad.options());
    const auto real = grad.options().dtype(at::kFloat);
    const Tensor weights_grad = args[2] == Py_None ? at::empty({kept.rows}, real) : at::empty({r.tokens, r.top_k}, real);
    void *h_data = h_grad.data_ptr(), *a_data = a.data_ptr();
    float* w_data = static_cast<float*>(weights_grad.data_ptr());
    place.Run([&](void* stream, char* error, size_t error_size) {
      return t0b_gated_backward(code, kept.rows, kept.width, kept.group, kept.codes, kept.scales, input.data,
                                input.stride, r.weights, r.rows, r.offsets, r.experts, h_data, a_data, w_data, stream,
                                error, error_size);
    });
    return Py_BuildValue("NNN", THPVariable_Wrap(h_grad), THPVariable_Wrap(a), THPVariable_Wrap(weights_grad));
  });
}

// (checkpoint, T0B_* code of the wanted type) -> values
PyObject* CheckpointLoad(PyObject*, Arguments args, Py_ssize_t count) {
  return Guarded(count, 2, [&]() -> PyObject* {
    Kept::Check(args[0]);
    const Tensor& codes = Get(PyTuple_GET_ITEM(args[0], 0), "checkpoint codes");
    const Place place(codes);
    const Kept kept(place, args[0]);
    const int32_t code = Small(args[1], "dtype");
    const at::ScalarType type = code == T0B_F32 ? at::kFloat : code == T0B_F16 ? at::kHalf : at::kBFloat16;
    const Tensor values = at::empty({kept.rows, 2 * int64_t{kept.width}}, codes.options().dtype(type));
    void* result = values.data_ptr();
    place.Run([&](void* stream, char* error, size_t error_size) {
      return t0b_checkpoint_load(code, kept.rows, kept.width, kept.group, kept.codes, kept.scales, result, stream, error,
                                 error_size);
    });
    return THPVariable_Wrap(values);
  });
}

// (x, codes, scales, group, routing, gather, out) -> rows
PyObject* RoutedMatvec(PyObject*, Arguments args, Py_ssize_t count) {
  return Guarded(count, 7, [&]() -> PyObject* {
    const Tensor &x = Get(args[0], "x"), &codes = Get(args[1], "4-bit weight codes");
    const Tensor& scales = Get(args[2], "4-bit weight scales");
    const Place place(x);
    const Routing r(place, args[4]);
    const int32_t code = HalfCode(x, "4-bit product operands"), group = Group(args[3], "weight group");
    if (x.dim() != 2 || x.size(1) % group != 0) {
      throw Refusal("weight group must divide the inner width");
    }
    if (codes.dim() != 3) throw Refusal("4-bit weight codes must be [experts, outer, inner / 2]");
    const int32_t inner = Width(x.size(1), "inner"), outer = Width(codes.size(1), "outer"), gather = Flag(args[5]);
    const uint8_t* code_data =
        Packed<uint8_t>(place, codes, {r.experts, outer, inner / 2}, at::kByte, "4-bit weight codes");
    const void* scale_data =
        Packed(place, scales, {r.experts, outer, inner / group}, x.scalar_type(), "4-bit weight scales");
    const int64_t x_rows = gather != 0 ? r.tokens : r.entries;
    const Rows rows = Matrix(place, x, x_rows, inner, "x", Kind(gather != 0));
    const Tensor out = Output(place, x, args[6], {r.entries, outer}, x.scalar_type());
    void* result = out.data_ptr();
    place.Run([&](void* stream, char* error, size_t error_size) {
      return t0b_routed_matvec4(code, r.entries, r.experts, r.top_k, inner, outer, group, gather, rows.data, x_rows,
                                rows.stride, code_data, scale_data, r.rows, r.offsets, result, stream, error, error_size);
    });
    return THPVariable_Wrap(out);
  });
}

#define T0B_METHOD(name, function) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(function)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {
    T0B_METHOD("route", Route),
    T0B_METHOD("route_backward", RouteBackward),
    T0B_METHOD("routed_matmul", RoutedMatmul),
    T0B_METHOD("routed_weight_grad", RoutedWeightGrad),
    T0B_METHOD("routed_sum", RoutedSum),
    T0B_METHOD("gated_save", GatedSave),
    T0B_METHOD("gated_backward", GatedBackward),
    T0B_METHOD("checkpoint_load", CheckpointLoad),
    T0B_METHOD("routed_matvec", RoutedMatvec),
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_routed", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__routed(void) { return PyModule_Create(&kModule); }

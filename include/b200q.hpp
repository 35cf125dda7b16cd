// C++ host shim over the C ABI of b200q.h with the shape of the reference's operator functions
// (mlx/ops.cpp: quantize :5208-5245, dequantize :5465-5517, quantized_matmul :4784-4834,
// gather_qmm :5553-5629; qqmm, the grouped products, routing and adapters in the same manner): same argument meaning, same validation (mlx/ops.cpp:110-181,
// 4704-4754), std::invalid_argument where the reference throws it and std::runtime_error for
// everything the library reports later.  Arrays are non-owning views of row-contiguous device
// memory; outputs and scratch are allocated by the caller (the reference's eval_gpu does that
// with its own allocator).  Header only; link with libb200q.so.
#pragma once

#include <cstdint>
#include <sstream>
#include <stdexcept>
#include <string>
#include <vector>

#include "b200q.h"

namespace b200q {

enum class Dtype : int { float32 = B200Q_F32, float16 = B200Q_F16, bfloat16 = B200Q_BF16, uint32 = 100, uint8 = 101, int32 = 102, int64 = 103 };

inline const char* name(Dtype t) {
  switch (t) {
    case Dtype::float32: return "float32";
    case Dtype::float16: return "float16";
    case Dtype::bfloat16: return "bfloat16";
    case Dtype::uint8: return "uint8";
    case Dtype::int32: return "int32";
    case Dtype::int64: return "int64";
    default: return "uint32";
  }
}
inline bool is_floating(Dtype t) { return (int)t < (int)Dtype::uint32; }

// Row-contiguous device array: shape + dtype + pointer.
struct ArrayView {
  void* data = nullptr;
  Dtype dtype = Dtype::float32;
  std::vector<int64_t> shape;
  int ndim() const { return (int)shape.size(); }
  int64_t dim(int i) const { return shape[i < 0 ? shape.size() + i : i]; }
  int64_t size() const {
    int64_t n = 1;
    for (auto d : shape) n *= d;
    return n;
  }
};

struct Workspace {  // scratch sized with b200q_*_workspace_bytes, zeroed once with b200q_workspace_init
  void* data = nullptr;
  size_t bytes = 0;
};

namespace detail {
inline std::string shape_str(const std::vector<int64_t>& s) {
  std::ostringstream o;
  o << "(";
  for (size_t i = 0; i < s.size(); ++i) o << (i ? "," : "") << s[i];
  o << ")";
  return o.str();
}
inline void check(int rc) {
  if (rc == B200Q_OK) return;
  if (rc == B200Q_ERR_INVALID_ARGUMENT) throw std::invalid_argument(b200q_last_error());
  throw std::runtime_error(b200q_last_error());
}
// mlx/ops.cpp:110-150
inline void validate_quantized_input(const char* tag, const ArrayView& w, const ArrayView& scales, const ArrayView& biases,
                                     int group_size, int bits) {
  if (w.dtype != Dtype::uint32) {
    std::ostringstream m;
    m << "[" << tag << "] The weight matrix should be uint32 but received " << name(w.dtype);
    throw std::invalid_argument(m.str());
  }
  if (scales.shape != biases.shape) {
    std::ostringstream m;
    m << "[" << tag << "] Scales and biases should have the same shape. Received scales with shape "
      << shape_str(scales.shape) << " and biases with " << shape_str(biases.shape);
    throw std::invalid_argument(m.str());
  }
  bool batch_ok = w.ndim() >= 2 && scales.ndim() == w.ndim();
  for (int i = 0; batch_ok && i < w.ndim() - 2; ++i) batch_ok = w.shape[i] == scales.shape[i];
  if (!batch_ok) {
    std::ostringstream m;
    m << "[" << tag << "] Weight and scales should have the same batch shape. Received weight with shape "
      << shape_str(w.shape) << ", scales with " << shape_str(scales.shape) << ".";
    throw std::invalid_argument(m.str());
  }
  if (w.dim(-1) * 32 / bits != scales.dim(-1) * group_size) {
    std::ostringstream m;
    m << "[" << tag << "] The shapes of the weight and scales are incompatible based on bits and group_size. "
      << "w.shape() == " << shape_str(w.shape) << " and scales.shape() == " << shape_str(scales.shape)
      << " with group_size=" << group_size << " and bits=" << bits;
    throw std::invalid_argument(m.str());
  }
}
// mlx/ops.cpp:152-181: returns {w_inner, w_outer}
inline std::pair<int64_t, int64_t> extract_dims(const char* tag, const ArrayView& x, const ArrayView& w, const ArrayView& scales,
                                                const ArrayView& biases, bool transpose, int group_size, int bits) {
  validate_quantized_input(tag, w, scales, biases, group_size, bits);
  if (x.ndim() < 1) throw std::invalid_argument(std::string("[") + tag + "] x must have at least one dimension");
  const int64_t x_inner = x.dim(-1);
  const int64_t w_inner = transpose ? w.dim(-1) * 32 / bits : w.dim(-2);
  const int64_t w_outer = transpose ? w.dim(-2) : w.dim(-1) * 32 / bits;
  if (w_inner != x_inner) {
    std::ostringstream m;
    m << "[" << tag << "] Last dimension of first input with shape (..., " << x_inner
      << ") does not match the expanded quantized matrix (" << w_inner << ", " << w_outer << ") computed from shape "
      << shape_str(w.shape) << " with group_size=" << group_size << ", bits=" << bits << " and transpose=" << transpose;
    throw std::invalid_argument(m.str());
  }
  return {w_inner, w_outer};
}
inline void validate_types(const char* tag, const ArrayView& x, const ArrayView& scales, const ArrayView& biases) {
  // mlx/ops.cpp:4704-4754: only real floating types; this shim does not promote: one dtype for all
  if (!is_floating(scales.dtype) || !is_floating(biases.dtype) || !is_floating(x.dtype)) {
    std::ostringstream m;
    m << "[" << tag << "] Only real floating types are supported but scales.dtype() == " << name(scales.dtype)
      << " and biases.dtype() == " << name(biases.dtype) << ".";
    throw std::invalid_argument(m.str());
  }
  if (x.dtype != scales.dtype || x.dtype != biases.dtype) {
    std::ostringstream m;
    m << "[" << tag << "] x, scales and biases must already have the result type (the reference casts them before the "
      << "primitive, mlx/ops.cpp:4816-4818); got " << name(x.dtype) << ", " << name(scales.dtype) << ", " << name(biases.dtype);
    throw std::invalid_argument(m.str());
  }
}
}  // namespace detail

// w [.., K] -> wq uint32 [.., K*bits/32], scales / biases [.., K/group_size]  (mlx/ops.cpp:5208-5245)
inline void quantize(const ArrayView& w, ArrayView& wq, ArrayView& scales, ArrayView& biases, int group_size = 64,
                     int bits = 4, void* stream = nullptr) {
  if (!is_floating(w.dtype))
    throw std::invalid_argument(std::string("[quantize] Only real floating types can be quantized but w has type ") + name(w.dtype) + ".");
  if (w.ndim() < 2) {
    std::ostringstream m;
    m << "[quantize] The matrix to be quantized must have at least 2 dimension but it has only " << w.ndim() << ".";
    throw std::invalid_argument(m.str());
  }
  const int64_t K = w.dim(-1), rows = K ? w.size() / K : 0;
  detail::check(b200q_quantize(w.data, (int)w.dtype, rows, K, group_size, bits, static_cast<uint32_t*>(wq.data), scales.data,
                               biases.data, stream));
}

// wq, scales, biases -> w [.., K]  (mlx/ops.cpp:5465-5517)
inline void dequantize(const ArrayView& wq, const ArrayView& scales, const ArrayView& biases, ArrayView& out, int group_size = 64,
                       int bits = 4, void* stream = nullptr) {
  detail::validate_quantized_input("dequantize", wq, scales, biases, group_size, bits);
  const int64_t K = wq.dim(-1) * 32 / bits, rows = wq.dim(-1) ? wq.size() / wq.dim(-1) : 0;
  detail::check(b200q_dequantize(static_cast<const uint32_t*>(wq.data), scales.data, biases.data, (int)scales.dtype, rows, K,
                                 group_size, bits, out.data, stream));
}

// out[i, :] = dequantize(row ids[i]) : QuantizedEmbedding.__call__ (python/mlx/nn/layers/quantized.py:149-158)
inline void quantized_embedding(const ArrayView& ids, const ArrayView& wq, const ArrayView& scales, const ArrayView& biases,
                                ArrayView& out, int group_size = 64, int bits = 4, void* stream = nullptr) {
  detail::validate_quantized_input("quantized_embedding", wq, scales, biases, group_size, bits);
  if (ids.dtype != Dtype::uint32) throw std::invalid_argument("[quantized_embedding] ids must be uint32.");
  if (wq.ndim() != 2) throw std::invalid_argument("[quantized_embedding] the table must be a 2-D packed matrix");
  const int64_t K = wq.dim(-1) * 32 / bits;
  detail::check(b200q_dequantize_rows(static_cast<const uint32_t*>(wq.data), scales.data, biases.data,
                                      static_cast<const uint32_t*>(ids.data), ids.size(), (int)scales.dtype, wq.dim(0), K,
                                      group_size, bits, out.data, stream));
}

// x [.., M, K] against one matrix w (2-D) or a stack of matrices with x's batch shape  (mlx/ops.cpp:4784-4834)
inline void quantized_matmul(const ArrayView& x, const ArrayView& w, const ArrayView& scales, const ArrayView& biases, ArrayView& out,
                             const Workspace& ws, bool transpose = true, int group_size = 64, int bits = 4,
                             void* stream = nullptr) {
  detail::validate_types("quantized_matmul", x, scales, biases);
  const auto dims = detail::extract_dims("quantized_matmul", x, w, scales, biases, transpose, group_size, bits);
  const int64_t K = dims.first, N = dims.second;
  const int64_t M = x.ndim() > 1 ? x.dim(-2) : 1;
  const int64_t batch = (M * K) ? x.size() / (M * K) : 0;
  const bool w_batched = w.ndim() > 2;
  detail::check(b200q_qmm(x.data, static_cast<const uint32_t*>(w.data), scales.data, biases.data, out.data, (int)x.dtype, batch, M,
                          N, K, group_size, bits, transpose ? 1 : 0, w_batched ? 1 : 0, ws.data, ws.bytes, stream));
}

// out[i] = x[lhs[i]] * dequant(w[rhs[i]]); indices uint32, already broadcast against each other  (mlx/ops.cpp:5553-5629)
inline void gather_qmm(const ArrayView& x, const ArrayView& w, const ArrayView& scales, const ArrayView& biases,
                       const ArrayView& lhs_indices, const ArrayView& rhs_indices, ArrayView& out, const Workspace& ws,
                       bool transpose = true, int group_size = 64, int bits = 4, bool sorted_indices = false,
                       void* stream = nullptr) {
  detail::validate_types("gather_qmm", x, scales, biases);
  const auto dims = detail::extract_dims("gather_qmm", x, w, scales, biases, transpose, group_size, bits);
  if (lhs_indices.dtype != Dtype::uint32 || rhs_indices.dtype != Dtype::uint32)
    throw std::invalid_argument("[gather_qmm] Got lhs_indices or rhs_indices with invalid dtype. Indices must be integral.");
  if (lhs_indices.shape != rhs_indices.shape)
    throw std::invalid_argument("[gather_qmm] lhs_indices and rhs_indices must be broadcast to one shape by the caller");
  if (x.ndim() < 2 || w.ndim() < 2)
    throw std::invalid_argument("[gather_qmm] x and w must have at least two dimensions");
  const int64_t K = dims.first, N = dims.second, M = x.dim(-2);
  const int64_t x_batch = (M * K) ? x.size() / (M * K) : 0;
  const int64_t E = w.size() / (w.dim(-1) * w.dim(-2));
  detail::check(b200q_gather_qmm(x.data, static_cast<const uint32_t*>(w.data), scales.data, biases.data,
                                 static_cast<const uint32_t*>(lhs_indices.data), static_cast<const uint32_t*>(rhs_indices.data),
                                 lhs_indices.size(), out.data, (int)x.dtype, x_batch, E, M, N, K, group_size, bits, transpose ? 1 : 0,
                                 sorted_indices ? 3 : 0, ws.data, ws.bytes, stream));
}

// ---- microscaled 4-bit floating point (b200q_fp4_quantize says how values are rounded)
enum class Fp4 : int { mxfp4 = B200Q_MXFP4, nvfp4 = B200Q_NVFP4 };
namespace detail {
inline int group(Fp4 mode) { return mode == Fp4::mxfp4 ? 32 : 16; }
// wq [.., K/8] uint32 and scales [.., K/group] uint8
inline void validate_fp4(const char* tag, const ArrayView& wq, const ArrayView& scales, Fp4 mode) {
  if (wq.dtype != Dtype::uint32 || scales.dtype != Dtype::uint8)
    throw std::invalid_argument(std::string("[") + tag + "] the weight matrix should be uint32 and its scales uint8 but are " + name(wq.dtype) +
                                " and " + name(scales.dtype));
  bool ok = wq.ndim() >= 2 && scales.ndim() == wq.ndim() && wq.dim(-1) * 8 == scales.dim(-1) * group(mode);
  for (int i = 0; ok && i < wq.ndim() - 1; ++i) ok = wq.shape[i] == scales.shape[i];
  if (!ok)
    throw std::invalid_argument(std::string("[") + tag + "] The shapes of the weight and scales are incompatible: " + shape_str(wq.shape) + " and " +
                                shape_str(scales.shape) + " with 4 bits in groups of " + std::to_string(group(mode)));
}
// A global scale (or an empty view: none): one float32, or one per matrix where `each` says how many there are.
inline const float* global_scale(const char* tag, const ArrayView& g, Fp4 mode, int64_t each) {
  if (!g.data) return nullptr;
  if (mode != Fp4::nvfp4 || g.dtype != Dtype::float32 || (g.size() != 1 && g.size() != each))
    throw std::invalid_argument(std::string("[") + tag + "] a global scale is one float32 (or one per matrix) and belongs to nvfp4");
  return static_cast<const float*>(g.data);
}
// A result that the library will write: as many elements of the right type as it writes.
inline void validate_result(const char* tag, const ArrayView& out, int64_t size, Dtype type) {
  if (out.dtype != type)
    throw std::invalid_argument(std::string("[") + tag + "] unsupported dtype of the result: " + name(out.dtype) + " instead of " + name(type));
  if (out.size() != size)
    throw std::invalid_argument(std::string("[") + tag + "] the result's shape " + shape_str(out.shape) + " does not have " + std::to_string(size) + " elements");
}
inline int64_t matrices(const ArrayView& a) {
  int64_t n = 1;
  for (int i = 0; i < a.ndim() - 2; ++i) n *= a.shape[i];
  return n;
}
inline int size_bytes(const char* tag, const ArrayView& sizes, int64_t groups) {
  if ((sizes.dtype != Dtype::int32 && sizes.dtype != Dtype::int64) || sizes.ndim() != 1 || sizes.dim(0) != groups)
    throw std::invalid_argument(std::string("[") + tag + "] one integral group size per expert is needed");
  return sizes.dtype == Dtype::int64 ? 8 : 4;
}
}  // namespace detail

// w [.., K] -> wq, scales
inline void quantize(const ArrayView& w, ArrayView& wq, ArrayView& scales, Fp4 mode, const ArrayView& global_scale = {}, void* stream = nullptr) {
  if (!is_floating(w.dtype))
    throw std::invalid_argument(std::string("[quantize] Only real floating types can be quantized but w has type ") + name(w.dtype) + ".");
  detail::validate_fp4("quantize", wq, scales, mode);
  bool ok = w.ndim() == wq.ndim() && w.dim(-1) == wq.dim(-1) * 8;
  for (int i = 0; ok && i < w.ndim() - 1; ++i) ok = w.shape[i] == wq.shape[i];
  if (!ok)
    throw std::invalid_argument("[quantize] w " + detail::shape_str(w.shape) + " does not match the packed matrix " + detail::shape_str(wq.shape));
  const int64_t K = w.dim(-1), rows = K ? w.size() / K : 0;
  const float* g = detail::global_scale("quantize", global_scale, mode, detail::matrices(w));
  detail::check(b200q_fp4_quantize(w.data, (int)w.dtype, rows, K, (int)mode, g, global_scale.size() == 1 || !g ? (rows ? rows : 1) : w.dim(-2),
                                   static_cast<uint32_t*>(wq.data), static_cast<uint8_t*>(scales.data), stream));
}

// wq, scales -> out [.., K] in out's type
inline void dequantize(const ArrayView& wq, const ArrayView& scales, ArrayView& out, Fp4 mode, const ArrayView& global_scale = {},
                       void* stream = nullptr) {
  detail::validate_fp4("dequantize", wq, scales, mode);
  const int64_t K = wq.dim(-1) * 8, rows = wq.dim(-1) ? wq.size() / wq.dim(-1) : 0;
  if (is_floating(out.dtype)) detail::validate_result("dequantize", out, rows * K, out.dtype);   // (any other type the library refuses)
  const float* g = detail::global_scale("dequantize", global_scale, mode, detail::matrices(wq));
  detail::check(b200q_fp4_dequantize(static_cast<const uint32_t*>(wq.data), static_cast<const uint8_t*>(scales.data), (int)mode, g,
                                     global_scale.size() == 1 || !g ? (rows ? rows : 1) : wq.dim(-2), (int)out.dtype, rows, K, out.data, stream));
}

// x [.., K] times the transpose of w [N, K/8], x quantized on the way
inline void qqmm(const ArrayView& x, const ArrayView& w, const ArrayView& scales, ArrayView& out, const Workspace& ws, Fp4 mode,
                 const ArrayView& global_scale_x = {}, const ArrayView& global_scale_w = {}, void* stream = nullptr) {
  detail::validate_fp4("qqmm", w, scales, mode);
  const int64_t K = w.dim(-1) * 8;
  if (w.ndim() != 2 || x.ndim() < 1 || x.dim(-1) != K || !is_floating(x.dtype))
    throw std::invalid_argument("[qqmm] x " + detail::shape_str(x.shape) + " does not match the matrix w " + detail::shape_str(w.shape));
  detail::validate_result("qqmm", out, (K ? x.size() / K : 0) * w.dim(0), x.dtype);
  detail::check(b200q_grouped_qqmm(x.data, static_cast<const uint32_t*>(w.data), static_cast<const uint8_t*>(scales.data), nullptr, 0, out.data,
                                   (int)x.dtype, K ? x.size() / K : 0, 1, w.dim(0), K, (int)mode,
                                   detail::global_scale("qqmm", global_scale_x, mode, 1), detail::global_scale("qqmm", global_scale_w, mode, 1), 0,
                                   ws.data, ws.bytes, stream));
}

// Rows of x [T, K] sorted by expert, w [E, N, K/8]; sizes [E] on the device
inline void grouped_qqmm(const ArrayView& x, const ArrayView& w, const ArrayView& scales, const ArrayView& sizes, ArrayView& out,
                         const Workspace& ws, Fp4 mode, const ArrayView& global_scale_x = {}, const ArrayView& global_scale_w = {},
                         void* stream = nullptr) {
  detail::validate_fp4("grouped_qqmm", w, scales, mode);
  if (w.ndim() != 3 || x.ndim() != 2 || x.dim(1) != w.dim(2) * 8 || !is_floating(x.dtype))
    throw std::invalid_argument("[grouped_qqmm] x " + detail::shape_str(x.shape) + " does not match the matrices w " + detail::shape_str(w.shape));
  const int bytes = detail::size_bytes("grouped_qqmm", sizes, w.dim(0));
  detail::validate_result("grouped_qqmm", out, x.dim(0) * w.dim(1), x.dtype);
  detail::check(b200q_grouped_qqmm(x.data, static_cast<const uint32_t*>(w.data), static_cast<const uint8_t*>(scales.data), sizes.data, bytes,
                                   out.data, (int)x.dtype, x.dim(0), w.dim(0), w.dim(1), x.dim(1), (int)mode,
                                   detail::global_scale("grouped_qqmm", global_scale_x, mode, 1),
                                   detail::global_scale("grouped_qqmm", global_scale_w, mode, w.dim(0)), global_scale_w.size() > 1, ws.data, ws.bytes,
                                   stream));
}

// Rows of x [T, K] sorted by expert, 16-bit w [E, N, K] (transpose) or [E, K, N]; sizes [E] on the device.  The gradient with respect
// to x is the same call on the cotangent with `transpose` inverted.
inline void grouped_mm(const ArrayView& x, const ArrayView& w, const ArrayView& sizes, ArrayView& out, const Workspace& ws, bool transpose = true,
                       void* stream = nullptr) {
  if (w.ndim() != 3 || x.ndim() != 2 || x.dim(1) != w.dim(transpose ? 2 : 1) || x.dtype != w.dtype)
    throw std::invalid_argument("[grouped_mm] x " + detail::shape_str(x.shape) + " does not match the matrices w " + detail::shape_str(w.shape));
  const int bytes = detail::size_bytes("grouped_mm", sizes, w.dim(0));
  detail::validate_result("grouped_mm", out, x.dim(0) * w.dim(transpose ? 1 : 2), x.dtype);
  detail::check(b200q_grouped_mm(x.data, w.data, sizes.data, bytes, out.data, (int)x.dtype, x.dim(0), w.dim(0), w.dim(transpose ? 1 : 2), x.dim(1),
                                 transpose ? 1 : 0, ws.data, ws.bytes, stream));
}

// The gradient of grouped_mm with respect to w, in w's layout
inline void grouped_mm_dw(const ArrayView& dy, const ArrayView& x, const ArrayView& sizes, ArrayView& dw, const Workspace& ws, bool transpose = true,
                          void* stream = nullptr) {
  if (dy.ndim() != 2 || x.ndim() != 2 || dy.dim(0) != x.dim(0) || dy.dtype != x.dtype || sizes.ndim() != 1)
    throw std::invalid_argument("[grouped_mm_dw] dy and x must be matrices of one type with as many rows");
  const int bytes = detail::size_bytes("grouped_mm_dw", sizes, sizes.dim(0));
  detail::validate_result("grouped_mm_dw", dw, sizes.dim(0) * dy.dim(1) * x.dim(1), x.dtype);
  const ArrayView &a = transpose ? dy : x, &b = transpose ? x : dy;
  detail::check(b200q_grouped_mm_dw(a.data, b.data, sizes.data, bytes, dw.data, (int)x.dtype, x.dim(0), sizes.dim(0), a.dim(1), b.dim(1), ws.data,
                                    ws.bytes, stream));
}

// ---- routing to experts, rows between tokens and experts, adapters (b200q_route and so on say what they compute)
enum class Scoring : int { softmax = B200Q_SOFTMAX, sigmoid = B200Q_SIGMOID };
// What route_experts writes: weights float32 [.., top]; experts, places int32 [.., top]; sizes int32 [E]; order int32 [tokens * top]
struct Routing {
  ArrayView weights, experts, sizes, places, order;
};
// What group_rows writes, int32: sizes [n], starts [n + 1], order [rows], tiles [b200q_group_rows_tiles(rows, n), 4]
struct RowGroups {
  ArrayView sizes, starts, order, tiles;
};
struct RouteOptions {
  Scoring scoring = Scoring::softmax;
  ArrayView bias = {};   // float32 [E]; empty: none
  int64_t groups = 1, top_groups = 1;
  int group_best = 1;
  bool renormalize = false;
  float scale = 1.0f;
};
namespace detail {
inline int32_t* i32(const ArrayView& a) { return static_cast<int32_t*>(a.data); }
inline float* f32(const ArrayView& a) { return static_cast<float*>(a.data); }
inline int64_t rows_of(const ArrayView& a) {
  int64_t n = 1;
  for (int i = 0; i < a.ndim() - 1; ++i) n *= a.shape[i];
  return n;
}
inline bool same_rows(const ArrayView& a, const ArrayView& b) {
  bool ok = a.ndim() >= 1 && a.ndim() == b.ndim();
  for (int i = 0; ok && i < a.ndim() - 1; ++i) ok = a.shape[i] == b.shape[i];
  return ok;
}
// places [.., top] and order [tokens * top]; -> top
inline int64_t plan(const char* tag, const Routing& r) {
  if (r.places.dtype != Dtype::int32 || r.order.dtype != Dtype::int32 || r.places.ndim() < 1 || r.order.ndim() != 1 || r.order.dim(0) != r.places.size())
    throw std::invalid_argument(std::string("[") + tag + "] places and order are int32, with one entry per pair each");
  return r.places.dim(-1);
}
inline void row_groups(const char* tag, const RowGroups& g, int64_t rows, int64_t n) {
  validate_result(tag, g.sizes, n, Dtype::int32);
  validate_result(tag, g.starts, n + 1, Dtype::int32);
  validate_result(tag, g.order, rows, Dtype::int32);
  validate_result(tag, g.tiles, 4 * b200q_group_rows_tiles(rows, n), Dtype::int32);
}
struct AdapterDims {
  int64_t T, L, N, K, r;
};
inline AdapterDims adapters(const char* tag, const ArrayView& y, const ArrayView& x, const ArrayView& a, const ArrayView& b, const RowGroups& g, const ArrayView& scales) {
  if (a.ndim() != 3 || b.ndim() != 3 || !same_rows(x, y) || a.dim(0) != b.dim(0) || a.dim(1) != b.dim(2) || x.dim(-1) != a.dim(2) || y.dim(-1) != b.dim(1))
    throw std::invalid_argument(std::string("[") + tag + "] The shapes of y " + shape_str(y.shape) + ", x " + shape_str(x.shape) + ", a " + shape_str(a.shape) + " and b " +
                                shape_str(b.shape) + " do not match");
  if (y.dtype != x.dtype || a.dtype != x.dtype || b.dtype != x.dtype) throw std::invalid_argument(std::string("[") + tag + "] y, x, a and b must be of one type");
  const AdapterDims d{rows_of(x), a.dim(0), b.dim(1), a.dim(2), a.dim(1)};
  row_groups(tag, g, d.T, d.L);
  if (scales.data) validate_result(tag, scales, d.L, Dtype::float32);
  return d;
}
inline void* inner(const char* tag, const Workspace& h, const AdapterDims& d) {
  if (h.bytes < b200q_add_adapters_inner_bytes(d.T, d.r)) throw std::runtime_error(std::string("[") + tag + "] the buffer of inner products is too small");
  return h.data;
}
}  // namespace detail

// logits [.., E] -> out
inline void route_experts(const ArrayView& logits, Routing& out, const Workspace& ws, const RouteOptions& o = {}, void* stream = nullptr) {
  if (!is_floating(logits.dtype) || logits.ndim() < 1 || !detail::same_rows(logits, out.experts))
    throw std::invalid_argument("[route_experts] logits " + detail::shape_str(logits.shape) + " do not match the experts " + detail::shape_str(out.experts.shape));
  const int64_t T = detail::rows_of(logits), E = logits.dim(-1), top = out.experts.dim(-1);
  detail::validate_result("route_experts", out.weights, T * top, Dtype::float32);
  for (const ArrayView* v : {&out.experts, &out.places, &out.order}) detail::validate_result("route_experts", *v, T * top, Dtype::int32);
  detail::validate_result("route_experts", out.sizes, E, Dtype::int32);
  if (o.bias.data) detail::validate_result("route_experts", o.bias, E, Dtype::float32);
  detail::check(b200q_route(logits.data, (int)logits.dtype, T, E, top, (int)o.scoring, detail::f32(o.bias), o.groups, o.top_groups, o.group_best, o.renormalize,
                            o.scale, detail::f32(out.weights), detail::i32(out.experts), detail::i32(out.sizes), detail::i32(out.places), detail::i32(out.order),
                            ws.data, ws.bytes, stream));
}

// The gradient with respect to the logits of the weights' gradient dw [.., top]
inline void route_dlogits(const ArrayView& dw, const ArrayView& logits, const ArrayView& experts, ArrayView& dlogits, const RouteOptions& o = {}, void* stream = nullptr) {
  if (!is_floating(logits.dtype) || logits.ndim() < 1 || !detail::same_rows(logits, experts) || experts.dtype != Dtype::int32)
    throw std::invalid_argument("[route_dlogits] logits " + detail::shape_str(logits.shape) + " do not match the experts " + detail::shape_str(experts.shape));
  detail::validate_result("route_dlogits", dw, experts.size(), Dtype::float32);
  detail::validate_result("route_dlogits", dlogits, logits.size(), logits.dtype);
  detail::check(b200q_route_dlogits(detail::f32(dw), logits.data, (int)logits.dtype, detail::i32(experts), detail::rows_of(logits), logits.dim(-1), experts.dim(-1),
                                    (int)o.scoring, o.renormalize, o.scale, dlogits.data, stream));
}

// x [.., D] -> xs [tokens * top, D]
inline void dispatch_rows(const ArrayView& x, const Routing& r, ArrayView& xs, void* stream = nullptr) {
  const int64_t top = detail::plan("dispatch_rows", r);
  if (!detail::same_rows(x, r.places)) throw std::invalid_argument("[dispatch_rows] x " + detail::shape_str(x.shape) + " does not have a row for every token");
  if (is_floating(x.dtype)) detail::validate_result("dispatch_rows", xs, r.order.size() * x.dim(-1), x.dtype);
  detail::check(b200q_dispatch_rows(x.data, (int)x.dtype, detail::rows_of(x), top, x.dim(-1), detail::i32(r.places), detail::i32(r.order), xs.data, stream));
}

// y [tokens * top, D] -> out [.., D]
inline void combine_rows(const ArrayView& y, const Routing& r, ArrayView& out, bool weighted = true, void* stream = nullptr) {
  const int64_t top = detail::plan("combine_rows", r);
  if (y.ndim() != 2 || y.dim(0) != r.order.dim(0)) throw std::invalid_argument("[combine_rows] y " + detail::shape_str(y.shape) + " does not have a row for every pair");
  if (weighted) detail::validate_result("combine_rows", r.weights, r.places.size(), Dtype::float32);
  if (is_floating(y.dtype)) detail::validate_result("combine_rows", out, detail::rows_of(r.places) * y.dim(1), y.dtype);
  detail::check(b200q_combine_rows(y.data, (int)y.dtype, detail::rows_of(r.places), top, y.dim(1), detail::i32(r.places), weighted ? detail::f32(r.weights) : nullptr,
                                   out.data, stream));
}

// Gradients of combine_rows; dys and dw may be empty views: not wanted
inline void combine_rows_grad(const ArrayView& dy, const ArrayView& y, const Routing& r, ArrayView& dys, ArrayView& dw, void* stream = nullptr) {
  const int64_t top = detail::plan("combine_rows_grad", r);
  if (y.ndim() != 2 || y.dim(0) != r.order.dim(0) || dy.dtype != y.dtype || dy.ndim() < 1 || dy.dim(-1) != y.dim(1) || !detail::same_rows(dy, r.places))
    throw std::invalid_argument("[combine_rows_grad] dy " + detail::shape_str(dy.shape) + " does not match the result of combine_rows");
  detail::validate_result("combine_rows_grad", r.weights, r.places.size(), Dtype::float32);
  if (dys.data) detail::validate_result("combine_rows_grad", dys, y.size(), y.dtype);
  if (dw.data) detail::validate_result("combine_rows_grad", dw, r.places.size(), Dtype::float32);
  detail::check(b200q_combine_rows_grad(dy.data, y.data, (int)y.dtype, detail::rows_of(r.places), top, y.dim(1), detail::i32(r.places), detail::i32(r.order),
                                        detail::f32(r.weights), dys.data, detail::f32(dw), stream));
}

// ids [..] int32 or int64 -> out
inline void group_rows(const ArrayView& ids, int64_t n, RowGroups& out, const Workspace& ws, void* stream = nullptr) {
  if (ids.dtype != Dtype::int32 && ids.dtype != Dtype::int64) throw std::invalid_argument(std::string("[group_rows] ids must be int32 or int64 but are ") + name(ids.dtype));
  if (n < 0) throw std::invalid_argument("[group_rows] a negative number of groups");
  detail::row_groups("group_rows", out, ids.size(), n);
  detail::check(b200q_group_rows(ids.data, ids.dtype == Dtype::int64 ? 8 : 4, ids.size(), n, detail::i32(out.sizes), detail::i32(out.starts), detail::i32(out.order),
                                 detail::i32(out.tiles), ws.data, ws.bytes, stream));
}

// y [.., N] + adapters of x [.., K] -> out (which may be y); a [L, r, K], b [L, N, r]; h: b200q_add_adapters_inner_bytes bytes, left for the gradient
inline void add_adapters(const ArrayView& y, const ArrayView& x, const ArrayView& a, const ArrayView& b, const RowGroups& groups, const Workspace& h, ArrayView& out,
                         const ArrayView& scales = {}, void* stream = nullptr) {
  const auto d = detail::adapters("add_adapters", y, x, a, b, groups, scales);
  if (is_floating(x.dtype)) detail::validate_result("add_adapters", out, d.T * d.N, x.dtype);
  detail::check(b200q_add_adapters(y.data, x.data, a.data, b.data, (int)x.dtype, d.T, d.L, d.N, d.K, d.r, detail::i32(groups.order), detail::i32(groups.tiles),
                                   detail::f32(scales), detail::inner("add_adapters", h, d), out.data, stream));
}

// Gradients of add_adapters (that of y is dy); dx, da and db may be empty views: not wanted.  h: what add_adapters left, for db alone; g: scratch as large, for dx and da
inline void add_adapters_grad(const ArrayView& dy, const ArrayView& x, const ArrayView& a, const ArrayView& b, const RowGroups& groups, const Workspace& h,
                              const Workspace& g, ArrayView& dx, ArrayView& da, ArrayView& db, const ArrayView& scales = {}, void* stream = nullptr) {
  const auto d = detail::adapters("add_adapters_grad", dy, x, a, b, groups, scales);
  if (dx.data) detail::validate_result("add_adapters_grad", dx, x.size(), x.dtype);
  if (da.data) detail::validate_result("add_adapters_grad", da, a.size(), x.dtype);
  if (db.data) detail::validate_result("add_adapters_grad", db, b.size(), x.dtype);
  detail::check(b200q_add_adapters_grad(dy.data, x.data, a.data, b.data, (int)x.dtype, d.T, d.L, d.N, d.K, d.r, detail::i32(groups.order), detail::i32(groups.starts),
                                        detail::i32(groups.tiles), detail::f32(scales), db.data ? detail::inner("add_adapters_grad", h, d) : h.data,
                                        dx.data || da.data ? detail::inner("add_adapters_grad", g, d) : nullptr, dx.data, da.data, db.data, stream));
}

}  // namespace b200q

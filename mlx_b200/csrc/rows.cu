// Rows between the tokens' order and the experts': dispatch_rows, combine_rows and their gradients.
//
//   dispatch  xs[places[t, j]] = x[t]
//   combine   y[t] = sum over j of w[t, j] ys[places[t, j]]   (without w: the gradient of dispatch)
//   its gradients  d ys[places[t, j]] = w[t, j] dy[t],  d w[t, j] = <dy[t], ys[places[t, j]]>
//
// Everything is bound by HBM, so a token's row is read from there (or written) once, the experts' rows once each,
// in pieces of 16 bytes.  Sums are fp32 in the order of j, rounded once.  A place outside [0, T top) is a pair without a row:
// it adds nothing and gets nothing.  Rows that no pair has are those whose `order` is negative, the last ones; they get zeros.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace b200q {
namespace {

template <typename T, int VEC>
struct alignas(VEC * sizeof(T)) Vec {
  T v[VEC];
};
constexpr int kThreads = 256;

struct RowsParams {
  const void *x, *y;       // tokens' rows; experts' rows
  void* out;
  const int *places, *order;
  const float* weights;
  float* dw;
  int64_t T, R;            // tokens, rows (T * top)
  int64_t D, pieces;       // width, pieces of 16 bytes per row
  int top;
};

// ---- rows that are whole pieces of 16 bytes on their boundaries.  dispatch and combine: a thread has a piece of a token and its pairs' pieces.  4096 tokens, 2 of 8
// experts, 4096 wide, bf16, by graph replay: dispatch 15.7 us (6.4 TB/s, 0.98 of the measured copy rate), combine 19.6 (5.1), without weights 19.0.
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) dispatch_kernel(const RowsParams p) {
  using V = Vec<T, VEC>;
  const V* x = static_cast<const V*>(p.x);
  V* xs = static_cast<V*>(p.out);
  const int64_t n = p.T * p.pieces, step = (int64_t)gridDim.x * kThreads;
  const bool left = p.order[p.R - 1] < 0;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += step) {
    const int64_t t = i / p.pieces, c = i - t * p.pieces;
    const V v = x[i];
    for (int j = 0; j < p.top; ++j) {
      const int64_t at = p.places[t * p.top + j];
      if (at >= 0 && at < p.R) xs[at * p.pieces + c] = v;
    }
    if (left)
      for (int64_t r = t * p.top; r < (t + 1) * p.top; ++r)
        if (p.order[r] < 0) xs[r * p.pieces + c] = V{};
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) combine_kernel(const RowsParams p) {
  using V = Vec<T, VEC>;
  const V* y = static_cast<const V*>(p.y);
  V* out = static_cast<V*>(p.out);
  const int64_t n = p.T * p.pieces, step = (int64_t)gridDim.x * kThreads;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += step) {
    const int64_t t = i / p.pieces, c = i - t * p.pieces;
    float acc[VEC] = {};
#pragma unroll 4
    for (int j = 0; j < p.top; ++j) {
      const int64_t at = p.places[t * p.top + j];
      if (at < 0 || at >= p.R) continue;
      const float w = p.weights ? p.weights[t * p.top + j] : 1.0f;
      const V v = y[at * p.pieces + c];
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] = fmaf(w, Elem<T>::to_float(v.v[k]), acc[k]);
    }
    V o;
#pragma unroll
    for (int k = 0; k < VEC; ++k) o.v[k] = Elem<T>::from_float(acc[k]);
    out[i] = o;
  }
}

// A block has a token, whose row stays in L1 for its pairs.  The same rows: 29.3 us (5.7 TB/s).
template <typename T, int VEC>
__global__ void __launch_bounds__(kThreads) combine_grad_kernel(const RowsParams p) {
  using V = Vec<T, VEC>;
  __shared__ float part[32][kThreads / 32];   // of d w, for 32 choices at a time
  const int64_t t = blockIdx.x;
  const V* dy = static_cast<const V*>(p.x) + t * p.pieces;
  const V* y = static_cast<const V*>(p.y);
  V* dys = static_cast<V*>(p.out);
  for (int j = 0; j < p.top; ++j) {
    const int64_t at = p.places[t * p.top + j];
    const bool has = at >= 0 && at < p.R;
    const float w = p.weights[t * p.top + j];
    float dot = 0.0f;
    if (has)
      for (int64_t c = threadIdx.x; c < p.pieces; c += kThreads) {
        const V g = dy[c];
        if (p.dw) {
          const V v = y[at * p.pieces + c];
#pragma unroll
          for (int k = 0; k < VEC; ++k) dot = fmaf(Elem<T>::to_float(g.v[k]), Elem<T>::to_float(v.v[k]), dot);
        }
        if (dys) {
          V o;
#pragma unroll
          for (int k = 0; k < VEC; ++k) o.v[k] = Elem<T>::from_float(w * Elem<T>::to_float(g.v[k]));
          dys[at * p.pieces + c] = o;
        }
      }
    for (int o = 16; o; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if ((threadIdx.x & 31) == 0) part[j & 31][threadIdx.x >> 5] = dot;
    if ((j & 31) == 31 || j == p.top - 1) {
      __syncthreads();
      const int j0 = j & ~31;
      if (p.dw && threadIdx.x <= (unsigned)(j - j0)) {
        float s = 0.0f;
        for (int q = 0; q < kThreads / 32; ++q) s += part[threadIdx.x][q];
        p.dw[t * p.top + j0 + threadIdx.x] = s;
      }
      __syncthreads();
    }
  }
  if (dys && p.order[p.R - 1] < 0)
    for (int64_t r = t * p.top; r < (t + 1) * p.top; ++r)
      if (p.order[r] < 0)
        for (int64_t c = threadIdx.x; c < p.pieces; c += kThreads) dys[r * p.pieces + c] = V{};
}

// ---- rows that start anywhere.  A block has a token.  What is written to a row goes by the pieces of 16 bytes of memory that it covers: whole ones by
// one store, those at its ends value by value.  What is read for a whole piece is 16 bytes from any address: two pieces of memory and a shift.  (Both hold bytes of
// the row, and memory is mapped by more than 16 bytes, so that nothing outside is touched that is not there.)  1531 tokens, 6 of 64 experts, 2047 wide, f16, by graph
// replay: dispatch 12.2 us (3.6 TB/s), combine 10.5, its gradients 18.2 (4.5); bound by instructions, the shifts and the rows' ends.
template <typename T>
__device__ __forceinline__ Vec<T, 16 / sizeof(T)> load_any(const T* p) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  const uint32_t off = a & 15;
  const uint4* q = reinterpret_cast<const uint4*>(a - off);
  const uint4 lo = q[0];
  uint4 hi = lo;
  if (off) hi = q[1];
  uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  if (off & 8) {
#pragma unroll
    for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
  }
  if (off & 4) {
#pragma unroll
    for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
  }
  union {
    uint32_t u[4];
    Vec<T, 16 / sizeof(T)> v;
  } r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r.u[i] = __funnelshift_r(w[i], w[i + 1], (off & 2) * 8);
  return r.v;
}
// For the row at `row`: whole(first column) for the pieces that this thread of a group has, one(column) for its values at the ends.
template <typename T, typename F, typename G>
__device__ __forceinline__ void for_pieces(const T* row, int64_t D, int id, int group, F whole, G one) {
  constexpr int VEC = 16 / sizeof(T);
  const int64_t head = min((int64_t)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) % 16 / sizeof(T)), D), tail = head + (D - head) / VEC * VEC;
  for (int64_t c = head + id * VEC; c < tail; c += group * VEC) whole(c);
  // the ends' values: with the last threads, which have the fewest pieces
  const int64_t ends = head + D - tail;
  for (int64_t i = group - 1 - id; i < ends; i += group) one(i < head ? i : tail + i - head);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) dispatch_any_kernel(const RowsParams p) {
  constexpr int VEC = 16 / sizeof(T);
  const int64_t t = blockIdx.x;
  const T* x = static_cast<const T*>(p.x) + t * p.D;
  T* xs = static_cast<T*>(p.out);
  const bool left = p.order[p.R - 1] < 0;
  for (int j = 0; j < p.top; ++j) {
    const int64_t at = p.places[t * p.top + j];
    if (at >= 0 && at < p.R)
      for_pieces(xs + at * p.D, p.D, threadIdx.x, blockDim.x, [&](int64_t c) { *reinterpret_cast<Vec<T, VEC>*>(xs + at * p.D + c) = load_any(x + c); },
                 [&](int64_t c) { xs[at * p.D + c] = x[c]; });
  }
  if (left)
    for (int64_t r = t * p.top; r < (t + 1) * p.top; ++r)
      if (p.order[r] < 0)
        for (int64_t c = threadIdx.x; c < p.D; c += blockDim.x) xs[r * p.D + c] = Elem<T>::from_float(0.0f);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) combine_any_kernel(const RowsParams p) {
  constexpr int VEC = 16 / sizeof(T);
  const int64_t t = blockIdx.x;
  const T* y = static_cast<const T*>(p.y);
  T* out = static_cast<T*>(p.out) + t * p.D;
  for_pieces(out, p.D, threadIdx.x, blockDim.x, [&](int64_t c) {
    float acc[VEC] = {};
#pragma unroll 4
    for (int j = 0; j < p.top; ++j) {
      const int64_t at = p.places[t * p.top + j];
      if (at < 0 || at >= p.R) continue;
      const float w = p.weights ? p.weights[t * p.top + j] : 1.0f;
      const auto v = load_any(y + at * p.D + c);
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[k] = fmaf(w, Elem<T>::to_float(v.v[k]), acc[k]);
    }
    Vec<T, VEC> o;
#pragma unroll
    for (int k = 0; k < VEC; ++k) o.v[k] = Elem<T>::from_float(acc[k]);
    *reinterpret_cast<Vec<T, VEC>*>(out + c) = o;
  }, [&](int64_t c) {
    float acc = 0.0f;
    for (int j = 0; j < p.top; ++j) {
      const int64_t at = p.places[t * p.top + j];
      if (at >= 0 && at < p.R) acc = fmaf(p.weights ? p.weights[t * p.top + j] : 1.0f, Elem<T>::to_float(y[at * p.D + c]), acc);
    }
    out[c] = Elem<T>::from_float(acc);
  });
}

// A group of threads has a pair (token, choice): a warp, or the block where rows are long and pairs few: up to 12 pairs for every 16 bytes of a row.  (Inputs not in L2, block /
// warp, us: rows of 2047, f16, 300 pairs 4.5 / 12.1, 2400 14.0 / 16.4, 3600 18.7 / 17.8, 9186 44.2 / 32.5; of 1023, f32, 2400 12.6 / 16.8, 3600 17.3 / 17.9, 4800 22.2 / 19.4; of 255,
// bf16, 300 2.8 / 2.8, 800 4.2 / 2.8; of 8191, bf16, 300 8.6 / 43, 9186 101 / 109.)  dy's row is read once from HBM and for the token's other pairs from L2.
template <typename T>
__global__ void __launch_bounds__(kThreads) combine_grad_any_kernel(const RowsParams p, int group) {
  constexpr int VEC = 16 / sizeof(T);
  using V = Vec<T, VEC>;
  __shared__ float part[kThreads / 32];
  const int id = threadIdx.x % group;
  const int64_t pair = (int64_t)blockIdx.x * (kThreads / group) + threadIdx.x / group;
  if (pair >= p.R) return;   // (a whole warp; blocks of one pair have none such)
  const int64_t at = p.places[pair];
  const T *dy = static_cast<const T*>(p.x) + pair / p.top * p.D, *y = static_cast<const T*>(p.y) + at * p.D;
  T *dys = static_cast<T*>(p.out), *d = dys + at * p.D;
  float dot = 0.0f;
  if (at >= 0 && at < p.R) {
    const float w = p.weights[pair];
    auto whole = [&](int64_t c) {
      const V g = load_any(dy + c);
      if (p.dw) {
        const V v = load_any(y + c);
#pragma unroll
        for (int k = 0; k < VEC; ++k) dot = fmaf(Elem<T>::to_float(g.v[k]), Elem<T>::to_float(v.v[k]), dot);
      }
      if (dys) {
        V o;
#pragma unroll
        for (int k = 0; k < VEC; ++k) o.v[k] = Elem<T>::from_float(w * Elem<T>::to_float(g.v[k]));
        *reinterpret_cast<V*>(d + c) = o;
      }
    };
    for_pieces(dys ? d : const_cast<T*>(y), p.D, id, group, whole, [&](int64_t c) {
      const float g = Elem<T>::to_float(dy[c]);
      if (p.dw) dot = fmaf(g, Elem<T>::to_float(y[c]), dot);
      if (dys) d[c] = Elem<T>::from_float(w * g);
    });
  }
  if (p.dw) {
    for (int o = 16; o; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if (group > 32) {
      if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = dot;
      __syncthreads();
      if (id == 0)
        for (int q = 1; q < kThreads / 32; ++q) dot += part[q];
    }
    if (id == 0) p.dw[pair] = dot;
  }
  if (dys && p.order[pair] < 0)   // a row that no pair has
    for (int64_t c = id; c < p.D; c += group) dys[pair * p.D + c] = Elem<T>::from_float(0.0f);
}

enum class Kind { Dispatch, Combine, Grad };

template <typename T>
int launch(Kind kind, RowsParams p, cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(T);
  const uintptr_t all = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.y) | reinterpret_cast<uintptr_t>(p.out) | (uintptr_t)(p.D * sizeof(T));
  p.pieces = p.D / VEC;
  const unsigned tokens = (unsigned)p.T, threads = (unsigned)std::min<int64_t>(kThreads, (p.pieces + 32) / 32 * 32);
  const int group = p.R < 12 * p.pieces ? kThreads : 32;
  const unsigned pairs = (unsigned)((p.R + kThreads / group - 1) / (kThreads / group));
  if (all % 16 == 0) {   // every piece of 16 bytes on its boundary
    const unsigned blocks = (unsigned)std::min<int64_t>((p.T * p.pieces + kThreads - 1) / kThreads, 148 * 8 * 16);
    switch (kind) {
      case Kind::Dispatch: dispatch_kernel<T, VEC><<<blocks, kThreads, 0, st>>>(p); break;
      case Kind::Combine: combine_kernel<T, VEC><<<blocks, kThreads, 0, st>>>(p); break;
      case Kind::Grad: combine_grad_kernel<T, VEC><<<tokens, kThreads, 0, st>>>(p); break;
    }
  } else {
    switch (kind) {
      case Kind::Dispatch: dispatch_any_kernel<T><<<tokens, threads, 0, st>>>(p); break;
      case Kind::Combine: combine_any_kernel<T><<<tokens, threads, 0, st>>>(p); break;
      case Kind::Grad: combine_grad_any_kernel<T><<<pairs, kThreads, 0, st>>>(p, group); break;
    }
  }
  B200Q_LAUNCH_OK("rows kernel");
  return B200Q_OK;
}

int run(Kind kind, const RowsParams& p, int dtype, cudaStream_t st) {
  switch (dtype) {
    case B200Q_F32: return launch<float>(kind, p, st);
    case B200Q_F16: return launch<__half>(kind, p, st);
    default: return launch<__nv_bfloat16>(kind, p, st);
  }
}

int check(const char* tag, int dtype, int64_t T, int64_t top, int64_t D) {
  if (dtype != B200Q_F32 && dtype != B200Q_F16 && dtype != B200Q_BF16)
    return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] unsupported dtype code %d", tag, dtype);
  if (T < 0 || top < 0 || D < 0) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] negative dimension.", tag);
  if (top > INT32_MAX || D > INT32_MAX || (top > 0 && T > INT32_MAX / top))
    return fail(B200Q_ERR_UNSUPPORTED, "[%s] No implementation for problem shape: more than 2^31 - 1 rows or elements in one.", tag);
  return B200Q_OK;
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" int b200q_dispatch_rows(const void* x, int dtype, int64_t T, int64_t top, int64_t D, const int32_t* places, const int32_t* order, void* xs,
                                   void* stream) {
  const char* tag = "dispatch_rows";
  if (int rc = check(tag, dtype, T, top, D)) return rc;
  if (T == 0 || top == 0 || D == 0) return B200Q_OK;
  if (!x || !places || !order || !xs) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] null pointer", tag);
  if (!on_boundaries({x, xs}, dtype_size(dtype)) || !on_boundaries({places, order}, 4)) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] misaligned pointer", tag);
  const RowsParams p{x, nullptr, xs, places, order, nullptr, nullptr, T, T * top, D, 0, (int)top};
  return run(Kind::Dispatch, p, dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int b200q_combine_rows(const void* y, int dtype, int64_t T, int64_t top, int64_t D, const int32_t* places, const float* weights, void* out,
                                  void* stream) {
  const char* tag = "combine_rows";
  if (int rc = check(tag, dtype, T, top, D)) return rc;
  if (T == 0 || D == 0) return B200Q_OK;
  if (!out || (top > 0 && (!y || !places))) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] null pointer", tag);
  if (!on_boundaries({y, out}, dtype_size(dtype)) || !on_boundaries({places, weights}, 4)) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] misaligned pointer", tag);
  const RowsParams p{nullptr, y, out, places, nullptr, weights, nullptr, T, T * top, D, 0, (int)top};
  return run(Kind::Combine, p, dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int b200q_combine_rows_grad(const void* dy, const void* y, int dtype, int64_t T, int64_t top, int64_t D, const int32_t* places,
                                       const int32_t* order, const float* weights, void* dys, float* dw, void* stream) {
  const char* tag = "combine_rows";
  if (int rc = check(tag, dtype, T, top, D)) return rc;
  if (T == 0 || top == 0 || (!dys && !dw)) return B200Q_OK;
  if (!on_boundaries({dy, y, dys}, dtype_size(dtype)) || !on_boundaries({places, order, weights, dw}, 4)) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] misaligned pointer", tag);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (D == 0) {
    if (dw) B200Q_CUDA_OK(cudaMemsetAsync(dw, 0, (size_t)T * top * 4, st));
    return B200Q_OK;
  }
  if (!dy || (dw && !y) || !places || !order || !weights) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] null pointer", tag);
  const RowsParams p{dy, y, dys, places, order, weights, dw, T, T * top, D, 0, (int)top};
  return run(Kind::Grad, p, dtype, st);
}
